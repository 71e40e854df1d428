"""Packed prompts through the C ABI against the definitions in 64 bits:
vxk_prompt_rope (rotary rows) and vxk_prompt_attention (attention within each
sequence: causal, windowed and whole, grouped heads, lengths from 0).

Tolerances.  h = torch.finfo(type).eps / 2 is the largest relative error of a
rounding to the type (f16 2^-11, bf16 2^-8), U = 2^-24 fp32's.

rope: x cos - y sin with fp32 cos, sin (U each) and three fp32 roundings is off by
4 U (|x| + |y|), then rounded: h |out|.

attention: the probabilities are rounded to the type (h each) for their product with
v while their sum is not, so the weighted mean is off by h M, M = sum_j p_j |v_j|, and
is then rounded, h |out|.  A score is a sum of head_dim exact products and its error
is at most head_dim 2 U A, A = scale sum |q_i k_i|, plus 4 U |s| for its scaling
and exponent: e^s is off by D = 2 U (head_dim A + 4 |s|) relative to itself, in the
numerator and in the sum: 2 D M.  The sums over n keys add n 2 U M.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F16, BF16 = 1, 30
U = 2.0 ** -24
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _type(dtype):
    import torch

    return torch.float16 if dtype == F16 else torch.bfloat16


def _stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def make(lens, heads, kv, dim, dtype, seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed + sum(lens) * 7 + heads)
    rows, t = max(1, sum(lens)), _type(dtype)
    q = (torch.randn(rows, heads, dim, generator=g, device="cuda") * 2).to(t)
    k = torch.randn(rows, kv, dim, generator=g, device="cuda").to(t)
    v = torch.randn(rows, kv, dim, generator=g, device="cuda").to(t)
    return q, k, v


def attend(vxk, q, k, v, lens, dtype, prompt=None, **cfg):
    import torch

    own = prompt is None
    prompt = prompt or vxk.Prompt(n_q_heads=q.shape[1], n_kv_heads=k.shape[1], head_dim=q.shape[2], max_seqs=len(lens),
                                  max_rows=max(1, sum(lens)), max_position=0, dtype=dtype, **cfg)
    prompt.plan(lens, cuda_stream=_stream())
    out = torch.full_like(q, 9.0)
    prompt.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _stream())
    prompt.sync(_stream())
    if own:
        prompt.close()
    return out


def check_attention(out, q, k, v, lens, dtype, causal=1, window=0, scale=None):
    """Every row of out against the definition, by sequence and kv head, on the GPU in 64 bits."""
    import torch

    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    scale = scale or dim ** -0.5
    h, at = HALF[dtype], 0
    for n in lens:
        i = torch.arange(n, device="cuda")
        allowed = torch.ones(n, n, dtype=torch.bool, device="cuda")
        if causal:
            back = i[:, None] - i[None, :]
            allowed = (back >= 0) & (back < (window or n + 1))
        for hk in range(k.shape[1] if n else 0):
            kk, vv = k[at: at + n, hk].double(), v[at: at + n, hk].double()
            for hq in range(hk * group, (hk + 1) * group):
                qq = q[at: at + n, hq].double()
                s = (qq @ kk.T * scale).masked_fill(~allowed, -float("inf"))
                p = torch.softmax(s, -1)
                a = (qq.abs() @ kk.abs().T * scale).masked_fill(~allowed, 0.0)
                d = 2 * U * (dim * a.max(-1, keepdim=True).values +
                             4 * s.masked_fill(~allowed, 0.0).abs().max(-1, keepdim=True).values)
                want, mean = p @ vv, p @ vv.abs()
                tol = h * (mean + want.abs()) * 1.01 + (2 * d + 2 * U * n) * mean + 2.0 ** -25
                off = (out[at: at + n, hq].double() - want).abs()
                assert bool((off <= tol).all()), (n, hq, float((off / tol).max()))
        at += n
    assert bool((out[at:] == 9.0).all()), "rows behind the last sequence were written"


LENS = [[1], [2, 1], [38], [64, 65, 63], [127, 128, 129], [0, 5, 0, 300, 0], [255, 256, 257, 1], [700], [31, 33, 32, 1000, 17]]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", LENS, ids=lambda l: "-".join(map(str, l)))
def test_causal(vxk, dtype, dim, lens):
    q, k, v = make(lens, 8, 2, dim, dtype)
    check_attention(attend(vxk, q, k, v, lens, dtype), q, k, v, lens, dtype)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (2, 1), (3, 1), (6, 2), (8, 1), (16, 1), (32, 1), (24, 2), (5, 5), (64, 1)])
def test_head_groups(vxk, heads, kv):
    lens = [70, 3, 260]
    for dim, dtype in ((128, F16), (64, BF16)):
        q, k, v = make(lens, heads, kv, dim, dtype)
        check_attention(attend(vxk, q, k, v, lens, dtype), q, k, v, lens, dtype)


@pytest.mark.parametrize("dim,heads,kv", [(64, 20, 20), (128, 8, 2)])
def test_whole(vxk, dim, heads, kv):
    for lens in ([1], [130, 0, 1, 500], [128, 256]):
        q, k, v = make(lens, heads, kv, dim, BF16)
        check_attention(attend(vxk, q, k, v, lens, BF16, causal=0), q, k, v, lens, BF16, causal=0)


@pytest.mark.parametrize("dim,heads,kv,lens,causal,window", [
    (64, 20, 20, [600] * 5 + [300, 129], 0, 0), (128, 32, 8, [200] * 13 + [1] * 9, 1, 0), (64, 12, 12, [500] * 7, 1, 140)])
def test_more_items_than_ctas(vxk, dim, heads, kv, lens, causal, window):
    """Several items a CTA, of every number of key tiles."""
    q, k, v = make(lens, heads, kv, dim, F16)
    out = attend(vxk, q, k, v, lens, F16, causal=causal, window=window)
    check_attention(out, q, k, v, lens, F16, causal=causal, window=window)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 128, 129, 300, 10000])
def test_window(vxk, window):
    lens = [500, 1, 129, 64]
    for dim, dtype, heads, kv in ((128, F16, 8, 2), (64, BF16, 3, 3)):
        q, k, v = make(lens, heads, kv, dim, dtype)
        out = attend(vxk, q, k, v, lens, dtype, window=window)
        check_attention(out, q, k, v, lens, dtype, window=window)


def test_scale_and_long_sequence(vxk):
    lens = [3001, 40]
    q, k, v = make(lens, 8, 2, 128, F16)
    check_attention(attend(vxk, q, k, v, lens, F16), q, k, v, lens, F16)
    check_attention(attend(vxk, q, k, v, lens, F16, scale=0.01), q, k, v, lens, F16, scale=float(np.float32(0.01)))


def test_large_scores_and_a_late_maximum(vxk):
    """Scores of hundreds, the largest at the end of the sequence: the running maximum has to follow."""
    import torch

    lens = [900, 300]
    q, k, v = make(lens, 4, 2, 128, BF16)
    k *= torch.linspace(0.1, 20, sum(lens), device="cuda")[:, None, None].to(k.dtype)
    check_attention(attend(vxk, q, k, v, lens, BF16), q, k, v, lens, BF16)
    q.zero_()  # equal scores: the mean
    check_attention(attend(vxk, q, k, v, lens, BF16), q, k, v, lens, BF16)


def test_neighbours_and_the_future_do_not_reach_a_row(vxk):
    """NaN and infinities in another sequence, in rows behind the last, and in a row's own future change nothing."""
    import torch

    lens = [70, 33, 200]
    for dim, dtype in ((128, BF16), (64, F16)):
        q, k, v = make(lens + [140], 8, 2, dim, dtype)
        clean = attend(vxk, q, k, v, lens, dtype)
        for bad in (float("nan"), float("inf")):
            k2, v2, q2 = k.clone(), v.clone(), q.clone()
            k2[70:103] = bad
            v2[70:103] = bad
            q2[70:103] = bad
            k2[303:] = bad
            v2[303:] = bad
            v2[103 + 150] = bad  # a row of the last sequence
            k2[103 + 160] = bad
            got = attend(vxk, q2, k2, v2, lens, dtype)
            assert torch.equal(got[:70], clean[:70])
            assert torch.equal(got[103: 103 + 150], clean[103: 103 + 150])
            assert bool((~torch.isfinite(got[103 + 150: 303].float())).all())
            assert bool((got[303:] == 9.0).all())


def test_minus_infinity_scores(vxk):
    """k rows whose score overflows to -inf have probability 0; a row with no other has NaN, as the formula."""
    import torch

    lens = [40]
    q, k, v = make(lens, 2, 1, 64, F16)
    q = q.abs() + 1
    k[:5] = -float("inf")
    out = attend(vxk, q, k, v, lens, F16)
    assert bool(torch.isnan(out[:5].float()).all())
    check_attention(out[5:], q[5:], k[5:], v[5:], [35], F16)


def test_repeats_graph_and_a_new_plan(vxk):
    import torch

    lens, dtype = [300, 20, 130], F16
    q, k, v = make(lens, 8, 2, 128, dtype)
    prompt = vxk.Prompt(n_q_heads=8, n_kv_heads=2, head_dim=128, max_seqs=8, max_rows=600, max_position=0, dtype=dtype)
    first = attend(vxk, q, k, v, lens, dtype, prompt=prompt)
    out = torch.full_like(q, 9.0)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        prompt.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                         torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    # the same graph under a smaller plan, and under one too large for its buffers
    prompt.plan([17, 200, 0, 33], cuda_stream=_stream())
    out.fill_(9.0)
    graph.replay()
    prompt.sync(_stream())
    check_attention(out, q, k, v, [17, 200, 0, 33], dtype)
    prompt.plan([451], cuda_stream=_stream())
    out.fill_(9.0)
    graph.replay()
    with pytest.raises(vxk.VxkError) as e:
        prompt.sync(_stream())
    assert e.value.status == vxk.BACKEND_ERROR and "plan" in str(e.value)
    assert bool((out == 9.0).all())
    prompt.sync(_stream())
    # planning inside a capture is refused
    with pytest.raises(vxk.VxkError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            prompt.plan([10], cuda_stream=torch.cuda.current_stream().cuda_stream)
    assert e.value.status == vxk.INVALID_STATE
    prompt.close()


def test_another_stream_and_an_empty_plan(vxk):
    import torch

    lens = [90, 200]
    q, k, v = make(lens, 4, 4, 64, BF16)
    prompt = vxk.Prompt(n_q_heads=4, n_kv_heads=4, head_dim=64, max_seqs=4, max_rows=300, max_position=0, dtype=BF16)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    prompt.plan(lens, cuda_stream=a.cuda_stream)
    b.wait_stream(a)
    for s in (a, b, a, b):  # calls of one prompt may overlap
        out = torch.full_like(q, 9.0)
        s.wait_stream(torch.cuda.current_stream())
        prompt.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), s.cuda_stream)
        outs.append(out)
    torch.cuda.synchronize()
    for out in outs:
        check_attention(out, q, k, v, lens, BF16)
    assert prompt.plan([0, 0], cuda_stream=_stream()) == 0
    out = torch.full_like(q, 9.0)
    prompt.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _stream())
    prompt.sync(_stream())
    assert bool((out == 9.0).all())
    prompt.close()


def test_offsets_beyond_32_bits(vxk):
    """530,000 rows of 32 heads of 128: more than 2^31 values of q and of the output."""
    import torch

    lens, heads, dim, dtype = [1000] * 529 + [937, 63], 32, 128, F16
    rows, tail = sum(lens), 1000
    g = torch.Generator(device="cuda").manual_seed(11)
    prompt = vxk.Prompt(n_q_heads=heads, n_kv_heads=1, head_dim=dim, max_seqs=len(lens), max_rows=rows, max_position=1000,
                        dtype=dtype)
    prompt.plan(lens, cuda_stream=_stream())
    q = torch.zeros(rows, heads, dim, device="cuda")
    k, v = torch.zeros(rows, 1, dim, device="cuda"), torch.zeros(rows, 1, dim, device="cuda")
    for x in (q, k, v):
        x[-tail:] = torch.randn(x[-tail:].shape, generator=g, device="cuda")
    q16, k16, v16 = (torch.full(x.shape, 9.0, dtype=torch.float16, device="cuda") for x in (q, k, v))
    prompt.rope(*(x.data_ptr() for x in (q, k, v, q16, k16, v16)), _stream())
    prompt.sync(_stream())
    small = vxk.Prompt(n_q_heads=heads, n_kv_heads=1, head_dim=dim, max_seqs=2, max_rows=tail, max_position=1000, dtype=dtype)
    small.plan([937, 63], cuda_stream=_stream())
    want = [torch.empty_like(x[-tail:]) for x in (q16, k16, v16)]
    small.rope(*(x[-tail:].contiguous().data_ptr() for x in (q, k, v)), *(x.data_ptr() for x in want), _stream())
    small.sync(_stream())
    for x, y in zip((q16, k16, v16), want):
        assert torch.equal(x[-tail:], y) and bool((x[: tail] == 0).all())
    del q
    out = torch.full_like(q16, 9.0)
    prompt.attention(q16.data_ptr(), k16.data_ptr(), v16.data_ptr(), out.data_ptr(), _stream())
    prompt.sync(_stream())
    check_attention(out[-tail:], q16[-tail:], k16[-tail:], v16[-tail:], [937, 63], dtype)
    assert bool((out[: -tail] == 0).all())
    prompt.close()
    small.close()


# ---- rotary rows --------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,first,heads,kv,dim", [
    ([1], [0], 1, 1, 64), ([38], None, 32, 8, 128), ([5, 0, 40], [7, 0, 99000], 3, 1, 128), ([130, 1], [4000, 0], 20, 20, 64),
    ([64], [1], 33, 11, 64)])
def test_rope(vxk, dtype, lens, first, heads, kv, dim):
    import torch

    rows, t, h = sum(lens), _type(dtype), HALF[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    q, k, v = (torch.randn(rows, n, dim, generator=g, device="cuda") for n in (heads, kv, kv))
    q[0, 0, :2] = torch.tensor([0.0, -0.0], device="cuda")
    prompt = vxk.Prompt(n_q_heads=heads, n_kv_heads=kv, head_dim=dim, max_seqs=len(lens), max_rows=rows + 3,
                        max_position=100000, dtype=dtype)
    assert prompt.plan(lens, first, _stream()) == rows
    outs = [torch.full((rows + 2, n, dim), 9.0, dtype=t, device="cuda") for n in (heads, kv, kv)]
    prompt.rope(q.data_ptr(), k.data_ptr(), v.data_ptr(), *(o.data_ptr() for o in outs), _stream())
    prompt.sync(_stream())
    pos = np.concatenate([(first[i] if first else 0) + np.arange(n) for i, n in enumerate(lens)]).astype(np.float64)
    angle = pos[:, None] * 1e6 ** (-np.arange(dim // 2) / (dim // 2))
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    for x, o in ((q, outs[0]), (k, outs[1])):
        x64 = x.double().cpu().numpy()
        a, b = x64[..., 0::2], x64[..., 1::2]
        want = np.stack((a * c - b * s, a * s + b * c), -1).reshape(x64.shape)
        size = np.repeat(np.abs(a) + np.abs(b), 2, -1).reshape(x64.shape)
        off = np.abs(o[:rows].double().cpu().numpy() - want)
        assert np.all(off <= h * np.abs(want) * 1.01 + 4 * U * size + 2.0 ** -25)
    assert torch.equal(outs[2][:rows], v.to(t))
    assert all(bool((o[rows:] == 9.0).all()) for o in outs)
    prompt.close()


def test_values_that_are_not_finite_among_many_items_of_one_tile(vxk):
    """Items with two tiles, each followed by dozens of one tile in the same CTA: a V row that is not finite reaches the
    rows that attend it and no others."""
    import torch

    lens, heads, kv, dtype = [64] * 160 + [20] * 2500, 8, 2, F16
    q, k, v = make(lens, heads, kv, 64, dtype)
    clean = attend(vxk, q, k, v, lens, dtype)
    assert bool(torch.isfinite(clean.float()).all())
    hit = torch.zeros(sum(lens), kv, dtype=torch.bool, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        if i % 7 == 0:
            row = at + (13 * i) % n
            v[row, i % kv, i % 64] = float("nan" if i % 2 else "inf")
            hit[row: at + n, i % kv] = True
        at += n
    got = attend(vxk, q, k, v, lens, dtype)
    hit = hit.repeat_interleave(heads // kv, 1)
    assert torch.equal(got[~hit], clean[~hit])
    assert bool((~torch.isfinite(got[hit].float())).any(-1).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("depth", [9.0, 12.0, 15.0, 17.5])
def test_many_small_probabilities_beside_a_large_one(vxk, dtype, dim, depth):
    """One key far above thousands of others, whose probabilities e^-depth are below f16's normal range.

    A probability is scaled before it is rounded so that the largest is at least 2^7; what f16 holds as a subnormal is
    then 2^-25 - 7 of the largest off, n 2^-32 of the largest |v| in all, besides the errors of check_attention.
    """
    import torch

    lens = [3000, 700]
    q, k, v = make(lens, 4, 2, dim, dtype)
    q.zero_()
    q[..., 0] = dim ** 0.5
    k.zero_()
    k[:, :, 0] = -depth
    v[:] = torch.rand(v.shape, device="cuda").to(v.dtype) + 0.5
    at = 0
    for n in lens:  # the first key of each: nearly all of the weight, and a v of 0
        k[at], v[at] = 0.0, 0.0
        at += n
    out, at = attend(vxk, q, k, v, lens, dtype), 0
    h = HALF[dtype]
    for n in lens:
        s = (q[at: at + n].double() * dim ** -0.5).transpose(0, 1) @ k[at: at + n].double().repeat_interleave(2, 1).permute(1, 2, 0)
        p = torch.softmax(s.masked_fill(torch.ones(n, n, device="cuda").triu(1) > 0, -float("inf")), -1)
        want = (p @ v[at: at + n].double().repeat_interleave(2, 1).transpose(0, 1)).transpose(0, 1)
        d = 2 * U * (dim + 4) * depth
        tol = 2.02 * h * want + (2 * d + 2 * U * n) * want + n * 2.0 ** -32 * 1.5 + 2.0 ** -25
        off = (out[at: at + n].double() - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())
        at += n
