"""Scores of rows of logits (vxk_head_score_logits) and of hidden rows
(vxk_head_score) through the C ABI against the definition in 64 bits: log
probability of the given token, entropy, and the top list with the lowest
index first among equal logits.

Tolerances.  U = 2^-24 is a rounding of fp32.  A thread adds at most L terms, all
positive, then a tree of ~20 joins; each term carries an ex2 error of 2 U and the
rounding of its exponent d = l - m (3 U |d|, and e^d |d| < 1/e of the largest
term), so s and t are off by at most (L + 64) U relative to themselves.  log s is
then off by (L + 64) U, the entropy log s - t / s by (L + 64) U (1 + 2 t / s), and
the log probability (l - m) - log s by (L + 64) U + 4 U |value|.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 30
U = 2.0 ** -24


def _stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def _torch_type(dtype):
    import torch

    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[dtype]


def reference(l, tokens, n_top):
    """Scores of float64 logits [rows][vocab]."""
    with np.errstate(all="ignore"):
        m = l.max(1, keepdims=True)
        base = np.where(np.isneginf(m), 0.0, m)
        d = l - base
        e = np.exp(d)
        s = e.sum(1)
        t = (e * np.where(e == 0, 0.0, d)).sum(1)
        lp = d - np.log(s)[:, None]
    order = np.argsort(-np.where(np.isnan(l), -np.inf, l), axis=1, kind="stable")[:, :n_top]
    given = np.where(tokens < 0, 0.0, np.take_along_axis(lp, np.maximum(tokens, 0)[:, None], 1)[:, 0])
    return given, np.log(s) - t / s, order, np.take_along_axis(lp, order, 1), t / s


def outputs(rows, n_top):
    import torch

    return (torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda"),
            torch.full((rows, n_top), -7, dtype=torch.int32, device="cuda"),
            torch.full((rows, n_top), 7.0, device="cuda"))


def ptrs(outs):
    return [o.data_ptr() if o.numel() else 0 for o in outs]


def score_logits(vxk, logits, vocab, tokens, n_top, dtype=None, head=None, sync=True):
    """logits: a CUDA tensor [rows][ld] (its first `vocab` columns count)."""
    import torch

    own = head is None
    head = head or vxk.Head(dim=64, vocab=vocab)
    outs = outputs(len(logits), n_top)
    tok = torch.from_numpy(np.asarray(tokens, np.int32)).cuda()
    dtype = dtype if dtype is not None else {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[logits.dtype]
    head.score_logits(logits.data_ptr(), dtype, logits.stride(0), len(logits), tok.data_ptr(), n_top, *ptrs(outs),
                      _stream())
    if sync:
        head.sync(_stream())
    got = [o.cpu().numpy() for o in outs]
    if own:
        head.close()
    return got


def check(got, l64, tokens, n_top):
    lp, ent, ids, top = got
    want_lp, want_ent, want_ids, want_top, ts = reference(l64, tokens, n_top)
    terms = l64.shape[1] / 32 + 17  # a warp a row at the least parallel
    tol = (terms + 64) * U
    assert np.array_equal(ids, want_ids)
    assert np.all(np.abs(lp - want_lp) <= tol + 4 * U * np.abs(want_lp))
    assert np.all(np.abs(ent - want_ent) <= tol * (1 + 2 * np.abs(ts)))
    fine = np.isfinite(want_top)
    assert np.array_equal(top[~fine], want_top[~fine])
    assert np.all(np.abs(top - want_top)[fine] <= tol + 4 * U * np.abs(want_top)[fine])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,pad,n_top", [
    (1, 1, 0, 1), (3, 7, 1, 5), (2, 33, 0, 16), (19, 511, 3, 1), (5, 4096, 0, 8), (9, 4097, 5, 16), (1, 131072, 0, 16),
    (3, 131071, 0, 4), (301, 12289, 2, 3), (700, 40, 7, 2), (64, 32003, 0, 0), (2, 300007, 1, 16),
    (500, 32003, 1, 5), (460, 70000, 0, 2)])
def test_logits_match_the_definition(vxk, dtype, rows, vocab, pad, n_top):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows * 31 + vocab)
    l = (torch.randn(rows, vocab + pad, generator=g, device="cuda") * 4).to(_torch_type(dtype))
    rng = np.random.default_rng(vocab)
    tokens = rng.integers(0, vocab, rows)
    tokens[:: 5] = -1 if rows > 1 else tokens[0]
    check(score_logits(vxk, l, vocab, tokens, n_top), l[:, :vocab].double().cpu().numpy(), tokens, n_top)


def test_offsets_beyond_32_bits(vxk):
    """17,000 rows of 131,072 logits: more than 2^31; all but a few rows are even."""
    import torch

    rows, vocab = 17000, 131072
    l = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    torch.manual_seed(9)
    some = [0, 8191, 16383, 16384, 16999]
    l[some] = torch.randn(len(some), vocab, device="cuda").bfloat16() * 3
    got = score_logits(vxk, l, vocab, np.full(rows, 77), 3)
    check([x[some] for x in got], l[some].double().cpu().numpy(), np.full(len(some), 77), 3)
    even = np.setdiff1d(np.arange(rows), some)
    assert np.allclose(got[0][even], -np.log(vocab), rtol=1e-5) and np.allclose(got[1][even], np.log(vocab), rtol=1e-5)
    assert np.array_equal(got[2][even], np.tile([0, 1, 2], (len(even), 1)))


def test_equal_logits_list_the_lowest_index_first(vxk):
    import torch

    vocab = 9001
    l = torch.zeros(4, vocab, device="cuda")          # one value everywhere
    l[1, 1::2] = -0.0                                  # -0 equals 0
    l[2, [8000, 17, 4097, 8999]] = 3.0                 # four ties across strips, warps and CTAs
    l[3] = -torch.arange(vocab, device="cuda", dtype=torch.float32) / 64
    tokens = np.array([0, 5, 17, 3])
    got = score_logits(vxk, l, vocab, tokens, 16)
    check(got, l.double().cpu().numpy(), tokens, 16)
    assert got[2][2, :4].tolist() == [17, 4097, 8000, 8999]


@pytest.mark.parametrize("vocab", [600, 9000])
def test_masked_infinite_and_nan_logits(vxk, vocab):
    import torch

    inf = float("inf")
    torch.manual_seed(3)
    l = torch.randn(8, vocab, device="cuda")
    l[0, ::3] = -inf                  # a masked vocabulary
    l[1, :] = -inf
    l[1, 77] = 2.5                    # one token left: certain
    l[2, :] = -inf                    # none left
    l[3, 400] = float("nan")
    l[4, 9] = inf
    l[5] = torch.finfo(torch.float32).min  # masked by the type's lowest value, everywhere
    l[6] = torch.finfo(torch.float32).min
    l[6, 33] = 1.0
    tokens = np.array([1, 77, 5, 2, 9, 4, 33, 8])
    lp, ent, ids, top = score_logits(vxk, l, vocab, tokens, 3)
    l64 = l.double().cpu().numpy()
    fine = [0, 1, 5, 6, 7]
    check([a[fine] for a in (lp, ent, ids, top)], l64[fine], tokens[fine], 3)
    assert lp[1] == 0 and ent[1] == 0 and ids[1].tolist() == [77, 0, 1]
    for r in (2, 3, 4):
        assert np.isnan(lp[r]) and np.isnan(ent[r])
        assert len(set(ids[r])) == 3 and ids[r].min() >= 0 and ids[r].max() < vocab
    # a masked token has probability 0
    l[0, 3] = -inf
    assert score_logits(vxk, l, vocab, np.array([3] * 8), 0)[0][0] == -inf


def test_optional_outputs_and_rows_behind_the_last(vxk):
    import torch

    torch.manual_seed(1)
    vocab, rows = 5000, 6
    l = torch.randn(rows, vocab, device="cuda")
    head = vxk.Head(dim=64, vocab=vocab)
    tok = torch.arange(rows, dtype=torch.int32, device="cuda")
    full = score_logits(vxk, l, vocab, np.arange(rows), 4, head=head)
    lp, ent, ids, top = outputs(rows + 2, 4)
    s = _stream()
    head.score_logits(l.data_ptr(), F32, vocab, rows, tok.data_ptr(), 4, lp.data_ptr(), 0, 0, 0, s)
    head.score_logits(l.data_ptr(), F32, vocab, rows, 0, 4, 0, ent.data_ptr(), 0, top.data_ptr(), s)
    head.score_logits(l.data_ptr(), F32, vocab, rows, 0, 4, 0, 0, ids.data_ptr(), 0, s)
    head.sync(s)
    for got, want, empty in zip((lp, ent, ids, top), full, (7, 7, -7, 7)):
        assert np.array_equal(got[:rows].cpu().numpy(), want)
        assert bool((got[rows:] == empty).all())
    head.close()


def test_a_token_outside_the_vocabulary_is_reported(vxk):
    import torch

    l = torch.zeros(3, 100, device="cuda")
    head = vxk.Head(dim=64, vocab=100)
    with pytest.raises(vxk.VxkError) as e:
        score_logits(vxk, l, 100, np.array([1, 100, 2]), 0, head=head)
    assert e.value.status == vxk.BACKEND_ERROR and "vocabulary" in str(e.value)
    got = score_logits(vxk, l, 100, np.array([1, 99, 2]), 0, head=head)  # usable afterwards
    assert np.allclose(got[0], -np.log(100.0), atol=1e-5)
    head.close()


def test_same_results_every_time_and_inside_a_graph(vxk):
    import torch

    torch.manual_seed(5)
    vocab, rows = 50000, 37
    l = torch.randn(rows, vocab, device="cuda").bfloat16()
    tokens = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    head = vxk.Head(dim=64, vocab=vocab)
    outs = outputs(rows, 5)

    def call():
        head.score_logits(l.data_ptr(), BF16, vocab, rows, tokens.data_ptr(), 5, *ptrs(outs),
                          torch.cuda.current_stream().cuda_stream)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(vxk.VxkError) as e:  # the first call allocates
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            call()
    assert e.value.status == vxk.INVALID_STATE
    call()
    torch.cuda.synchronize()
    first = [o.clone() for o in outs]
    with torch.cuda.graph(graph, stream=side):
        call()
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))
    l.copy_(torch.randn(rows, vocab, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    got = [o.cpu().numpy() for o in outs]
    check(got, l.double().cpu().numpy(), tokens.cpu().numpy(), 5)
    head.close()


# ---- from hidden rows ---------------------------------------------------------

# The product's logits add two errors: the tensor core's sums (products of 16-bit
# values are exact in fp32; a step adds 16 of them to the running sum, dropping bits
# below 2^-23 = 2 U of it, for 16 steps a 256-column piece in f16 and 32 steps a
# 512-column piece in bf16; the pieces are added in fp32, U each, dim / 256 of them at
# most; giving back the mean of what is dropped adds no more than was dropped at most),
# so at most (32 + dim / 256 + 2) 2 U A with A = sum |x_i w_i| of the logit, and
# none for x's rounding to W's type, which belongs to the definition.  A logit off by D
# moves a log probability by 2 D at most (its own and log s), the entropy by
# 2 D (1 + H + log s...) <= 2 D (2 + the largest |log p| that matters).

def logit_error(x64, w64):
    a = np.abs(x64) @ np.abs(w64).T
    return (32 + x64.shape[1] / 256 + 2) * 2 * U * a.max()


def run_head(vxk, w, x, tokens, n_top, dtype, head=None):
    import torch

    own = head is None
    head = head or vxk.Head(dim=x.shape[1], vocab=len(w), dtype=dtype)
    outs = outputs(len(x), n_top)
    tok = torch.from_numpy(np.asarray(tokens, np.int32)).cuda()
    head.score(w.data_ptr(), x.data_ptr(), len(x), tok.data_ptr(), n_top, *ptrs(outs), _stream())
    head.sync(_stream())
    got = [o.cpu().numpy() for o in outs]
    if own:
        head.close()
    return got


def check_head(got, l64, tokens, n_top, err):
    lp, ent, ids, top = got
    want_lp, want_ent, want_ids, want_top, ts = reference(l64, tokens, n_top)
    tol = (l64.shape[1] + 64) * U + 2 * err
    assert np.all(np.abs(lp - want_lp) <= tol + 4 * U * np.abs(want_lp))
    assert np.all(np.abs(ent - want_ent) <= tol * (3 + 2 * np.abs(ts)))
    for r in range(len(l64)):
        assert len(set(ids[r])) == n_top
        listed = l64[r, ids[r]]
        # the listed logits are the largest ones up to the error, and in order up to it
        assert np.all(np.abs(listed - l64[r, want_ids[r]]) <= 2 * err)
        assert np.all(np.abs(top[r] - (want_top[r] + listed - l64[r, want_ids[r]])) <= tol + 4 * U * np.abs(want_top[r]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,vocab,dim,n_top", [
    (1, 1, 64, 1), (1, 257, 64, 4), (2, 5003, 1280, 5), (37, 1000, 576, 16), (128, 4096, 512, 0), (129, 777, 128, 3),
    (300, 20001, 1088, 8), (2100, 600, 192, 2), (17, 131072, 256, 6)])
def test_hidden_rows_match_the_definition(vxk, dtype, rows, vocab, dim, n_top):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows + vocab + dim)
    t = _torch_type(dtype)
    w = (torch.randn(vocab, dim, generator=g, device="cuda") * dim ** -0.5).to(t)
    x = torch.randn(rows, dim, generator=g, device="cuda") * 4
    tokens = np.random.default_rng(dim).integers(0, vocab, rows)
    if rows > 2:
        tokens[1] = -1
    got = run_head(vxk, w, x, tokens, n_top, dtype)
    x64, w64 = x.to(t).double().cpu().numpy(), w.double().cpu().numpy()
    check_head(got, x64 @ w64.T, tokens, n_top, logit_error(x64, w64))


def test_hidden_rows_agree_with_their_logits(vxk):
    """Equal rows of W give equal logits: the lowest index comes first, across tiles and CTAs."""
    import torch

    torch.manual_seed(2)
    vocab, dim, rows = 9000, 256, 3
    w = (torch.randn(vocab, dim, device="cuda") * 0.01).half()
    x = torch.randn(rows, dim, device="cuda")
    for r, places in enumerate(([8000, 31, 8500], [7000, 4000, 4001], [255, 256, 8999])):
        w[places] = (torch.sign(x[r]) * 0.5).half()
    got = run_head(vxk, w, x, np.zeros(rows), 3, F16)
    assert got[2].tolist() == [[31, 8000, 8500], [4000, 4001, 7000], [255, 256, 8999]]
    assert np.all(got[3][:, 0] == got[3][:, 1]) and np.all(got[3][:, 1] == got[3][:, 2])


def test_hidden_rows_with_nan_stay_apart(vxk):
    import torch

    torch.manual_seed(4)
    vocab, dim, rows = 3001, 192, 70
    w = (torch.randn(vocab, dim, device="cuda") * 0.05).bfloat16()
    x = torch.randn(rows, dim, device="cuda")
    tokens = np.arange(rows)
    clean = run_head(vxk, w, x, tokens, 4, BF16)
    x[3, 5] = float("nan")
    x[64, 0] = float("inf")
    got = run_head(vxk, w, x, tokens, 4, BF16)
    for r in range(rows):
        if r in (3, 64):
            assert np.isnan(got[0][r]) and np.isnan(got[1][r])
        else:
            assert all(np.array_equal(a[r], b[r]) for a, b in zip(got, clean))


def test_hidden_rows_same_every_time_and_inside_a_graph(vxk):
    import torch

    torch.manual_seed(6)
    vocab, dim, rows = 20000, 512, 200
    w = (torch.randn(vocab, dim, device="cuda") * 0.05).half()
    x = torch.randn(rows, dim, device="cuda")
    tokens = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    head = vxk.Head(dim=dim, vocab=vocab)
    outs = outputs(rows, 5)

    def call():
        head.score(w.data_ptr(), x.data_ptr(), rows, tokens.data_ptr(), 5, *ptrs(outs),
                   torch.cuda.current_stream().cuda_stream)

    call()
    head.sync(_stream())
    first = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call()
        call()
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))
    head.sync(_stream())
    head.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lists_of_rising_falling_and_equal_logits(vxk, dtype):
    """Rows whose every strip beats the last (or ties with it), and strips full of candidates."""
    import torch

    vocab, n_top = 70001, 16
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    l = torch.stack([i / 64, -i / 64, torch.zeros_like(i), torch.floor(i / 5000), -torch.floor(i / 5000),
                     torch.where(i % 4096 < 3000, i, -i) / 128, (i % 7 == 3).float(),
                     torch.where(i > 60000, torch.full_like(i, 5.0), i * 0)]).to(_torch_type(dtype))
    tokens = np.arange(8) * 7000
    check(score_logits(vxk, l, vocab, tokens, n_top), l.double().cpu().numpy(), tokens, n_top)


def test_hidden_rows_with_equal_logits(vxk):
    """Zero rows make every logit 0: the lowest indices are listed and the distribution is even."""
    import torch

    vocab, dim, rows = 9001, 128, 140
    w = torch.randn(vocab, dim, device="cuda").half()
    x = torch.randn(rows, dim, device="cuda")
    x[::3] = 0.0
    for n_top in (1, 4, 16):
        lp, ent, ids, top = run_head(vxk, w, x, np.arange(rows), n_top, F16)
        assert np.array_equal(ids[::3], np.tile(np.arange(n_top), (len(ids[::3]), 1)))
        assert np.allclose(lp[::3], -np.log(vocab), rtol=1e-6) and np.allclose(ent[::3], np.log(vocab), rtol=1e-6)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n_top", [2, 5, 16])
def test_lists_of_a_masked_vocabulary(vxk, dtype, n_top):
    """Rows with few logits left: the list goes on with the lowest of the masked indices."""
    import torch

    vocab = 70001
    l = torch.full((4, vocab), -float("inf"), device="cuda")
    l[0, [3, 40000, 69999]] = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    l[1, 65536] = 0.0
    l[2, 20000:20012] = torch.arange(12, device="cuda", dtype=torch.float32)
    l[3, ::4099] = 1.5
    tokens = np.array([3, 65536, 20011, 4099])
    l = l.to(_torch_type(dtype))
    check(score_logits(vxk, l, vocab, tokens, n_top), l.double().cpu().numpy(), tokens, n_top)


def test_rows_with_hardly_a_number(vxk):
    """NaN nearly everywhere: NaN outputs, and a list of indices that differ."""
    import torch

    vocab = 30000
    l = torch.full((2, vocab), float("nan"), device="cuda")
    l[0, 29999] = 1.0
    lp, ent, ids, _ = score_logits(vxk, l, vocab, np.array([5, 5]), 6)
    assert np.all(np.isnan(lp)) and np.all(np.isnan(ent)) and ids[0, 0] == 29999
    for r in range(2):
        assert len(set(ids[r])) == 6 and ids[r].min() >= 0 and ids[r].max() < vocab
