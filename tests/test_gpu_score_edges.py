"""Scores of logits and of hidden rows at the edges of their definition, through the C ABI.

Tolerances.  U = 2^-24 is a rounding of fp32.  Where the logits are exact (sums of integers) their differences
l - m are too, so a log probability is one rounding U |value| from exact behind the error of log s: at most L
terms in one thread and a tree of joins, (L + 64) U.
"""
from __future__ import annotations

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


def _outputs(rows, n_top):
    import torch

    return (torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda"),
            torch.full((rows, n_top), -7, dtype=torch.int32, device="cuda"), torch.full((rows, n_top), 7.0, device="cuda"))


def _score_logits(vxk, l, dtype, vocab, tokens, n_top):
    import torch

    head = vxk.Head(dim=64, vocab=vocab)
    outs = _outputs(len(l), n_top)
    tok = torch.as_tensor(tokens, dtype=torch.int32, device="cuda")
    head.score_logits(l.data_ptr(), dtype, l.stride(0), len(l), tok.data_ptr(), n_top, *(o.data_ptr() for o in outs), _stream())
    head.sync(_stream())
    head.close()
    return outs


def _score(vxk, w, x, dtype, tokens, n_top):
    import torch

    head = vxk.Head(dim=x.shape[1], vocab=len(w), dtype=dtype)
    outs = _outputs(len(x), n_top)
    tok = torch.as_tensor(tokens, dtype=torch.int32, device="cuda")
    head.score(w.data_ptr(), x.data_ptr(), len(x), tok.data_ptr(), n_top, *(o.data_ptr() for o in outs), _stream())
    head.sync(_stream())
    head.close()
    return outs


def _lowest_first(l, n_top):
    import torch

    return torch.sort(l.float(), dim=1, descending=True, stable=True)[1][:, :n_top].int()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_top", [1, 2, 3, 16])
@pytest.mark.parametrize("rows,vocab", [(500, 70001), (460, 70003), (160, 133333)])
def test_ties_with_the_ragged_end_of_a_row(vxk, dtype, n_top, rows, vocab):
    """Runs of many strips, the first of them lower, all behind it equal up to the row's last element."""
    import torch

    l = torch.zeros(rows, vocab, device="cuda")
    l[:, :4096] = -1.0
    l[1::4, : 3 * 4096 + 5] = -1.0
    l[2::4, 20000:] = 1.0
    l[3::4] = torch.randint(0, 3, l[3::4].shape, device="cuda").float()
    l = l.to(_torch_type(dtype))
    ids = _score_logits(vxk, l, dtype, vocab, torch.zeros(rows), n_top)[2]
    assert torch.equal(ids, _lowest_first(l, n_top))
    assert ids[0, 0] == 4096 and ids[1, 0] == 3 * 4096 + 5 and ids[2, 0] == 20000


def _valid(ids, vocab):
    ids = ids.cpu().numpy()
    return ids.min() >= 0 and ids.max() < vocab and all(len(set(r)) == len(r) for r in ids)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [7, 600, 601, 4096, 4097, 30000])
def test_lists_of_rows_with_hardly_a_number(vxk, dtype, vocab):
    """NaN nearly everywhere: indices that exist and differ, the numbers first."""
    import torch

    nan, n_top = float("nan"), min(6, vocab)
    l = torch.full((6, vocab), nan, device="cuda")
    l[1, vocab - 1] = 1.0
    l[2, vocab // 2] = -float("inf")
    l[3, : vocab // 3] = 2.0
    l[4, ::5] = -3.0
    l[5, [2, 4]] = torch.tensor([1.0, 2.0], device="cuda")
    l = l.to(_torch_type(dtype))
    lp, ent, ids, _ = _score_logits(vxk, l, dtype, vocab, torch.zeros(6), n_top)
    assert bool(torch.isnan(lp).all()) and bool(torch.isnan(ent).all())
    assert _valid(ids, vocab)
    assert ids[1, 0] == vocab - 1 and ids[2, 0] == vocab // 2 and ids[3, 0] == 0 and ids[5, :2].tolist() == [4, 2]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_top", [1, 2, 4, 16])
@pytest.mark.parametrize("rows,vocab", [(1, 3001), (70, 40000), (200, 40000)])
def test_lists_of_hidden_rows_over_a_matrix_with_nan(vxk, dtype, n_top, rows, vocab):
    """Whole groups of W's rows NaN beside the largest logits: indices that exist and differ, the numbers first."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    t = _torch_type(dtype)
    x = torch.rand(rows, 64, generator=g, device="cuda") + 0.5
    w = torch.rand(vocab, 64, generator=g, device="cuda").to(t)
    for numbers in ([], list(range(8)), list(range(16, 24)), list(range(0, vocab, 131)), [5, vocab - 1]):
        broken = torch.full_like(w, float("nan"))
        broken[numbers] = w[numbers]
        lp, ent, ids, _ = _score(vxk, broken, x, dtype, torch.zeros(rows), n_top)
        assert bool(torch.isnan(lp).all()) and bool(torch.isnan(ent).all())
        assert _valid(ids, vocab)
        first = min(n_top, len(numbers))
        assert bool(torch.isin(ids[:, :first].cpu(), torch.tensor(numbers, dtype=torch.int32)).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim", [(2, 4096), (17, 2048), (130, 4096), (40, 576)])
@pytest.mark.parametrize("kind", ["few", "early", "dense"])
def test_sums_that_are_exact_stay_exact(vxk, dtype, rows, dim, kind):
    """Integer products whose sums need no more than 12 bits: no step of them rounds, so neither may the logits."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    t, vocab, n_top = _torch_type(dtype), 2000, 8
    w = torch.randint(-8, 9, (vocab, dim), generator=g, device="cuda").to(t)
    x = torch.zeros(rows, dim, device="cuda")
    if kind == "dense":
        x = torch.randint(0, 2, (rows, dim), generator=g, device="cuda").float() * 2 - 1
    else:
        for r in range(rows):
            at = torch.randperm(dim if kind == "few" else 64, generator=g, device="cuda")[:5]
            x[r, at] = 16.0 * torch.randint(-3, 4, (5,), generator=g, device="cuda")
            x[r, at[0]] = 48.0
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    lp, ent, ids, top = _score(vxk, w, x, dtype, tokens, n_top)
    l = x.double() @ w.double().T
    assert float(l.abs().max()) < 4096
    want = torch.log_softmax(l, 1)
    p = want.exp()
    tol = (16 + 64) * U  # 2000 columns over the CTAs are a tile of 32 each, 16 of them a thread's

    def near(got, to):
        return bool(((got.double() - to).abs() <= tol + 1.01 * U * to.abs()).all())

    assert torch.equal(ids, _lowest_first(l, n_top))
    assert near(lp, want.gather(1, tokens[:, None])[:, 0])
    assert near(top, want.gather(1, ids.long()))
    t_s = (p * (l - l.amax(1, keepdim=True))).sum(1).abs()  # the entropy is log s + this
    assert bool(((ent.double() + (p * want).sum(1)).abs() <= tol * (1 + 2 * t_s)).all())


def test_the_first_call_of_a_head_waits_for_no_other_stream(vxk):
    """Its scratch is allocated and cleared while another stream is busy for a second."""
    import time

    import torch

    l = torch.randn(5, 9000, device="cuda")
    tok = torch.zeros(5, dtype=torch.int32, device="cuda")
    outs = _outputs(5, 3)
    side = torch.cuda.Stream()

    def call(head):
        head.score_logits(l.data_ptr(), F32, 9000, 5, tok.data_ptr(), 3, *(o.data_ptr() for o in outs), side.cuda_stream)

    warm, head = vxk.Head(dim=64, vocab=9000), vxk.Head(dim=64, vocab=9000)
    call(warm)
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    torch.cuda.synchronize()
    torch.cuda._sleep(int(1.9e9))  # the legacy stream, about a second
    t = time.perf_counter()
    call(head)
    took = time.perf_counter() - t
    torch.cuda.synchronize()
    busy = time.perf_counter() - t
    assert busy > 0.4 and took < busy / 4, (took, busy)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    warm.close()
    head.close()
