"""vxk_decoder_score: every row of a batch scored (packed prompts, the attention
within them, final norm, log probabilities), and the operators of that pass in a
chain of their own.

Against the oracle's decoder with the packed attention plugged in
(vxk_prompt_rope + vxk_prompt_attention on the oracle's q, k, v), so that everything
else follows the oracle.  As in the tests of vxk_decoder_forward a row whose activations
met no rounding step differently agrees to ~1e-6, and one such event decorrelates it at
the 1e-2 level: logits are held to 5e-2 of the largest, and log probabilities, which
are a logit less a log-sum-exp, to twice that.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

STEP_BAR = 5e-2
EXACT_BAR = 1e-4


def _stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


class PackedAttention:
    """The packed attention for the oracle: whole prompts only."""

    def __init__(self, vxk, max_rows):
        self.prompt = vxk.Prompt(max_seqs=64, max_rows=max_rows, max_position=1024)

    def begin(self, batch):
        self.prompt.plan([n for _, n in batch], cuda_stream=_stream())

    def layer(self, l, q, k, v):
        import torch

        d = [torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda() for x in (q, k, v)]
        h = [torch.empty(x.shape, dtype=torch.float16, device="cuda") for x in d]
        out = torch.empty_like(h[0])
        self.prompt.rope(*(x.data_ptr() for x in d), *(x.data_ptr() for x in h), _stream())
        self.prompt.attention(*(x.data_ptr() for x in h), out.data_ptr(), _stream())
        self.prompt.sync(_stream())
        return out.float().cpu().numpy()

    def end(self):
        pass


def _setup(vxk, tmp_path, seed, untied=False, max_rows=128, max_streams=16, cache=1):
    import decoder_model

    path = tmp_path / f"s{seed}.gguf"
    tensors = decoder_model.build(path, seed, types=decoder_model.Q4_K_M, untied_f16_head=untied)
    g = vxk.Gguf(path)
    pool = vxk.Pool(n_layers=2, n_blocks=24 * max_streams, capacity=512, max_streams=max_streams, max_rows=max_rows,
                    max_position=1024, dtype=cache)
    dec = vxk.Decoder(g, pool, audio_capacity=32, enc_capacity=16)
    g.close()
    return tensors, pool, dec


def _score(dec, tokens, slots, given, n_top):
    import torch

    n = len(tokens)
    outs = (torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda"),
            torch.full((n, n_top), -7, dtype=torch.int32, device="cuda"), torch.full((n, n_top), 7.0, device="cuda"))
    dec.score(tokens, slots, given, n_top, *(o.data_ptr() for o in outs), _stream())
    dec.sync(_stream())
    return [o.cpu().numpy() for o in outs]


def _log_softmax(l):
    m = l.max(-1, keepdims=True)
    return l - m - np.log(np.exp(l - m).sum(-1, keepdims=True))


@pytest.mark.parametrize("untied", [False, True], ids=["q6_k head", "f16 head"])
def test_prompts_are_scored_like_the_oracle(vxk, tmp_path, untied):
    """The prefixes of one text as the streams of one batch: position i of every prefix is the last of prefix i + 1."""
    import vx_decoder as vd

    tensors, pool, dec = _setup(vxk, tmp_path, 31 + untied, untied)
    rng = np.random.default_rng(5)
    text = [int(t) for t in rng.integers(0, dec.info["vocab"], 12)]
    given = [int(t) for t in rng.integers(0, dec.info["vocab"], 12)]
    streams = [pool.open_stream() for _ in text]
    tokens = [t for n in range(1, 13) for t in text[:n]]
    want_given = [t for n in range(1, 13) for t in given[:n]]
    want_given[3] = -1
    pool.plan(streams, list(range(1, 13)), _stream())
    lp, ent, ids, top = _score(dec, tokens, [0] * 78, want_given, 3)
    pool.commit()
    ref = vd.Decoder(tensors, 2, capacity=512, attention=PackedAttention(vxk, 128))
    _, logits, _ = ref.forward([(s, text[: n + 1]) for n, s in enumerate(streams)], np.zeros((78, dec.info["dim"])))
    want = _log_softmax(logits)
    size = np.abs(logits).max()
    errs = []
    r = 0
    for n in range(1, 13):
        for i in range(n):
            e = abs(lp[r] - want[i, given[i]]) if want_given[r] >= 0 else abs(lp[r])
            assert e <= 2 * STEP_BAR * size
            assert np.all(np.abs(top[r] - want[i, ids[r]]) <= 2 * STEP_BAR * size)
            assert np.all(np.sort(logits[i])[-1] - logits[i, ids[r]][0] <= 2 * STEP_BAR * size)
            assert abs(ent[r] - -(np.exp(want[i]) * want[i]).sum()) <= 2 * STEP_BAR * size
            errs.append(e)
            r += 1
    assert lp[3] == 0
    assert np.median(errs) <= 2 * EXACT_BAR * size or min(errs) <= EXACT_BAR * size
    dec.close()
    pool.close()


def test_streams_with_a_past_are_scored_over_the_cache(vxk, tmp_path):
    """Aborted and planned again, the forward's own logits of the last rows give the same log probabilities."""
    import torch

    for untied in (False, True):
        _, pool, dec = _setup(vxk, tmp_path, 41 + untied, untied)
        rng = np.random.default_rng(8)
        vocab = dec.info["vocab"]
        a, b = pool.open_stream(), pool.open_stream()
        amax = torch.zeros(2, dtype=torch.int32, device="cuda")
        pool.plan([a, b], [5, 2], _stream())
        dec.forward([int(t) for t in rng.integers(0, vocab, 7)], [0] * 7, amax.data_ptr(), cuda_stream=_stream())
        dec.sync(_stream())
        pool.commit()
        for n_new in ([3, 4], [1, 1]):
            tokens = [int(t) for t in rng.integers(0, vocab, sum(n_new))]
            given = [int(t) for t in rng.integers(0, vocab, sum(n_new))]
            pool.plan([a, b], n_new, _stream())
            lp, _, ids, top = _score(dec, tokens, [0] * len(tokens), given, 4)
            pool.abort()
            pool.plan([a, b], n_new, _stream())
            logits = torch.empty(2, vocab, device="cuda")
            dec.forward(tokens, [0] * len(tokens), amax.data_ptr(), logits.data_ptr(), cuda_stream=_stream())
            dec.sync(_stream())
            pool.commit()
            l = logits.cpu().numpy().astype(np.float64)
            want = _log_softmax(l)
            for s, r in enumerate((n_new[0] - 1, sum(n_new) - 1)):
                assert abs(lp[r] - want[s, given[r]]) <= EXACT_BAR * np.abs(l).max()
                assert np.all(np.abs(top[r] - want[s, ids[r]]) <= EXACT_BAR * np.abs(l).max())
        dec.close()
        pool.close()


@pytest.mark.parametrize("cache,past", [(0, 0), (1, 5)], ids=["f32 cache", "one stream with a past"])
def test_prompts_that_are_not_packed(vxk, tmp_path, cache, past):
    """Whole prompts of an F32 cache, and ones beside a stream with a past, are attended over the
    cache: the forward's own log probabilities."""
    import torch

    _, pool, dec = _setup(vxk, tmp_path, 71 + past, cache=cache)
    rng = np.random.default_rng(10)
    vocab = dec.info["vocab"]
    streams, lens = [pool.open_stream(), pool.open_stream()], [60, 11]
    amax = torch.zeros(2, dtype=torch.int32, device="cuda")
    if past:
        pool.plan(streams[1:], [past], _stream())
        dec.forward([3] * past, [0] * past, amax.data_ptr(), cuda_stream=_stream())
        dec.sync(_stream())
        pool.commit()
    tokens = [int(t) for t in rng.integers(0, vocab, 71)]
    given = [int(t) for t in rng.integers(0, vocab, 71)]
    pool.plan(streams, lens, _stream())
    lp, _, _, _ = _score(dec, tokens, [0] * 71, given, 0)
    pool.abort()
    pool.plan(streams, lens, _stream())
    logits = torch.empty(2, vocab, device="cuda")
    dec.forward(tokens, [0] * 71, amax.data_ptr(), logits.data_ptr(), cuda_stream=_stream())
    dec.sync(_stream())
    pool.commit()
    l = logits.cpu().numpy().astype(np.float64)
    want = _log_softmax(l)
    for s, r in enumerate((59, 70)):
        assert abs(lp[r] - want[s, given[r]]) <= EXACT_BAR * np.abs(l).max()
    dec.close()
    pool.close()


def test_decoding_goes_on_behind_a_scored_prompt(vxk, tmp_path):
    """The caches of a scored prompt are those of a prefill: the first layer's bytes, and the next token's logits."""
    import torch

    _, pool, dec = _setup(vxk, tmp_path, 51)
    rng = np.random.default_rng(9)
    vocab = dec.info["vocab"]
    a, b = pool.open_stream(), pool.open_stream()
    text = [int(t) for t in rng.integers(0, vocab, 70)]
    pool.plan([a], [70], _stream())
    first = _score(dec, text, [0] * 70, text[1:] + [-1], 0)
    pool.commit()
    pool.plan([b], [70], _stream())
    amax = torch.zeros(2, dtype=torch.int32, device="cuda")
    dec.forward(text, [0] * 70, amax.data_ptr(), cuda_stream=_stream())
    dec.sync(_stream())
    pool.commit()
    for x, y in zip(pool.read_rows(0, a, 0, 70, _stream()), pool.read_rows(0, b, 0, 70, _stream())):
        assert np.array_equal(x, y)
    pool.plan([a, b], [1, 1], _stream())
    logits = torch.empty(2, vocab, device="cuda")
    dec.forward([7, 7], [0, 0], amax.data_ptr(), logits.data_ptr(), cuda_stream=_stream())
    dec.sync(_stream())
    pool.commit()
    assert float((logits[0] - logits[1]).abs().max()) <= STEP_BAR * float(logits.abs().max())
    # the same prompt once more, aborted: no trace, the same scores
    c = pool.open_stream()
    for _ in range(2):
        pool.plan([c], [70], _stream())
        again = _score(dec, text, [0] * 70, text[1:] + [-1], 0)
        pool.abort()
        assert all(np.array_equal(x, y) for x, y in zip(first, again))
    assert pool.ring(c).next_absolute_position == 0
    dec.close()
    pool.close()


def test_refusals(vxk, tmp_path):
    _, pool, dec = _setup(vxk, tmp_path, 61)
    s = pool.open_stream()

    def status(*args):
        with pytest.raises(vxk.VxkError) as e:
            dec.score(*args)
        return e.value.status

    assert status([1], [0], [1], 0) == vxk.INVALID_STATE  # nothing planned
    pool.plan([s], [2], _stream())
    vocab = dec.info["vocab"]
    assert status([1, 2], [0, 0], [1, vocab], 0) == vxk.INVALID_ARGUMENT
    assert status([1, vocab], [0, 0], [1, 1], 0) == vxk.INVALID_ARGUMENT
    assert status([1, 2], [0, 0], [1, 1], 17) == vxk.INVALID_ARGUMENT
    assert status([1, 2], [0, 0], [1, 1], -1) == vxk.INVALID_ARGUMENT
    assert status([1, 2], [0, 0], [1], 0) == vxk.INVALID_ARGUMENT
    dec.score([1, 2], [0, 0], [-1, -1], 0, cuda_stream=_stream())  # nothing wanted is fine
    dec.sync(_stream())
    pool.abort()
    dec.close()
    pool.close()


def test_the_operators_in_a_chain(vxk):
    """Projections' rows -> rope -> attention -> hidden rows -> scores, against the same in 64 bits.

    h = 2^-11 (f16): rounding q, k and v moves a score by at most about 2 h |q||k| scale, a weight by that
    relative to itself, the mean by h for v and h for the output besides; the hidden row is one head-mix of it
    and is rounded once more (h).  With |score| <= 8 that is 20 h of the row, so a logit is off by at most
    25 h sum |x w|, a log probability by twice that.
    """
    import torch

    torch.manual_seed(3)
    lens, heads, kv, dim, vocab = [40, 0, 129, 7], 4, 2, 64, 3000
    rows, width = sum(lens), heads * dim
    q, k, v = (torch.randn(rows, n, dim, device="cuda") * 0.7 for n in (heads, kv, kv))
    w = (torch.randn(vocab, width, device="cuda") * width ** -0.5).half()
    tokens = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    prompt = vxk.Prompt(n_q_heads=heads, n_kv_heads=kv, head_dim=dim, max_seqs=4, max_rows=rows, max_position=200)
    head = vxk.Head(dim=width, vocab=vocab)
    prompt.plan(lens, [3, 0, 0, 50], _stream())
    h = [torch.empty(x.shape, dtype=torch.float16, device="cuda") for x in (q, k, v)]
    out = torch.empty_like(h[0])
    lp = torch.empty(rows, device="cuda")
    prompt.rope(*(x.data_ptr() for x in (q, k, v)), *(x.data_ptr() for x in h), _stream())
    prompt.attention(*(x.data_ptr() for x in h), out.data_ptr(), _stream())
    hidden = out.float().reshape(rows, width)
    head.score(w.data_ptr(), hidden.data_ptr(), rows, tokens.data_ptr(), 0, lp.data_ptr(), 0, 0, 0, _stream())
    prompt.sync(_stream())
    head.sync(_stream())

    def turned(x, first, n, at):
        pos = torch.arange(first, first + n, device="cuda", dtype=torch.float64)
        angle = pos[:, None] * 1e6 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2))
        c = torch.view_as_complex(x[at: at + n].double().reshape(n, -1, dim // 2, 2).contiguous())
        return torch.view_as_real(c * torch.polar(torch.ones_like(angle), angle)[:, None]).reshape(n, -1, dim)

    at, want = 0, []
    for n, first in zip(lens, [3, 0, 0, 50]):
        if n:
            qq, kk = turned(q, first, n, at), turned(k, first, n, at)
            vv = v[at: at + n].double()
            mask = torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1)
            o = [torch.softmax((qq[:, i] @ kk[:, i // 2].T / dim ** 0.5).masked_fill(mask, -float("inf")), -1) @ vv[:, i // 2]
                 for i in range(heads)]
            want.append(torch.stack(o, 1).reshape(n, width))
        at += n
    x = torch.cat(want)
    logits = x @ w.double().T
    ref = torch.log_softmax(logits, 1).gather(1, tokens.long()[:, None])[:, 0]
    tol = 2 * 25 * 2.0 ** -11 * (x.abs() @ w.double().abs().T).amax(1)
    assert bool(((lp.double() - ref).abs() <= tol).all())
    prompt.close()
    head.close()


@pytest.mark.parametrize("cache", [8, 1], ids=["q8_0 cache", "f16 cache"])
@pytest.mark.parametrize("lens", [[60, 11], [30, 25], [128]], ids=str)
def test_scores_are_the_forwards_own(vxk, tmp_path, cache, lens):
    """Whole prompts on both sides of the packed form's 64 rows against the logits that vxk_decoder_forward gives for
    the same batch.  A Q8_0 cache is attended as it is stored, at every size; an f16 cache's packed rows differ from it
    by roundings of q and the probabilities to f16, which one step of the products' activation rounding can carry to the
    1e-2 level."""
    import torch

    _, pool, dec = _setup(vxk, tmp_path, 81, cache=cache)
    rng = np.random.default_rng(12)
    vocab, rows = dec.info["vocab"], sum(lens)
    streams = [pool.open_stream() for _ in lens]
    amax = torch.zeros(len(lens), dtype=torch.int32, device="cuda")
    tokens = [int(t) for t in rng.integers(0, vocab, rows)]
    given = [int(t) for t in rng.integers(0, vocab, rows)]
    pool.plan(streams, lens, _stream())
    lp, ent, ids, top = _score(dec, tokens, [0] * rows, given, 4)
    pool.abort()
    pool.plan(streams, lens, _stream())
    logits = torch.empty(len(lens), vocab, device="cuda")
    dec.forward(tokens, [0] * rows, amax.data_ptr(), logits.data_ptr(), cuda_stream=_stream())
    dec.sync(_stream())
    pool.commit()
    l = logits.cpu().numpy().astype(np.float64)
    want = _log_softmax(l)
    bar = (EXACT_BAR if cache == 8 or rows < 64 else 2 * STEP_BAR) * np.abs(l).max()
    for s, r in enumerate(np.cumsum(lens) - 1):
        assert abs(lp[r] - want[s, given[r]]) <= bar
        assert np.all(np.abs(top[r] - want[s, ids[r]]) <= bar)
        assert abs(ent[r] + (np.exp(want[s]) * want[s]).sum()) <= bar
    dec.close()
    pool.close()


def test_a_decode_step_behind_a_scored_batch_waits_as_before(vxk, tmp_path):
    """vxk_decoder_sync of a step that uses no packed attention makes the calls that it made before any was used."""
    import torch
    from torch.profiler import ProfilerActivity, profile

    _, pool, dec = _setup(vxk, tmp_path, 91)
    a = pool.open_stream()
    amax = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step():
        pool.plan([a], [1], _stream())
        dec.forward([7], [0], amax.data_ptr(), cuda_stream=_stream())
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            dec.sync(_stream())
        pool.commit()
        return sum(e.count for e in p.key_averages() if "Memcpy DtoH" in e.key)

    step()
    before = step()
    assert before > 0
    b = pool.open_stream()
    pool.plan([b], [70], _stream())
    _score(dec, [3] * 70, [0] * 70, [4] * 70, 0)
    pool.commit()
    assert step() == before
    dec.close()
    pool.close()


def test_handles_of_their_own_on_several_threads(vxk):
    """Eight host threads, each with a prompt, a head and a stream of its own, make and use them at once."""
    import threading

    import torch

    lens, heads, dim, vocab = [40, 90], 4, 64, 5000
    rows, width = sum(lens), heads * dim
    torch.manual_seed(4)
    q, k, v = (torch.randn(rows, n, dim, device="cuda").half() for n in (heads, 2, 2))
    w, tokens = torch.randn(vocab, width, device="cuda").half(), torch.arange(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    got, errors, start = [None] * 8, [], threading.Barrier(8)

    def work(i):
        try:
            s = torch.cuda.Stream()
            out, x, lp = (torch.empty(n, dtype=t, device="cuda") for n, t in
                          ((q.shape, torch.float16), ((rows, width), torch.float32), (rows, torch.float32)))
            start.wait()
            prompt = vxk.Prompt(n_q_heads=heads, n_kv_heads=2, head_dim=dim, max_seqs=2, max_rows=rows, max_position=0)
            head = vxk.Head(dim=width, vocab=vocab)
            prompt.plan(lens, cuda_stream=s.cuda_stream)
            with torch.cuda.stream(s):
                prompt.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), s.cuda_stream)
                x.copy_(out.reshape(rows, width))
                head.score(w.data_ptr(), x.data_ptr(), rows, tokens.data_ptr(), 0, lp.data_ptr(), cuda_stream=s.cuda_stream)
            prompt.sync(s.cuda_stream)
            head.sync(s.cuda_stream)
            got[i] = lp.cpu()
            prompt.close()
            head.close()
        except Exception as e:  # noqa: BLE001 - reported by the test
            errors.append(e)
            start.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(torch.equal(g, got[0]) for g in got) and bool(torch.isfinite(got[0]).all())


def test_scoring_inside_a_capture_is_refused(vxk, tmp_path):
    """It uploads what the host gives it, which a replay would not do again: refused, and usable afterwards."""
    import torch

    _, pool, dec = _setup(vxk, tmp_path, 95)
    a = pool.open_stream()
    side = torch.cuda.Stream()
    for rows in (2, 70):
        for warm in (False, True):
            pool.plan([a], [rows], _stream())
            torch.cuda.synchronize()
            with pytest.raises(vxk.VxkError) as e:
                with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                    dec.score([3] * rows, [0] * rows, [4] * rows, 0, cuda_stream=torch.cuda.current_stream().cuda_stream)
            assert e.value.status == vxk.INVALID_STATE
            first = _score(dec, [3] * rows, [0] * rows, [4] * rows, 2)
            again = _score(dec, [3] * rows, [0] * rows, [4] * rows, 2)
            assert all(np.array_equal(x, y) for x, y in zip(first, again))
            pool.abort()
    dec.close()
    pool.close()
