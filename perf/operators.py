"""Scoring packed prompts: the cases by which its four operators are measured.

A recogniser's hypotheses or prompts lie packed behind one another, a row per token, and each
token gets its log probability.  The operators that such a pass needs besides the products:

  rope    the q and k rows of the projections rotated to their positions (pairs (2i, 2i + 1)) and
          rounded, with v, to the 16-bit rows that the attention reads
  attend  attention within every packed sequence, causal, windowed or whole, with grouped heads
  logits  log probability of each row's given token, entropy and the top alternatives, from logits
  head    the same from hidden rows and the embedding matrix, the logits never written

`run` is the plain form where `own` is false and the framework's call where it is true.
"""
import math
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GGML = {"f16": 1, "bf16": 30, "f32": 0}
THETA = 1e6


# ---------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one stream's 38-token prompt: the smallest call, all launch latency
        dict(name="rope 38", op="rope", lens="38", first=0, heads=32, kv=8, dim=128, type="f16"),
        # a training-size batch of ragged transcripts at far positions, bandwidth
        dict(name="rope ragged 13k", op="rope", lens="4096,1,511,0,2048,1777,385,3000,38,1100,77", first=30000,
             heads=32, kv=8, dim=128, type="bf16"),
        # the 38-token prompts of 64 streams that open together
        dict(name="attend 64x38", op="attend", lens=",".join(["38"] * 64), heads=32, kv=8, dim=128, type="f16",
             causal=True, window=0),
        # hypotheses of every length, from nothing to two thousand tokens
        dict(name="attend ragged", op="attend", lens="2011,1,383,0,957,64,129,1500,38,700,5,2048,311,1211,450,127",
             heads=32, kv=8, dim=128, type="bf16", causal=True, window=0),
        # one long transcript, as long as the decoder's cache
        dict(name="attend 8192", op="attend", lens="8192", heads=32, kv=8, dim=128, type="f16", causal=True, window=0),
        # four 30-second windows of encoder frames, every frame attending to every other
        dict(name="attend 4x1500 whole", op="attend", lens="1500,1500,1500,1500", heads=20, kv=20, dim=64, type="bf16",
             causal=False, window=0),
        # a decode step of four streams: the alternatives of one token each
        dict(name="logits 4", op="logits", rows=4, vocab=131072, pad=0, type="f32", top=5),
        # a long transcript's logits
        dict(name="logits 600", op="logits", rows=600, vocab=131072, pad=0, type="f32", top=8),
        # 16-bit logits of an odd vocabulary in padded rows: ties everywhere
        dict(name="logits 333 odd", op="logits", rows=333, vocab=32003, pad=5, type="bf16", top=16),
        # a few rows over a small matrix: latency
        dict(name="head 5 small", op="head", rows=5, vocab=32000, dim=1280, type="f16", top=4),
        # one 30-second window's tokens over the whole vocabulary: the matrix is read once
        dict(name="head 100", op="head", rows=100, vocab=131072, dim=2048, type="bf16", top=4),
        # a batch of transcripts: the matrix product bounds it
        dict(name="head 2000", op="head", rows=2000, vocab=131072, dim=4096, type="bf16", top=4),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_lens(rng, most, longest):
    lens, total = [], 0
    for _ in range(_log_uniform(rng, 1, 64)):
        n = 0 if rng.random() < 0.05 else _log_uniform(rng, 1, longest)
        if total + n <= most:
            lens.append(n)
            total += n
    return lens if total else [rng.randint(1, 64)]


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "logits", "head"])
    kind = rng.choice(["f16", "bf16"])
    if op in ("rope", "attend"):
        dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8, 20 if dim == 64 else 8])
        heads = kv * (rng.choice([1, 2, 3, 4, 6, 8]) if kv <= 4 else rng.choice([1, 2, 4]) if kv == 8 else 1)
        if op == "rope":
            lens = _draw_lens(rng, 13000, 6000)
            return dict(op=op, lens=",".join(map(str, lens)), first=_log_uniform(rng, 1, 60000) - 1, heads=heads, kv=kv,
                        dim=dim, type=kind)
        lens = _draw_lens(rng, 10000, _log_uniform(rng, 32, 5000))
        while len(lens) * max(lens) ** 2 > 4096 ** 2 * 3:  # what the plain form pads to
            lens.remove(max(lens))
        causal = rng.random() < 0.75
        window = _log_uniform(rng, 1, 1500) if causal and rng.random() < 0.3 else 0
        return dict(op=op, lens=",".join(map(str, lens)), heads=heads, kv=kv, dim=dim, type=kind, causal=causal,
                    window=window)
    if op == "logits":
        vocab = _log_uniform(rng, 50, 131072)
        rows = _log_uniform(rng, 1, min(20000, 600 * 131072 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8, 61]),
                    type=rng.choice(["f32", "f32", kind]), top=rng.randint(0, 16))
    return dict(op=op, rows=_log_uniform(rng, 1, 2000), vocab=_log_uniform(rng, 1000, 131072),
                dim=64 * rng.randint(16, 64), type=kind, top=rng.randint(0, 4))


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def work(case):
    if case["op"] == "rope":
        n = sum(_lens(case)) * (case["heads"] + 2 * case["kv"]) * case["dim"]
        return {"bytes": n * 4 + n * 2, "flops": n * 3}
    if case["op"] == "attend":
        rows, pairs = sum(_lens(case)), 0
        for n in _lens(case):
            if not case["causal"]:
                pairs += n * n
            else:
                w = min(n, case["window"] or n)
                pairs += w * (w + 1) // 2 + (n - w) * w
        return {"bytes": rows * (2 * case["heads"] + 2 * case["kv"]) * case["dim"] * 2,
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    outputs = case["rows"] * (4 + 4 + 4 + 8 * case["top"])
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + outputs, "flops": 5 * n}
    return {"bytes": case["vocab"] * case["dim"] * 2 + case["rows"] * case["dim"] * 4 + outputs,
            "flops": 2 * case["rows"] * case["vocab"] * case["dim"] + 5 * case["rows"] * case["vocab"]}


# --------------------------------------------------------------------------------------- inputs

def _framework():
    if "voxtral.cpp_b200" not in sys.path:
        sys.path.insert(0, "voxtral.cpp_b200")
    import vxk

    return vxk


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    def integers(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] in ("rope", "attend"):
        lens, dim, t = _lens(case), case["dim"], TYPES[case["type"]]
        rows, heads, kv = sum(lens), case["heads"], case["kv"]
        first = [case.get("first", 0)] * len(lens)
        s["lens"] = lens
        # where each row stands in its sequence, and each sequence's rows in a padded batch
        counts = torch.tensor(lens, device="cuda")
        starts = torch.cumsum(counts, 0) - counts
        s["within"] = torch.arange(rows, device="cuda") - torch.repeat_interleave(starts, counts)
        s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), counts)
        if case["op"] == "rope":
            s["positions"] = s["within"] + case["first"]
            s["q"], s["k"], s["v"] = normal(rows, heads, dim), normal(rows, kv, dim), normal(rows, kv, dim)
            s["outs"] = tuple(torch.empty(x.shape, dtype=t, device="cuda") for x in (s["q"], s["k"], s["v"]))
        else:
            # scores of a few units, as trained heads have them
            s["q"], s["k"] = normal(rows, heads, dim, std=2.0, dtype=t), normal(rows, kv, dim, dtype=t)
            s["v"] = normal(rows, kv, dim, dtype=t)
            s["out"] = torch.empty(rows, heads, dim, dtype=t, device="cuda")
        if own:
            vxk = _framework()
            s["prompt"] = vxk.Prompt(
                device=torch.cuda.current_device(), n_q_heads=heads, n_kv_heads=kv, head_dim=dim,
                max_seqs=len(lens), max_rows=rows, dtype=GGML[case["type"]], rope_theta=THETA,
                max_position=(max(lens) + case["first"]) if case["op"] == "rope" else 0,
                causal=int(case.get("causal", True)), window=case.get("window", 0))
            s["prompt"].plan(lens, first, _stream())
        return s

    rows, vocab, top, t = case["rows"], case["vocab"], case["top"], TYPES[case["type"]]
    if case["op"] == "logits":
        ld = vocab + case["pad"]
        s["logits"] = normal(rows, ld, std=2.5, dtype=t)
        # a model is sure of most of its tokens
        peak = integers(0, vocab, rows, 1)
        s["logits"].scatter_(1, peak, 8 + normal(rows, 1, std=4.0, dtype=t))
        s["tokens"] = torch.where(integers(0, 4, rows) > 0, peak[:, 0], integers(0, vocab, rows)).int()
        dim = 64
    else:
        dim = case["dim"]
        s["w"] = normal(vocab, dim, std=dim ** -0.5, dtype=t)
        # hidden rows that point at a few tokens, each well behind the one before it
        chosen = integers(0, vocab, rows, 4)
        share = 12 * 0.7 ** torch.arange(4, device="cuda", dtype=torch.float32)
        s["x"] = torch.einsum("j,rjd->rd", share, s["w"][chosen].float()) + normal(rows, dim, std=0.1)
        s["tokens"] = torch.where(integers(0, 4, rows) > 0, chosen[:, 0], integers(0, vocab, rows)).int()
    s["outs"] = (torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
                 torch.empty(rows, top, dtype=torch.int32, device="cuda"), torch.empty(rows, top, device="cuda"))
    if own:
        s["head"] = _framework().Head(device=torch.cuda.current_device(), dim=dim, vocab=vocab,
                                      dtype=GGML[case["type"]] if case["op"] == "head" else GGML["f16"])
    return s


# -------------------------------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case = s["case"]
    if case["op"] == "rope":
        q, k, v = s["outs"]
        s["prompt"].rope(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), q.data_ptr(), k.data_ptr(),
                         v.data_ptr(), _stream())
        return s["outs"]
    if case["op"] == "attend":
        s["prompt"].attention(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), _stream())
        return s["out"]
    logprob, entropy, ids, top = s["outs"]
    outs = (logprob.data_ptr(), entropy.data_ptr(), ids.data_ptr(), top.data_ptr())
    if case["op"] == "logits":
        s["head"].score_logits(s["logits"].data_ptr(), GGML[case["type"]], s["logits"].stride(0), case["rows"],
                               s["tokens"].data_ptr(), case["top"], *outs, _stream())
    else:
        s["head"].score(s["w"].data_ptr(), s["x"].data_ptr(), case["rows"], s["tokens"].data_ptr(), case["top"], *outs,
                        _stream())
    return s["outs"]


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(x.shape)


def _score(logits, tokens, top):
    """Log probabilities of the tokens, entropies, and the `top` largest (the lowest index first among equals)."""
    below = logits - logits.amax(1, keepdim=True)
    e = below.exp()
    total = e.sum(1)
    entropy = total.log() - (e * below).sum(1) / total
    logprobs = below - total.log()[:, None]
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top] if top else logits.new_empty(len(logits), 0).long()
    return logprobs.gather(1, tokens.long()[:, None])[:, 0], entropy, ids.int(), logprobs.gather(1, ids)


def _run_plain(s):
    case = s["case"]
    if case["op"] == "rope":
        t, half = TYPES[case["type"]], case["dim"] // 2
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        angle = s["positions"].double()[:, None] * THETA ** (-i / half)  # far positions need 64 bits
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        return _rotate(s["q"], cos, sin).to(t), _rotate(s["k"], cos, sin).to(t), s["v"].to(t)
    if case["op"] == "attend":
        n, longest, group = len(s["lens"]), max(s["lens"]), case["heads"] // case["kv"]
        at = (s["seq"], s["within"])

        def padded(x):
            y = x.new_zeros(n, longest, *x.shape[1:], dtype=torch.float32)
            y[at] = x.float()
            return y.transpose(1, 2)

        q, k, v = padded(s["q"]), padded(s["k"]), padded(s["v"])
        q = q.reshape(n, case["kv"], group, longest, case["dim"])
        scores = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(case["dim"] ** -0.5)
        i = torch.arange(longest, device="cuda")
        allowed = i[None, None, :] < torch.tensor(s["lens"], device="cuda")[:, None, None]
        if case["causal"]:
            back = i[:, None] - i[None, :]
            allowed = allowed & (back >= 0) & (back < (case["window"] or longest))
        scores.masked_fill_(~allowed[:, None, None], -math.inf)
        scores -= scores.amax(-1, keepdim=True).clamp_min(-1e30)
        scores.exp_()
        total = scores.sum(-1, keepdim=True)
        out = torch.matmul(scores, v[:, :, None]) / total
        out = out.reshape(n, case["heads"], longest, case["dim"]).transpose(1, 2)
        return out[at].to(s["q"].dtype)
    if case["op"] == "logits":
        return _score(s["logits"][:, : case["vocab"]].float(), s["tokens"], case["top"])
    x = s["x"].to(s["w"].dtype).float()  # hidden rows take the matrix's type, as in the greedy head
    return _score(torch.matmul(x, s["w"].float().t()), s["tokens"], case["top"])


# ------------------------------------------------------------------------------ in 64 bits, apart

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        half = case["dim"] // 2
        turns = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.zeros((), dtype=torch.float64, device="cuda"))
        freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(THETA) / half))
        turns = turns * torch.exp(1j * torch.outer(s["positions"].double(), freq))[:, None]
        spin = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(*x.shape[:-1], half, 2)) * turns).reshape(x.shape)  # noqa: E731
        return spin(s["q"]), spin(s["k"]), s["v"].double()
    if case["op"] == "attend":
        out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        group = case["heads"] // case["kv"]
        for n in s["lens"]:
            i = torch.arange(n, device="cuda")
            bias = torch.zeros(n, n, dtype=torch.float64, device="cuda")
            if case["causal"]:
                bias[i[:, None] < i[None, :]] = -math.inf
                if case["window"]:
                    bias[i[:, None] - i[None, :] >= case["window"]] = -math.inf
            for h in range(case["heads"] if n else 0):
                q, k, v = (x[at : at + n, j].double() for x, j in ((s["q"], h), (s["k"], h // group), (s["v"], h // group)))
                out[at : at + n, h] = torch.softmax(q @ k.t() / math.sqrt(case["dim"]) + bias, -1) @ v
            at += n
        return out
    parts = []
    for r in range(0, case["rows"], 256):
        if case["op"] == "logits":
            l = s["logits"][r : r + 256, : case["vocab"]].double()
        else:
            l = s["x"][r : r + 256].to(s["w"].dtype).double() @ s["w"].double().t()
        lp = torch.log_softmax(l, 1)
        best = torch.sort(l, dim=1, descending=True, stable=True)[1][:, : case["top"]]
        given = s["tokens"][r : r + 256].long()[:, None]
        parts.append((lp.gather(1, given)[:, 0], torch.special.entr(lp.exp()).sum(1), best.int(), lp.gather(1, best)))
    return tuple(torch.cat(p) for p in zip(*parts))
