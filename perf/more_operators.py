"""Serving from a cache held in 4 bits, as measurable cases.

A step of an engine whose cache is held in 4 bits is made of four operators:

  prompt  causal attention of whole prompts, packed, over their own keys and values
  store   keys and values into the 4-bit pool (and the values they stand for, back)
  attend  attention of single tokens and chunks over the 4-bit pool
  logits  penalties, biases and grammar masks before a token is chosen

Each case is one call of one of them (a store and its reading back are two) at
shapes of this repository's configurations, tests and benchmark, or generic ones of
the same range.

What a pool of 4 bits holds: 32 neighbouring channels of a token's key (value) in
one head are a group, with m its smallest element in f16 and
s = f16((largest - m) / 15), the subtraction and division in f32; element x is held
as c = round((x - m) / s) in 0 .. 15 (ties to even, 0 where s = 0) and stands for
m + s c.
"""
import math
import os
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
GROUP = 32

LLAMA_1B = (32, 8, 64)
TINYLLAMA = (32, 4, 64)
LLAMA_8B = (32, 8, 128)
LLAMA_70B = (64, 8, 128)
QWEN_05B = (14, 2, 64)
WIDE = (16, 8, 256)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _prompt(name, model, dtype, seqs, lo, hi, packed, lens):
    h, kv, hd = model
    return {"name": name, "kind": "prompt", "dtype": dtype, "heads": h, "kv_heads": kv,
            "head_dim": hd, "seqs": seqs, "lo": lo, "hi": hi, "packed": packed, "lens": lens}


def _store(name, model, dtype, tokens, spread, lens, block=16):
    h, kv, hd = model
    return {"name": name, "kind": "store", "dtype": dtype, "kv_heads": kv, "head_dim": hd,
            "tokens": tokens, "spread": spread, "block": block, "lens": lens}


def _attend(name, model, dtype, seqs, ctx_lo, ctx_hi, q_lo, q_hi, lens, block=16):
    h, kv, hd = model
    return {"name": name, "kind": "attend", "dtype": dtype, "heads": h, "kv_heads": kv,
            "head_dim": hd, "block": block, "seqs": seqs, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "q_lo": q_lo, "q_hi": q_hi, "lens": lens}


def _logits(name, dtype, batch, vocab, hist_lo, hist_hi, bias, masks, lens):
    return {"name": name, "kind": "logits", "dtype": dtype, "batch": batch, "vocab": vocab,
            "hist_lo": hist_lo, "hist_hi": hist_hi, "bias": bias, "masks": masks, "lens": lens}


def listed():
    return [
        # A few short chat turns arrive at once: latency.
        _prompt("prompt_tiny", TINYLLAMA, "f16", 5, 1, 90, True, 41),
        # The engine's own type, a ratio of 7, paragraphs.
        _prompt("prompt_qwen_f32", QWEN_05B, "f32", 4, 200, 900, False, 42),
        # An admission round of an 8B server; q, k and v are columns of one projection.
        _prompt("prompt_8b_packed", LLAMA_8B, "bf16", 6, 300, 2600, True, 43),
        # One long document.
        _prompt("prompt_70b_long", LLAMA_70B, "bf16", 1, 8000, 8000, False, 44),
        # A decode step's new tokens, one in each of 256 sequences.
        _store("store_8b_step", LLAMA_8B, "bf16", 256, True, 45),
        # Prompts of some 60 thousand tokens in all, block after block.
        _store("store_70b_prompts", LLAMA_70B, "f16", 60001, False, 46),
        # Eight chats on a small model: few rows, the work has to be spread and joined.
        _attend("attend_1b_8", LLAMA_1B, "f16", 8, 600, 9000, 1, 1, 47),
        # The decode step of the headline batch.
        _attend("attend_8b_256", LLAMA_8B, "bf16", 256, 512, 4096, 1, 1, 48),
        # Long contexts, what a cache of 4 bits is for.
        _attend("attend_8b_long", LLAMA_8B, "bf16", 48, 12000, 32000, 1, 1, 49),
        # Decodes, drafted chunks and prompt chunks over earlier contexts in one call.
        _attend("attend_70b_chunks", LLAMA_70B, "bf16", 12, 500, 8000, 1, 200, 50),
        # A few requests, f32 logits.
        _logits("logits_f32_6", "f32", 6, 32000, 1, 2000, 20, 2, 51),
        # A full batch, half of it under a grammar, long histories.
        _logits("logits_bf16_128", "bf16", 128, 128256, 50, 8000, 300, 16, 52),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: any of the models, types and options, sizes
    spread over their logarithm."""
    kind = rng.choice(["prompt", "prompt", "store", "attend", "attend", "attend", "logits"])
    lens = rng.randrange(1 << 20)
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    model = rng.choice([LLAMA_1B, TINYLLAMA, LLAMA_8B, LLAMA_70B, QWEN_05B, WIDE])
    h, kv, hd = model
    block = rng.choice([16, 16, 16, 32, 64])
    if kind == "prompt":
        hi = _log(rng, 1, 4000 if dtype == "f32" else 8000)
        most = (1 << 30) if dtype == "f32" else (4 << 30)  # (scores of the padded batch)
        seqs = _log(rng, 1, max(1, min(40, most // (h * hi * hi))))
        c = _prompt("", model, dtype, seqs, max(1, int(hi * rng.random())), hi,
                    rng.random() < 0.5, lens)
    elif kind == "store":
        c = _store("", model, dtype, _log(rng, 1, 120_000_000 // (kv * hd * 2)),
                   rng.random() < 0.5, lens, block)
    elif kind == "attend":
        hi = _log(rng, 1, 32000)
        q = rng.choice([1, 1, 1, 5, _log(rng, 1, 500)])
        rows = 1_000_000 if q <= 8 else 60_000_000 // (h * q)
        seqs = _log(rng, 1, max(1, min(256, min(rows, 1_500_000 * 8 * 128 // (kv * hd)) // (hi + q))))
        c = _attend("", model, dtype, seqs, int(hi * rng.random()), hi, rng.randint(1, q), q, lens,
                    block)
    else:
        vocab = rng.choice([32000, 128256, _log(rng, 100, 128000)])
        hist = _log(rng, 1, 8000)
        c = _logits("", dtype, _log(rng, 1, 64 if dtype == "f32" else 128), vocab,
                    int(hist * rng.random()), hist, rng.choice([0, _log(rng, 1, 300)]),
                    rng.choice([0, _log(rng, 1, 16)]), lens)
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _ints(case, salt, n, lo, hi):
    r = random.Random(case["lens"] * 131 + salt)
    return [r.randint(lo, hi) for _ in range(n)]


def _prompts(case):
    return _ints(case, 1, case["seqs"], case["lo"], case["hi"])


def _q_lens(case):
    return _ints(case, 2, case["seqs"], case["q_lo"], case["q_hi"])


def _ctx_lens(case):
    """Keys of a sequence, its new tokens among them."""
    return [c + q for c, q in zip(_ints(case, 1, case["seqs"], case["ctx_lo"], case["ctx_hi"]),
                                  _q_lens(case))]


def _hist(case):
    return _ints(case, 3, case["batch"], case["hist_lo"], case["hist_hi"])


def _biased(case):
    return _ints(case, 4, case["batch"], 0, case["bias"])


def _cu(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _centres(g, kv, hd):
    """Channels of keys have centres of their own, a few of them far out."""
    c = _normal(g, (kv, hd))
    far = torch.rand((kv, hd), generator=g, device=DEV) < 0.03
    return torch.where(far, c * 6.0, c * 0.7)


def _pieces(g, n, kv, hd, dtype):
    """Keys and values of tokens 0 .. n - 1 in pieces of at most 65,536 tokens."""
    c = _centres(g, kv, hd)
    for i in range(0, n, 1 << 16):
        m = min(n - i, 1 << 16)
        yield i, m, (_normal(g, (m, kv, hd)) + c).to(dtype), _normal(g, (m, kv, hd), dtype)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tables(g, case):
    """Block tables over a shuffled pool, and its number of blocks."""
    bs = case["block"]
    need = [-(-c // bs) for c in _ctx_lens(case)]
    nb = int(1.1 * sum(need)) + 1
    perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    tables = torch.zeros((len(need), max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    return tables, nb


def _inputs(case, seed):
    """The plain tensors of a case, but for the keys and values of a pool."""
    g, d = _gen(seed), {}
    if case["kind"] == "logits":
        b, v, hist, bias = case["batch"], case["vocab"], _hist(case), _biased(case)
        x = _normal(g, (b, v)) * 3.0
        x[:, v // 2] = -math.inf  # a token that no request may take
        d["logits"] = x.to(DT[case["dtype"]])
        n = sum(hist)
        # words come back: a few tokens make up most of a text
        u = torch.rand(n, generator=g, device=DEV)
        d["tokens"] = (v * u ** 4).long().clamp(max=v - 1).to(torch.int32)
        d["cu"] = _i32(_cu(hist))
        d["prompt"] = _i32([int(m * f) for m, f in zip(hist, [0.0, 0.3, 1.0, 0.7] * len(hist))])
        d["rep"] = torch.rand(b, generator=g, device=DEV) * 0.4 + 0.9
        d["rep"][::3] = 1.0
        d["pres"] = torch.rand(b, generator=g, device=DEV) * 2.0 - 0.5
        d["freq"] = torch.rand(b, generator=g, device=DEV) * 0.6 - 0.1
        m = sum(bias)
        d["bias_tokens"] = torch.randint(0, v, (m,), generator=g, device=DEV).to(torch.int32)
        d["bias_values"] = _normal(g, (m,)) * 4.0
        d["cu_bias"] = _i32(_cu(bias))
        words = (v + 31) // 32
        if case["masks"]:
            allow = torch.rand((case["masks"], words * 32), generator=g, device=DEV)
            share = torch.rand((case["masks"], 1), generator=g, device=DEV) ** 3  # most are narrow
            bit = torch.ones(1, dtype=torch.int64, device=DEV) << torch.arange(32, device=DEV)
            w = ((allow < share).view(-1, words, 32) * bit).sum(2)
            d["mask"] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
            d["mask_rows"] = _i32([m if m < case["masks"] else -1 for m in
                                   _ints(case, 5, b, 0, 2 * case["masks"])])
        else:
            d["mask"] = d["mask_rows"] = None
        d["out"] = torch.empty_like(d["logits"])
        return d
    kv, hd, dt = case["kv_heads"], case["head_dim"], DT[case["dtype"]]
    if case["kind"] == "prompt":
        h, n = case["heads"], _prompts(case)
        x = _normal(g, (sum(n), h + 2 * kv, hd), dt)
        x[:, h:h + kv] += _centres(g, kv, hd).to(dt) * 0.3
        q, k, v = x.split((h, kv, kv), 1)  # columns of one projection, or tensors of their own
        d["q"], d["k"], d["v"] = (q, k, v) if case["packed"] else \
            (q.contiguous(), k.contiguous(), v.contiguous())
        d["cu"] = _i32(_cu(n))
        return d
    if case["kind"] == "store":
        n, bs = case["tokens"], case["block"]
        d["num_blocks"] = n + 3 if case["spread"] else int(1.2 * n) // bs + 3
        perm = torch.randperm(d["num_blocks"], generator=g, device=DEV)
        at = torch.arange(n, device=DEV)
        if case["spread"]:
            d["slots"] = perm[:n] * bs + at % bs
        else:
            d["slots"] = perm[at // bs] * bs + at % bs
        d["slots"] = d["slots"].to(torch.int32)
        c = _centres(g, kv, hd)
        d["k"] = (_normal(g, (n, kv, hd)) + c).to(dt)
        d["v"] = _normal(g, (n, kv, hd), dt)
        return d
    ctx, q = _ctx_lens(case), _q_lens(case)
    d["tables"], d["num_blocks"] = _tables(g, case)
    d["ctx"] = _i32(ctx)
    d["cu"] = _i32(_cu(q)) if max(q) > 1 or min(q) < 1 else None
    d["q"] = _normal(g, (sum(q), case["heads"], hd), dt)
    return d


def _hold(x):
    """x (n, kv, hd) in 4 bits: codes, two to a byte, and (m, s) of each group."""
    y = x.unflatten(2, (-1, GROUP))
    low, high = y.amin(3), y.amax(3)
    m = low.half()
    s = ((high.float() - m.float()) / torch.full_like(high, 15.0, dtype=torch.float32)).half()
    step = torch.where(s > 0, s, 1.0).double()[..., None]
    c = ((y.double() - m.double()[..., None]) / step).round().clamp(0, 15)
    c = torch.where(s[..., None] > 0, c, 0.0).to(torch.uint8).flatten(2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack((m, s), 3)


def _stands_for(codes, ms, dtype):
    """The values that codes and (m, s) stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, GROUP))
    return (ms[..., 0, None].to(dtype) + ms[..., 1, None].to(dtype) * c.to(dtype)).flatten(-2)


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case["kind"] == "prompt":
        d["longest"] = max(_prompts(case))
    if case["kind"] in ("store", "attend"):
        kv, hd, bs, nb = case["kv_heads"], case["head_dim"], case["block"], d["num_blocks"]
        if own:  # the pool that the program keeps
            d["cache"] = _package().PagedKvCache(1, nb, bs, kv, hd, _package().Q4)
            d["pool"] = d["cache"].layer(0)
        else:
            d["held"] = [(torch.zeros((nb * bs, kv, hd // 2), dtype=torch.uint8, device=DEV),
                          torch.zeros((nb * bs, kv, hd // GROUP, 2), dtype=torch.float16,
                                      device=DEV)) for _ in range(2)]
    if case["kind"] == "attend":
        d["q_max"], d["ctx_max"] = max(_q_lens(case)), max(_ctx_lens(case))
        for i, m, k, v in _pieces(_gen(seed + (1 << 40)), nb * bs, kv, hd, DT[case["dtype"]]):
            if own:
                d["pool"].q4_append(k, v, torch.arange(i, i + m, dtype=torch.int32, device=DEV))
            else:
                for (codes, ms), x in zip(d["held"], (k, v)):
                    codes[i:i + m], ms[i:i + m] = _hold(x)
        torch.cuda.synchronize()
    return d


def _package():
    at = os.path.join(os.getcwd(), "ai-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pagedkv
    return pagedkv


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s, kind)
    return {"prompt": _plain_prompt, "store": _plain_store, "attend": _plain_attend,
            "logits": _plain_logits}[kind](s, s["case"])


def _own(s, kind):
    if kind == "prompt":
        return _package().prompt_attention(s["q"], s["k"], s["v"], s["cu"], max_len=s["longest"])
    if kind == "store":
        s["pool"].q4_append(s["k"], s["v"], s["slots"])
        k, v = s["pool"].q4_gather(s["slots"], out_dtype=s["k"].dtype)
        return {"k": k, "v": v}
    if kind == "attend":
        return s["pool"].q4_attention(s["q"], s["tables"], s["ctx"], cu_q_lens=s["cu"],
                                      max_q_len=s["q_max"], max_context_len=s["ctx_max"])
    return _package().adjust_logits(
        s["logits"], tokens=s["tokens"], cu_tokens=s["cu"], prompt_lens=s["prompt"],
        repetition=s["rep"], presence=s["pres"], frequency=s["freq"],
        bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], cu_bias=s["cu_bias"],
        mask=s["mask"], mask_rows=s["mask_rows"], out=s["out"])


def _softmax_rows(x, ok):
    """softmax over the last axis of scores x where ok; rows without any are zero."""
    x = x.masked_fill_(~ok, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_prompt(s, case):
    """Token i of a prompt attends its tokens 0 .. i; the batch is padded."""
    h, kv, hd, n = case["heads"], case["kv_heads"], case["head_dim"], s["longest"]
    cu = s["cu"].long()
    t = cu.shape[0] - 1
    seq = torch.searchsorted(cu[1:], torch.arange(s["q"].shape[0], device=DEV), right=True)
    at = torch.arange(s["q"].shape[0], device=DEV) - cu[seq]

    def padded(x):
        out = torch.zeros((t, n, x.shape[1], hd), dtype=torch.float32, device=DEV)
        out[seq, at] = x.float()
        return out.transpose(1, 2).unflatten(1, (kv, -1))  # t kv group n hd

    q, k, v = padded(s["q"]) / math.sqrt(hd), padded(s["k"]), padded(s["v"])
    causal = torch.ones((n, n), dtype=torch.bool, device=DEV).tril()
    p = _softmax_rows(q @ k.transpose(3, 4).contiguous(), causal)
    o = (p @ v).flatten(1, 2).transpose(1, 2)  # t n h hd
    return o[seq, at].reshape(-1, h * hd).to(s["q"].dtype)


def _plain_store(s, case):
    slots, out = s["slots"].long(), {}
    for name, (codes, ms) in zip("kv", s["held"]):
        codes[slots], ms[slots] = _hold(s[name])
        out[name] = _stands_for(codes[slots], ms[slots], torch.float32).to(s[name].dtype)
    return out


def _plain_attend(s, case):
    """softmax(q k / sqrt(hd)) v over each row's context, the batch padded."""
    bs, kv, hd = case["block"], case["kv_heads"], case["head_dim"]
    ctx, n, m = s["ctx"].long(), s["ctx_max"], s["q_max"]
    t, rows = ctx.shape[0], s["q"].shape[0]
    at = torch.arange(rows, device=DEV)
    if s["cu"] is None:
        seq, i, first = at, at - at, ctx - 1
    else:
        cu = s["cu"].long()
        seq = torch.searchsorted(cu[1:], at, right=True)
        i, first = at - cu[seq], ctx - (cu[1:] - cu[:-1])
    q = torch.zeros((t, m, case["heads"], hd), dtype=torch.float32, device=DEV)
    q[seq, i] = s["q"].float() / math.sqrt(hd)
    q = q.unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # t kv (group m) hd
    key = torch.arange(n, device=DEV)
    slot = s["tables"].long()[:, key // bs] * bs + key % bs
    k, v = ((_stands_for(c[slot], ms[slot], torch.float32)).transpose(1, 2)
            for c, ms in s["held"])  # t kv n hd
    ok = key <= first[:, None, None] + torch.arange(m, device=DEV)[None, :, None]  # t m n
    ok = ok & (key < ctx[:, None, None])
    x = q @ k.transpose(2, 3).contiguous()
    p = _softmax_rows(x.unflatten(2, (-1, m)), ok[:, None, None])
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, m)).permute(0, 3, 1, 2, 4)  # t m kv group hd
    return o[seq, i].reshape(rows, -1).to(s["q"].dtype)


def _plain_logits(s, case):
    """Repetition: logits of tokens seen are divided (positive ones) or multiplied by
    r; then frequency times the count among generated tokens and presence are
    taken off, biases added (the last of a token's entries counts), and tokens
    without a bit in their request's mask row excluded."""
    b, v = s["logits"].shape
    cu, x = s["cu"].long(), s["logits"].float()
    at = torch.arange(s["tokens"].numel(), device=DEV)
    req = torch.searchsorted(cu[1:], at, right=True)
    where = req * v + s["tokens"].long()
    new = at - cu[req] >= s["prompt"].long()[req]
    zero = torch.zeros(b * v, dtype=torch.int32, device=DEV)
    count = zero.index_add(0, where, new.to(torch.int32)).view(b, v)
    seen = zero.index_fill(0, where, 1).view(b, v) > 0
    r = s["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["freq"][:, None] * count
    x = x - torch.where(count > 0, s["pres"][:, None], 0.0)
    if s["bias_tokens"].numel():
        cb = s["cu_bias"].long()
        j = torch.arange(s["bias_tokens"].numel(), device=DEV)
        where = torch.searchsorted(cb[1:], j, right=True) * v + s["bias_tokens"].long()
        last = torch.full((b * v,), -1, device=DEV).scatter_reduce(0, where, j, "amax").view(b, v)
        x = torch.where(last >= 0, x + s["bias_values"][last.clamp(min=0)], x)
    if s["mask"] is not None:
        t = torch.arange(v, device=DEV)
        rows = s["mask_rows"].long()
        word = s["mask"][rows.clamp(min=0)][:, t // 32]
        ok = ((word >> (t % 32).to(torch.int32)) & 1).bool() | (rows < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
    s["out"].copy_(x)
    return s["out"]


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "logits":
        b, v = case["batch"], case["vocab"]
        return {"bytes": 2 * b * v * e + 4 * sum(_hist(case)) + 8 * sum(_biased(case))
                + case["masks"] * ((v + 31) // 32) * 4 + 28 * b, "flops": 4 * b * v}
    kv, hd = case["kv_heads"], case["head_dim"]
    held = kv * (hd // 2 + hd // GROUP * 4)  # bytes of a token's key or value in 4 bits
    if case["kind"] == "store":
        n = case["tokens"]
        return {"bytes": 4 * n * (kv * hd * e + held) + 8 * n, "flops": 12 * n * kv * hd}
    h = case["heads"]
    if case["kind"] == "prompt":
        n = _prompts(case)
        return {"bytes": sum(n) * (2 * h + 2 * kv) * hd * e,
                "flops": 2 * h * hd * sum(m * (m + 1) for m in n)}
    ctx, q = _ctx_lens(case), _q_lens(case)
    return {"bytes": sum(ctx) * 2 * held + 2 * sum(q) * h * hd * e,
            "flops": 4 * h * hd * sum(m * c - m * (m - 1) // 2 for c, m in zip(ctx, q))}


def _exact_held(x):
    """What a pool of 4 bits gives back for x, in 64 bits, group by group of channels."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for j in range(0, x.shape[-1], GROUP):
        g = x[..., j:j + GROUP].float()
        m = g.min(-1, keepdim=True).values.to(torch.float16).float()
        span = g.max(-1, keepdim=True).values - m
        s = torch.div(span, torch.full_like(span, 15)).to(torch.float16).double()
        c = torch.round((g.double() - m.double()) / s).clamp(0, 15).nan_to_num(0.0)
        out[..., j:j + GROUP] = m.double() + s * torch.where(s > 0, c, 0.0)
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(case, d)
    if case["kind"] == "store":
        return {"k": _exact_held(d["k"]), "v": _exact_held(d["v"])}
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    group = h // kv
    if case["kind"] == "prompt":
        out = torch.empty(d["q"].shape, dtype=torch.float64, device=DEV)
        cu = _cu(_prompts(case))
        for a, b in zip(cu, cu[1:]):
            above = torch.arange(b - a, device=DEV)
            above = above[None, :] > above[:, None]
            for j in range(h):
                x = d["q"][a:b, j].double() @ d["k"][a:b, j // group].double().T * hd ** -0.5
                x[above] = -math.inf
                out[a:b, j] = torch.softmax(x, 1) @ d["v"][a:b, j // group].double()
        return out.reshape(cu[-1], -1)
    bs, ctx, q = case["block"], _ctx_lens(case), _q_lens(case)
    n = d["num_blocks"] * bs
    k = torch.empty((n, kv, hd), dtype=DT[case["dtype"]], device=DEV)
    v = torch.empty_like(k)
    for i, m, a, b in _pieces(_gen(seed + (1 << 40)), n, kv, hd, DT[case["dtype"]]):
        k[i:i + m], v[i:i + m] = a, b
    out = torch.empty(d["q"].shape, dtype=torch.float64, device=DEV)
    r = 0
    for i, (c, m) in enumerate(zip(ctx, q)):
        pos = torch.arange(c, device=DEV)
        at = d["tables"][i].long()[pos // bs] * bs + pos % bs
        kk, vv = _exact_held(k[at]), _exact_held(v[at])
        hidden = pos[None, :] > c - m + torch.arange(m, device=DEV)[:, None]
        for j in range(h):
            x = d["q"][r:r + m, j].double() @ kk[:, j // group].T * hd ** -0.5
            x[hidden] = -math.inf
            out[r:r + m, j] = torch.softmax(x, 1) @ vv[:, j // group]
        r += m
    return out.reshape(r, -1)


def _exact_logits(case, d):
    """Row by row, from lists."""
    v = case["vocab"]
    out = d["logits"].double()
    rep, pres, freq = (d[n].double().tolist() for n in ("rep", "pres", "freq"))
    cu, cb, prompt = d["cu"].tolist(), d["cu_bias"].tolist(), d["prompt"].tolist()
    tokens, bt = d["tokens"].long(), d["bias_tokens"].tolist()
    bv = d["bias_values"].double().tolist()
    rows = d["mask_rows"].tolist() if d["mask"] is not None else None
    for i in range(case["batch"]):
        x = out[i]
        mine = tokens[cu[i]:cu[i + 1]]
        t = torch.unique(mine)
        y = x[t]
        x[t] = torch.where(y > 0, y / rep[i], y * rep[i])
        n = torch.bincount(mine[prompt[i]:], minlength=v)
        x -= freq[i] * n + pres[i] * (n > 0)
        bias = dict(zip(bt[cb[i]:cb[i + 1]], bv[cb[i]:cb[i + 1]]))
        if bias:
            x[torch.tensor(list(bias), device=DEV)] += torch.tensor(
                list(bias.values()), dtype=torch.float64, device=DEV)
        if rows and rows[i] >= 0:
            bits = (d["mask"][rows[i]][:, None] >> torch.arange(32, device=DEV).to(torch.int32)) & 1
            x[bits.flatten()[:v] == 0] = -math.inf
    return out
