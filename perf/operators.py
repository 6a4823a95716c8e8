"""Timed cases of the 4-bit K/V cache and of packed prompt attention.

A case is one call of one of three operators, beside its plain form in
elementary torch operations:

- "append4": F32 K and V rows into a cache held in 4 bits, and the values the
  cache then stands for back out (what a program that hands a session on, or
  compares it, reads);
- "attend4": attention of a layer over such a cache: one token (decode), a
  session batch of 2 to 16 tokens, a prompt chunk, sliding windows over rings;
- "packed": attention over several whole prompts or texts laid end to end, each
  over its own keys: causal prompts in BF16, bidirectional texts in F32 (the
  embedding call of several texts).

A cache's block is 32 consecutive elements of a row: with lo and hi its least
and largest element, s = f16((hi - lo) / 15), z = f16(lo), an element x is the
whole number c = rint((x - z) / s) within 0 .. 15 (0 where s is 0) and stands
for f16(c s + z), rounded once. (Elements are first brought within +-65280, so
that no value overflows f16.)

Head shapes are those of the models this repository's benchmark and tests
name, and a few others. Cached keys have the per-channel offsets that make a
block's range one-sided; q and k are normalised per head.
"""
import math

import torch

own = False

DEV = "cuda"

LLAMA = dict(n_head=32, n_kv=8, head_dim=64)
QWEN = dict(n_head=32, n_kv=8, head_dim=128)
GEMMA_1B = dict(n_head=4, n_kv=1, head_dim=256)
GEMMA_4B = dict(n_head=8, n_kv=4, head_dim=256)
EMBED = dict(n_head=3, n_kv=1, head_dim=256)
SHAPES = [LLAMA, QWEN, GEMMA_1B, GEMMA_4B, EMBED, dict(n_head=14, n_kv=2, head_dim=64),
          dict(n_head=6, n_kv=2, head_dim=96), dict(n_head=16, n_kv=16, head_dim=128)]


def _append4(shape, n_tok, pos0, rows):
    return dict(kind="append4", n_tok=n_tok, pos0=pos0, rows=rows, kv_dim=shape["n_kv"] * shape["head_dim"])


def _attend4(shape, n_tok, pos0, window=0):
    return dict(kind="attend4", n_tok=n_tok, pos0=pos0, window=window, **shape)


def _packed(shape, lens, dtype, causal=True, window=0):
    return dict(kind="packed", lens=",".join(map(str, lens)), dtype=dtype, causal=causal, window=window, **shape)


def listed():
    return [
        # A decode step's append: one row of one layer, all latency.
        dict(_append4(QWEN, 1, 4000, 8192), name="append_token"),
        # A prompt's rows of one layer.
        dict(_append4(QWEN, 4096, 0, 32768), name="append_prompt"),
        # The shortest decode call: one KV head, a thousand keys.
        dict(_attend4(GEMMA_1B, 1, 1023), name="decode_gemma_1k"),
        # Decode at long context.
        dict(_attend4(QWEN, 1, 32767), name="decode_qwen_32k"),
        # Decode at the context that a cache in 4 bits makes room for.
        dict(_attend4(LLAMA, 1, 131071), name="decode_llama_128k"),
        # A forward pass of a session that verifies drafts, odd in tokens and keys.
        dict(_attend4(QWEN, 13, 20011), name="session_qwen_20k"),
        # The last chunk of a 4096-token prompt.
        dict(_attend4(QWEN, 512, 3584), name="chunk_qwen_4k"),
        # A chunk of a long prompt on a sliding layer, its ring wrapped.
        dict(_attend4(GEMMA_4B, 1024, 15360, 1024), name="chunk_gemma_window"),
        # A few short requests at once: latency.
        dict(_packed(QWEN, [1, 37, 16, 90], "bf16"), name="packed_tiny"),
        # Texts to embed, bidirectional with the model's window, F32 as its cache is.
        dict(_packed(EMBED, [212, 7, 640, 33, 1024, 58, 391, 1500, 129, 86, 777, 5], "f32", causal=False, window=512),
             name="packed_texts"),
        # Ragged prompts of several requests.
        dict(_packed(QWEN, [1303, 2048, 77, 512, 1, 1790, 901, 258], "bf16"), name="packed_prompts"),
        # One long prompt beside short ones.
        dict(_packed(LLAMA, [300, 8192, 45], "bf16"), name="packed_long"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append4", "decode", "decode", "session", "chunk", "packed", "packed", "packed"])
    shape = rng.choice(SHAPES)
    if kind == "append4":
        n = rng.choice([1, rng.randint(2, 16), _log_int(rng, 20, 4000)])
        return _append4(shape, n, _log_int(rng, 1, 30000), 32 * _log_int(rng, (n + 31) // 32, 1000))
    if kind == "decode":
        return _attend4(shape, 1, _log_int(rng, 1, 60000), rng.choice([0, 0, 512, 1024]))
    if kind == "session":
        return _attend4(shape, rng.randint(2, 16), _log_int(rng, 10, 16000), rng.choice([0, 0, 512, 1024]))
    if kind == "chunk":
        return _attend4(shape, _log_int(rng, 17, 900), rng.choice([0, _log_int(rng, 20, 8000)]), rng.choice([0, 0, 512]))
    dtype = rng.choice(["bf16", "f32"])
    longest = _log_int(rng, 16, 2000)
    lens = [longest] + [_log_int(rng, 1, longest) for _ in range(rng.randint(0, 9))]
    rng.shuffle(lens)
    return _packed(shape, lens, dtype, causal=rng.random() < 0.7, window=rng.choice([0, 0, 256, 512]))


# ---- inputs: from the seed alone, in plain torch --------------------------------------

def _randn(seed, path, *shape):
    s = seed & 0x7FFFFFFF
    for p in path:
        s = (s * 1000003 + p + 1) & 0x7FFFFFFFFFFF
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(s), device=DEV, dtype=torch.float32)


def _heads_normed(x, head_dim):
    h = x.view(x.shape[0], -1, head_dim)
    return (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)).reshape(x.shape)


def _kv_rows(seed, n, kv_dim, head_dim):
    """K rows with offsets per channel, normalised per head, and V rows."""
    k = _randn(seed, (1,), n, kv_dim) + _randn(seed, (3,), 1, kv_dim)
    return _heads_normed(k, head_dim), _randn(seed, (2,), n, kv_dim)


def _quantised(x):
    """(codes, two to a byte: elements i and i + 16 of a block in byte i; scale; offset) of F32 rows."""
    b = x.clamp(-65280.0, 65280.0).view(x.shape[0], -1, 32)
    lo, hi = b.amin(-1), b.amax(-1)
    s, z = ((hi - lo) / 15.0).half(), lo.half()
    c = torch.where(s[..., None] > 0, torch.round((b - z.float()[..., None]) / s.float()[..., None]), torch.zeros_like(b))
    c = c.clamp(0, 15).to(torch.uint8)
    return c[..., :16] | (c[..., 16:] << 4), s, z


def _values(q):
    """What the codes stand for, F32. The product has at most 15 significant bits, and no product of a code and a
    scale is near enough to a border of f16's steps for the 32-bit sum to move it there."""
    codes, s, z = q
    c = torch.cat([codes & 15, codes >> 4], -1).float()
    return (c * s.float()[..., None] + z.float()[..., None]).half().float().view(codes.shape[0], -1)


# ---- the append -----------------------------------------------------------------------

def _prepare_append4(case, seed):
    n, d = case["n_tok"], case["kv_dim"]
    k, v = _kv_rows(seed, n, d, 32)
    s = dict(case=case, k=k, v=v)
    if own:
        from libllmcpu_amd import KVCache

        s.update(kv=KVCache([case["rows"]], [d], q4=True), k_out=torch.empty(n, d, device=DEV),
                 v_out=torch.empty(n, d, device=DEV))
    torch.cuda.synchronize()
    return s


def _run_append4(s):
    c = s["case"]
    if own:
        kv, n, k_out, v_out = s["kv"], c["n_tok"], s["k_out"], s["v_out"]
        kv.append_f32_device(0, s["k"].data_ptr(), s["v"].data_ptr(), pos0=c["pos0"], n_tok=n)
        first = c["pos0"] % c["rows"]
        m = min(n, c["rows"] - first)  # rows before the ring wraps
        kv.read_f32_device(0, first, m, k_out.data_ptr(), v_out.data_ptr())
        if m < n:
            kv.read_f32_device(0, 0, n - m, k_out.data_ptr() + 4 * m * c["kv_dim"], v_out.data_ptr() + 4 * m * c["kv_dim"])
        return {"k": k_out, "v": v_out}
    return {"k": _values(_quantised(s["k"])), "v": _values(_quantised(s["v"]))}


def _work_append4(case):
    n = 2 * case["n_tok"] * case["kv_dim"]
    return dict(bytes=int(n * (4 + 0.625 + 4)), flops=8 * n)


def _exact_values(x):
    """The cache's values in 64 bits, from the definition: codes by comparison with the borders between them.
    A border is (c + 1/2) s + z; an element on it goes to the even code. The quotient of the definition is a 32-bit
    one, so where the element is within its rounding of a border it is that quotient that decides."""
    b = x.view(x.shape[0], -1, 32).double()
    lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
    s = ((hi - lo).float() / 15.0).half().double()
    z = lo.float().half().double()
    c = torch.zeros_like(b)
    t32 = (b - z).float() / s.float().clamp_min(1e-30)
    for j in range(15):
        above = t32 > j + 0.5 if j % 2 == 0 else t32 >= j + 0.5
        c += (above & (s > 0)).double()
    return (c * s + z).float().half().double().view(x.shape)


def _exact_append4(case, seed):
    k, v = _kv_rows(seed, case["n_tok"], case["kv_dim"], 32)
    return {"k": _exact_values(k), "v": _exact_values(v)}


# ---- attention over the cache -----------------------------------------------------------

def _prepare_attend4(case, seed):
    hd, n = case["head_dim"], case["pos0"] + case["n_tok"]
    q = _heads_normed(_randn(seed, (0,), case["n_tok"], case["n_head"] * hd), hd)
    k, v = _kv_rows(seed, n, case["n_kv"] * hd, hd)
    if own:
        from libllmcpu_amd import KVCache, kv_rows

        rows = kv_rows((n + 255) // 256 * 256, case["window"], case["n_tok"])
        kv = KVCache([rows], [case["n_kv"] * hd], q4=True)
        torch.cuda.synchronize()
        for p in range(max(0, n - rows), n, rows):
            m = min(rows, n - p)
            kv.append_f32_device(0, k[p].data_ptr(), v[p].data_ptr(), pos0=p, n_tok=m)
        kv.sync()
        return dict(case=case, q=q, kv=kv, out=torch.empty_like(q))
    s = dict(case=case, q=q, k=_quantised(k), v=_quantised(v))
    torch.cuda.synchronize()
    return s


def _seen(pos, n, causal, window):
    """[len(pos), n]: whether position pos attends to key 0 .. n - 1."""
    key = torch.arange(n, device=DEV)
    if causal:
        ok = key[None, :] <= pos[:, None]
        return ok & (key[None, :] > pos[:, None] - window) if window else ok
    return (key[None, :] - pos[:, None]).abs() <= window // 2 if window else torch.ones(len(pos), n, device=DEV, dtype=torch.bool)


def _attend(q, k, v, seen, shape):
    """Softmax attention of q [n, n_head * hd] over k, v [m, n_kv * hd], in 32 bits."""
    h, kv, hd = shape["n_head"], shape["n_kv"], shape["head_dim"]
    n, m, g = q.shape[0], k.shape[0], h // kv
    qh = q.float().view(n, kv, g, hd).permute(1, 0, 2, 3).reshape(kv, n * g, hd)
    kh, vh = (x.float().view(m, kv, hd).permute(1, 0, 2).contiguous() for x in (k, v))
    s = torch.bmm(qh, kh.transpose(1, 2)).mul_(1.0 / math.sqrt(hd)).view(kv, n, g, m)
    s.masked_fill_(~seen[None, :, None, :], -math.inf)
    s = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    o = torch.bmm((s / s.sum(-1, keepdim=True)).view(kv, n * g, m), vh)
    return o.view(kv, n, g, hd).permute(1, 0, 2, 3).reshape(n, h * hd)


def _run_attend4(s):
    c = s["case"]
    scale = 1.0 / math.sqrt(c["head_dim"])
    if own:
        s["kv"].attend_device(0, s["q"].data_ptr(), s["out"].data_ptr(), n_tok=c["n_tok"], pos0=c["pos0"],
                              window=c["window"], n_head=c["n_head"], n_kv=c["n_kv"], head_dim=c["head_dim"], scale=scale)
        return s["out"]
    n = c["pos0"] + c["n_tok"]
    seen = _seen(torch.arange(c["pos0"], n, device=DEV), n, True, c["window"])
    return _attend(s["q"], _values(s["k"]), _values(s["v"]), seen, c)


def _span_sum(lens, pos0, n_tok, causal, window):
    """Attended (query, key) pairs of queries pos0 .. pos0 + n_tok - 1 of a sequence of `lens` keys."""
    pos = torch.arange(pos0, pos0 + n_tok)
    if causal:
        first, last = (torch.clamp(pos + 1 - window, min=0) if window else torch.zeros_like(pos)), pos
    elif window:
        first, last = torch.clamp(pos - window // 2, min=0), torch.clamp(pos + window // 2, max=lens - 1)
    else:
        first, last = torch.zeros_like(pos), torch.full_like(pos, lens - 1)
    return int((last - first + 1).sum()), int(last[-1] - first[0] + 1)


def _work_attend4(case):
    pairs, keys = _span_sum(case["pos0"] + case["n_tok"], case["pos0"], case["n_tok"], True, case["window"])
    qd, kd = case["n_head"] * case["head_dim"], case["n_kv"] * case["head_dim"]
    return dict(bytes=int(2 * keys * kd * 0.625) + 8 * case["n_tok"] * qd, flops=4 * qd * pairs)


def _exact_softmax(q, k, v, pos0, causal, window, shape):
    """Attention in 64 bits of queries at pos0 .. of one sequence, a KV head and some rows at a time."""
    hd, g = shape["head_dim"], shape["n_head"] // shape["n_kv"]
    n, m = q.shape[0], k.shape[0]
    out = torch.empty(n, q.shape[1], device=DEV, dtype=torch.float64)
    key = torch.arange(m, device=DEV)
    rows = max(1, (1 << 26) // m)
    for h in range(shape["n_head"]):
        kh, vh = (x[:, (h // g) * hd:(h // g + 1) * hd].double() for x in (k, v))
        for r in range(0, n, rows):
            p = torch.arange(pos0 + r, pos0 + min(r + rows, n), device=DEV)[:, None]
            if causal:
                dead = (key > p) | (key <= p - window) if window else key > p
            else:
                dead = (key - p).abs() > window // 2 if window else torch.zeros(len(p), m, dtype=torch.bool, device=DEV)
            s = (q[r:r + rows, h * hd:(h + 1) * hd].double() @ kh.t() / math.sqrt(hd)).masked_fill(dead, -math.inf)
            out[r:r + rows, h * hd:(h + 1) * hd] = torch.softmax(s, -1) @ vh
    return out


def _exact_attend4(case, seed):
    hd, n = case["head_dim"], case["pos0"] + case["n_tok"]
    q = _heads_normed(_randn(seed, (0,), case["n_tok"], case["n_head"] * hd), hd)
    k, v = _kv_rows(seed, n, case["n_kv"] * hd, hd)
    return _exact_softmax(q, _exact_values(k), _exact_values(v), case["pos0"], True, case["window"], case)


# ---- packed prompts -----------------------------------------------------------------------

def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _packed_inputs(case, seed):
    hd, n = case["head_dim"], sum(_lens(case))
    q = _heads_normed(_randn(seed, (0,), n, case["n_head"] * hd), hd)
    k, v = _kv_rows(seed, n, case["n_kv"] * hd, hd)
    return [x.bfloat16() if case["dtype"] == "bf16" else x for x in (q, k, v)]


def _prepare_packed(case, seed):
    q, k, v = _packed_inputs(case, seed)
    s = dict(case=case, q=q, k=k, v=v)
    lens = _lens(case)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    if own:
        from libllmcpu_amd import KVCache

        s.update(kv=KVCache([32], [64]), out=torch.empty_like(q), starts=starts)
    else:
        # which row of which sequence a row is
        at = torch.tensor(starts, device=DEV)
        s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device=DEV), at[1:] - at[:-1])
        s["pos"] = torch.arange(sum(lens), device=DEV) - at[s["seq"]]
    torch.cuda.synchronize()
    return s


def _run_packed(s):
    c = s["case"]
    if own:
        s["kv"].attend_packed_device(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(),
                                     starts=s["starts"], bf16=c["dtype"] == "bf16", window=c["window"], causal=c["causal"],
                                     n_head=c["n_head"], n_kv=c["n_kv"], head_dim=c["head_dim"],
                                     scale=1.0 / math.sqrt(c["head_dim"]))
        return s["out"]
    # the sequences side by side, each padded to the longest
    h, kv, hd = c["n_head"], c["n_kv"], c["head_dim"]
    lens = _lens(c)
    b, n, g = len(lens), max(lens), h // kv
    seq, pos = s["seq"], s["pos"]

    def padded(x):
        y = torch.zeros(b, n, x.shape[1], device=DEV)
        y[seq, pos] = x.float()
        return y

    qh = padded(s["q"]).view(b, n, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(b * kv, n * g, hd)
    kh, vh = (padded(x).view(b, n, kv, hd).permute(0, 2, 1, 3).reshape(b * kv, n, hd) for x in (s["k"], s["v"]))
    key = torch.arange(n, device=DEV)
    real = key[None, :] < torch.tensor(lens, device=DEV)[:, None]
    seen = _seen(key, n, c["causal"], c["window"])[None] & real[:, None, :]  # [b, query, key]
    seen |= ~real[:, :, None] & (key == 0)  # (a padding row, not kept, sees one key)
    w = torch.bmm(qh, kh.transpose(1, 2)).mul_(1.0 / math.sqrt(hd)).view(b, kv, n, g, n)
    w.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True)))
    w = w / w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(b * kv, n * g, n), vh).view(b, kv, n, g, hd).permute(0, 2, 1, 3, 4).reshape(b, n, h * hd)
    return o[seq, pos].to(s["q"].dtype)


def _work_packed(case):
    lens, size = _lens(case), 2 if case["dtype"] == "bf16" else 4
    qd, kd = case["n_head"] * case["head_dim"], case["n_kv"] * case["head_dim"]
    pairs = sum(_span_sum(n, 0, n, case["causal"], case["window"])[0] for n in lens)
    return dict(bytes=size * sum(lens) * (2 * qd + 2 * kd), flops=4 * qd * pairs)


def _exact_packed(case, seed):
    q, k, v = _packed_inputs(case, seed)
    out, at = [], 0
    for n in _lens(case):
        out.append(_exact_softmax(*(x[at:at + n] for x in (q, k, v)), 0, case["causal"], case["window"], case))
        at += n
    return torch.cat(out)


_KINDS = {"append4": (_prepare_append4, _run_append4, _work_append4, _exact_append4),
          "attend4": (_prepare_attend4, _run_attend4, _work_attend4, _exact_attend4),
          "packed": (_prepare_packed, _run_packed, _work_packed, _exact_packed)}


def prepare(case, seed):
    return _KINDS[case["kind"]][0](case, seed)


def run(state):
    return _KINDS[state["case"]["kind"]][1](state)


def work(case):
    return _KINDS[case["kind"]][2](case)


def exact(case, seed):
    return _KINDS[case["kind"]][3](case, seed)
