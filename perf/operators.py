"""Measured calls of the rollout's 8-bit key/value cache and of the per-token statistics of logits.

Four operators: appending new keys and values to the paged 8-bit cache, attention over that cache, the log-probability /
entropy / top alternatives of given tokens, and the gradient of those.  ``run`` computes them in elementary torch
operations (``own`` false) or through ``chatlearn_b200.ops`` (``own`` true).
"""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_MIN, SCALE_MAX = 2.0 ** -24, 2.0 ** 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of one layer: 128 sequences, one new token each, keys and values are views of the qkv rows
        dict(name="append_step_128", op="append", dtype="bf16", seqs=128, nq=32, nkv=8, dim=128, block=64, lo=128, hi=2600, new_lo=1, new_hi=1),
        # a prefill step of one layer: 16 prompts of about a thousand tokens
        dict(name="append_prefill_16", op="append", dtype="bf16", seqs=16, nq=32, nkv=8, dim=128, block=64, lo=900, hi=1152, new_lo=900, new_hi=1152),
        # small pages, fp32 rows, continuation chunks of odd lengths, some sequences without new tokens
        dict(name="append_chunks_fp32", op="append", dtype="fp32", seqs=13, nq=8, nkv=4, dim=64, block=16, lo=40, hi=333, new_lo=0, new_hi=37),
        # one sequence alone: the smallest call, where latency counts
        dict(name="decode_1_short", op="attend", dtype="bf16", seqs=1, nq=32, nkv=8, dim=128, block=64, lo=700, hi=777, new_lo=1, new_hi=1),
        # the decode step of a rollout batch with ragged contexts
        dict(name="decode_128", op="attend", dtype="bf16", seqs=128, nq=32, nkv=8, dim=128, block=64, lo=128, hi=2600, new_lo=1, new_hi=1),
        # few rows, long contexts: the sequence axis has to be split
        dict(name="decode_4_long", op="attend", dtype="bf16", seqs=4, nq=32, nkv=8, dim=128, block=64, lo=30001, hi=65500, new_lo=1, new_hi=1),
        # 16 query heads over 2 key/value heads of 256, pages of 32
        dict(name="decode_48_dim256", op="attend", dtype="bf16", seqs=48, nq=16, nkv=2, dim=256, block=32, lo=1, hi=6000, new_lo=1, new_hi=1),
        # continuation chunks of prompts that are prefilled in pieces, causal inside the chunk
        dict(name="chunk_8x512", op="attend", dtype="bf16", seqs=8, nq=32, nkv=8, dim=128, block=64, lo=3800, hi=4300, new_lo=512, new_hi=512),
        # statistics of the sampled tokens of one decode step: fp32 logits of a 152 k vocabulary
        dict(name="logprob_step_128", op="logprob", dtype="fp32", rows=128, vocab=151936, pad=0, top=8, temp=0.8, masked=0.0, grad=False),
        # one row of an odd vocabulary cut out of padded logits, most alternatives that a server hands out
        dict(name="logprob_1_odd", op="logprob", dtype="fp32", rows=1, vocab=32001, pad=63, top=20, temp=1.0, masked=0.2, grad=False),
        # a training chunk: forward and gradient with alternatives (distillation on a teacher's top choices)
        dict(name="logprob_train_1024", op="logprob", dtype="bf16", rows=1024, vocab=151936, pad=0, top=16, temp=1.0, masked=0.0, grad=True),
        # small ragged rows with masked vocabulary entries and wholly masked rows, forward and gradient
        dict(name="logprob_train_odd", op="logprob", dtype="fp32", rows=301, vocab=32001, pad=0, top=5, temp=1.3, masked=0.3, grad=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "chunk", "logprob", "grad"])
    if op in ("logprob", "grad"):
        rows, vocab = _spread(rng, 1, 1024), _spread(rng, 1000, 151936)
        return dict(op="logprob", dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8, 64]),
                    top=rng.randint(0, 32), temp=round(rng.uniform(0.5, 1.5), 3), masked=rng.choice([0.0, 0.0, 0.25]), grad=op == "grad")
    nkv, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16])
    dim, block = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    seqs = _spread(rng, 1, 160)
    room = min(60000, 200_000_000 // (seqs * nkv * dim))         # tokens a sequence, so that no case outgrows the listed ones
    if op == "chunk":
        room = min(room, 4000)
        new_hi = max(1, min(room, 2_000_000 // (seqs * nkv * rep * dim)))
        new_hi = _spread(rng, 1, min(new_hi, 600))
    elif op == "append":
        room = min(room, 3000)
        new_hi = rng.choice([1, _spread(rng, 1, room)])
    else:
        new_hi = 1
    hi = _spread(rng, max(new_hi, 8), max(room, new_hi + 8))
    lo = rng.randint(min(new_hi, hi), hi)
    new_lo = rng.randint(0 if seqs > 3 else 1, new_hi) if new_hi > 1 else 1
    return dict(op="append" if op == "append" else "attend", dtype=rng.choice(["bf16", "bf16", "fp16"]), seqs=seqs, nq=nkv * rep, nkv=nkv, dim=dim,
                block=block, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi)


# ------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """Lengths and new tokens of every sequence, on the host (the engine's scheduler knows them).  The new tokens go by the
    case alone, so that a case has one number of rows."""
    g = torch.Generator().manual_seed(case["seqs"] * 7919 + case["new_hi"])
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (case["seqs"],), generator=g)
    g.manual_seed(seed)
    lens = torch.randint(case["lo"], case["hi"] + 1, (case["seqs"],), generator=g)
    return torch.maximum(lens, new), new


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logprob":
        R, V = case["rows"], case["vocab"]
        z = torch.empty(R, V + case["pad"], device=dev, dtype=dt)
        z.copy_(torch.randn(R, V + case["pad"], device=dev, generator=g) * 2.5)
        z = z[:, :V]
        tok = torch.randint(0, V, (R,), device=dev, generator=g)
        # a sampled token is mostly a likely one
        likely = z.float().argmax(-1)
        tok = torch.where(torch.rand(R, device=dev, generator=g) < 0.6, likely, tok)
        if case["masked"]:
            z.masked_fill_(torch.rand(R, V, device=dev, generator=g) < case["masked"], -math.inf)
            if R > 8:
                z[R // 3] = -math.inf                    # a row that its mask leaves nothing of
                tok[R // 2] = -1                         # a row without a token
        n = case["top"]
        grads = [torch.randn(R, device=dev, generator=g) / R, 0.01 * torch.randn(R, device=dev, generator=g) / R,
                 torch.randn(R, n, device=dev, generator=g) / R]
        return dict(case=case, z=z, tok=tok, grads=grads)
    lens, new = _lengths(case, seed)
    B, bs, nkv, D, nq = case["seqs"], case["block"], case["nkv"], case["dim"], case["nq"]
    # pages in no order, room for every sequence at its longest
    width = (max(case["hi"], case["new_hi"]) + bs - 1) // bs
    nb = B * width + 3
    perm = torch.randperm(nb, device=dev, generator=g).to(torch.int32)
    tables = perm[:B * width].view(B, width)
    T = int(new.sum())
    # rows as the qkv projection leaves them: queries, keys and values side by side, a few channels much larger
    gain = torch.ones(D, device=dev)
    gain[torch.randperm(D, device=dev, generator=g)[:4]] = 6.0
    qkv = torch.randn(T, nq + 2 * nkv, D, device=dev, generator=g) * gain
    qkv[:, :nq] *= 0.5
    qkv = qkv.to(dt).view(T, -1)
    q, k, v = (x.view(T, -1, D) for x in qkv.split([nq * D, nkv * D, nkv * D], dim=1))
    # what earlier steps left in the cache: codes that use their page's range, and the page's power-of-two scale
    powers = torch.tensor([2.0 ** -8, 2.0 ** -7, 2.0 ** -6, 2.0 ** -5], device=dev)
    ks = powers[torch.randint(1, 4, (nb, nkv), device=dev, generator=g)]
    vs = powers[torch.randint(0, 3, (nb, nkv), device=dev, generator=g)]
    kc = torch.empty(nb, nkv, bs, D, dtype=torch.float8_e4m3fn, device=dev)
    vc = torch.empty_like(kc)
    step = max(1, 50_000_000 // (nkv * bs * D))
    for s in range(0, nb, step):
        m = min(step, nb - s)
        kc[s:s + m] = (torch.randn(m, nkv, bs, D, device=dev, generator=g) * (32.0 * gain)).clamp_(-448, 448).to(kc.dtype)
        vc[s:s + m] = (torch.randn(m, nkv, bs, D, device=dev, generator=g) * 96.0).clamp_(-448, 448).to(kc.dtype)
    return dict(case=case, q=q, k=k, v=v, kc=kc, vc=vc, ks=ks, vs=vs, tables=tables, lens=lens.to(dev, torch.int32),
                new=new.to(dev, torch.int32), T=T, max_len=int(lens.max()), max_new=int(new.max()))


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "logprob": _plain_logprob}[case["op"]](state)


def _run_own(state):
    from chatlearn_b200 import ops
    case = state["case"]
    if case["op"] == "logprob":
        z = state["z"]
        if not case["grad"]:
            return tuple(ops.token_logprobs(z, state["tok"], case["top"], case["temp"]))
        z = z.detach().requires_grad_(True)
        out = ops.token_logprobs(z, state["tok"], case["top"], case["temp"])
        some = 3 if case["top"] else 2
        dz, = torch.autograd.grad(out[:some], z, state["grads"][:some])
        return tuple(t.detach() for t in out) + (dz,)
    cache = ops.Q8KVCache(state["kc"], state["vc"], state["ks"], state["vs"])
    new = None if case["new_lo"] == case["new_hi"] == 1 else state["new"]
    if case["op"] == "append":
        ops.kv_append_q8(state["k"], state["v"], cache, state["tables"], state["lens"], new)
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    return ops.paged_attention_q8(state["q"], cache, state["tables"], state["lens"], new)


def _rows(state):
    """Sequence and position of every row."""
    new, lens = state["new"].long(), state["lens"].long()
    row = torch.arange(state["T"], device=new.device)
    ends = torch.cumsum(new, 0)
    b = torch.searchsorted(ends, row, right=True)
    return b, lens[b] - ends[b] + row


def _needed(amax):
    """The smallest power of two s with amax <= 448 s (amax = m 2^e with 0.5 <= m < 1; amax / m is exact)."""
    m, _ = torch.frexp(amax)
    s = torch.where(m > 0, amax / m, 0.0) * torch.where(m <= 0.875, 2.0 ** -9, 2.0 ** -8)
    return s.clamp(SCALE_MIN, SCALE_MAX)


def _append_one(x, codes, scale, page, off):
    nb, nkv, bs, D = codes.shape
    x = x.float()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)                                       # [T, nkv]
    need = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, nkv), _needed(amax), "amax")
    first = torch.full((nb,), bs, device=x.device).scatter_reduce_(0, page, off, "amin")          # first new row of a page
    old = torch.where((first == 0)[:, None], 0.0, scale)
    touched = first < bs
    s = torch.where(touched[:, None], torch.maximum(old, need), scale)
    pages = touched.nonzero().squeeze(1)
    raw = codes.view(torch.uint8)
    was, grow = raw[pages].view(codes.dtype).float(), (old / s)[pages][:, :, None, None]
    kept = torch.arange(bs, device=x.device)[None, None, :, None] < first[pages][:, None, None, None]
    raw[pages] = torch.where(kept, was * grow, was).to(codes.dtype).view(torch.uint8)
    raw[page, :, off] = (x / s[page][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(codes.dtype).view(torch.uint8)
    scale.copy_(s)


def _plain_append(state):
    b, pos = _rows(state)
    bs = state["case"]["block"]
    page, off = state["tables"][b, pos // bs].long(), pos % bs
    _append_one(state["k"], state["kc"], state["ks"], page, off)
    _append_one(state["v"], state["vc"], state["vs"], page, off)
    return state["kc"], state["vc"], state["ks"], state["vs"]


def _plain_attend(state):
    case = state["case"]
    q, tables, lens, new = state["q"], state["tables"].long(), state["lens"].long(), state["new"].long()
    B, W = tables.shape
    nkv, D, bs, N = case["nkv"], case["dim"], case["block"], state["max_new"]
    rep = case["nq"] // nkv
    codes = lambda c: c.view(torch.uint8)[tables].view(c.dtype).float()  # noqa: E731
    k = (codes(state["kc"]) * state["ks"][tables][..., None, None]).transpose(1, 2).reshape(B, nkv, 1, W * bs, D)
    v = (codes(state["vc"]) * state["vs"][tables][..., None, None]).transpose(1, 2).reshape(B, nkv, 1, W * bs, D)
    b, pos = _rows(state)
    j = pos - (lens - new)[b]                                                                      # row inside its sequence
    rows = torch.zeros(B, N, case["nq"], D, device=q.device)
    rows[b, j] = q.float()
    rows = rows.view(B, N, nkv, rep, D).permute(0, 2, 3, 1, 4)                                     # [B, nkv, rep, N, D]
    s = torch.matmul(rows.reshape(B, nkv, 1, rep * N, D), k.transpose(-1, -2)).view(B, nkv, rep, N, W * bs) / math.sqrt(D)
    last = (lens - new)[:, None] + torch.arange(N, device=q.device)                                # [B, N]
    seen = torch.arange(W * bs, device=q.device)[None, None, :] <= last[:, :, None]
    seen &= torch.arange(W * bs, device=q.device)[None, None, :] < lens[:, None, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, nkv, 1, rep * N, W * bs), v).view(B, nkv, rep, N, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, N, case["nq"], D)[b, j].to(q.dtype)


def _plain_logprob(state):
    case = state["case"]
    tok, n, inv = state["tok"], case["top"], 1.0 / case["temp"]
    raw = state["z"].float()
    z = raw * inv
    top = z.amax(-1, keepdim=True)
    some = top > -math.inf                                                                         # a row with anything left
    e = torch.where(some, (z - top).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    lse = torch.where(some, top + total.log(), -math.inf)
    p = torch.where(some, e / total, 0.0)
    logp = torch.where(z > -math.inf, z - lse, -math.inf)
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    has = (tok >= 0) & (tok < z.shape[1])
    at = tok.clamp(0, z.shape[1] - 1)[:, None]
    lp = torch.where(has, logp.gather(1, at).squeeze(1), 0.0)
    # the n largest logits, ties by the lowest index: unique whole-number keys
    bits = (raw + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)) * (1 << 20) + ((1 << 20) - 1 - torch.arange(z.shape[1], device=z.device))
    ids = torch.topk(key, n, dim=1).indices
    tops = logp.gather(1, ids)
    if not case["grad"]:
        return lp, ent, tops, ids
    g_lp, g_ent, g_top = state["grads"]
    g_lp = torch.where(has & some.squeeze(1), g_lp, 0.0)
    g_top = torch.where(some, g_top, 0.0)
    dz = -p * (g_lp + g_top.sum(-1))[:, None] - torch.where(p > 0, p * (logp + ent[:, None]), 0.0) * g_ent[:, None]
    dz.scatter_add_(1, at, g_lp[:, None])
    dz.scatter_add_(1, ids, g_top)
    return lp, ent, tops, ids, (dz * inv).to(state["z"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "logprob":
        size = case["rows"] * case["vocab"] * (4 if case["dtype"] == "fp32" else 2)
        return dict(bytes=size * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top"]), flops=case["rows"] * case["vocab"] * (8 if case["grad"] else 4))
    lens, new = _lengths(case, 0)
    T, size = float(new.sum()), 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "append":
        return dict(bytes=T * case["nkv"] * 2 * case["dim"] * (size + 1), flops=T * case["nkv"] * 2 * case["dim"] * 2)
    pairs = float((new * lens - new * (new - 1) // 2).sum())
    read = float(torch.where(new > 0, lens, 0).sum()) * case["nkv"] * 2 * case["dim"]
    return dict(bytes=read + 2 * T * case["nq"] * case["dim"] * size, flops=4.0 * pairs * case["nq"] * case["dim"])


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprob":
        return _exact_logprob(case, s)
    lens, new = (t.tolist() for t in _lengths(case, seed))
    return (_exact_append if case["op"] == "append" else _exact_attend)(case, s, lens, new)


def _exact_append(case, s, lens, new):
    """Codes before they are rounded to 8 bits; scales as they have to be."""
    bs, tables = case["block"], s["tables"].tolist()
    outs = []
    for x, codes, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        codes, scale, x = codes.double(), scale.double(), x.double()
        row = 0
        for b in range(len(lens)):
            pos, end = lens[b] - new[b], lens[b]
            while pos < end:
                m = min(bs - pos % bs, end - pos)
                page, off = tables[b][pos // bs], pos % bs
                part = x[row:row + m].transpose(0, 1)                                              # [nkv, m, D]
                big = part.abs().amax((1, 2))
                need = torch.full_like(big, SCALE_MIN)
                while bool((big > E4M3_MAX * need).any()):
                    need = torch.where(big > E4M3_MAX * need, 2 * need, need)
                if off:
                    grown = torch.maximum(scale[page], need)
                    codes[page, :, :off] *= (scale[page] / grown)[:, None, None]
                    need = grown
                scale[page] = need
                codes[page, :, off:off + m] = part / need[:, None, None]
                pos, row = pos + m, row + m
        outs.append((codes, scale))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]


def _exact_attend(case, s, lens, new):
    nkv, D, bs, nq = case["nkv"], case["dim"], case["block"], case["nq"]
    out, row = torch.zeros(s["T"], nq, D, dtype=torch.float64, device="cuda"), 0
    for b in range(len(lens)):
        L, n = lens[b], new[b]
        if n == 0:
            continue
        pages = s["tables"][b, :(L + bs - 1) // bs].long()
        k = (s["kc"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s["ks"][pages].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(nkv, -1, D)[:, :L]
        v = (s["vc"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s["vs"][pages].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(nkv, -1, D)[:, :L]
        q = s["q"][row:row + n].double().view(n, nkv, nq // nkv, D)
        a = torch.einsum("nhrd,hld->hrnl", q, k) * D ** -0.5
        late = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
        p = torch.softmax(a.masked_fill(late, -math.inf), -1)
        out[row:row + n] = torch.einsum("hrnl,hld->nhrd", p, v).reshape(n, nq, D)
        row += n
    return out


def _exact_logprob(case, s):
    R, V, n, T = case["rows"], case["vocab"], case["top"], case["temp"]
    lp, ent = torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    tops = torch.zeros(R, n, dtype=torch.float64)
    dz = torch.zeros(R, V, dtype=torch.float64, device="cuda") if case["grad"] else None
    tok = s["tok"].tolist()
    g_lp, g_ent, g_top = (g.double() for g in s["grads"])
    for r in range(R):
        z = s["z"][r].double() / T
        order = torch.sort(s["z"][r].float(), descending=True, stable=True).indices[:n]
        lse = torch.logsumexp(z, 0)
        if not bool(lse > -math.inf):
            lp[r] = -math.inf if tok[r] >= 0 else 0.0
            tops[r] = -math.inf
            continue
        logp = z - lse
        p = logp.exp()
        plogp = torch.nan_to_num(p * logp, nan=0.0)
        h = -plogp.sum()
        lp[r], ent[r], tops[r] = logp[tok[r]] if tok[r] >= 0 else 0.0, h, logp[order]
        if dz is not None:
            a = g_lp[r] if tok[r] >= 0 else 0.0 * g_lp[r]
            d = -p * (a + g_top[r].sum()) - g_ent[r] * (plogp + p * h)
            if tok[r] >= 0:
                d[tok[r]] += a
            d[order] += g_top[r]
            dz[r] = d / T
    return (lp, ent, tops, None) + ((dz,) if case["grad"] else ())
