"""Measured cases of the latent-attention operators around the 8-bit paged cache.

Four operators: appending tokens to the cache (latent norm, position rotation,
quantisation), single-token attention over it in absorbed form, reading a
sequence's rows back for re-expansion, and prompt attention in expanded form.

The 8-bit cache holds, per token, R latent values in e4m3 and P rotated key
values in bf16, both divided by the token's scale, a power of two:
    row = scale * [e4m3 latent (R) | bf16 rope key (P)]
`cache` is uint8 [n_blocks, 64, R + 2P], `scales` fp32 [n_blocks, 64].
"""

import math

import numpy as np
import torch

own = False

PAGE = 64
THETA = 10000.0
EPS = 1e-6

# head layouts of the repository's model configurations: the DeepSeek-V3 and
# DeepSeek-V2-Lite shapes and the tiny test model
V3 = dict(H=128, R=512, P=64, nope=128, vd=128)
V2_LITE = dict(H=16, R=512, P=64, nope=128, vd=128)
TINY = dict(H=8, R=128, P=32, nope=64, vd=64)


def listed():
    return [
        # one user generating with V2-Lite: the smallest call, all latency
        dict(name="append v2lite token", op="append", **V2_LITE, rows=1, lo=512, hi=512, ragged=1, pad=0),
        # a decode step's batch at the V3 target's 32 sequences a GPU, 4k context
        dict(name="append v3 batch", op="append", **V3, rows=32, lo=2048, hi=4200, ragged=2, pad=0),
        # a whole prefill chunk (the engine's most rows a call) of ragged prompts, its end padded
        dict(name="append v3 chunk", op="append", **V3, rows=4096, lo=0, hi=4095, ragged=3, pad=37),
        # one V2-Lite sequence in the middle of a chat
        dict(name="decode v2lite one", op="decode", **V2_LITE, B=1, lo=777, hi=777, ragged=4),
        # the V2-Lite throughput workload: 32 sequences of 512-token prompts and up to 256 new tokens
        dict(name="decode v2lite batch", op="decode", **V2_LITE, B=32, lo=513, hi=768, ragged=5),
        # the isolated V3 attention workload: 64 sequences, context uniform in [1024, 8192]
        dict(name="decode v3 batch", op="decode", **V3, B=64, lo=1024, hi=8192, ragged=6),
        # few long documents: the split over a long axis
        dict(name="decode v3 long", op="decode", **V3, B=3, lo=60000, hi=131072, ragged=7),
        # one sequence's history before its next chunk
        dict(name="read v2lite one", op="read", R=512, P=64, B=1, lo=700, hi=700, ragged=8),
        # several histories of a chunk with mixed prompts
        dict(name="read v3 batch", op="read", R=512, P=64, B=16, lo=1, hi=8192, ragged=9),
        # the V2-Lite workload's prompts: 32 of about 512 tokens
        dict(name="prefill v2lite prompts", op="prefill", **V2_LITE, B=32, lo=400, hi=512, ragged=10, past=0),
        # a V3 chunk of 1024 new tokens behind 3000 cached ones
        dict(name="prefill v3 behind history", op="prefill", **V3, B=1, lo=1024, hi=1024, ragged=11, past=3000),
        # a long V3 prompt in one chunk
        dict(name="prefill v3 prompt", op="prefill", **V3, B=1, lo=4096, hi=4096, ragged=12, past=0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "read", "prefill", "prefill"])
    shape = dict(rng.choice([V3, V2_LITE, TINY]))
    ragged = rng.randrange(1 << 20)
    if op == "append":
        shape["H"] = rng.choice([shape["H"], rng.randint(1, shape["H"])])
        rows = _log_int(rng, 1, 4096)
        hi = _log_int(rng, 1, 8192)
        return dict(op=op, **shape, rows=rows, lo=rng.randint(0, hi), hi=hi, ragged=ragged, pad=rng.randint(0, min(5, rows - 1)))
    if op == "decode":
        shape["H"] = rng.choice([shape["H"], rng.randint(1, 128)])
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, max(64, min(65536, 262144 // B)))
        return dict(op=op, **shape, B=B, lo=rng.randint(0, hi), hi=hi, ragged=ragged)
    if op == "read":
        B = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 131072 // B)
        return dict(op=op, R=shape["R"], P=shape["P"], B=B, lo=rng.randint(0, hi), hi=hi, ragged=ragged)
    shape["H"] = rng.choice([shape["H"], rng.randint(1, shape["H"])])
    B = _log_int(rng, 1, 16)
    hi = _log_int(rng, 1, int(4096 / math.sqrt(B)))
    past = rng.choice([0, 0, rng.randint(1, 2000)])
    past = 0 if hi * (hi + 2 * past) * B > 4096 * 4096 else past
    return dict(op=op, **shape, B=B, lo=rng.randint(1, hi), hi=hi, ragged=ragged, past=past)


# ------------------------------------------------------------------ inputs


def _lens(case, n):
    """n ragged lengths of a case, the first the largest allowed (a fixed choice of the case, not of the seed)."""
    r = np.random.default_rng(case["ragged"])
    v = r.integers(case["lo"], case["hi"] + 1, size=n)
    v[0] = case["hi"]
    return v.astype(np.int64)


def _append_rows(case):
    """Sequence, position (-1: padding) of each row, and the number of sequences: runs of consecutive positions."""
    rows, pad = case["rows"], case["pad"]
    seq, pos, b, left = [], [], 0, rows - pad
    r = np.random.default_rng(case["ragged"])
    while left > 0:
        # decode batches append one token a sequence, chunks whole runs
        n = 1 if rows <= 256 else int(min(left, r.integers(1, 1024)))
        start = case["hi"] if b == 0 and n == 1 else int(r.integers(case["lo"], case["hi"] + 1))
        seq += [b] * n
        pos += range(start, start + n)
        b, left = b + 1, left - n
    return np.array(seq + [0] * pad), np.array(pos + [-1] * pad), b


def _pages(rng, lens):
    """A block table over a random permutation of just enough pages for these lengths."""
    pages = (np.asarray(lens) + PAGE - 1) // PAGE
    n_blocks, width = max(1, int(pages.sum())), max(1, int(pages.max()))
    table = np.zeros((len(pages), width), np.int32)
    perm, at = rng.permutation(n_blocks), 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), n_blocks


def _quantise(c):
    """e4m3 codes and power-of-two scale of rows c: the smallest scale that keeps the row within 448."""
    amax = c.abs().amax(-1).float()
    m, e = torch.frexp(amax)
    s = torch.where(m <= 0.875, e - 9, e - 8).clamp(-64, 64)
    scale = torch.where(amax > 0, torch.exp2(s.double()), torch.ones((), dtype=torch.float64, device=c.device))
    return (c / scale[..., None].to(c.dtype)).float().to(torch.float8_e4m3fn), scale.float()


def _cache(g, n_blocks, R, P):
    """A cache whose rows hold normed latents (unit variance under a norm weight near 1) and rotated keys."""
    w = 1 + 0.2 * torch.randn(R, generator=g, device="cuda")
    c = torch.randn(n_blocks, PAGE, R, generator=g, device="cuda") * w
    kr = torch.randn(n_blocks, PAGE, P, generator=g, device="cuda")
    q8, scale = _quantise(c)
    kr = (kr.bfloat16().float() / scale[..., None]).bfloat16()
    return torch.cat([q8.view(torch.uint8), kr.view(torch.uint8)], -1), scale


def _cu(lens):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    rng = np.random.default_rng(seed * 1000003 + 29)

    def randn(*shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case=case, op=case["op"])
    P = case["P"]
    R = case["R"]
    if case["op"] == "append":
        seq, pos, n_seq = _append_rows(case)
        T, H, qh = case["rows"], case["H"], case["nope"] + P
        last = np.zeros(n_seq, np.int64)
        np.maximum.at(last, seq[pos >= 0], pos[pos >= 0] + 1)
        s["block_table"], s["n_blocks"] = _pages(rng, last)
        s["kv_a"] = randn(T, R + P, dtype=torch.float32, std=1.3)
        s["w_norm"] = 1 + 0.2 * randn(R, dtype=torch.float32)
        s["q"] = randn(T, H * qh)
        s["positions"] = torch.from_numpy(pos.astype(np.int32)).cuda()
        s["seq_ids"] = torch.from_numpy(seq.astype(np.int32)).cuda()
        s["cache"], s["scales"] = _cache(g, s["n_blocks"], R, P)
        s["q_rope"] = torch.zeros(T, H, P, dtype=torch.bfloat16, device="cuda")
    elif case["op"] == "decode":
        lens = _lens(case, case["B"])
        s["block_table"], n_blocks = _pages(rng, lens)
        s["seq_lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        s["cache"], s["scales"] = _cache(g, n_blocks, R, P)
        s["q_lat"], s["q_rope"] = randn(case["B"], case["H"], R), randn(case["B"], case["H"], P)
        s["scale"] = 1.0 / math.sqrt(case["nope"] + P)
    elif case["op"] == "read":
        lens = _lens(case, case["B"])
        s["block_table"], n_blocks = _pages(rng, lens)
        s["cu"], s["total"] = _cu(lens), int(lens.sum())
        s["cache"], s["scales"] = _cache(g, n_blocks, R, P)
    else:
        lq = _lens(case, case["B"])
        lk = lq + case["past"]
        H, nope, vd = case["H"], case["nope"], case["vd"]
        s["cu_q"], s["cu_k"], s["max_q"], s["max_k"] = _cu(lq), _cu(lk), int(lq.max()), int(lk.max())
        # as the projections leave them: the nope parts inside [T, H, nope + P] queries and [T, H, nope + vd] keys|values
        q, kv = randn(int(lq.sum()), H, nope + P), randn(int(lk.sum()), H, nope + vd)
        s["q_nope"], s["q_rope"] = q[..., :nope], randn(int(lq.sum()), H, P)
        s["k_nope"], s["v"], s["k_rope"] = kv[..., :nope], kv[..., nope:], randn(int(lk.sum()), P)
        s["scale"] = 1.0 / math.sqrt(nope + P)
    return s


# --------------------------------------------------------- the framework's calls

_ctx = None


def _context():
    """The context that a program keeps for its GPU, on torch's default stream."""
    global _ctx
    if _ctx is None:
        import deepseek_cpp_infer_b200 as dsb

        _ctx = dsb.Context(torch.cuda.current_device())
        _ctx.use_legacy_stream()
    return _ctx


def _run_own(s):
    ctx, c = _context(), s["case"]
    if s["op"] == "append":
        ctx.kv_norm_rope_append_fp8(
            s["kv_a"], s["w_norm"], s["q"], s["positions"], s["block_table"], c["H"], c["nope"], c["R"], c["P"], EPS,
            THETA, s["cache"], s["scales"], s["q_rope"], seq_ids=s["seq_ids"])
        return _append_outputs(s)
    if s["op"] == "decode":
        out = torch.empty_like(s["q_lat"])
        ctx.mla_decode_fp8(s["q_lat"], s["q_rope"], s["cache"], s["scales"], s["block_table"], s["seq_lens"],
                           s["scale"], out)
        return out
    if s["op"] == "read":
        lat = torch.empty(s["total"], c["R"], dtype=torch.bfloat16, device="cuda")
        rope = torch.empty(s["total"], c["P"], dtype=torch.bfloat16, device="cuda")
        ctx.mla_cache_read_fp8(s["cache"], s["scales"], s["block_table"], s["cu"], lat, rope)
        return lat, rope
    T = s["q_nope"].shape[0]
    out = torch.empty(T, c["H"], c["vd"], dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(T, c["H"], dtype=torch.float32, device="cuda")
    ctx.mla_prefill(s["q_nope"], s["q_rope"], s["k_nope"], s["k_rope"], s["v"], s["cu_q"], s["cu_k"], s["max_q"],
                    s["scale"], out, lse=lse)
    return out, lse


# ------------------------------------------------------------- plain forms


def _append_outputs(s):
    """The whole cache, as the values its bytes hold, its scales and the rotated queries."""
    R = s["case"]["R"]
    return dict(latent=s["cache"][..., :R].view(torch.float8_e4m3fn), rope=s["cache"][..., R:].view(torch.bfloat16),
                scales=s["scales"], q_rope=s["q_rope"])


def _rotate(x, cos, sin):
    """Rotates the interleaved pairs of the last dimension."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _run_append(s):
    c = s["case"]
    R, P, nope = c["R"], c["P"], c["nope"]
    live = s["positions"] >= 0
    pos = s["positions"].clamp_min(0).long()
    # 64 bits: angles of far positions, and latents next to a rounding border
    x = s["kv_a"][:, :R].double()
    lat = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["w_norm"].double()
    q8, scale = _quantise(lat)
    freq = THETA ** (-torch.arange(0, P, 2, dtype=torch.float64, device="cuda") / P)
    ang = pos[:, None].double() * freq
    cos, sin = ang.cos().float(), ang.sin().float()
    kr = (_rotate(s["kv_a"][:, R:], cos, sin).bfloat16().float() / scale[:, None]).bfloat16()
    q = s["q"].view(len(pos), c["H"], nope + P)[..., nope:].float()
    q = _rotate(q, cos[:, None], sin[:, None]).bfloat16()
    at = s["block_table"][s["seq_ids"].long(), pos // PAGE].long() * PAGE + pos % PAGE
    rows = torch.cat([q8.view(torch.uint8), kr.view(torch.uint8)], -1)
    s["cache"].view(-1, R + 2 * P)[at[live]] = rows[live]
    s["scales"].view(-1)[at[live]] = scale[live]
    s["q_rope"].copy_(torch.where(live[:, None, None], q, s["q_rope"]))
    return _append_outputs(s)


def _rows32(s, table):
    """The cached rows of a block table, [B, width * 64, R] and [.., P] in 32 bits."""
    R = s["case"]["R"]
    page, scale = s["cache"][table.long()].flatten(1, 2), s["scales"][table.long()].flatten(1, 2)[..., None]
    return page[..., :R].view(torch.float8_e4m3fn).float() * scale, page[..., R:].view(torch.bfloat16).float() * scale


def _softmax(scores, mask):
    """Masked softmax over the last dimension (a row with nothing left: zeros), and its log-sum-exp."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    return p / total.clamp_min(1e-30), (top + total.log()).squeeze(-1)


def _run_decode(s):
    lat, rope = _rows32(s, s["block_table"])
    mask = torch.arange(lat.shape[1], device="cuda")[None, None] < s["seq_lens"][:, None, None]
    scores = (s["q_lat"].float() @ lat.mT + s["q_rope"].float() @ rope.mT) * s["scale"]
    return (_softmax(scores, mask)[0] @ lat).bfloat16()


def _of_rows(cu, width):
    """Row indices [B, width] of the sequences of cu, and which of them are theirs."""
    at = torch.arange(width, device="cuda")[None] + cu[:-1, None].long()
    mine = at < cu[1:, None]
    return torch.where(mine, at, torch.zeros_like(at)), mine


def _run_read(s):
    at = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], at, right=True) - 1
    t = at - s["cu"][b]
    row = s["block_table"][b, (t // PAGE).long()].long() * PAGE + t % PAGE
    R = s["case"]["R"]
    rows, scale = s["cache"].flatten(0, 1)[row], s["scales"].flatten()[row][:, None]
    lat = rows[:, :R].contiguous().view(torch.float8_e4m3fn).float() * scale
    rope = rows[:, R:].contiguous().view(torch.bfloat16).float() * scale
    return lat.bfloat16(), rope.bfloat16()


def _run_prefill(s):
    iq, mq = _of_rows(s["cu_q"], s["max_q"])
    ik, mk = _of_rows(s["cu_k"], s["max_k"])
    q = torch.cat([s["q_nope"], s["q_rope"]], -1)[iq].float().transpose(1, 2)
    k = torch.cat([s["k_nope"], s["k_rope"][:, None].expand(-1, s["case"]["H"], -1)], -1)[ik].float().transpose(1, 2)
    v = s["v"][ik].float().transpose(1, 2)
    behind = (s["cu_k"].diff() - s["cu_q"].diff())[:, None, None]
    mask = torch.arange(s["max_k"], device="cuda") <= torch.arange(s["max_q"], device="cuda")[:, None] + behind
    p, lse = _softmax((q @ k.mT) * s["scale"], (mask & mk[:, None])[:, None])
    return (p @ v).transpose(1, 2)[mq].bfloat16(), lse.transpose(1, 2)[mq]


def run(s):
    if own:
        return _run_own(s)
    return dict(append=_run_append, decode=_run_decode, read=_run_read, prefill=_run_prefill)[s["op"]](s)


# ------------------------------------------------------------------ 64 bits


def _row64(s, b, n):
    """The first n cached rows of sequence b in 64 bits."""
    R = s["case"]["R"]
    pages = s["block_table"][b, :(n + PAGE - 1) // PAGE].long()
    sc = s["scales"][pages].reshape(-1)[:n, None].double()
    raw = s["cache"][pages].reshape(-1, s["cache"].shape[-1])[:n]
    lat = raw[:, :R].contiguous().view(torch.float8_e4m3fn).to(torch.float32).double() * sc
    return lat, raw[:, R:].contiguous().view(torch.bfloat16).double() * sc


def exact(case, seed):
    s = prepare(case, seed)
    R, P = case["R"], case["P"]
    if case["op"] == "append":
        # what is held in 8 bits stands for a rounded value: only the scales and the rotations have one in 64 bits
        live = s["positions"] >= 0
        rope = s["cache"][..., R:].contiguous().view(torch.bfloat16).double().flatten(0, 1)
        scales = s["scales"].double().flatten()
        k = torch.arange(P // 2, dtype=torch.float64, device="cuda")
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(len(live), P // 2),
                        s["positions"].double()[:, None] * torch.exp(-2 * k / P * math.log(THETA)))

        def turn(x):
            return torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (P // 2, 2)).contiguous()) * z_of(x)).flatten(-2)

        def z_of(x):
            return z if x.dim() == 2 else z[:, None]

        x = s["kv_a"][:, :R].double()
        lat = x / (x.pow(2).sum(-1, keepdim=True) / R + EPS).sqrt() * s["w_norm"].double()
        e = torch.ceil(torch.log2(lat.abs().max(-1).values / 448))
        pos, seq = s["positions"].long().clamp_min(0), s["seq_ids"].long()
        at = (s["block_table"][seq, pos // PAGE].long() * PAGE + pos % PAGE)[live]
        scales[at] = torch.exp2(e)[live]
        rope[at] = (turn(s["kv_a"][:, R:]) / torch.exp2(e)[:, None])[live]
        q = s["q"].unflatten(-1, (case["H"], case["nope"] + P))[..., case["nope"]:]
        q = torch.where(live[:, None, None], turn(q), s["q_rope"].double())
        return dict(latent=None, rope=rope.view(*s["cache"].shape[:2], P), scales=scales.view_as(s["scales"]), q_rope=q)
    if case["op"] == "decode":
        out = torch.zeros(*s["q_lat"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["seq_lens"].tolist()):
            if n > 0:
                lat, rope = _row64(s, b, n)
                a = s["q_lat"][b].double() @ lat.T + s["q_rope"][b].double() @ rope.T
                out[b] = torch.softmax(a * s["scale"], -1) @ lat
        return out
    if case["op"] == "read":
        cu = s["cu"].tolist()
        rows = [_row64(s, b, cu[b + 1] - cu[b]) for b in range(case["B"])]
        return torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
    H = case["H"]
    out = torch.zeros(*s["q_nope"].shape[:2], case["vd"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(*s["q_nope"].shape[:2], dtype=torch.float64, device="cuda")
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(case["B"]):
        q, k = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        nq, nk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
        for h in range(H):
            a = s["q_nope"][q, h].double() @ s["k_nope"][k, h].double().T + s["q_rope"][q, h].double() @ s["k_rope"][k].double().T
            a = (a * s["scale"]).masked_fill(hidden, -math.inf)
            lse[q, h] = torch.logsumexp(a, -1)
            out[q, h] = torch.softmax(a, -1) @ s["v"][k, h].double()
    return out, lse


# --------------------------------------------------------------------- work


def work(case):
    P, R = case["P"], case["R"]
    row = R + 2 * P + 4  # a cached token: latents, rope key, scale
    if case["op"] == "append":
        live, H = case["rows"] - case["pad"], case["H"]
        return {"bytes": live * (4 * (R + P) + row + 12 + 4 * H * P) + 4 * R, "flops": live * (6 * R + 3 * P * (H + 1))}
    if case["op"] == "decode":
        n, q = int(_lens(case, case["B"]).sum()), case["B"] * case["H"]
        return {"bytes": n * row + n // PAGE * 4 + q * (2 * (R + P) + 2 * R), "flops": 2 * n * case["H"] * (2 * R + P)}
    if case["op"] == "read":
        n = int(_lens(case, case["B"]).sum())
        return {"bytes": max(1, n * (row + 2 * (R + P))), "flops": n * (R + P)}
    lq = _lens(case, case["B"])
    lk, H, dq, vd = lq + case["past"], case["H"], case["nope"] + P, case["vd"]
    pairs = int((lq * (lk - lq) + lq * (lq + 1) // 2).sum())
    return {"bytes": int(lq.sum()) * H * (2 * dq + 2 * vd + 4) + int(lk.sum()) * (H * 2 * (case["nope"] + vd) + 2 * P),
            "flops": 2 * pairs * H * (dq + vd)}
