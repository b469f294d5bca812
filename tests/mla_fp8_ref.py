"""Plain 64-bit implementations of the 8-bit latent cache operators, and
builders of their inputs (used by tests/test_mla_fp8_gpu.py and
tests/test_mla_prefill_gpu.py).

Rounding bounds follow from the types: a rounding is off by at most half a
step, 2^-8 of the value for bf16 and 2^-4 for e4m3.
"""

import math

import numpy as np

PAGE = 64


def quantise(c):
    """Rows c (float64 torch) -> e4m3 codes (uint8) and the row's power-of-two scale (float32)."""
    import torch

    amax = c.abs().amax(-1).float()
    m, e = torch.frexp(amax)  # m in [0.5, 1): amax = m 2^e, 448 = 0.875 * 2^9
    s = torch.where(m <= 0.875, e - 9, e - 8).clamp(-64, 64)
    scale = torch.where(amax > 0, torch.exp2(s.double()), torch.ones_like(amax, dtype=torch.float64))
    codes = (c / scale[..., None]).float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scale.float()


def make_cache(n_blocks, R, P, seed, device="cuda", std=1.0):
    """A full 8-bit cache of N(0, std) latents and N(0, 1) rope keys: (cache, scales)."""
    import torch

    g = torch.Generator(device=device)
    g.manual_seed(seed)
    c = torch.randn(n_blocks, PAGE, R, generator=g, device=device, dtype=torch.float64) * std
    kr = torch.randn(n_blocks, PAGE, P, generator=g, device=device, dtype=torch.float32)
    codes, scale = quantise(c)
    kr = (kr.bfloat16().float() / scale[..., None]).bfloat16()
    return torch.cat([codes, kr.view(torch.uint8)], -1).contiguous(), scale


def make_table(lens, seed, device="cuda", extra=0, max_blocks=None):
    """A block table over a random permutation of pages; unused slots hold -1.  (table, n_blocks)"""
    import torch

    pages = (np.asarray(lens, np.int64) + PAGE - 1) // PAGE
    n_blocks = max(1, int(pages.sum()) + extra)
    width = max_blocks or max(1, int(pages.max()))
    t = np.full((len(pages), width), -1, np.int32)
    perm, at = np.random.default_rng(seed).permutation(n_blocks), 0
    for b, n in enumerate(pages):
        t[b, :n] = perm[at:at + n]
        at += n
    return torch.from_numpy(t).to(device), n_blocks


def rows64(cache, scales, table, b, n, R):
    """The first n rows of sequence b in 64 bits: latents [n, R], rope keys [n, P]."""
    import torch

    pages = table[b, :(n + PAGE - 1) // PAGE].long()
    raw = cache[pages].reshape(-1, cache.shape[-1])[:n]
    sc = scales[pages].reshape(-1)[:n, None].double()
    lat = raw[:, :R].contiguous().view(torch.float8_e4m3fn).float().double()
    return lat * sc, raw[:, R:].contiguous().view(torch.bfloat16).double() * sc


def decode64(q_lat, q_rope, cache, scales, table, lens, scale):
    """out [B, H, R] in 64 bits, the probability-weighted magnitude of the latents [B, H, R] and the largest
    latent [B] (both for the tolerance)."""
    import torch

    B, H, R = q_lat.shape
    out = torch.zeros(B, H, R, dtype=torch.float64, device=q_lat.device)
    mag, top = torch.zeros_like(out), torch.zeros(B, dtype=torch.float64, device=q_lat.device)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        lat, rope = rows64(cache, scales, table, b, int(n), R)
        s = (q_lat[b].double() @ lat.T + q_rope[b].double() @ rope.T) * scale
        p = torch.softmax(s, -1)
        out[b], mag[b], top[b] = p @ lat, p @ lat.abs(), lat.abs().max()
    return out, mag, top


def decode_tol(out, mag, top):
    """Elementwise bound of |kernel - out|.  The output's bf16 rounding: 2^-8 |out|.  A probability is held as the
    sum of two e4m3 digits, the second rounding the first's remainder (2^-4 of it, itself at most 2^-4 of the
    probability): 2^-8 of each term, so 2^-8 mag.  Below the digits' range each is off by at most 2^-14 of its tile's
    largest (2^-10 at 64 heads a CTA), upwards or downwards; the terms of a sequence must cancel to 2^-11 top, which is
    stricter than their worst case.  Scores carry fp32 sums of exact products (the two digits of
    a query are exact to 2^-18 of its largest value): 2^-12 mag covers sum |q k| scale up to about 500."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -12) * mag + 2.0 ** -11 * top[:, None, None] + 1e-30


def append64(kv_a, w_norm, q, positions, H, nope, R, P, eps, theta):
    """codes, scale, rope key (unrounded, unscaled), rotated queries (unrounded), each in 64 bits."""
    import torch

    x = kv_a[:, :R].double()
    c = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w_norm.double()
    codes, scale = quantise(c)
    k = torch.arange(P // 2, dtype=torch.float64, device=kv_a.device)
    ang = positions.double()[:, None] * torch.exp(-2 * k / P * math.log(theta))

    def turn(v, ang):
        a, b = v[..., 0::2].double(), v[..., 1::2].double()
        return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2)

    kr = turn(kv_a[:, R:R + P], ang)
    qr = turn(q.reshape(len(positions), H, nope + P)[..., nope:], ang[:, None])
    return codes, scale, kr, qr


def prefill64(q_nope, q_rope, k_nope, k_rope, v, cu_q, cu_k, scale, causal=True):
    """out, lse, sum_j p |v| and the row's largest sum |q k| scale, in 64 bits."""
    import torch

    Tq, H, _ = q_nope.shape
    dev = q_nope.device
    out = torch.zeros(Tq, H, v.shape[2], dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    lse = torch.full((Tq, H), -math.inf, dtype=torch.float64, device=dev)
    sab = torch.zeros(Tq, H, dtype=torch.float64, device=dev)
    for b in range(len(cu_q) - 1):
        q, k = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if nq <= 0 or nk <= 0:
            continue
        Q = torch.cat([q_nope[q], q_rope[q]], -1).double().transpose(0, 1)
        K = torch.cat([k_nope[k], k_rope[k][:, None].expand(-1, H, -1)], -1).double().transpose(0, 1)
        V = v[k].double().transpose(0, 1)
        s = Q @ K.transpose(1, 2) * scale
        sab[q] = (Q.abs() @ K.abs().transpose(1, 2) * abs(scale)).amax(-1).T
        if causal:
            hidden = torch.ones(nq, nk, dtype=torch.bool, device=dev).triu(nk - nq + 1)
            s = s.masked_fill(hidden, -math.inf)
        l = torch.logsumexp(s, -1)
        p = torch.where(l[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - l[..., None]))
        out[q], mag[q], lse[q] = (p @ V).transpose(0, 1), (p @ V.abs()).transpose(0, 1), l.T
    return out, lse, mag, sab
