"""The 8-bit paged latent cache on the GPU: appending, absorbed decode
attention and reading back, against plain 64-bit implementations
(tests/mla_fp8_ref.py)."""

import math

import numpy as np
import pytest

import mla_fp8_ref as ref
from deepseek_cpp_infer_b200 import DSB_EINVAL, DSB_EUNSUPPORTED as DSB_UNSUP, Context, DsbError

pytestmark = pytest.mark.gpu

BIG, SMALL = (512, 64, 128), (128, 32, 64)  # (R, P, nope)
THETA, EPS = 10000.0, 1e-6


# ------------------------------------------------------------------ append


def append_case(rows, H, shape, seed, ld_pad=0):
    import torch

    R, P, nope = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kv = torch.randn(rows, R + P + ld_pad, generator=g, device="cuda")
    w = 1 + 0.2 * torch.randn(R, generator=g, device="cuda")
    q = torch.randn(rows, H * (nope + P) + 2 * ld_pad, generator=g, device="cuda").bfloat16()
    return kv, w, q


def run_append(ctx, kv, w, q, pos, table, n_blocks, H, shape, seq_ids=None, fill=0xA5):
    import torch

    R, P, nope = shape
    cache = torch.full((n_blocks, 64, R + 2 * P), fill, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_blocks, 64), -7.0, device="cuda")
    q_rope = torch.full((len(pos), H, P), -7.0, dtype=torch.bfloat16, device="cuda")
    ctx.kv_norm_rope_append_fp8(kv, w, q, pos, table, H, nope, R, P, EPS, THETA, cache, scales, q_rope,
                                seq_ids=seq_ids)
    ctx.sync()
    return cache, scales, q_rope


def check_append(kv, w, q, pos, seq, table, H, shape, cache, scales, q_rope):
    import torch

    R, P, nope = shape
    live = pos >= 0
    codes, scale, kr, qr = ref.append64(kv[:, :R + P], w, q[:, :H * (nope + P)], pos.clamp_min(0), H, nope, R, P, EPS,
                                        THETA)
    at = table[seq.long(), pos.clamp_min(0).long() // 64].long() * 64 + pos.clamp_min(0).long() % 64
    flat, fs = cache.view(-1, R + 2 * P), scales.view(-1)
    assert torch.equal(fs[at[live]], scale[live])
    assert torch.equal(flat[at[live]][:, :R], codes[live])
    got = flat[at[live]][:, R:].contiguous().view(torch.bfloat16).double() * scale[live, None].double()
    # the bf16 rounding, and fp32 products and sines (a few 2^-24 of either input)
    pair = kv[live, R:R + P].double().abs().unflatten(-1, (P // 2, 2)).sum(-1).repeat_interleave(2, -1)
    assert ((got - kr[live]).abs() <= 2.0 ** -8 * kr[live].abs() + 2.0 ** -20 * pair + 1e-38).all()
    qin = q[:, :H * (nope + P)].reshape(len(pos), H, nope + P)[..., nope:].double().abs()
    pair = qin.unflatten(-1, (P // 2, 2)).sum(-1).repeat_interleave(2, -1)[live]
    assert ((q_rope[live].double() - qr[live]).abs() <= 2.0 ** -8 * qr[live].abs() + 2.0 ** -20 * pair + 1e-38).all()
    # nothing else was written
    rest = torch.ones(flat.shape[0], dtype=torch.bool, device="cuda")
    rest[at[live]] = False
    assert (flat[rest] == 0xA5).all() and (fs[rest] == -7.0).all() and (q_rope[~live] == -7.0).all()


@pytest.mark.parametrize("shape", [BIG, SMALL])
@pytest.mark.parametrize("rows,H", [(1, 16), (1, 1), (3, 5), (32, 128), (65, 17)])
def test_append_one_token_per_sequence(gpu_ctx, rows, H, shape):
    import torch

    rng = np.random.default_rng(rows)
    lens = rng.integers(1, 300, size=rows)
    table, n_blocks = ref.make_table(lens, seed=rows, extra=2)
    pos = torch.from_numpy((lens - 1).astype(np.int32)).cuda()
    kv, w, q = append_case(rows, H, shape, seed=rows + 100)
    got = run_append(gpu_ctx, kv, w, q, pos, table, n_blocks, H, shape)
    check_append(kv, w, q, pos, torch.arange(rows, device="cuda"), table, H, shape, *got)


@pytest.mark.parametrize("shape,H", [(BIG, 128), (SMALL, 8)])
def test_append_chunk_with_padding_and_pitches(gpu_ctx, shape, H):
    """Runs of several sequences in one call, padded rows in the middle and at the end, wider row pitches."""
    import torch

    seq, pos = [], []
    for b, (p0, n) in enumerate([(0, 700), (130, 1), (63, 66), (0, 1), (1000, 333)]):
        seq += [b] * n + [0] * (b % 2)
        pos += list(range(p0, p0 + n)) + [-1] * (b % 2)
    seq += [99, -5]
    pos += [-1, -3]
    table, n_blocks = ref.make_table([700, 131, 129, 1, 1333], seed=3, extra=1)
    kv, w, q = append_case(len(seq), H, shape, seed=4, ld_pad=4)
    seq_t = torch.tensor(seq, dtype=torch.int32, device="cuda")
    pos_t = torch.tensor(pos, dtype=torch.int32, device="cuda")
    got = run_append(gpu_ctx, kv, w, q, pos_t, table, n_blocks, H, shape, seq_ids=seq_t)
    check_append(kv, w, q, pos_t, seq_t.clamp(0, 4), table, H, shape, *got)


def test_append_extreme_rows(gpu_ctx):
    """Zero rows, amax on a scale border, tiny and huge norm weights, far positions."""
    import torch

    R, P, nope = shape = BIG
    H, rows = 2, 6
    kv, w, q = append_case(rows, H, shape, seed=8)
    kv[0, :R] = 0
    kv[1, :R] = 0
    kv[1, 5] = 1.0  # c = sqrt(R) w at one place
    kv[2] *= 1e-18
    kv[3] *= 1e15
    w[:3] = torch.tensor([1e-20, 1e20, 0.0])
    pos = torch.tensor([0, 1, 163839, 99999, 131071, 64], dtype=torch.int32, device="cuda")
    table = torch.full((rows, 163840 // 64), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(rows), pos.cpu().long() // 64] = torch.arange(rows, dtype=torch.int32, device="cuda").flip(0)
    got = run_append(gpu_ctx, kv, w, q, pos, table, rows, H, shape)
    check_append(kv, w, q, pos, torch.arange(rows, device="cuda"), table, H, shape, *got)


def test_append_out_of_table_is_reported(gpu_ctx):
    """A position past the table, a page id outside the pool, a sequence outside the table: the row's cache write is
    skipped and dsb_sync reports it; the other rows are written."""
    import torch

    R, P, nope = shape = SMALL
    H = 2
    table = torch.tensor([[0, 9], [1, -1], [2, 2]], dtype=torch.int32, device="cuda")
    for bad_pos, bad_seq in [(128, 0), (64, 0), (64, 1), (3, 3), (3, -1)]:
        kv, w, q = append_case(2, H, shape, seed=9)
        pos = torch.tensor([bad_pos, 5], dtype=torch.int32, device="cuda")
        seq = torch.tensor([bad_seq, 2], dtype=torch.int32, device="cuda")
        cache = torch.full((3, 64, R + 2 * P), 0xA5, dtype=torch.uint8, device="cuda")
        scales = torch.full((3, 64), -7.0, device="cuda")
        q_rope = torch.empty(2, H, P, dtype=torch.bfloat16, device="cuda")
        gpu_ctx.kv_norm_rope_append_fp8(kv, w, q, pos, table, H, nope, R, P, EPS, THETA, cache, scales, q_rope,
                                        seq_ids=seq)
        with pytest.raises(DsbError) as e:
            gpu_ctx.sync()
        assert e.value.code == DSB_EINVAL
        gpu_ctx.sync()  # reported once
        mine = torch.zeros(3, 64, dtype=torch.bool, device="cuda")
        mine[2, 5] = True
        assert (scales[~mine] == -7.0).all() and (cache[~mine] == 0xA5).all() and scales[2, 5] > 0


# ------------------------------------------------------------------ decode


def decode_inputs(lens, H, shape, seed, max_blocks=None, q_std=1.0):
    import torch

    R, P, nope = shape
    table, n_blocks = ref.make_table(lens, seed, extra=1, max_blocks=max_blocks)
    cache, scales = ref.make_cache(n_blocks, R, P, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    B = len(lens)
    q_lat = (torch.randn(B, H, R, generator=g, device="cuda") * q_std).bfloat16()
    q_rope = (torch.randn(B, H, P, generator=g, device="cuda") * q_std).bfloat16()
    return q_lat, q_rope, cache, scales, table, 1 / math.sqrt(nope + P)


def run_decode(ctx, q_lat, q_rope, cache, scales, table, lens, scale):
    import torch

    out = torch.full_like(q_lat, 7.0)
    seq_lens = lens if isinstance(lens, torch.Tensor) else torch.tensor(lens, dtype=torch.int32, device="cuda")
    ctx.mla_decode_fp8(q_lat, q_rope, cache, scales, table, seq_lens, scale, out)
    return out


def check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale):
    want, mag, top = ref.decode64(q_lat, q_rope, cache, scales, table, lens, scale)
    err = (out.double() - want).abs()
    tol = ref.decode_tol(want, mag, top)
    assert (err <= tol).all(), float((err / tol).max())


LENS = [1, 63, 64, 65, 127, 128, 129, 777, 0, 2048]


@pytest.mark.parametrize("shape", [BIG, SMALL])
@pytest.mark.parametrize("H", [1, 8, 16, 17, 32, 33, 64, 65, 100, 128])
def test_decode_ragged(gpu_ctx, H, shape):
    x = decode_inputs(LENS, H, shape, seed=H)
    out = run_decode(gpu_ctx, *x[:5], LENS, x[5])
    gpu_ctx.sync()
    check_decode(out, *x[:5], LENS, x[5])
    assert (out[LENS.index(0)] == 0).all()


@pytest.mark.parametrize("lens,H", [([1], 16), ([0], 16), ([5000], 16), ([40000], 128), ([131072, 1, 60000], 16),
                                    ([300] * 150, 16), ([1024] * 40 + [0] * 40, 128), ([16] * 400, 20)])
def test_decode_splits(gpu_ctx, lens, H):
    """One sequence over many SMs, many sequences per SM, and both."""
    x = decode_inputs(lens, H, BIG, seed=len(lens))
    out = run_decode(gpu_ctx, *x[:5], lens, x[5])
    gpu_ctx.sync()
    check_decode(out, *x[:5], lens, x[5])


@pytest.mark.parametrize("shape", [BIG, SMALL])
@pytest.mark.parametrize("B,H", [(31, 16), (32, 16), (40, 51), (40, 53), (64, 33), (33, 128), (700, 3)])
def test_decode_merges(gpu_ctx, B, H, shape):
    """Sequences cut by several runs, whole ones and empty ones, on both sides of the sizes at which the merge of the
    cut ones changes its shape (32 sequences; 2048 rows)."""
    lens = [(0, 1500, 40, 129, 333)[i % 5] + i % 3 for i in range(B)]
    lens[0] = 0
    x = decode_inputs(lens, H, shape, seed=B + H)
    out = run_decode(gpu_ctx, *x[:5], lens, x[5])
    gpu_ctx.sync()
    check_decode(out, *x[:5], lens, x[5])
    assert (out[0] == 0).all()


def test_decode_ignores_what_lies_past_a_length(gpu_ctx):
    """Rows behind a length hold e4m3 NaN codes, infinite rope keys and NaN scales; table slots behind it are -1."""
    import torch

    lens = [1, 70, 128, 200, 0]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=5, max_blocks=6)
    clean = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    used = torch.zeros(cache.shape[0], 64, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for i in range(n):
            used[table[b, i // 64].long(), i % 64] = True
    cache[~used] = 0x7F  # e4m3 NaN; bf16 0x7f7f is 3.4e38
    cache[:, :, 512:][~used] = 0xFF  # bf16 NaN
    scales[~used] = float("nan")
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    assert torch.equal(out.view(torch.int16), clean.view(torch.int16))
    check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale)


def test_decode_attention_sink(gpu_ctx):
    """One token holds most of the probability, thousands share the rest: their contribution must survive."""
    import torch

    n, R = 40000, 512
    q_lat, q_rope, cache, scales, table, scale = decode_inputs([n], 16, BIG, seed=6)
    q_lat.zero_()
    q_rope.zero_()
    q_rope[..., 0] = 1.0
    kr = torch.zeros(cache.shape[0], 64, 64, device="cuda")
    kr[table[0, 0].long(), 0, 0] = 11.0 / scale  # exp(11) against 40000 tokens of weight 1
    codes, sc = ref.quantise(torch.randn(cache.shape[0], 64, R, device="cuda", dtype=torch.float64) * 0.1 + 1.0)
    cache[..., :R], scales[:] = codes, sc
    cache[..., R:] = (kr / sc[..., None]).bfloat16().view(torch.uint8)
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, [n], scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, [n], scale)


@pytest.mark.parametrize("H", [16, 64])
def test_decode_equal_tail_beside_a_peak_in_every_tile(gpu_ctx, H):
    """Equal probabilities whose digits all round the same way, in tiles whose largest is at the low end of the digits'
    window.  Up to 32 heads their floor is 2^-14 of the window's unit and the common bound holds; at 64 each may be
    off by 2^-10 of a unit that is at most its tile's largest: 2^-10 sum_j top(tile of j) |latent_j| more."""
    import torch

    B, n, R = torch.cuda.get_device_properties(0).multi_processor_count, 1024, 512  # a sequence of 8 tiles for every SM
    lens = [n] * B
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, H, BIG, seed=8)
    q_lat.zero_()
    q_rope.zero_()
    q_rope[..., 0] = 1.0
    # the first tile's largest probability is 16 units, the others' 1.05, the tail 8.5 steps of 2^-9
    unit = torch.full((n,), 8.5 * 2.0 ** -9, dtype=torch.float64)
    unit[5::128] = 1.05
    unit[5] = 16.0
    kr = torch.zeros(cache.shape[0], 64, 64, device="cuda")
    kr[table.long(), :, 0] = (unit.log() / scale).float().cuda().view(1, -1, 64).expand(B, -1, -1)
    codes, sc = ref.quantise(torch.randn(cache.shape[0], 64, R, device="cuda", dtype=torch.float64) * 0.1 + 1.0)
    sc.fill_(2.0 ** -8)  # (any power of two: the codes stand for other values then)
    cache[..., :R], scales[:] = codes, sc
    cache[..., R:] = (kr / sc[..., None]).bfloat16().view(torch.uint8)
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    want, mag, top = ref.decode64(q_lat, q_rope, cache, scales, table, lens, scale)
    tol = ref.decode_tol(want, mag, top)
    if H == 64:
        for b in range(B):
            lat, rope = ref.rows64(cache, scales, table, b, n, R)
            p = torch.softmax(rope[:, 0] * scale, -1).view(-1, 128)
            tol[b] += 2.0 ** -10 * (p.amax(1, keepdim=True).expand(-1, 128).reshape(-1) @ lat.abs())
    err = (out.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("lead", [1.0, 2.0, 3.9, 15.0])
@pytest.mark.parametrize("tail", [17.0, 0.9, 0.9 * 2.0 ** -2, 0.9 * 2.0 ** -5])
@pytest.mark.parametrize("H", [16, 32, 64, 128])
def test_decode_tail_below_the_digits_of_its_tile(gpu_ctx, H, tail, lead):
    """A peak in every tile and 127 equal probabilities beside it, `tail` 2^-10 of the peak: around half a step of the
    digits, where all can be lost together, and far below it; the first tile's peak is `lead` times the others'.  What
    lies below the digits' steps costs a sequence at most 2^-8 of its probabilities (2^-10 up to 32 heads): at most
    that much of a tile's mean latent."""

    import torch

    B, n, R = torch.cuda.get_device_properties(0).multi_processor_count, 1024, 512
    lens = [n] * B
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, H, BIG, seed=9)
    q_lat.zero_()
    q_rope.zero_()
    q_rope[..., 0] = 1.0
    unit = torch.full((n,), tail * 2.0 ** -10, dtype=torch.float64)
    unit[5::128] = 1.0
    unit[5] = lead
    kr = torch.zeros(cache.shape[0], 64, 64, device="cuda")
    kr[table.long(), :, 0] = (unit.log() / scale).float().cuda().view(1, -1, 64).expand(B, -1, -1)
    codes, sc = ref.quantise(torch.randn(cache.shape[0], 64, R, device="cuda", dtype=torch.float64) * 0.1 + 1.0)
    sc.fill_(2.0 ** -8)
    cache[..., :R], scales[:] = codes, sc
    cache[..., R:] = (kr / sc[..., None]).bfloat16().view(torch.uint8)
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    want, mag, _ = ref.decode64(q_lat, q_rope, cache, scales, table, lens, scale)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag + 1e-30
    for b in range(B):
        lat, _ = ref.rows64(cache, scales, table, b, n, R)
        tol[b] += 2.0 ** (-8 if H > 32 else -10) * lat.abs().view(-1, 128, R).mean(1).amax(0)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


def test_decode_scales_far_apart(gpu_ctx):
    """Token scales over 20 octaves and queries over 8: the largest tokens' latents dominate the output."""
    import torch

    lens = [500, 130]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=7)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    f = torch.exp2(torch.randint(-20, 1, scales.shape, generator=g, device="cuda").float())
    scales *= f
    q_lat *= torch.exp2(torch.randint(-8, 1, q_lat.shape[:2], generator=g, device="cuda").float())[..., None]
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale)


@pytest.mark.parametrize("q_std", [0.0, 1e-3, 8.0])
def test_decode_flat_and_peaked(gpu_ctx, q_std):
    lens = [900, 64, 3]
    x = decode_inputs(lens, 128, BIG, seed=11, q_std=q_std)
    out = run_decode(gpu_ctx, *x[:5], lens, x[5])
    gpu_ctx.sync()
    check_decode(out, *x[:5], lens, x[5])


def test_decode_zero_and_negative_scale(gpu_ctx):
    lens = [300, 64]
    for scale in (0.0, -0.07):
        x = decode_inputs(lens, 16, BIG, seed=12)
        out = run_decode(gpu_ctx, *x[:5], lens, scale)
        gpu_ctx.sync()
        check_decode(out, *x[:5], lens, scale)


def test_decode_page_order_and_repeats_are_bitwise(gpu_ctx):
    import torch

    lens = [1500, 64, 4000, 333]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 128, BIG, seed=13)
    a = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    assert torch.equal(a, run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale))
    perm = torch.randperm(cache.shape[0], device="cuda")
    c2, s2 = torch.empty_like(cache), torch.empty_like(scales)
    c2[perm], s2[perm] = cache, scales
    t2 = torch.where(table >= 0, perm[table.clamp_min(0).long()].int(), table)
    b = run_decode(gpu_ctx, q_lat, q_rope, c2, s2, t2, lens, scale)
    gpu_ctx.sync()
    assert torch.equal(a, b)


def test_decode_one_page_shared_by_sequences(gpu_ctx):
    """Two sequences with the same first page (a shared prefix)."""
    lens = [100, 150]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=14)
    table[1, 0] = table[0, 0]
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale)


def test_decode_far_pages(gpu_ctx):
    """Page offsets past 2^32 bytes."""
    import torch

    n_blocks, R, P = 110000, 512, 64
    cache = torch.zeros(n_blocks, 64, R + 2 * P, dtype=torch.uint8, device="cuda")
    scales = torch.ones(n_blocks, 64, device="cuda")
    q_lat, q_rope, small, sc, table, scale = decode_inputs([200, 70], 16, BIG, seed=15)
    far = torch.tensor([[109999, 5, 108000, 60000], [54000, 109000, -1, -1]], dtype=torch.int32, device="cuda")
    for b in range(2):
        for i in range(table.shape[1]):
            if table[b, i] >= 0:
                cache[far[b, i].long()], scales[far[b, i].long()] = small[table[b, i].long()], sc[table[b, i].long()]
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, far, [200, 70], scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, far, [200, 70], scale)


def test_decode_captured_and_replayed_with_other_lengths(gpu_ctx):
    import torch

    stream = torch.cuda.Stream()
    ctx = Context(0)
    ctx.set_stream(stream.cuda_stream)
    lens = [900, 1, 2000]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=16)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q_lat)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ctx.mla_decode_fp8(q_lat, q_rope, cache, scales, table, seq_lens, scale, out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.mla_decode_fp8(q_lat, q_rope, cache, scales, table, seq_lens, scale, out)
    for lens2 in ([900, 1, 2000], [0, 1, 129], [64, 0, 1999]):
        seq_lens.copy_(torch.tensor(lens2, dtype=torch.int32))
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_decode(out, q_lat, q_rope, cache, scales, table, lens2, scale)
    ctx.sync()
    del graph
    ctx.close()


def test_decode_bad_lengths_and_pages_are_reported(gpu_ctx):
    """A negative length, a length past the table and a page id outside the pool set the status; the other
    sequences are computed."""
    for what in ("negative", "long", "page", "page_negative"):
        lens = [100, 300, 64]
        q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=17)
        given = list(lens)
        if what == "negative":
            given[1] = -4
        elif what == "long":
            given[1] = table.shape[1] * 64 + 1
        else:
            table[1, 2] = cache.shape[0] if what == "page" else -1
        out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, given, scale)
        with pytest.raises(DsbError) as e:
            gpu_ctx.sync()
        assert e.value.code == DSB_EINVAL
        for b in (0, 2):
            check_decode(out[b:b + 1], q_lat[b:b + 1], q_rope[b:b + 1], cache, scales, table[b:b + 1], [lens[b]], scale)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_decode_non_finite_query_stays_in_its_head(gpu_ctx, value):
    """Its scores are infinite or NaN, so its softmax is NaN; the other heads and sequences are as without it."""
    lens = [300, 200]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=19)
    bad_lat, bad_rope = q_lat.clone(), q_rope.clone()
    bad_lat[0, 3, 100] = value
    bad_rope[1, 9, 5] = value
    out = run_decode(gpu_ctx, bad_lat, bad_rope, cache, scales, table, lens, scale)
    clean = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    assert out[0, 3].isnan().all() and out[1, 9].isnan().all()
    out[0, 3], out[1, 9] = clean[0, 3], clean[1, 9]
    assert (out == clean).all()
    check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale)


@pytest.mark.parametrize("B", [1, 31, 32, 40])
@pytest.mark.parametrize("tiles", [[0], [3], [0, 5], [7]])
def test_decode_nan_tile_of_a_cut_sequence(gpu_ctx, B, tiles):
    """A tile of 128 tokens with NaN rope keys, each tile of its sequence in a run of its own: the sequence's output is
    NaN whichever merge joins the runs, the other sequences' as without it."""
    import torch

    lens = [1000] + [1] * (B - 1)
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=50 + B)
    clean = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    for t in tiles:
        cache[table[0, 2 * t:2 * t + 2].long(), :, 512:] = 0xFF  # bf16 NaN
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    assert out[0].isnan().all()
    assert torch.equal(out[1:], clean[1:]) and clean.isfinite().all()


@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("e", [26, 60, 90, 105, 107, 112, 119])
def test_decode_queries_of_any_finite_size(gpu_ctx, H, e):
    """Queries near the end of the type's range: all weight on the best token, as in 64 bits, over several tiles."""
    import torch

    lens = [1000] * 45 + [64, 1]  # several tiles a run
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, H, BIG, seed=70)
    q_lat *= 2.0 ** e
    q_rope *= 2.0 ** e
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens, scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, lens, scale)


@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("n,none", [(1000, [0]), (1000, [0, 1, 2]), (1000, [3]), (1000, [7]), (260, [0, 1]), (19000, [0, 100])])
def test_decode_tiles_of_infinitely_low_scores(gpu_ctx, H, n, none):
    """Tiles whose scores are all -inf (infinite rope keys) weigh nothing and leave no mark on the others, whose scores
    lie 200 below zero; in a run with others, in runs of their own, and in a whole sequence (NaN, as 0 / 0)."""
    import torch

    lens = [n, 300, 256] + [0] * 300  # (few runs a sequence, and runs with several sequences)
    for B in (3, 303):
        q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens[:B], H, BIG, seed=60)
        q_rope.zero_()
        q_rope[..., 0] = 1.0
        kr = torch.zeros(cache.shape[0], 64, 64, device="cuda")
        kr[..., 0] = -200.0 / scale
        for t in none:
            kr[table[0, 2 * t:2 * t + 2].long(), :, 0] = -math.inf
        kr[table[2, :4].long(), :, 0] = -math.inf
        cache[..., 512:] = (kr / scales[..., None]).bfloat16().view(torch.uint8)
        out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, lens[:B], scale)
        gpu_ctx.sync()
        assert out[2].isnan().all()
        check_decode(out[:2], q_lat[:2], q_rope[:2], cache, scales, table[:2], lens[:2], scale)


def test_decode_length_beyond_32_bit_positions_is_reported(gpu_ctx):
    """A table of 2^24 + 1 pages would hold it; positions past 2^30 are refused instead of wrapping."""
    import torch

    q_lat, q_rope, cache, scales, _, scale = decode_inputs([64], 16, SMALL, seed=18)
    table = torch.zeros(1, (1 << 24) + 1, dtype=torch.int32, device="cuda")
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, [(1 << 30) + 1], scale)
    with pytest.raises(DsbError) as e:
        gpu_ctx.sync()
    assert e.value.code == DSB_EINVAL
    assert (out == 0).all()


# -------------------------------------------------------------------- read


@pytest.mark.parametrize("shape", [BIG, SMALL])
@pytest.mark.parametrize("lens", [[1], [64, 1, 65, 0, 130], [0, 0, 7], [700, 3]])
def test_read_back_is_exact(gpu_ctx, lens, shape):
    import torch

    R, P, _ = shape
    table, n_blocks = ref.make_table(lens, seed=1)
    cache, scales = ref.make_cache(n_blocks, R, P, seed=2)
    T = sum(lens)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    lat = torch.full((T + 3, R + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.full((T + 3, P + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu_ctx.mla_cache_read_fp8(cache, scales, table, cu, lat[:, :R], rope[:, :P])
    gpu_ctx.sync()
    want = [ref.rows64(cache, scales, table, b, n, R) for b, n in enumerate(lens)]
    assert torch.equal(lat[:T, :R].double(), torch.cat([w[0] for w in want]))
    assert torch.equal(rope[:T, :P].double(), torch.cat([w[1] for w in want]))
    # rows behind the last sequence and columns past the row are left as they were
    assert (lat[T:] == 7.0).all() and (rope[T:] == 7.0).all() and (lat[:, R:] == 7.0).all() and (rope[:, P:] == 7.0).all()


@pytest.mark.parametrize("shape", [BIG, SMALL])
def test_read_of_one_part(gpu_ctx, shape):
    """Only the latents, or only the rope keys."""
    import torch

    R, P, _ = shape
    lens = [70, 1, 200]
    table, n_blocks = ref.make_table(lens, seed=5)
    cache, scales = ref.make_cache(n_blocks, R, P, seed=6)
    cu = torch.tensor([0, 70, 71, 271], dtype=torch.int32, device="cuda")
    lat, rope = torch.zeros(271, R, dtype=torch.bfloat16, device="cuda"), torch.zeros(271, P, dtype=torch.bfloat16, device="cuda")
    gpu_ctx.mla_cache_read_fp8(cache, scales, table, cu, lat, None)
    gpu_ctx.mla_cache_read_fp8(cache, scales, table, cu, None, rope)
    gpu_ctx.sync()
    want = [ref.rows64(cache, scales, table, b, n, R) for b, n in enumerate(lens)]
    assert torch.equal(lat.double(), torch.cat([w[0] for w in want]))
    assert torch.equal(rope.double(), torch.cat([w[1] for w in want]))


def test_read_every_code(gpu_ctx):
    """All 256 e4m3 codes (NaN among them) and scales from 2^-64 to 2^64."""
    import torch

    cache = torch.arange(512, device="cuda").to(torch.uint8).repeat(1, 64, 1)
    cache = torch.cat([cache, torch.zeros(1, 64, 128, dtype=torch.uint8, device="cuda")], -1).contiguous()
    scales = torch.exp2(torch.linspace(-64, 64, 64, device="cuda").round())[None].contiguous()
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lat = torch.zeros(64, 512, dtype=torch.bfloat16, device="cuda")
    rope = torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
    gpu_ctx.mla_cache_read_fp8(cache, scales, table, torch.tensor([0, 64], dtype=torch.int32, device="cuda"), lat, rope)
    gpu_ctx.sync()
    want = cache[0, :, :512].contiguous().view(torch.float8_e4m3fn).float() * scales[0][:, None]
    assert torch.equal(torch.nan_to_num(lat.float(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def test_read_bad_pages_are_reported(gpu_ctx):
    import torch

    table = torch.tensor([[0, 5], [1, 2]], dtype=torch.int32, device="cuda")
    cache, scales = ref.make_cache(3, 128, 32, seed=3)
    lat = torch.full((300, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.full((300, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    for cu in ([0, 70, 80], [0, 10, 145]):  # a page outside the pool, a length past the table
        lat.fill_(7.0)
        gpu_ctx.mla_cache_read_fp8(cache, scales, table, torch.tensor(cu, dtype=torch.int32, device="cuda"), lat, rope)
        with pytest.raises(DsbError) as e:
            gpu_ctx.sync()
        assert e.value.code == DSB_EINVAL
        good = ref.rows64(cache, scales, table, 0, min(64, cu[1]), 128)[0]
        assert torch.equal(lat[:len(good)].double(), good)
        assert (lat[64:70] == 7.0).all() if cu[1] == 70 else (lat[138:145] == 7.0).all()


def test_read_more_rows_than_the_buffers_hold_is_reported(gpu_ctx):
    import torch

    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    cache, scales = ref.make_cache(2, 128, 32, seed=4)
    lat = torch.full((90, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.full((90, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu_ctx.mla_cache_read_fp8(cache, scales, table, torch.tensor([0, 81], dtype=torch.int32, device="cuda"), lat[:80],
                               rope[:80])
    with pytest.raises(DsbError) as e:
        gpu_ctx.sync()
    assert e.value.code == DSB_EINVAL
    want = ref.rows64(cache, scales, table, 0, 80, 128)
    assert torch.equal(lat[:80].double(), want[0]) and torch.equal(rope[:80].double(), want[1])
    assert (lat[80:] == 7.0).all() and (rope[80:] == 7.0).all()


# ---------------------------------------------------------------- refusals


def test_decode_table_past_32_bits_is_refused(gpu_ctx):
    """65536 sequences of 32768 pages: an index into the table would not fit an int."""
    d = {k: 16 for k in ("q_lat", "q_rope", "cache", "scales", "table", "lens", "out")}
    args = (gpu_ctx.h, d["q_lat"], d["q_rope"], d["cache"], d["scales"], 1, d["table"], 1 << 15, d["lens"], 1 << 16, 16,
            512, 64, 0.1, d["out"])
    assert gpu_ctx._l.dsb_mla_decode_fp8(*args) == DSB_EINVAL


def test_refusals(gpu_ctx):
    """At the C entry points (the bindings' own checks come before some of these: they raise ValueError)."""
    import torch

    lens = [100]
    q_lat, q_rope, cache, scales, table, scale = decode_inputs(lens, 16, BIG, seed=1)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q_lat)
    kv, w, q = append_case(2, 16, BIG, seed=1)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    qr2 = torch.empty(2, 16, 64, dtype=torch.bfloat16, device="cuda")
    lat = torch.empty(100, 512, dtype=torch.bfloat16, device="cuda")
    rope = torch.empty(100, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 100], dtype=torch.int32, device="cuda")

    def p(t):
        return t.data_ptr()

    l, h, n = gpu_ctx._l, gpu_ctx.h, cache.shape[0]
    dec = dict(ctx=h, q_lat=p(q_lat), q_rope=p(q_rope), cache=p(cache), scales=p(scales), n_blocks=n, table=p(table),
               max_blocks=table.shape[1], lens=p(sl), B=1, H=16, R=512, P=64, scale=scale, out=p(out))
    app = dict(ctx=h, kv=p(kv), ld_kv=kv.stride(0), w=p(w), q=p(q), ldq=q.stride(0), pos=p(pos), seq=None,
               table=p(table), n_seqs=2, max_blocks=table.shape[1], B=2, H=16, nope=128, R=512, P=64, eps=EPS,
               theta=THETA, cache=p(cache), scales=p(scales), n_blocks=n, q_rope=p(qr2))
    read = dict(ctx=h, cache=p(cache), scales=p(scales), n_blocks=n, table=p(table), max_blocks=table.shape[1],
                cu=p(cu), B=1, T=100, R=512, P=64, lat=p(lat), ld_lat=512, rope=p(rope), ld_rope=64)
    for f, args, bad in (
            (l.dsb_mla_decode_fp8, dec,
             [(DSB_EINVAL, k, None) for k in ("ctx", "q_lat", "q_rope", "cache", "scales", "table", "lens", "out")]
             + [(DSB_EINVAL, "scale", float("nan")), (DSB_EINVAL, "scale", float("inf")), (DSB_UNSUP, "R", 256),
                (DSB_UNSUP, "P", 32), (DSB_EINVAL, "H", 0), (DSB_EINVAL, "H", 129), (DSB_EINVAL, "B", 0),
                (DSB_EINVAL, "max_blocks", 0), (DSB_EINVAL, "n_blocks", 0), (DSB_EINVAL, "n_blocks", 1 << 25),
                (DSB_EINVAL, "B", 65537), (DSB_EINVAL, "out", p(out) + 2), (DSB_EINVAL, "q_lat", p(q_lat) + 8), (DSB_EINVAL, "cache", p(cache) + 1)]),
            (l.dsb_kv_norm_rope_append_fp8, app,
             [(DSB_EINVAL, k, None) for k in ("ctx", "kv", "w", "q", "pos", "table", "cache", "scales", "q_rope")]
             + [(DSB_UNSUP, "R", 256), (DSB_UNSUP, "P", 128), (DSB_EINVAL, "nope", 100), (DSB_EINVAL, "nope", -8),
                (DSB_EINVAL, "theta", 0.0), (DSB_EINVAL, "theta", float("inf")), (DSB_EINVAL, "eps", -1.0),
                (DSB_EINVAL, "ldq", 16 * 192 - 8), (DSB_EINVAL, "ld_kv", 575), (DSB_EINVAL, "ld_kv", 578),
                (DSB_EINVAL, "n_seqs", 1), (DSB_EINVAL, "H", 0), (DSB_EINVAL, "B", 0), (DSB_EINVAL, "kv", p(kv) + 4),
                (DSB_EINVAL, "n_blocks", 0)]),
            (l.dsb_mla_cache_read_fp8, read,
             [(DSB_EINVAL, k, None) for k in ("ctx", "cache", "scales", "table", "cu")]
             + [(DSB_UNSUP, "R", 64), (DSB_EINVAL, "T", -1), (DSB_EINVAL, "B", 0), (DSB_EINVAL, "ld_lat", 504),
                (DSB_EINVAL, "ld_lat", 516), (DSB_EINVAL, "ld_rope", 56), (DSB_EINVAL, "lat", p(lat) + 2)])):
        for code, k, v in bad:
            assert f(*{**args, k: v}.values()) == code, (f.__name__, k, v)
    for args in ((q_lat, q_rope, cache, scales, table, sl.long(), scale, out),
                 (q_lat.transpose(1, 2).contiguous().transpose(1, 2), q_rope, cache, scales, table, sl, scale, out),
                 (q_lat, q_rope, cache, scales[:1], table, sl, scale, out),
                 (q_lat, q_rope, cache, scales, table.cpu(), sl, scale, out),
                 (q_lat.float(), q_rope, cache, scales, table, sl, scale, out)):
        with pytest.raises(ValueError):
            gpu_ctx.mla_decode_fp8(*args)
    gpu_ctx.sync()


# --------------------------------------------------- moving references, streams


@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("pattern", ["rising", "falling", "alternating", "spike", "first", "late_sink"])
def test_decode_scores_move_between_tiles(gpu_ctx, pattern, H):
    """Per-tile score levels hundreds apart (logits up to 900): the reference of the probabilities moves up, moves
    down, and past the range in which maxima are compared in half precision.  q_rope is one-hot, so a level is a
    single exact product."""
    import torch

    n, R, P = 9 * 128 - 20, 512, 64
    q_lat, q_rope, cache, scales, table, scale = decode_inputs([n], H, BIG, seed=30)
    q_lat *= 0.25
    q_rope.zero_()
    q_rope[..., 0] = 1.0
    tile = torch.arange(n, device="cuda") // 128
    level = {"rising": 100.0 * tile, "falling": 800.0 - 100.0 * tile, "alternating": 900.0 * (tile % 2),
             "spike": 900.0 * (torch.arange(n, device="cuda") == 600), "first": 12.0 * (torch.arange(n, device="cuda") == 0),
             "late_sink": 11.0 * (torch.arange(n, device="cuda") == n - 1)}[pattern]
    kr = torch.zeros(cache.shape[0], 64, P, device="cuda")
    idx = table[0][(torch.arange(n, device="cuda") // 64)].long()
    kr[idx, torch.arange(n, device="cuda") % 64, 0] = level / scale
    cache[..., R:] = (kr / scales[..., None]).bfloat16().view(torch.uint8)
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, [n], scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, [n], scale)


def test_decode_rows_never_written(gpu_ctx):
    """A cache as it is created (zero codes, zero scales) behind two written rows: they count as zero rows."""
    import torch

    n = 200
    q_lat, q_rope, cache, scales, table, scale = decode_inputs([n], 16, BIG, seed=31)
    page = table[0].long()
    cache[page[0], 2:] = 0
    scales[page[0], 2:] = 0
    cache[page[1:]] = 0
    scales[page[1:]] = 0
    out = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, [n], scale)
    gpu_ctx.sync()
    check_decode(out, q_lat, q_rope, cache, scales, table, [n], scale)


def test_decode_two_contexts_at_once(gpu_ctx):
    """Two contexts on two streams, calls in flight together: each has its own scratch."""
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [Context(0) for _ in range(2)]
    cases = [decode_inputs([5000, 300], 64, BIG, seed=32), decode_inputs([40, 7000, 129], 16, BIG, seed=33)]
    lens = [[5000, 300], [40, 7000, 129]]
    dev = [torch.tensor(l, dtype=torch.int32, device="cuda") for l in lens]
    outs = [torch.empty_like(c[0]) for c in cases]
    torch.cuda.synchronize()
    for c, s in zip(ctxs, streams):
        c.set_stream(s.cuda_stream)
    for _ in range(20):
        for i in range(2):
            ctxs[i].mla_decode_fp8(*cases[i][:5], dev[i], cases[i][5], outs[i])
    for i in range(2):
        ctxs[i].sync()
        check_decode(outs[i], *cases[i][:5], lens[i], cases[i][5])
        ctxs[i].close()


def test_decode_growing_batches_on_one_context(gpu_ctx):
    """The same context with very different calls in a row: nothing of an earlier call is left in the scratch."""
    for lens, H in (([3000] * 3, 128), ([1] * 200, 16), ([0, 0, 5], 64), ([9000], 17), ([64] * 33, 128)):
        x = decode_inputs(lens, H, BIG, seed=34)
        out = run_decode(gpu_ctx, *x[:5], lens, x[5])
        gpu_ctx.sync()
        check_decode(out, *x[:5], lens, x[5])


def test_append_captured_and_replayed(gpu_ctx):
    import torch

    R, P, nope = shape = BIG
    H, rows = 16, 5
    stream, ctx = torch.cuda.Stream(), Context(0)
    ctx.set_stream(stream.cuda_stream)
    table, n_blocks = ref.make_table([300] * rows, seed=40)
    kv, w, q = append_case(rows, H, shape, seed=41)
    pos = torch.tensor([0, 10, 64, 299, 128], dtype=torch.int32, device="cuda")
    cache = torch.full((n_blocks, 64, R + 2 * P), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_blocks, 64), -7.0, device="cuda")
    q_rope = torch.full((rows, H, P), -7.0, dtype=torch.bfloat16, device="cuda")
    args = (kv, w, q, pos, table, H, nope, R, P, EPS, THETA, cache, scales, q_rope)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.kv_norm_rope_append_fp8(*args)
    for p in ([0, 10, 64, 299, 128], [1, -1, 65, 200, 7]):
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        cache.fill_(0xA5)
        scales.fill_(-7.0)
        q_rope.fill_(-7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_append(kv, w, q, pos, torch.arange(rows, device="cuda"), table, H, shape, cache, scales, q_rope)
    ctx.sync()
    del graph
    ctx.close()
