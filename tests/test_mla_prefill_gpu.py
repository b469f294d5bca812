"""Prompt attention in expanded form (dsb_mla_prefill) against a plain 64-bit
implementation, and the latent-attention operators as a model runs them:
append, read back, expand, attend over a prompt, then decode."""

import math

import numpy as np
import pytest

import mla_fp8_ref as ref
from deepseek_cpp_infer_b200 import DSB_EINVAL, DSB_EUNSUPPORTED, Context, DsbError

pytestmark = pytest.mark.gpu

BIG, SMALL = (128, 64, 128), (64, 32, 64)  # (nope, P, vd)


def cu_of(lens):
    import torch

    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def inputs(lq, lk, H, dims, seed, packed=True, std=1.0, extra=0):
    """Queries and keys of ragged sequences; packed: k_nope and v as halves of one projection."""
    import torch

    nope, P, vd = dims
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def r(*s):
        return (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()

    Tq, Tk = sum(lq) + extra, max(1, sum(lk) + extra)
    if packed:
        q, kv = r(Tq, H, nope + P), r(Tk, H, nope + vd)
        qn, kn, v = q[..., :nope], kv[..., :nope], kv[..., nope:]
    else:
        qn, kn, v = r(Tq, H, nope), r(Tk, H, nope), r(Tk, H, vd)
    return qn, r(Tq, H, P), kn, r(Tk, P), v, 1 / math.sqrt(nope + P)


def run(ctx, x, lq, lk, causal=True, max_q=None, lse=True, out=None):
    import torch

    qn, qr, kn, kr, v, scale = x
    if out is None:
        out = torch.full((qn.shape[0], qn.shape[1], v.shape[2]), 7.0, dtype=torch.bfloat16, device="cuda")
    l = torch.full(qn.shape[:2], 7.0, device="cuda") if lse else None
    ctx.mla_prefill(qn, qr, kn, kr, v, cu_of(lq), cu_of(lk), max(lq) if max_q is None else max_q, scale, out,
                    causal=causal, lse=l)
    return out, l


def check(out, lse, x, lq, lk, causal=True):
    """Bounds: the output's bf16 rounding, 2^-8 |out|; each probability rounded to bf16 before its product with v,
    2^-8 sum p |v|; the scores' fp32 sums of n products, at most n 2^-24 sum |q k| scale each, and the exponential
    (a few 2^-22): that much more of p (twice: numerator and denominator) and of lse."""
    n, T = x[0].shape[2] + x[1].shape[2], sum(lq)
    want, wl, mag, sab = ref.prefill64(*x[:5], np.concatenate([[0], np.cumsum(lq)]).tolist(),
                                       np.concatenate([[0], np.cumsum(lk)]).tolist(), x[5], causal)
    ds = n * 2.0 ** -24 * sab + 2.0 ** -20
    err = (out[:T].double() - want[:T]).abs()
    tol = 2.0 ** -8 * want[:T].abs() + (2.0 ** -8 + 2 * ds[:T, :, None]) * mag[:T] + 1e-30
    assert (err <= tol).all(), float((err / tol).max())
    assert (out[T:] == 7.0).all()  # rows behind the last sequence
    if lse is not None:
        a, b = lse[:T].double(), wl[:T]
        none = b == -math.inf
        assert (a[none] == -math.inf).all() and (out[:T][none] == 0).all()
        assert ((a - b).abs() <= ds[:T] + 2.0 ** -21 * b.abs())[~none].all(), float((a - b).abs()[~none].max())
        assert (lse[T:] == 7.0).all()


@pytest.mark.parametrize("dims", [BIG, SMALL])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 700])
def test_one_prompt(gpu_ctx, n, dims):
    x = inputs([n], [n], 3, dims, seed=n)
    out, lse = run(gpu_ctx, x, [n], [n])
    gpu_ctx.sync()
    check(out, lse, x, [n], [n])


@pytest.mark.parametrize("dims,H", [(BIG, 16), (BIG, 1), (SMALL, 8), (BIG, 5)])
@pytest.mark.parametrize("lq,lk", [([5, 1, 300, 129], [5, 1, 300, 129]), ([1, 1, 1], [1, 500, 64]),
                                   ([130, 7], [1000, 135]), ([0, 64, 0, 200], [0, 64, 3, 257])])
def test_ragged_and_behind_history(gpu_ctx, lq, lk, H, dims):
    x = inputs(lq, lk, H, dims, seed=H + len(lq), extra=3)
    out, lse = run(gpu_ctx, x, lq, lk)
    gpu_ctx.sync()
    check(out, lse, x, lq, lk)


def test_rows_that_see_nothing(gpu_ctx):
    """More queries than keys: the first rows of a sequence see none; a sequence without keys."""
    lq, lk = [200, 300, 4], [70, 0, 9]
    x = inputs(lq, lk, 2, BIG, seed=1)
    out, lse = run(gpu_ctx, x, lq, lk)
    gpu_ctx.sync()
    check(out, lse, x, lq, lk)
    out, lse = run(gpu_ctx, x, lq, lk, causal=False)
    gpu_ctx.sync()
    check(out, lse, x, lq, lk, causal=False)


@pytest.mark.parametrize("dims", [BIG, SMALL])
def test_full_attention(gpu_ctx, dims):
    lq, lk = [77, 300], [513, 31]
    x = inputs(lq, lk, 4, dims, seed=2, packed=False)
    out, lse = run(gpu_ctx, x, lq, lk, causal=False)
    gpu_ctx.sync()
    check(out, lse, x, lq, lk, causal=False)


@pytest.mark.parametrize("std", [0.0, 0.05, 6.0])
def test_flat_and_peaked(gpu_ctx, std):
    x = inputs([400], [400], 4, BIG, seed=3, std=std)
    out, lse = run(gpu_ctx, x, [400], [400])
    gpu_ctx.sync()
    check(out, lse, x, [400], [400])


def test_rising_scores(gpu_ctx):
    """Scores that grow along the keys: the running maximum moves in every tile."""
    import torch

    n = 1000
    x = list(inputs([n], [n], 2, BIG, seed=4))
    x[0].zero_()
    x[1].zero_()
    x[1][..., 0] = 8.0
    x[3].zero_()
    x[3][:, 0] = (torch.arange(n, device="cuda") / 4).bfloat16()
    out, lse = run(gpu_ctx, x, [n], [n])
    gpu_ctx.sync()
    check(out, lse, x, [n], [n])


@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_zero_and_negative_scale(gpu_ctx, scale):
    x = inputs([300], [300], 2, BIG, seed=5)[:5] + (scale,)
    out, lse = run(gpu_ctx, x, [300], [300])
    gpu_ctx.sync()
    check(out, lse, x, [300], [300])


def test_values_past_a_sequence_do_not_leak(gpu_ctx):
    """Keys and values of the neighbouring sequence, and rows past the last one, hold infinities and NaN."""
    import torch

    lq = lk = [100, 90]
    x = inputs(lq, lk, 3, BIG, seed=6, extra=50)
    clean, lc = run(gpu_ctx, x, lq, lk)
    for t, bad in ((x[2], float("inf")), (x[3], float("nan")), (x[4], float("nan"))):
        t[100:] = bad
    x[0][100:] = float("nan")
    out, lse = run(gpu_ctx, x, lq, lk)
    gpu_ctx.sync()
    assert torch.equal(out[:100], clean[:100]) and torch.equal(lse[:100], lc[:100])


def test_masked_future_infinities_do_not_leak(gpu_ctx):
    """Within one sequence, rows before a poisoned key stay finite and unchanged."""
    import torch

    n, at = 300, 150
    x = inputs([n], [n], 2, BIG, seed=7)
    clean, lc = run(gpu_ctx, x, [n], [n])
    x[2][at:] = float("inf")
    x[4][at:] = float("nan")
    out, lse = run(gpu_ctx, x, [n], [n])
    gpu_ctx.sync()
    assert torch.equal(out[:at], clean[:at]) and torch.equal(lse[:at], lc[:at])


@pytest.mark.parametrize("lq,lk,keys,causal", [
    (300, 300, [10, 50, 120], True),      # one bordering step
    (300, 300, [100, 128, 255], True),    # over the steps that one item's border crosses
    (200, 500, [310, 390, 480], True),    # behind a history
    (256, 511, [254, 400, 510], True),    # the widest border: keys 256 .. 510, and one that every row sees
    (130, 300, [0, 260, 299], True), (40, 333, [257, 300, 332], False)])
def test_non_finite_values_reach_the_rows_that_see_them_only(gpu_ctx, lq, lk, keys, causal):
    """Each column holds up to three of +inf, -inf and NaN at different keys, in every order.  A row's column is what
    the values that the row sees make of it: NaN from a NaN or from both infinities, the infinity from one, the
    clean result from none."""
    import itertools

    import torch

    inf, nan = float("inf"), float("nan")
    x = inputs([lq], [lk], 2, BIG, seed=lq + lk)
    clean, lc = run(gpu_ctx, x, [lq], [lk], causal=causal)
    order = list(itertools.permutations([inf, -inf, nan, None], 3))
    want, row = clean.clone(), torch.arange(lq, device="cuda")
    for col, kinds in enumerate(order):
        total = torch.zeros(lq, device="cuda")
        for key, value in zip(keys, kinds):
            if value is not None:
                x[4][key, :, col] = value
                total += torch.where((row + lk - lq >= key) | (not causal), value, 0.0)
        want[:lq, :, col] = torch.where((total == 0)[:, None], want[:lq, :, col], total[:, None].bfloat16())
    out, lse = run(gpu_ctx, x, [lq], [lk], causal=causal)
    gpu_ctx.sync()
    assert torch.equal(lse, lc)
    cut = len(order)
    assert torch.equal(out[:, :, cut:], clean[:, :, cut:])
    got, want = out[:lq, :, :cut].float(), want[:lq, :, :cut].float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[~want.isnan()].sign(), want[~want.isnan()].sign())
    # (a value that a row does not see has no weight there, whatever it was)
    assert torch.equal(got[want.isfinite()], want[want.isfinite()])


def test_long_prompt_and_repeats_are_bitwise(gpu_ctx):
    import torch

    x = inputs([2500], [4300], 4, BIG, seed=8)
    out, lse = run(gpu_ctx, x, [2500], [4300])
    gpu_ctx.sync()
    check(out, lse, x, [2500], [4300])
    again, l2 = run(gpu_ctx, x, [2500], [4300])
    assert torch.equal(out, again) and torch.equal(lse, l2)


def test_output_pitch_and_no_lse(gpu_ctx):
    import torch

    lq = [130, 40]
    x = inputs(lq, lq, 3, BIG, seed=9)
    wide = torch.full((170, 5 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, :384].unflatten(-1, (3, 128))
    run(gpu_ctx, x, lq, lq, lse=False, out=out)
    gpu_ctx.sync()
    check(out, None, x, lq, lq)
    assert (wide[:, 384:] == 7.0).all()


@pytest.mark.parametrize("T,H", [(1, 4), (1, 1), (70, 1)])
def test_one_row_or_head_of_any_stride(gpu_ctx, T, H):
    """Dimensions of one element whose strides (1) are no pitches."""
    import torch

    x = inputs([T], [T], H, BIG, seed=16)
    out, lse = run(gpu_ctx, x, [T], [T])
    odd = [torch.as_strided(t, t.shape, [1 if n == 1 else s for n, s in zip(t.shape, t.stride())], t.storage_offset())
           for t in x[:5]]
    out2, lse2 = run(gpu_ctx, (*odd, x[5]), [T], [T])
    gpu_ctx.sync()
    check(out2, lse2, x, [T], [T])
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_max_q_too_small_is_reported(gpu_ctx):
    lq = [100, 300]
    x = inputs(lq, lq, 2, BIG, seed=10)
    run(gpu_ctx, x, lq, lq, max_q=200)
    with pytest.raises(DsbError) as e:
        gpu_ctx.sync()
    assert e.value.code == DSB_EINVAL


def test_max_q_of_zero_is_reported(gpu_ctx):
    lq = [100, 3]
    x = inputs(lq, lq, 2, BIG, seed=13)
    run(gpu_ctx, x, lq, lq, max_q=0)
    with pytest.raises(DsbError) as e:
        gpu_ctx.sync()
    assert e.value.code == DSB_EINVAL
    run(gpu_ctx, x, [0, 0], lq, max_q=0)
    gpu_ctx.sync()


def test_no_keys_and_no_queries_at_all(gpu_ctx):
    """Tensors without memory: zero rows and lse = -inf, or nothing to do."""
    import torch

    x = inputs([5, 0], [0, 0], 2, BIG, seed=14)
    x = (*x[:2], x[2][:0], x[3][:0], x[4][:0], x[5])
    out, lse = run(gpu_ctx, x, [5, 0], [0, 0])
    gpu_ctx.sync()
    assert (out == 0).all() and torch.isneginf(lse).all() and out.shape[0] == 5
    x = inputs([0, 0], [5, 200], 2, BIG, seed=15)
    out, _ = run(gpu_ctx, x, [0, 0], [5, 200])
    gpu_ctx.sync()
    assert out.shape[0] == 0


def test_captured_and_replayed(gpu_ctx):
    import torch

    stream, ctx = torch.cuda.Stream(), Context(0)
    ctx.set_stream(stream.cuda_stream)
    lens = [200, 77]
    x = inputs(lens, lens, 4, BIG, seed=11)
    out, lse = torch.zeros(277, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(277, 4, device="cuda")
    cu = cu_of(lens)
    args = (*x[:5], cu, cu, 200, x[5], out)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ctx.mla_prefill(*args, lse=lse)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.mla_prefill(*args, lse=lse)
    for lens2 in (lens, [77, 200], [150, 0]):
        cu.copy_(cu_of(lens2))
        out.fill_(7.0)
        lse.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, lse, x, lens2, lens2)
    ctx.sync()
    del graph
    ctx.close()


def test_refusals(gpu_ctx):
    x = inputs([10], [10], 2, BIG, seed=12)
    qn, qr, kn, kr, v, scale = x

    def refused(code, *a):
        import torch

        out = torch.empty(10, 2, a[4].shape[2], dtype=torch.bfloat16, device="cuda")
        with pytest.raises(DsbError) as e:
            gpu_ctx.mla_prefill(*a, cu_of([10]), cu_of([10]), 10, scale if len(a) == 5 else a[5], out)
        assert e.value.code == code

    refused(DSB_EUNSUPPORTED, qn[..., :64], qr, kn[..., :64], kr, v)
    refused(DSB_EUNSUPPORTED, qn, qr, kn, kr, v[..., :64])
    import torch

    shifted = torch.empty(10 * 2 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(10, 2, 128)  # 2-byte aligned
    refused(DSB_EINVAL, shifted, qr, kn, kr, v)
    odd = torch.empty(10, 2, 132, dtype=torch.bfloat16, device="cuda")[..., :128]  # head pitch 132
    refused(DSB_EINVAL, qn, qr, odd, kr, v)
    with pytest.raises(DsbError) as e:
        gpu_ctx.mla_prefill(qn, qr, kn, kr, v, cu_of([10]), cu_of([10]), 10, float("nan"),
                            torch.empty(10, 2, 128, dtype=torch.bfloat16, device="cuda"))
    assert e.value.code == DSB_EINVAL
    with pytest.raises(ValueError):  # the binding: strided innermost dimension, wrong type
        gpu_ctx.mla_prefill(qn.transpose(1, 2).contiguous().transpose(1, 2), qr, kn, kr, v, cu_of([10]), cu_of([10]), 10,
                            scale, torch.empty(10, 2, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        gpu_ctx.mla_prefill(qn, qr, kn, kr, v.half(), cu_of([10]), cu_of([10]), 10, scale,
                            torch.empty(10, 2, 128, dtype=torch.bfloat16, device="cuda"))
    gpu_ctx.sync()


# ------------------------------------------- more items than SMs (each CTA takes several)


def crowd(name):
    """(lq, lk, H, dims): calls with several work items (256 query rows of a head) for every SM."""
    import torch

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rng = np.random.default_rng(len(name))
    if name == "ragged":  # about eight items a CTA, dead ones (short and empty prompts) between live ones
        lq = [0, 1, *rng.integers(100, 513, size=28).tolist(), 0, 257]
        return lq, lq, (4 * sms + len(lq) - 1) // len(lq), BIG
    if name == "groups":  # head groups of two items an SM, the last one short
        return [600], [600], 128, BIG
    if name == "sees_nothing":  # more queries than keys: tiles and whole items without keys beside ones with
        lq, lk = [600, 300, 256, 40, 700, 129], [100, 301, 90, 0, 40, 513]
        return lq, lk, (3 * sms + 17) // 18 + 1, BIG
    if name == "history":
        lq = rng.integers(1, 300, size=12).tolist()
        return lq, [n + int(p) for n, p in zip(lq, rng.integers(0, 900, size=12))], (3 * sms + 11) // 12, BIG
    lq = [0, 1, *rng.integers(100, 700, size=20).tolist(), 3]
    return lq, lq, (4 * sms + len(lq) - 1) // len(lq), SMALL


CROWDS = ["ragged", "groups", "sees_nothing", "history", "small"]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("name", CROWDS)
def test_several_items_per_cta(gpu_ctx, name, causal):
    import torch

    lq, lk, H, dims = crowd(name)
    x = inputs(lq, lk, H, dims, seed=100, extra=5)
    out, lse = run(gpu_ctx, x, lq, lk, causal=causal)
    gpu_ctx.sync()
    check(out, lse, x, lq, lk, causal=causal)
    again, l2 = run(gpu_ctx, x, lq, lk, causal=causal)
    assert torch.equal(out, again) and torch.equal(lse, l2)


@pytest.mark.parametrize("name", ["ragged", "history", "small"])
def test_several_items_per_cta_with_non_finite_values(gpu_ctx, name):
    """A NaN in some sequences' border and none in others, so that items with and without one follow each other on a
    CTA: only its column, and only in rows that see it."""
    import torch

    lq, lk, H, dims = crowd(name)
    x = inputs(lq, lk, H, dims, seed=101)
    clean, lc = run(gpu_ctx, x, lq, lk)
    want, q0, k0 = clean.clone(), 0, 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        key = m - 1 - (7 * b) % max(1, n)  # the last n keys are bordering ones
        if b % 3 != 0 and n > 0:
            for h in range(b % 2, H, 2):
                col = (5 * b + h) % x[4].shape[2]
                x[4][k0 + key, h, col] = float("nan")
                want[q0 + max(0, key - (m - n)):q0 + n, h, col] = float("nan")
        q0, k0 = q0 + n, k0 + m
    out, lse = run(gpu_ctx, x, lq, lk)
    gpu_ctx.sync()
    assert torch.equal(lse, lc) and torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[~want.isnan()], want[~want.isnan()])


# ------------------------------------------------------------- as a model runs them


@pytest.mark.parametrize("H,dims,R", [(16, BIG, 512), (8, SMALL, 128)])
def test_prompt_then_decode(gpu_ctx, H, dims, R):
    """Two prompts in two chunks, then three single tokens each, through the 8-bit cache.  Every chunk appends its
    rows, reads its sequences' whole history back, expands it to keys and values (kv_b projection) and attends;
    every single token appends and attends in absorbed form.  Each step is compared with the 64-bit attention over
    what the cache holds; the last prompt row's expanded output and an absorbed decode of the same row agree."""
    import torch

    nope, P, vd = dims
    g = torch.Generator(device="cuda")
    g.manual_seed(20)

    def r(*s, std=1.0):
        return torch.randn(*s, generator=g, device="cuda") * std

    w_uk, w_uv = r(H, nope, R, std=R ** -0.5).bfloat16(), r(H, vd, R, std=R ** -0.5).bfloat16()
    w_kv = torch.cat([w_uk, w_uv], 1).reshape(H * (nope + vd), R).contiguous()
    w_norm = 1 + 0.1 * r(R)
    scale = 1 / math.sqrt(nope + P)
    total, chunks, n_new = [150, 67], [[70, 60], [80, 7]], 3
    table, n_blocks = ref.make_table([t + n_new for t in total], seed=21)
    cache = torch.zeros(n_blocks, 64, R + 2 * P, dtype=torch.uint8, device="cuda")
    scales = torch.ones(n_blocks, 64, device="cuda")
    have = [0, 0]

    def append(lens):
        T = sum(lens)
        kv_a, q = r(T, R + P), r(T, H * (nope + P)).bfloat16()
        seq = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([have[b] + i for b, n in enumerate(lens) for i in range(n)], dtype=torch.int32, device="cuda")
        q_rope = torch.empty(T, H, P, dtype=torch.bfloat16, device="cuda")
        gpu_ctx.kv_norm_rope_append_fp8(kv_a, w_norm, q, pos, table, H, nope, R, P, 1e-6, 10000.0, cache, scales,
                                        q_rope, seq_ids=seq)
        for b, n in enumerate(lens):
            have[b] += n
        return q.view(T, H, nope + P)[..., :nope], q_rope

    def absorb(q_nope):
        return torch.einsum("thn,hnr->thr", q_nope.float(), w_uk.float()).bfloat16().contiguous()

    for lens in chunks:
        q_nope, q_rope = append(lens)
        T = sum(have)
        lat = torch.empty(T, R, dtype=torch.bfloat16, device="cuda")
        rope = torch.empty(T, P, dtype=torch.bfloat16, device="cuda")
        gpu_ctx.mla_cache_read_fp8(cache, scales, table, cu_of(have), lat, rope)
        kv = torch.empty(T, H * (nope + vd), dtype=torch.bfloat16, device="cuda")
        gpu_ctx.linear(w_kv, lat, kv, M=H * (nope + vd), K=R)
        kv = kv.view(T, H, nope + vd)
        x = (q_nope, q_rope, kv[..., :nope], rope, kv[..., nope:], scale)
        out, lse = run(gpu_ctx, x, lens, have)
        gpu_ctx.sync()
        check(out, lse, x, lens, have)
        want = torch.cat([ref.rows64(cache, scales, table, b, n, R)[0] for b, n in enumerate(have)])
        assert torch.equal(lat.double(), want)
    # the last prompt rows in absorbed form: keys and values are not rounded to bf16 there, the absorbed query is
    last = torch.tensor([lens[0] - 1, sum(lens) - 1], device="cuda")
    o = run_decode(gpu_ctx, absorb(q_nope[last]), q_rope[last].contiguous(), cache, scales, table, have, scale)
    o = torch.einsum("bhr,hvr->bhv", o.float(), w_uv.float())
    d = (o - out[last].float()).norm() / o.norm()
    assert d <= 2.0 ** -6, float(d)  # a few bf16 roundings of keys, values, queries and outputs
    for _ in range(n_new):
        q_nope, q_rope = append([1, 1])
        q_lat = absorb(q_nope)
        o = run_decode(gpu_ctx, q_lat, q_rope, cache, scales, table, have, scale)
        gpu_ctx.sync()
        want, mag, top = ref.decode64(q_lat, q_rope, cache, scales, table, have, scale)
        assert ((o.double() - want).abs() <= ref.decode_tol(want, mag, top)).all()


def run_decode(ctx, q_lat, q_rope, cache, scales, table, lens, scale):
    import torch

    out = torch.empty_like(q_lat)
    ctx.mla_decode_fp8(q_lat, q_rope, cache, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale,
                       out)
    return out
