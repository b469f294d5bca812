"""Host-side checks of the 8-bit latent cache and prompt-attention entry
points: no GPU is used."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

import deepseek_cpp_infer_b200 as dsb
import mla_fp8_ref as ref


def test_null_context_is_refused():
    l = dsb.lib()
    z = ctypes.c_void_p()
    assert l.dsb_mla_decode_fp8(z, z, z, z, z, 1, z, 1, z, 1, 16, 512, 64, 1.0, z) == dsb.DSB_EINVAL
    assert l.dsb_kv_norm_rope_append_fp8(z, z, 576, z, z, 16 * 192, z, z, z, 1, 1, 1, 16, 128, 512, 64, 1e-6, 1e4, z, z, 1,
                                         z) == dsb.DSB_EINVAL
    assert l.dsb_mla_cache_read_fp8(z, z, z, 1, z, 1, z, 1, 1, 512, 64, z, 512, z, 64) == dsb.DSB_EINVAL
    assert l.dsb_mla_prefill(z, ctypes.byref(dsb.MlaPrefillArgs())) == dsb.DSB_EINVAL


def test_prefill_args_match_the_header(tmp_path):
    names = [n for n, _ in dsb.MlaPrefillArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsb/dsb.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof(dsb_mla_prefill_args, {n}));\n' for n in names)
                   + '  printf("%zu\\n", sizeof(dsb_mla_prefill_args));\n  return 0;\n}\n')
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{inc}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [getattr(dsb.MlaPrefillArgs, n).offset for n in names] + [ctypes.sizeof(dsb.MlaPrefillArgs)]
    assert got == want


def _e4m3_table():
    """All 256 e4m3 values from the format's definition."""
    v = np.zeros(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (e, m) == (15, 7) else (-x if s else x)
    return v


def test_reference_quantiser():
    """Codes are the nearest e4m3 values of c / scale; the scale is the least power of two that keeps 448."""
    import torch

    rng = np.random.default_rng(0)
    c = rng.standard_normal((40, 128)) * np.exp(rng.uniform(-20, 20, (40, 1)))
    c[0] = 0
    c[1, 3], c[1, 4:] = 448 * 2.0 ** 5, 1.0  # amax on the border
    c[2, :] = np.minimum(c[2], 0.1)
    c[2, 0] = 448 * 2.0 ** 5 * (1 + 2.0 ** -20)  # and just above it
    codes, scale = ref.quantise(torch.from_numpy(c))
    scale = scale.double().numpy()
    assert scale[0] == 1 and scale[1] == 2.0 ** 5 and scale[2] == 2.0 ** 6
    amax = np.abs(c).max(1)
    assert (amax <= 448 * scale * (1 + 1e-7))[1:].all() and (amax > 224 * scale * (1 - 1e-7))[1:].all()
    table = _e4m3_table()
    finite = np.sort(np.unique(table[np.isfinite(table)]))
    x = c / scale[:, None]
    near = finite[np.abs(finite[None, None] - x[..., None]).argmin(-1)]
    got = table[codes.numpy()]
    assert (np.abs(got - x) <= np.abs(near - x) + 1e-6 * np.abs(x)).all()


def test_every_cached_value_is_exact_in_bf16():
    """An e4m3 value has 4 significant bits and the scale is a power of two."""
    import torch

    table = torch.from_numpy(_e4m3_table()).float()
    table = table[torch.isfinite(table)]
    for e in (-64, -17, -1, 0, 9, 64):
        v = table * 2.0 ** e
        assert torch.equal(v.bfloat16().float(), v)


class _Recorder:
    """Stands in for the library: every entry point notes its arguments and succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return dsb.DSB_OK

        return call


def binding():
    """A Context whose calls end before the library; its tensors lie on the host (device -1)."""
    ctx = object.__new__(dsb.Context)
    ctx._l, ctx.h, ctx.device = _Recorder(), None, -1
    return ctx


def append_args(H=2, B=3, R=128, P=32, nope=64):
    import torch

    return dict(kv_a=torch.zeros(B, R + P), w_norm=torch.ones(R), q=torch.zeros(B, H * (nope + P)).bfloat16(),
                positions=torch.zeros(B, dtype=torch.int32), block_table=torch.zeros(B, 1, dtype=torch.int32), H=H,
                nope=nope, R=R, P=P, eps=1e-6, theta=1e4, cache=torch.zeros(4, 64, R + 2 * P, dtype=torch.uint8),
                scales=torch.ones(4, 64), q_rope=torch.zeros(B, H, P).bfloat16())


@pytest.mark.parametrize("name,cut", [("kv_a", slice(64, None)), ("kv_a", slice(0, 156)), ("q", slice(96, None)),
                                      ("q", slice(0, 184))])
@pytest.mark.parametrize("B", [1, 3])
def test_append_refuses_rows_narrower_than_a_token(name, cut, B):
    """A view of part of each row has the whole row's pitch: only its width shows that the kernel would read the next
    row's values, and behind the last row what follows the allocation."""
    a = append_args(B=B)
    ctx = binding()
    ctx.kv_norm_rope_append_fp8(**a)
    assert len(ctx._l.calls) == 1
    with pytest.raises(ValueError, match=name):
        ctx.kv_norm_rope_append_fp8(**{**a, name: a[name][:, cut]})
    assert len(ctx._l.calls) == 1


def read_args(T, R=128, P=32):
    import torch

    return dict(cache=torch.zeros(4, 64, R + 2 * P, dtype=torch.uint8), scales=torch.ones(4, 64),
                block_table=torch.zeros(1, 1, dtype=torch.int32), cu_seqlens=torch.tensor([0, T], dtype=torch.int32),
                latent=torch.zeros(T, R).bfloat16(), k_rope=torch.zeros(T, P).bfloat16())


def test_read_of_one_part():
    """Either output may be left out, as at the C entry point; not both."""
    import torch

    ctx, a = binding(), read_args(5)
    ctx.mla_cache_read_fp8(**a)
    ctx.mla_cache_read_fp8(**{**a, "latent": None})
    ctx.mla_cache_read_fp8(**{**a, "k_rope": None})
    both, rope, lat = (c[1] for c in ctx._l.calls)
    assert both[8:11] == rope[8:11] == lat[8:11] == (5, 128, 32)  # T, R, P
    assert rope[11] is None and rope[13:] == both[13:]
    assert lat[13] is None and lat[11:13] == both[11:13]
    with pytest.raises(ValueError):
        ctx.mla_cache_read_fp8(**{**a, "latent": None, "k_rope": None})
    with pytest.raises(ValueError):  # 192 bytes a row: R + 2P
        ctx.mla_cache_read_fp8(**{**a, "k_rope": None, "latent": torch.zeros(5, 129).bfloat16()})


def odd_row(t, stride=1):
    """The same single row with a first stride that says nothing (as after a transposition)."""
    import torch

    assert t.shape[0] == 1
    return torch.as_strided(t, t.shape, (stride, *t.stride()[1:]))


@pytest.mark.parametrize("stride", [1, 3, 8])
def test_one_row_of_any_stride(stride):
    """The stride of a dimension of one element is arbitrary: the library gets the row's own width."""
    import torch

    ctx, a = binding(), append_args(B=1)
    ctx.kv_norm_rope_append_fp8(**a)
    ctx.kv_norm_rope_append_fp8(**{**a, "kv_a": odd_row(a["kv_a"], stride), "q": odd_row(a["q"], stride)})
    ctx.kv_norm_rope_append_fp8(**{**a, "kv_a": torch.zeros(1, 161)[:, :160], "q": torch.zeros(1, 193).bfloat16()})
    first, second, third = (c[1] for c in ctx._l.calls)
    assert first == second and first[2] == third[2] == 160 and first[5] == third[5] == 192
    ctx, a = binding(), read_args(1)
    ctx.mla_cache_read_fp8(**a)
    ctx.mla_cache_read_fp8(**{**a, "latent": odd_row(a["latent"], stride), "k_rope": odd_row(a["k_rope"], stride)})
    assert ctx._l.calls[0][1] == ctx._l.calls[1][1]


def test_one_prompt_row_or_head_of_any_stride():
    import torch

    def x(*shape):
        return torch.zeros(*shape).bfloat16()

    cu, seen = torch.tensor([0, 1], dtype=torch.int32), []
    for T, H in ((1, 4), (1, 1), (5, 1)):
        kv = x(T, H, 128)
        a = dict(q_nope=x(T, H, 64), q_rope=x(T, H, 32), k_nope=kv[..., :64], k_rope=x(T, 32), v=kv[..., 64:],
                 cu_q=cu, cu_k=cu, max_q=T, softmax_scale=0.1, out=x(T, H, 64))
        for odd in (False, True):
            b = dict(a)
            if odd:  # the dimensions of one element get a stride of 1
                for k, t in a.items():
                    if isinstance(t, torch.Tensor) and t.dtype == torch.bfloat16:
                        b[k] = torch.as_strided(t, t.shape, [1 if n == 1 else s for n, s in zip(t.shape, t.stride())],
                                                t.storage_offset())
            ctx = binding()
            ctx.mla_prefill(**b)
            p = ctx._l.calls[0][1][1]._obj
            for name, dim, heads in (("q_nope", 64, H), ("q_rope", 32, H), ("k_nope", 64, H), ("k_rope", 32, 1), ("v", 64, H)):
                ld, hd = getattr(p, "ld_" + name), getattr(p, "hd_" + name) if name != "k_rope" else dim
                assert ld % 8 == 0 and hd % 8 == 0 and hd >= dim and ld >= (heads - 1) * hd + dim, (T, H, odd, name)
                if heads > 1:
                    assert hd == a[name].stride(1)
                if T > 1:
                    assert ld == a[name].stride(0)
            assert p.ld_out == H * 64
