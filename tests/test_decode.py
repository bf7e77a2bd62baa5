"""The decode step's operators without a GPU: their float64 references against independent
forms (complex rotation, autograd and differences, the list of all e4m3 values, dense
attention), their tables, and the C ABI's refusals before any device call."""

import ctypes
import math

import pytest
import torch

from kernelpilot_b200 import ext, registry
from kernelpilot_b200 import specs_decode as sd

CPU = torch.device("cpu")


# ---------------------------------------------------------------- norm and rotation

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 2, 10, 16])
def test_norm_rope_reference_is_a_complex_rotation(rot, interleaved):
    q, k, wq, wk, _, pos = sd._rope_inputs((5, 3, 2, 16), torch.float32, CPU, 0)
    table = sd.rope_table(4096, rot, CPU)
    got = sd.qk_norm_rope_reference(q, k, wq, wk, table, pos, 1e-6, interleaved)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        x = x.double()
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        i = torch.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        turn = torch.complex(table[:, :rot // 2].double(), table[:, rot // 2:].double())[pos]
        z = torch.complex(n[..., a], n[..., b]) * turn[:, None]
        want = n.clone()
        want[..., a], want[..., b] = z.real, z.imag
        torch.testing.assert_close(y, want, rtol=1e-12, atol=1e-12)


def test_rope_table_keeps_far_angles():
    table = sd.rope_table(100_000, 8, CPU)
    for pos in (1, 99_999):
        for i in range(4):
            ang = pos * 10000.0 ** (-2.0 * i / 8)
            assert float(table[pos, i]) == pytest.approx(math.cos(ang), abs=1e-7)
            assert float(table[pos, 4 + i]) == pytest.approx(math.sin(ang), abs=1e-7)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_backward_reference_is_autograd_and_differences(interleaved):
    gq, gk, q, k, wq, wk, _, pos = sd._rope_backward_inputs((4, 3, 2, 12), torch.float32, CPU, 1)
    table = sd.rope_table(4096, 8, CPU)
    xs = [t.double().requires_grad_() for t in (q, k, wq, wk)]

    def loss(q, k, wq, wk):
        a, b = sd.qk_norm_rope_reference(q, k, wq, wk, table, pos, 1e-3, interleaved)
        return (a * gq).sum() + (b * gk).sum()

    want = torch.autograd.grad(loss(*xs), xs)
    got = sd.qk_norm_rope_backward_reference(gq, gk, q, k, wq, wk, table, pos, 1e-3, interleaved)
    for a, b in zip(got, want, strict=True):
        torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-12)
    h = 1e-5
    for n, at in ((0, (1, 2, 5)), (1, (3, 0, 11)), (2, (7,)), (3, (0,))):
        lo, hi = ([t.detach().clone() for t in xs] for _ in range(2))
        lo[n][at] -= h
        hi[n][at] += h
        assert float((loss(*hi) - loss(*lo)) / (2 * h)) == pytest.approx(float(got[n][at]),
                                                                        rel=1e-6, abs=1e-8)


# ---------------------------------------------------------------- e4m3 rows

def _all_e4m3():
    v = torch.arange(256, dtype=torch.uint8).view(sd.E4M3).float()
    return v[torch.isfinite(v)].double().unique()


@pytest.mark.parametrize("size", [1e-30, 2e-3, 1.0, 448.0, 448.5, 1e4, 3e38])
def test_e4m3_rows_take_the_smallest_power_of_two_and_the_nearest_code(size):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 33, generator=g)
    x = (x / x.abs().amax(-1, keepdim=True) * size).float()
    codes, scale = sd.e4m3_rows(x)
    m, _ = torch.frexp(scale)
    assert torch.all(m == 0.5)  # a power of two
    top = x.double().abs().amax(-1)
    assert torch.all(top <= 448 * scale) and torch.all(top > 224 * scale)
    err = (codes.float().double() * scale[:, None] - x.double()).abs()
    best = ((_all_e4m3()[None, None] * scale[:, None, None]) - x.double()[..., None]).abs().amin(-1)
    assert torch.equal(err, best)


def test_e4m3_rows_of_zeros_tiny_values_and_values_that_are_not_finite():
    x = torch.zeros(5, 4)
    x[1, 2] = 2.0 ** -140
    x[2, 0] = float("inf")
    x[3, 3] = float("nan")
    x[4] = 448.0
    codes, scale = sd.e4m3_rows(x)
    assert scale[0] == 1.0 and scale[1] == 2.0 ** -126 and scale[4] == 1.0
    assert torch.isnan(scale[2]) and torch.isnan(scale[3])
    codes = codes.float()
    assert torch.all(codes[[0, 2, 3]] == 0) and torch.all(codes[4] == 448)


# ---------------------------------------------------------------- cache and attention

@pytest.mark.parametrize("e4m3", [0, 1])
def test_cache_references_round_trip(e4m3):
    k, v, slots, *caches = sd._write_inputs((9, 2, 8, 4, e4m3), torch.bfloat16, CPU, 0)
    slots[3] = -1
    kc, vc, ks, vs = (*sd._kv_cache_write(k, v, slots, *caches), None, None)[:4]
    out_k, out_v = sd.kv_cache_read_reference(kc, vc, slots, ks, vs)
    for x, y in ((k, out_k), (v, out_v)):
        assert torch.all(y[3] == 0)
        live = slots >= 0
        if e4m3:  # three fraction bits: half a step is 2^-4 of the value, or of the smallest normal
            mag = x[live].double().abs()
            step = torch.maximum(mag, mag.amax(-1, True) / 2 ** 14)
            assert torch.all((y[live] - x[live].double()).abs() <= step * 2.0 ** -4)
        else:
            assert torch.equal(y[live], x[live].double())
    untouched = torch.ones(kc.shape[0] * kc.shape[2], dtype=torch.bool)
    untouched[slots[slots >= 0]] = False
    rest = untouched.nonzero()[:, 0]
    assert torch.equal(kc[rest // 4, :, rest % 4].float(),
                       caches[0][rest // 4, :, rest % 4].float())


@pytest.mark.parametrize("e4m3", [0, 1])
def test_paged_reference_is_dense_attention(e4m3):
    q, kc, vc, table, lens, ks, vs = sd.paged_inputs((3, 4, 2, 8, 21, 5, e4m3), torch.float32,
                                                     CPU, 0, lens=[21, 1, 0])
    (out,) = sd.paged_attention_reference(q, kc, vc, table, lens, ks, vs)
    assert torch.all(out[2] == 0)
    for b in (0, 1):
        n = int(lens[b])
        rows = []
        for c, s in ((kc, ks), (vc, vs)):
            x = c.float().double() if s is None else c.float().double() * s.double()[..., None]
            flat = torch.stack([x[int(table[b, j // 5]), :, j % 5] for j in range(n)], dim=1)
            rows.append(flat.repeat_interleave(2, dim=0))
        want = torch.nn.functional.scaled_dot_product_attention(
            q[b].double()[:, None], rows[0], rows[1])[:, 0]
        torch.testing.assert_close(out[b], want, rtol=1e-12, atol=1e-12)


def test_reference_and_baseline_agree_on_every_spec():
    for spec in sd.DECODE_SPECS.values():
        for shape in spec.test_shapes[:3]:
            assert len(shape) == len(spec.shape_names)
            ins = spec.make_inputs(shape, torch.float32, CPU, 2)
            tol = spec.tolerance(shape, torch.float32)
            for a, b in zip(spec.baseline(*ins), spec.reference(*ins), strict=True):
                lim = tol if spec.name != "kv_cache_read" or not shape[-1] else \
                    sd.Tolerance(0.0, 2.0 ** -8)  # its baseline reads e4m3 rows as bf16
                torch.testing.assert_close(a.float().double(), b, rtol=lim.rtol, atol=lim.atol)
        for shape in spec.bench_shapes:
            for dt in spec.dtypes:
                assert spec.flops(shape) > 0 and spec.bytes_moved(shape, dt) > 0


# ---------------------------------------------------------------- tables and refusals

def test_every_decode_operator_has_stages_a_spec_and_variants():
    lib = ext.capi()
    assert set(registry.DECODE_STAGES) == set(sd.DECODE_SPECS)
    for op, stages in registry.DECODE_STAGES.items():
        assert lib.kpb_num_variants(op.encode()) == len(stages)
        assert op not in registry.CUDA_STAGES


P = ctypes.c_void_p(4096)  # an aligned address that no refused call follows
ODD = ctypes.c_void_p(4097)


def _rope(L, variant=1, dtype=2, T=4, Hq=2, Hkv=1, D=64, rot=64, q=P, pos=P):
    return L.kpb_qk_norm_rope(variant, dtype, q, P, P, P, P, pos, P, P, T, Hq, Hkv, D, rot, 100,
                              Hq * 64, Hkv * 64, 1e-6, 0, None)


def _rope_back(L, variant=1, dtype=2, T=4, D=64, rot=64, ws=P, ws_bytes=1 << 30, gq=P, dwq=P):
    return L.kpb_qk_norm_rope_backward(variant, dtype, gq, P, P, P, P, P, P, P, P, P, dwq, P, T, 2,
                                       1, D, rot, 100, 128, 64, 128, 64, 1e-6, 0, ws, ws_bytes,
                                       None)


def _write(L, variant=1, dtype=2, cache=2, T=4, H=2, D=64, pages=3, page=16, stride=None,
           kc=P, vc=ctypes.c_void_p(8192), ks=P, vs=ctypes.c_void_p(8192), k=P):
    stride = H * page * D if stride is None else stride
    return L.kpb_kv_cache_write(variant, dtype, cache, k, P, P, kc, vc, ks, vs, T, H, D, pages,
                                page, H * D, H * D, stride, None)


def _read(L, variant=1, dtype=2, cache=2, T=4, H=2, D=64, pages=3, page=16, stride=None, kc=P,
          ks=P, slots=P):
    stride = H * page * D if stride is None else stride
    return L.kpb_kv_cache_read(variant, dtype, cache, kc, P, slots, ks, P, P, P, T, H, D, pages,
                               page, stride, None)


def _paged(L, variant=1, dtype=2, cache=2, B=2, Hq=4, H=2, D=64, pages=3, page=16, width=4,
           table=P, lens=P, q=P, ks=P, ws=P, ws_bytes=1 << 30, stride=None):
    stride = H * page * D if stride is None else stride
    return L.kpb_paged_attention(variant, dtype, cache, q, P, P, table, lens, ks, P, P, B, Hq, H,
                                 D, pages, page, width, Hq * D, stride, width, 0.1, ws, ws_bytes,
                                 None)


@pytest.mark.parametrize("call,needle", [
    (lambda L: _rope(L, variant=2), "variant"),
    (lambda L: _rope(L, dtype=3), "dtype"),
    (lambda L: _rope(L, D=0, rot=0), "D must be"),
    (lambda L: _rope(L, D=257), "D must be"),
    (lambda L: _rope(L, rot=63), "rot must be"),
    (lambda L: _rope(L, rot=66), "rot must be"),
    (lambda L: _rope(L, T=-1), "T, heads"),
    (lambda L: _rope(L, T=1 << 30, Hq=2), "T, heads"),
    (lambda L: _rope(L, q=None), "null"),
    (lambda L: _rope(L, pos=None), "null"),
    (lambda L: _rope(L, q=ODD), "aligned"),
    (lambda L: _rope(L, pos=ctypes.c_void_p(4100)), "aligned"),
    (lambda L: _rope_back(L, variant=-1), "variant"),
    (lambda L: _rope_back(L, rot=3), "rot must be"),
    (lambda L: _rope_back(L, gq=None), "null"),
    (lambda L: _rope_back(L, dwq=None, T=0), "null"),
    (lambda L: _rope_back(L, gq=ODD), "aligned"),
    (lambda L: _rope_back(L, ws=None), "workspace"),
    (lambda L: _rope_back(L, ws_bytes=8), "workspace"),
    (lambda L: _rope_back(L, ws=ctypes.c_void_p(4104)), "16-byte"),
    (lambda L: _write(L, variant=2), "variant"),
    (lambda L: _write(L, dtype=3, cache=3), "dtype"),
    (lambda L: _write(L, cache=1), "cache dtype"),
    (lambda L: _write(L, cache=4), "cache dtype"),
    (lambda L: _write(L, page=0), "page_size"),
    (lambda L: _write(L, pages=-1), "num_pages"),
    (lambda L: _write(L, D=300), "D must be"),
    (lambda L: _write(L, stride=16 * 64), "page_stride"),
    (lambda L: _write(L, T=1 << 31), "T and T * Hkv"),
    (lambda L: _write(L, kc=None), "null"),
    (lambda L: _write(L, k=None), "null"),
    (lambda L: _write(L, cache=3, ks=None), "k_scale"),
    (lambda L: _write(L, cache=3, vs=ODD), "aligned"),
    (lambda L: _write(L, kc=ODD), "aligned"),
    (lambda L: _write(L, vc=P), "differ"),
    (lambda L: _write(L, cache=3, vs=P), "differ"),
    (lambda L: _read(L, variant=2), "variant"),
    (lambda L: _read(L, cache=0), "cache dtype"),
    (lambda L: _read(L, slots=None), "null"),
    (lambda L: _read(L, slots=ctypes.c_void_p(4100)), "aligned"),
    (lambda L: _read(L, cache=3, ks=None), "k_scale"),
    (lambda L: _read(L, page=1 << 31), "page_size"),
    (lambda L: _read(L, H=1 << 20, page=1 << 12), "Hkv * page_size"),
    (lambda L: _paged(L, variant=2), "variant"),
    (lambda L: _paged(L, dtype=0, cache=2), "cache dtype"),
    (lambda L: _paged(L, Hq=3), "multiple"),
    (lambda L: _paged(L, H=0), "multiple"),
    (lambda L: _paged(L, D=512), "D must be"),
    (lambda L: _paged(L, B=-1), "B, heads"),
    (lambda L: _paged(L, width=1 << 28), "max_pages"),
    (lambda L: _paged(L, table=None), "null"),
    (lambda L: _paged(L, lens=None), "null"),
    (lambda L: _paged(L, lens=ODD), "aligned"),
    (lambda L: _paged(L, q=ODD), "aligned"),
    (lambda L: _paged(L, cache=3, ks=None), "k_scale"),
    (lambda L: _paged(L, stride=1), "page_stride"),
])
def test_bad_arguments_are_refused_without_a_device(call, needle):
    lib = ext.capi()
    assert call(lib) == 1  # KPB_EINVAL
    assert needle in lib.kpb_last_error().decode()


def test_empty_calls_succeed_without_a_device():
    lib = ext.capi()
    assert _rope(lib, T=0, pos=None, q=None) == 0
    assert _write(lib, T=0, k=None) == 0
    assert _read(lib, T=0, slots=None) == 0
    assert _paged(lib, B=0, q=None, lens=None, table=None) == 0


def test_workspace_queries_of_the_decode_operators():
    lib = ext.capi()
    assert lib.kpb_qk_norm_rope_backward_workspace_bytes(1, 1, 1, 64) >= 2 * 64 * 4
    assert lib.kpb_qk_norm_rope_backward_workspace_bytes(1, 1, 1, 1000) == 0
    assert lib.kpb_paged_attention_workspace_bytes(0, 4, 8, 2, 64, 1000) == 0
    assert lib.kpb_paged_attention_workspace_bytes(5, 4, 8, 2, 64, 1000) == 0
    assert lib.kpb_paged_attention_workspace_bytes(1, 0, 8, 2, 64, 1000) == 0
