"""The decode step's kernels on a GPU, every variant, against the float64 references of
``specs_decode``: types, head counts, odd sizes, strides and alignments; empty, masked and
non-finite rows; indices outside their tables; repeated, captured and concurrent calls; and
a few decode steps run together.

Tolerances count roundings: an output is off by half a step of its type, plus an fp32 part
bounded from the float64 magnitudes of what was added up."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from kernelpilot_b200 import ext, registry
from kernelpilot_b200 import specs_decode as sd
from kernelpilot_b200.specs import randn

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
VARIANTS = [0, 1]
U24, U23 = 2.0 ** -24, 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(got, want, fp32_part, name=""):
    """|got - want| <= half a step of the output + the fp32 part, NaN where NaN."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g, w = got.double(), want
    assert torch.equal(torch.isnan(g), torch.isnan(w)), f"{name}: NaN in other places"
    lim = half_step(got.dtype) * (w.abs() + fp32_part) + fp32_part + tiny(got.dtype)
    bad = ((g - w).abs() > lim) & ~torch.isnan(w)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, first at "
                           f"{bad.nonzero()[0].tolist()}: {g[bad][0]} for {w[bad][0]}")


def device_errors():
    bits = ctypes.c_uint(0)
    ext.capi_check(ext.capi().kpb_device_errors(ctypes.byref(bits)))
    return bits.value


def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------- norm and rotation

ROPE_SHAPES = [(1, 1, 1, 2), (1, 32, 8, 128), (3, 5, 1, 7), (17, 4, 4, 64), (33, 6, 2, 80),
               (2, 64, 8, 128), (130, 3, 1, 256), (5, 2, 2, 33), (9, 7, 3, 96), (700, 32, 8, 128),
               (11, 0, 3, 64), (6, 3, 0, 64), (40, 1, 1, 1), (2100, 4, 2, 64),
               # enough rows for several heads a turn and many turns, heads no multiple of four
               (3001, 27, 3, 128), (1301, 30, 2, 80)]


def rope_limits(q, k, wq, wk):
    """fp32 part of a forward output: |y| <= |x| r |w|, two of them per output, and less than
    16 roundings each (square, sum, mean, rsqrt at 2 ulp, three products, the rotation)."""
    out = []
    for x, w in ((q, wq), (k, wk)):
        x = x.double()
        r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        depth = 16 + x.shape[-1] / 8  # a row's sum of squares, halved by the root
        top = (x * r * w.double()).abs().amax(-1, keepdim=True) if x.numel() else x
        out.append(2 * depth * U24 * top)
    return out


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROPE_SHAPES, ids=str)
def test_norm_rope(shape, dtype, variant):
    D = shape[-1]
    ins = sd._rope_inputs(shape, dtype, DEV, 0)
    for rot in {D - D % 2, (D // 2) & ~1}:
        table = sd.rope_table(4096, rot, DEV)
        for inter in (False, True):
            args = (*ins[:4], table, ins[5])
            got = ext.ops().qk_norm_rope(*args, 1e-6, inter, variant)
            want = sd.qk_norm_rope_reference(*args, 1e-6, inter)
            for g, w, lim in zip(got, want, rope_limits(*ins[:4]), strict=True):
                assert g.dtype == dtype and g.is_contiguous()
                check(g, w, lim, f"rot {rot} interleaved {inter}")


def backward_limits(gq, gk, q, k, wq, wk):
    out, dws = [], []
    for g, x, w in ((gq, q, wq), (gk, k, wk)):
        g, x, w = g.double(), x.double(), w.double()
        r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        xn = (x * r).abs()
        if not x.numel():
            out.append(x)
            dws.append(torch.zeros_like(w))
            continue
        # |dy| <= |a| + |b| of the pair <= 2 max |g|
        dy = 2 * g.abs().amax(-1, keepdim=True)
        dn = dy * w.abs().amax()
        depth = 24 + x.shape[-1] / 8
        out.append(depth * U24 * r * dn * (1 + xn.amax(-1, keepdim=True)
                                           * xn.mean(-1, keepdim=True)))
        # each term to `depth` roundings; added up lane by lane: rows / (8 warps x CTAs) in a
        # row and at most 8 * 148 partial sums after them, 64 at a time
        rows = x.shape[0] * x.shape[1]
        dws.append((depth + 200 + rows / 64) * U24 * (dy * xn).sum((0, 1)))
    return (*out, *dws)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROPE_SHAPES, ids=str)
def test_norm_rope_backward(shape, dtype, variant):
    D = shape[-1]
    ins = sd._rope_backward_inputs(shape, dtype, DEV, 0)
    lims = backward_limits(*ins[:6])
    for rot in {D - D % 2, (D // 2) & ~1}:
        table = sd.rope_table(4096, rot, DEV)
        for inter in (False, True):
            args = (*ins[:6], table, ins[7])
            got = ext.ops().qk_norm_rope_backward(*args, 1e-6, inter, variant)
            want = sd.qk_norm_rope_backward_reference(*args, 1e-6, inter)
            for g, w, lim, name in zip(got, want, lims, ("dq", "dk", "dwq", "dwk"), strict=True):
                assert g.dtype == dtype
                check(g, w, lim, f"{name} rot {rot} interleaved {inter}")


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_norm_rope_takes_slices_of_a_fused_projection(offset, variant):
    # q and k inside (T, (Hq + 2 Hkv) D + pad) rows; the pad and the offset put tokens and
    # heads off 16-byte boundaries
    T, Hq, Hkv, D = 21, 8, 2, 64
    for dtype in (torch.float32, torch.bfloat16):
        width = (Hq + 2 * Hkv) * D + offset
        flat = randn((T * width + offset,), dtype, DEV, generator(0), 2.0)[offset:]
        rows = flat.view(T, width)
        q, k = rows[:, :Hq * D].view(T, Hq, D), rows[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        _, _, wq, wk, table, pos = sd._rope_inputs((T, Hq, Hkv, D), dtype, DEV, 1)
        ins = (q, k, wq, wk, table, pos)
        got = ext.ops().qk_norm_rope(*ins, 1e-6, False, variant)
        for g, w, lim in zip(got, sd.qk_norm_rope_reference(*ins), rope_limits(q, k, wq, wk),
                             strict=True):
            check(g, w, lim)
        grads = (k.expand(T, Hkv, D)[:, :1].repeat(1, Hq, 1), k)  # one contiguous, one a slice
        got = ext.ops().qk_norm_rope_backward(*grads, *ins, 1e-6, False, variant)
        want = sd.qk_norm_rope_backward_reference(*grads, *ins)
        for g, w, lim in zip(got, want, backward_limits(*grads, q, k, wq, wk), strict=True):
            check(g, w, lim)


@pytest.mark.parametrize("variant", VARIANTS)
def test_norm_rope_weights_off_their_alignment(variant):
    T, Hq, Hkv, D = 5, 4, 2, 64
    q, k, wq, wk, table, pos = sd._rope_inputs((T, Hq, Hkv, D), torch.bfloat16, DEV, 0)
    wq = torch.cat([wq[:1], wq])[1:]
    flat = torch.cat([table.flatten()[:1], table.flatten()])[1:]
    table = flat.view(-1, D)
    got = ext.ops().qk_norm_rope(q, k, wq, wk, table, pos, 1e-6, False, variant)
    for g, w, lim in zip(got, sd.qk_norm_rope_reference(q, k, wq, wk, table, pos),
                         rope_limits(q, k, wq, wk), strict=True):
        check(g, w, lim)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("D", [64, 33])
def test_norm_rope_positions_outside_the_table(D, variant):
    T, Hq, Hkv = 6, 3, 2
    ins = list(sd._rope_backward_inputs((T, Hq, Hkv, D), torch.float32, DEV, 0))
    ins[6] = sd.rope_table(10, D - D % 2, DEV)
    ins[7] = torch.tensor([0, 9, 10, -1, 5, 2 ** 40], device=DEV)
    device_errors()
    q_out, k_out = ext.ops().qk_norm_rope(*ins[2:], 1e-6, False, variant)
    bad = torch.tensor([2, 3, 5], device=DEV)
    good = torch.tensor([0, 1, 4], device=DEV)
    assert device_errors() == 4
    want = sd.qk_norm_rope_reference(*(t[good] for t in ins[2:4]), *ins[4:7], ins[7][good])
    for out, w, lim in zip((q_out, k_out), want,
                           rope_limits(ins[2][good], ins[3][good], *ins[4:6]), strict=True):
        assert torch.isnan(out[bad]).all()
        check(out[good], w, lim)
    dq, dk, dwq, dwk = ext.ops().qk_norm_rope_backward(*ins, 1e-6, False, variant)
    assert device_errors() == 4
    for d in (dq, dk):
        assert torch.isnan(d[bad]).all() and not torch.isnan(d[good]).any()
    assert torch.isnan(dwq).all() and torch.isnan(dwk).all()


@pytest.mark.parametrize("variant", VARIANTS)
def test_norm_rope_of_special_rows(variant):
    # zeros (r = 1/sqrt(eps), all finite), huge values, an infinity and a NaN in one row each
    T, D = 5, 64
    q, k, wq, wk, table, pos = sd._rope_inputs((T, 2, 1, D), torch.float32, DEV, 0)
    q[0] = 0.0
    q[1] *= 1e17
    q[2, 0, 3] = float("inf")
    q[3, 1, 5] = float("nan")
    got = ext.ops().qk_norm_rope(q, k, wq, wk, table, pos, 1e-6, False, variant)[0]
    assert torch.equal(got[0], torch.zeros_like(got[0]))
    want = sd.qk_norm_rope_reference(q, k, wq, wk, table, pos)[0]
    check(got[[0, 1, 4]], want[[0, 1, 4]], rope_limits(q, k, wq, wk)[0][[0, 1, 4]])
    assert torch.isnan(got[2, 0]).any() and torch.isnan(got[3, 1]).all()
    check(got[2, 1], want[2, 1], rope_limits(q, k, wq, wk)[0][2, 1])


@pytest.mark.parametrize("variant", VARIANTS)
def test_norm_rope_gradient_against_differences(variant):
    ins = list(sd._rope_backward_inputs((3, 2, 1, 64), torch.float32, DEV, 4))
    got = ext.ops().qk_norm_rope_backward(*ins, 1e-6, False, variant)
    gq, gk = ins[0].double(), ins[1].double()

    def loss(q, k, wq, wk):
        a, b = sd.qk_norm_rope_reference(q, k, wq, wk, ins[6], ins[7])
        return float((a * gq).sum() + (b * gk).sum())

    h = 1e-5
    for n, at in ((0, (0, 1, 3)), (0, (2, 0, 63)), (1, (1, 0, 40)), (2, (9,)), (3, (50,))):
        lo, hi = ([t.double().clone() for t in ins[2:6]] for _ in range(2))
        lo[n][at] -= h
        hi[n][at] += h
        want = (loss(*hi) - loss(*lo)) / (2 * h)
        # differences are off by h^2 / 6 times a third derivative of some tens: 1e-8
        assert abs(float(got[n][at]) - want) <= 1e-7 + 64 * U24 * (abs(want) + 8.0)


# ---------------------------------------------------------------- the cache

CACHE_SHAPES = [(1, 1, 1, 1), (1, 8, 128, 16), (33, 2, 64, 7), (100, 4, 80, 16), (65, 3, 33, 5),
                (129, 1, 256, 64), (70, 2, 96, 1), (3000, 8, 128, 16), (40, 2, 48, 24)]


def same(a, b):
    """Equal bits, any NaN equal to any other."""
    a, b = (t.float() if t.dtype == sd.E4M3 else t for t in (a, b))
    return torch.equal(torch.nan_to_num(a.double(), nan=1e300),
                       torch.nan_to_num(b.double(), nan=1e300))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", CACHE_SHAPES, ids=str)
def test_cache_write_and_read(shape, dtype, e4m3, variant):
    k, v, slots, *caches = sd._write_inputs((*shape, e4m3), dtype, DEV, 0)
    if shape[0] > 2:
        slots[1] = -1
        slots[-1] = -7
    # rows of very different sizes, one of zeros, and one at the border of two scales
    k *= torch.exp2(torch.randint(-12, 8, k.shape[:2], generator=generator(1), device=DEV)
                    .to(dtype))[..., None]
    k[0, 0] = 0.0
    v[0] = 448.0 if dtype != torch.bfloat16 else 1.75
    want = sd.kv_cache_write_reference(k, v, slots, *caches)
    ext.ops().kv_cache_write(k, v, slots, *caches, variant)
    for c, w in zip(caches[:2 + 2 * e4m3], want, strict=True):
        assert same(c, w)  # every byte of the pool: rows behind the last one stay as they were
    for out in (dtype,) if not e4m3 else DTYPES:
        got = ext.ops().kv_cache_read(*caches[:2], slots, *caches[2:], out, variant)
        ref = sd.kv_cache_read_reference(*caches[:2], slots, *caches[2:])
        for g, w in zip(got, ref, strict=True):
            assert g.dtype == out and same(g, w.to(out))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_cache_calls_on_strided_tokens_and_pages(offset, e4m3, variant):
    # keys and values as slices of a fused projection, both caches in one allocation (pages
    # twice a page apart), each off 16-byte boundaries for odd offsets
    T, H, D, page, pages, dt = 40, 2, 64, 8, 9, torch.bfloat16
    flat = randn((T, 3 * H * D + offset), dt, DEV, generator(0))
    k, v = (flat[:, i * H * D + offset:(i + 1) * H * D + offset].view(T, H, D) for i in (1, 2))
    slots = torch.randperm(pages * page, generator=generator(1), device=DEV)[:T]
    ct = sd.E4M3 if e4m3 else dt
    pool = torch.zeros(pages * 2 * H * page * D + offset, dtype=torch.uint8 if e4m3 else dt,
                       device=DEV)[offset:].view(ct).view(pages, 2, H, page, D)
    kc, vc = pool[:, 0], pool[:, 1]
    scales = [torch.ones(pages, H, page, device=DEV) for _ in range(2)] if e4m3 else [None, None]
    want = sd.kv_cache_write_reference(k, v, slots, kc, vc, *scales)
    ext.ops().kv_cache_write(k, v, slots, kc, vc, *scales, variant)
    for c, w in zip((kc, vc, *scales)[:2 + 2 * e4m3], want, strict=True):
        assert same(c, w)
    got = ext.ops().kv_cache_read(kc, vc, slots, *scales, dt, variant)
    for g, w in zip(got, sd.kv_cache_read_reference(kc, vc, slots, *scales), strict=True):
        assert same(g, w.to(dt))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("D", [64, 33])
def test_e4m3_rows_that_are_not_finite_or_tiny(D, variant):
    k = randn((6, 1, D), torch.float32, DEV, generator(0))
    k[0, 0, 5] = float("inf")
    k[1, 0, 6] = float("-inf")
    k[2, 0, 7] = float("nan")
    k[3] *= 2.0 ** -140
    k[4] = 3e38
    caches = [torch.zeros(1, 1, 6, D, device=DEV).to(sd.E4M3) for _ in range(2)]
    scales = [torch.zeros(1, 1, 6, device=DEV) for _ in range(2)]
    slots = torch.arange(6, device=DEV)
    want = sd.kv_cache_write_reference(k, k, slots, *caches, *scales)
    ext.ops().kv_cache_write(k, k, slots, *caches, *scales, variant)
    for c, w in zip((*caches, *scales), want, strict=True):
        assert same(c, w)
    rows = ext.ops().kv_cache_read(*caches, slots, *scales, torch.float32, variant)[0]
    assert torch.isnan(rows[:3]).all() and torch.isfinite(rows[3:]).all()


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("D", [64, 33])
def test_slots_outside_the_cache(D, variant):
    k = randn((4, 2, D), torch.float32, DEV, generator(0))
    kc, vc = (torch.full((3, 2, 4, D), 7.0, device=DEV) for _ in range(2))
    slots = torch.tensor([11, 12, 2 ** 40, -1], device=DEV)
    device_errors()
    ext.ops().kv_cache_write(k, k + 1, slots, kc, vc, None, None, variant)
    assert device_errors() == 4
    for c, x in ((kc, k), (vc, k + 1)):
        assert torch.equal(c[2, :, 3], x[0])
        c[2, :, 3] = 7.0
        assert torch.all(c == 7.0)
    got = ext.ops().kv_cache_read(kc, vc, slots, None, None, torch.float32, variant)
    assert device_errors() == 4
    for g in got:
        assert torch.all(g[0] == 7.0) and torch.isnan(g[1:3]).all() and torch.all(g[3] == 0)


# ---------------------------------------------------------------- attention

def attention_limit(q, kc, vc, table, lens, ks, vs, scale=None):
    """fp32 part of the output, per head: a score is a sum of D products, each off by up to
    2^-23 of their magnitudes' sum per addition; a weight carries that twice (its own and the
    sum's), and 2^-15 where the weights enter the products as two 16-bit parts (bf16 cut
    towards zero leaves up to 2^-7 of the weight, and that is rounded to 2^-8 of itself); the
    sum over keys adds at most n / 4 + 32 roundings in a row."""
    B, Hq, D = q.shape
    Hkv, page = kc.shape[1:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, 1, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        pages = table[b].long()[j // page]
        k, v = (sd._values(c, s, pages, j % page, torch.float64).transpose(0, 1)
                for c, s in ((kc, ks), (vc, vs)))
        qq = q[b].double().view(Hkv, -1, D)
        a = (qq.abs() @ k.abs().transpose(1, 2)).amax(-1) * scale
        w = torch.softmax(qq @ k.transpose(1, 2) * scale, dim=-1)
        av = (w @ v.abs()).amax(-1)
        out[b, :, 0] = ((4 * (D + 16) * U23 * a + 2.0 ** -15 + (n / 4 + 32) * U23)
                        * av).reshape(Hq)
    return out


def run_paged(ins, variant, scale=None):
    return ext.ops().paged_attention(*ins, scale, variant)


def check_paged(ins, variant, scale=None):
    got = run_paged(ins, variant, scale)
    (want,) = sd.paged_attention_reference(*ins, scale)
    check(got, want, attention_limit(*ins, scale), f"variant {variant}")
    return got


# (B, Hq, Hkv, D, max_len, page): one head and many, group sizes 1..20, head dims odd and
# even, pages of one token, pages that end inside any tile, lengths from 1 on
PAGED_SHAPES = [(1, 1, 1, 16, 1, 1), (1, 8, 2, 64, 100, 16), (3, 32, 8, 128, 257, 16),
                (5, 6, 2, 80, 70, 7), (2, 3, 3, 33, 50, 24), (4, 16, 1, 256, 130, 64),
                (2, 20, 1, 128, 333, 100), (1, 32, 8, 128, 1037, 16), (7, 8, 8, 64, 900, 32),
                (2, 24, 2, 96, 515, 48), (1, 4, 4, 128, 5000, 16), (130, 4, 2, 64, 90, 16),
                (3, 9, 3, 8, 64, 3), (2, 40, 1, 64, 200, 128), (2, 4, 1, 256, 700, 16),
                (1, 1, 1, 1, 65, 2), (2, 34, 2, 128, 400, 16), (1, 10, 10, 112, 150, 16),
                (1, 8, 1, 128, 40000, 16)]


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", PAGED_SHAPES, ids=str)
def test_paged_attention(shape, dtype, e4m3, variant):
    check_paged(sd.paged_inputs((*shape, e4m3), dtype, DEV, 0), variant)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 0], [0, 5, 0, 200, 1, 0], [63, 64, 65, 128],
                                  [15, 16, 17, 31, 33], [3000] + [1] * 40, [1] * 40 + [3000],
                                  [0] * 300 + [33, 1] + [0] * 300 + [90] * 100,
                                  [5, 64, 0, 33] * 400],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_paged_attention_of_ragged_and_empty_sequences(lens, e4m3, variant):
    for dtype in (torch.float32, torch.bfloat16):
        ins = sd.paged_inputs((len(lens), 8, 2, 64, max(max(lens), 1), 16, e4m3), dtype, DEV, 1,
                              lens=lens)
        got = check_paged(ins, variant)
        for b, n in enumerate(lens):
            if n == 0:
                assert torch.all(got[b] == 0)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
def test_nothing_behind_a_sequence_is_read(e4m3, variant):
    # NaN in every row that no sequence holds, and table entries that point nowhere
    for dtype, D in ((torch.bfloat16, 128), (torch.float32, 40)):
        lens = [100, 0, 17, 48]
        ins = sd.paged_inputs((4, 4, 2, D, 100, 16, e4m3), dtype, DEV, 2, lens=lens)
        want = run_paged(ins, variant)
        q, kc, vc, table, _, ks, vs = ins
        held = torch.zeros(kc.shape[0], kc.shape[2], dtype=torch.bool, device=DEV)
        for b, n in enumerate(lens):
            j = torch.arange(n, device=DEV)
            held[table[b].long()[j // 16], j % 16] = True
        out = ~held[:, None].expand(-1, 2, -1)
        if e4m3:
            ks[out] = float("nan")
            vs[out] = float("nan")
            kc.view(torch.uint8)[out] = 0x7f
            vc.view(torch.uint8)[out] = 0xff
        else:
            kc[out] = float("nan")
            vc[out] = float("inf")
        table[table < 0] = 2 ** 31 - 1
        device_errors()
        assert torch.equal(run_paged(ins, variant), want)
        assert device_errors() == 0


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_that_are_not_finite_follow_the_softmax(dtype, variant):
    # sequence 0: a key whose score is -inf has no weight; 1: a NaN key; 2: a +inf score
    # (inf - inf); 3: all scores -inf (0 / 0); 4: an infinite value
    B, D, n = 5, 64, 40
    q, kc, vc, table, lens, *_ = sd.paged_inputs((B, 2, 1, D, n, 16, 0), dtype, DEV, 3,
                                                 lens=[n] * B)
    q[..., 0] = 1.0

    def row(cache, b, j):
        return cache[int(table[b, j // 16]), 0, j % 16]

    row(kc, 0, 20)[0] = float("-inf")
    row(kc, 1, 21)[3] = float("nan")
    row(kc, 2, 22)[0] = float("inf")
    for j in range(n):
        row(kc, 3, j)[0] = float("-inf")
    row(vc, 4, 7)[9] = float("inf")
    ins = (q, kc, vc, table, lens, None, None)
    got = run_paged(ins, variant)
    (want,) = sd.paged_attention_reference(*ins)
    assert torch.isnan(got[1:4]).all() and torch.isnan(want[1:4]).all()
    live = torch.arange(D, device=DEV) != 9
    assert torch.all(got[4, :, 9] == float("inf"))
    clean = (q, kc.nan_to_num(neginf=0.0), vc.nan_to_num(posinf=0.0), table, lens, None, None)
    lim = attention_limit(*clean)
    check(got[0], want[0], lim[0])
    check(got[4][:, live], want[4][:, live], lim[4])


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
def test_pages_and_lengths_outside_the_cache(e4m3, variant):
    for dtype, D in ((torch.bfloat16, 64), (torch.float32, 33)):
        lens = [50, 90, 33, 64]
        ins = list(sd.paged_inputs((4, 4, 2, D, 96, 16, e4m3), dtype, DEV, 4, lens=lens))
        ins[3][1, 2] = ins[1].shape[0]  # one past the last page, in the middle of sequence 1
        ins[3][3, 0] = -5
        device_errors()
        got = run_paged(ins, variant)
        assert device_errors() == 4
        assert torch.isnan(got[[1, 3]]).all()
        ok = [0, 2]
        sub = (ins[0][ok], ins[1], ins[2], ins[3][ok], ins[4][ok], ins[5], ins[6])
        (want,) = sd.paged_attention_reference(*sub)
        check(got[ok], want, attention_limit(*sub))
        # a length past the table is cut to it, a negative one is none
        ins = list(sd.paged_inputs((2, 4, 2, D, 96, 16, e4m3), dtype, DEV, 5, lens=[96, 96]))
        (want,) = sd.paged_attention_reference(*ins)
        ins[4] = torch.tensor([1000, -3], dtype=torch.int32, device=DEV)
        got = run_paged(ins, variant)
        assert device_errors() == 4
        full = (*ins[:4], torch.tensor([96, 96], dtype=torch.int32, device=DEV), *ins[5:])
        check(got[:1], want[:1], attention_limit(*full)[:1])
        assert torch.all(got[1] == 0)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_paged_attention_on_strides_and_alignments(offset, e4m3, variant):
    # q a slice of a wider projection, both caches in one pool, the table a window of a wider one
    B, Hq, H, D, page, dt = 3, 8, 2, 64, 16, torch.bfloat16
    q, kc, vc, table, lens, ks, vs = sd.paged_inputs((B, Hq, H, D, 100, page, e4m3), dt, DEV, 6)
    wide = randn((B, (Hq + 4) * D + offset), dt, DEV, generator(0))
    qs = wide[:, offset:offset + Hq * D].view(B, Hq, D)
    pages = kc.shape[0]
    bt = torch.uint8 if e4m3 else dt
    pool = torch.zeros(pages * 2 * H * page * D + offset, dtype=bt, device=DEV)[offset:]
    pool = pool.view(pages, 2, H, page, D)
    pool[:, 0], pool[:, 1] = kc.view(bt), vc.view(bt)
    pool = pool.view(kc.dtype)
    tables = torch.full((B, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    tables[:, 3:3 + table.shape[1]] = table
    ins = (qs, pool[:, 0], pool[:, 1], tables[:, 3:3 + table.shape[1]], lens, ks, vs)
    check_paged(ins, variant, scale=0.2)


@pytest.mark.parametrize("variant", VARIANTS)
def test_large_and_small_scores(variant):
    # scores of some hundreds: one key takes all the weight, whichever part of the cache holds it
    for dtype in (torch.float32, torch.bfloat16):
        ins = list(sd.paged_inputs((2, 8, 2, 128, 700, 16, 0), dtype, DEV, 7))
        for scale in (20.0, 1e-4, 0.0):
            check_paged(ins, variant, scale=scale)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_e4m3_scales_of_very_different_sizes(dtype, variant):
    # values from 2^-20 to 2^6 in one sequence; scales that are no powers of two too
    ins = list(sd.paged_inputs((2, 4, 1, 64, 300, 16, 1), dtype, DEV, 8))
    e = torch.randint(-20, 6, ins[6].shape, generator=generator(2), device=DEV)
    ins[6] = torch.exp2(e.float()) * (1 + torch.rand(ins[6].shape, generator=generator(3),
                                                     device=DEV))
    check_paged(ins, variant)
    ins[0] = ins[0] * 2.0 ** -10  # small queries keep their bits
    check_paged(ins, variant, scale=40.0)


@pytest.mark.parametrize("variant", VARIANTS)
def test_offsets_past_32_bits(variant):
    # one page of 2^31 + elements in: the table points at both ends of the pool
    H, page, D = 2, 64, 128
    pages = 2 ** 31 // (H * page * D) + 3
    dt = torch.bfloat16
    kc, vc = (torch.empty(pages, H, page, D, dtype=dt, device=DEV) for _ in range(2))
    ends = [0, pages - 1, pages - 2, 1]
    for i, p in enumerate(ends):
        kc[p], vc[p] = (randn((H, page, D), dt, DEV, generator(10 + 2 * i + j)) for j in (0, 1))
    table = torch.tensor([ends], dtype=torch.int32, device=DEV)
    lens = torch.tensor([250], dtype=torch.int32, device=DEV)
    q = randn((1, 8, D), dt, DEV, generator(9))
    check_paged((q, kc, vc, table, lens, None, None), variant)
    slots = torch.tensor([(pages - 1) * page + 5, 3, pages * page - 1], device=DEV)
    k = randn((3, H, D), dt, DEV, generator(30))
    ext.ops().kv_cache_write(k, k + 1, slots, kc, vc, None, None, variant)
    assert torch.equal(kc[pages - 1, :, 5], k[0]) and torch.equal(vc[0, :, 3], k[1] + 1)
    got = ext.ops().kv_cache_read(kc, vc, slots, None, None, dt, variant)
    assert torch.equal(got[0], k) and torch.equal(got[1], k + 1)


# ---------------------------------------------------------------- calls among others

def op_calls(variant, seed=0):
    """One call of each operator on fixed inputs; the write returns its caches."""
    ops = ext.ops()
    rope = sd._rope_inputs((70, 8, 2, 64), torch.bfloat16, DEV, seed)
    back = sd._rope_backward_inputs((700, 8, 2, 64), torch.bfloat16, DEV, seed)
    k, v, slots, *caches = sd._write_inputs((50, 2, 64, 16, 1), torch.bfloat16, DEV, seed)
    paged = sd.paged_inputs((9, 8, 2, 64, 2000, 16, 0), torch.bfloat16, DEV, seed)
    paged8 = sd.paged_inputs((9, 8, 2, 64, 700, 16, 1), torch.bfloat16, DEV, seed)

    def write():
        ops.kv_cache_write(k, v, slots, *caches, variant)
        return caches

    return {
        "qk_norm_rope": lambda: ops.qk_norm_rope(*rope, 1e-6, False, variant),
        "qk_norm_rope_backward": lambda: ops.qk_norm_rope_backward(*back, 1e-6, False, variant),
        "kv_cache_write": write,
        "kv_cache_read": lambda: ops.kv_cache_read(*caches[:2], slots, *caches[2:],
                                                   torch.bfloat16, variant),
        "paged_attention": lambda: (ops.paged_attention(*paged, None, variant),
                                    ops.paged_attention(*paged8, None, variant)),
    }


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("op", list(registry.DECODE_STAGES))
def test_calls_repeat_replay_and_run_beside_others(op, variant):
    call = op_calls(variant)[op]
    first = [t.clone() for t in call()]

    def equal(outs):
        return all(torch.equal(a.float(), b.float()) for a, b in zip(first, outs, strict=True))

    for _ in range(3):
        assert equal(call())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one call, each with its own workspace
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=side):
            outs.append(call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams, strict=True):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert equal(o)
    with torch.cuda.stream(streams[0]):  # a stream that is not the inputs' own
        streams[0].wait_stream(torch.cuda.default_stream())
        side = call()
    torch.cuda.synchronize()
    assert equal(side)


@pytest.mark.parametrize("variant", VARIANTS)
def test_a_captured_step_follows_new_lengths_pages_and_slots(variant):
    # one graph of write and attention; between replays the host changes what they read
    B, H, D, page, width = 6, 2, 64, 16, 40
    q, kc, vc, table, lens, *_ = sd.paged_inputs((B, 8, H, D, width * page, page, 0),
                                                 torch.bfloat16, DEV, 0, lens=[width * page] * B)
    k, v = (randn((B, H, D), torch.bfloat16, DEV, generator(i)) for i in (1, 2))
    slots = torch.full((B,), -1, device=DEV, dtype=torch.int64)
    ops = ext.ops()
    graph = torch.cuda.CUDAGraph()
    ops.paged_attention(q, kc, vc, table, lens, None, None, None, variant)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv_cache_write(k, v, slots, kc, vc, None, None, variant)
        out = ops.paged_attention(q, kc, vc, table, lens, None, None, None, variant)
    for step, new in enumerate([[1, 1, 1, 1, 1, 1], [640, 0, 3, 17, 0, 600], [0] * 6,
                                [64, 65, 63, 128, 1, 2]]):
        lens.copy_(torch.tensor(new))
        table.copy_(torch.stack([table[(b + 1) % B] for b in range(B)]))
        q.copy_(randn(q.shape, q.dtype, DEV, generator(50 + step)))
        at = (lens.long() - 1).clamp(min=0)
        slots.copy_(torch.where(lens > 0, table.long().gather(1, (at // page)[:, None])[:, 0]
                                * page + at % page, -1))
        graph.replay()
        ins = (q, kc, vc, table, lens, None, None)
        check(out, sd.paged_attention_reference(*ins)[0], attention_limit(*ins))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_and_a_few_decode_steps(dtype, e4m3, variant):
    """The operators as a model's attention block uses them: the prompt's q and k normed and
    rotated, its keys and values written, and per new token norm, write and attention; then
    the cached prefix read back for dense attention (kp.attention_causal) over it."""
    ops = ext.ops()
    B, Hq, H, D, page, n0, steps = 3, 4, 2, 64, 16, 37, 5
    width = -(-(n0 + steps) // page)
    pages = B * width
    table = torch.randperm(pages, generator=generator(0), device=DEV).to(torch.int32).view(B, width)
    ct = sd.E4M3 if e4m3 else dtype
    kc, vc = (torch.zeros(pages, H, page, D, device=DEV).to(ct) for _ in range(2))
    scales = [torch.ones(pages, H, page, device=DEV) for _ in range(2)] if e4m3 else [None, None]
    cos_sin = sd.rope_table(64, D, DEV)
    wq, wk = (randn((D,), dtype, DEV, generator(i)) for i in (1, 2))

    def block(tokens, positions, seed):
        """q, k, v of `tokens` new tokens per sequence, keys and values written."""
        T = B * tokens
        qkv = randn((T, (Hq + 2 * H) * D), dtype, DEV, generator(seed))
        q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, H * D, H * D], dim=1))
        pos = positions.expand(B, tokens).contiguous()
        slots = (table.long().gather(1, pos // page) * page + pos % page).flatten()
        qr, kr = ops.qk_norm_rope(q, k, wq, wk, cos_sin, pos.flatten(), 1e-6, False, variant)
        want = sd.qk_norm_rope_reference(q, k, wq, wk, cos_sin, pos.flatten())
        for g, w, lim in zip((qr, kr), want, rope_limits(q, k, wq, wk), strict=True):
            check(g, w, lim)
        ops.kv_cache_write(kr, v, slots, kc, vc, *scales, variant)
        return qr, kr, v, slots

    _, kr, v, slots = block(n0, torch.arange(n0, device=DEV), 10)
    keys, values = [kr.view(B, n0, H, D)], [v.reshape(B, n0, H, D)]
    for i in range(steps):
        qr, kr, v, _ = block(1, torch.full((1,), n0 + i, device=DEV), 20 + i)
        keys.append(kr.view(B, 1, H, D))
        values.append(v.reshape(B, 1, H, D))
        lens = torch.full((B,), n0 + i + 1, dtype=torch.int32, device=DEV)
        ins = (qr, kc, vc, table, lens, *scales)
        out = check_paged(ins, variant)
        if not e4m3:  # and against dense attention over the tokens themselves
            k_all, v_all = (torch.cat(t, 1).double().transpose(1, 2).repeat_interleave(
                Hq // H, dim=1) for t in (keys, values))
            s = (qr.double()[:, :, None] @ k_all.transpose(2, 3)) / math.sqrt(D)
            dense = (torch.softmax(s, -1) @ v_all)[:, :, 0]
            check(out, dense, attention_limit(*ins))
    # the prefix back: rows as written, ready for attention over the whole prompt
    k_back, v_back = ops.kv_cache_read(kc, vc, slots, *scales, dtype, variant)
    rows = []
    for back, sent in ((k_back, keys[0]), (v_back, values[0])):
        sent = sent.reshape(B * n0, H, D)
        if e4m3:
            codes, s = sd.e4m3_rows(sent)
            sent = (codes.float() * s.float()[..., None]).to(dtype)
        assert same(back, sent)
        rows.append(back.view(B, n0, H, D).transpose(1, 2).contiguous())
    q = randn((B, H, n0, D), dtype, DEV, generator(40))
    dense = ops.attention_causal(q, *rows, 1)
    last = ops.paged_attention(q[:, :, -1].contiguous(), kc, vc, table,
                               torch.full((B,), n0, dtype=torch.int32, device=DEV), *scales, None,
                               variant)
    tol = 1e-5 if dtype == torch.float32 else 2e-3  # attention_causal's own tolerance
    torch.testing.assert_close(dense[:, :, -1].float(), last.float(), atol=tol,
                               rtol=1e-4 if dtype == torch.float32 else 1e-2 + 2 ** -8)


# ---------------------------------------------------------------- refusals of the operators

def test_the_operators_refuse_what_they_do_not_take():
    ops = ext.ops()
    q, k, wq, wk, table, pos = sd._rope_inputs((4, 4, 2, 64), torch.bfloat16, DEV, 0)

    def refuse(match, fn, *args):
        with pytest.raises(RuntimeError, match=match):
            fn(*args)

    rope = ops.qk_norm_rope
    refuse("variant", rope, q, k, wq, wk, table, pos, 1e-6, False, 2)
    refuse("dtype", rope, q, k.float(), wq, wk, table, pos, 1e-6, False, 1)
    refuse("dtype", rope, q, k, wq.float(), wk, table, pos, 1e-6, False, 1)
    refuse("size", rope, q, k, wq[:5], wk, table, pos, 1e-6, False, 1)
    refuse("float32", rope, q, k, wq, wk, table.double(), pos, 1e-6, False, 1)
    refuse("Long", rope, q, k, wq, wk, table, pos.int(), 1e-6, False, 1)
    refuse("one per token", rope, q, k, wq, wk, table, pos[:3], 1e-6, False, 1)
    refuse("contiguously", rope, q.transpose(0, 1), k, wq, wk, table, pos, 1e-6, False, 1)
    refuse("match", rope, q, k[:3], wq, wk, table, pos, 1e-6, False, 1)
    refuse("rot must", rope, q, k, wq, wk, table[:, :63].contiguous(), pos, 1e-6, False, 1)
    refuse("GPU tensor", rope, q, k, wq, wk, table, pos.cpu(), 1e-6, False, 1)
    refuse("shapes", ops.qk_norm_rope_backward, q[:, :2], k, q, k, wq, wk, table, pos, 1e-6,
           False, 1)

    k, v, slots, kc, vc, ks, vs = sd._write_inputs((4, 2, 64, 16, 1), torch.bfloat16, DEV, 0)
    write, read = ops.kv_cache_write, ops.kv_cache_read
    refuse("go with", write, k, v, slots, kc, vc, None, None, 1)
    refuse("go with", write, k, v, slots, kc.to(k.dtype), vc.to(k.dtype), ks, vs, 1)
    refuse("heads", write, k[:, :1], v[:, :1], slots, kc, vc, ks, vs, 1)
    refuse("of one dtype", write, k, v, slots, kc, vc.to(k.dtype), ks, vs, 1)
    refuse("k's dtype", write, k, v, slots, kc.float(), vc.float(), None, None, 1)
    refuse("Long", write, k, v, slots.int(), kc, vc, ks, vs, 1)
    refuse("scales must", write, k, v, slots, kc, vc, ks[:1], vs, 1)
    refuse("differ", write, k, v, slots, kc, kc, ks, vs, 1)
    refuse("differ", write, k, v, slots, kc, vc, ks, ks, 1)
    refuse("must be contiguous", write, k, v, slots, kc.transpose(1, 2), vc.transpose(1, 2),
           ks, vs, 1)
    refuse("float32, float16 and bfloat16", read, kc, vc, slots, ks, vs, torch.float64, 1)
    refuse("own dtype", read, kc.to(k.dtype), vc.to(k.dtype), slots, None, None,
           torch.float32, 1)

    q, kc, vc, table, lens, ks, vs = sd.paged_inputs((2, 4, 2, 64, 40, 16, 0), torch.bfloat16,
                                                     DEV, 0)
    paged = ops.paged_attention
    refuse("multiple", paged, q[:, :3], kc, vc, table, lens, None, None, None, 1)
    refuse("head dim", paged, q[..., :32].contiguous(), kc, vc, table, lens, None, None, None, 1)
    refuse("q's dtype", paged, q.half(), kc, vc, table, lens, None, None, None, 1)
    refuse("Int", paged, q, kc, vc, table.long(), lens, None, None, None, 1)
    refuse("Int", paged, q, kc, vc, table, lens.long(), None, None, None, 1)
    refuse("sequences", paged, q, kc, vc, table[:1], lens, None, None, None, 1)
    refuse("one per sequence", paged, q, kc, vc, table, lens[:1], None, None, None, 1)
    refuse("variant", paged, q, kc, vc, table, lens, None, None, None, -1)
    refuse("page stride", paged, q, torch.cat([kc, kc], 1)[:, :2], vc, table, lens, None, None,
           None, 1)


@pytest.mark.parametrize("variant", VARIANTS)
def test_empty_inputs(variant):
    ops = ext.ops()
    q, k, wq, wk, table, pos = sd._rope_inputs((0, 4, 2, 64), torch.bfloat16, DEV, 0)
    a, b = ops.qk_norm_rope(q, k, wq, wk, table, pos, 1e-6, False, variant)
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(q, k, q, k, wq, wk, table, pos, 1e-6, False,
                                                 variant)
    assert dq.shape == q.shape and torch.all(dwq == 0) and torch.all(dwk == 0)
    k, v, slots, *caches = sd._write_inputs((3, 2, 64, 16, 0), torch.bfloat16, DEV, 0)
    before = caches[0].clone()
    ops.kv_cache_write(k[:0], v[:0], slots[:0], *caches, variant)
    assert torch.equal(caches[0], before)
    assert ops.kv_cache_read(*caches[:2], slots[:0], None, None, k.dtype, variant)[0].shape == \
        (0, 2, 64)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    q = randn((2, 4, 64), torch.bfloat16, DEV, generator(0))
    none = torch.empty(2, 0, dtype=torch.int32, device=DEV)  # no sequence has a page
    assert torch.all(ops.paged_attention(q, *caches[:2], none, lens, None, None, None,
                                         variant) == 0)
    assert ops.paged_attention(q[:0], *caches[:2], none[:0], lens[:0], None, None, None,
                               variant).shape == (0, 4, 64)
    # a cache without pages: every page of a sequence is outside it
    device_errors()
    pool = [c[:0] for c in caches[:2]]
    lens[1] = 3
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    got = ops.paged_attention(q, *pool, table, lens, None, None, None, variant)
    assert torch.all(got[0] == 0) and torch.isnan(got[1]).all() and device_errors() == 4
    rows = ops.kv_cache_read(*pool, slots[:2], None, None, k.dtype, variant)
    assert all(torch.isnan(r).all() for r in rows) and device_errors() == 4
    ops.kv_cache_write(k[:2], v[:2], slots[:2], *pool, None, None, variant)
    assert device_errors() == 4


def test_registry_runs_the_operators():
    for name, spec in sd.DECODE_SPECS.items():
        impls = registry.get_impls(name)
        assert set(impls) == {"torch", *(f"cuda:{s}" for s in registry.DECODE_STAGES[name])}
        for shape in spec.test_shapes:
            for dtype in DTYPES:
                tol = spec.tolerance(shape, dtype)
                for impl in (*impls, "best"):
                    fn = registry.best(name) if impl == "best" else impls[impl]
                    ins = spec.make_inputs(shape, dtype, DEV, 0)
                    want = spec.reference(*ins)
                    got = fn(*ins)
                    if name == "kv_cache_write":
                        got = [t for t in ins[3:] if t is not None] if got is None else got
                    elif name == "paged_attention" and impl != "torch":
                        got = (got,)
                    for g, w in zip(got, want, strict=True):
                        if name == "kv_cache_read":
                            w = w.to(g.dtype).double()
                        torch.testing.assert_close(g.float().double(), w, atol=tol.atol,
                                                   rtol=tol.rtol)


def test_no_call_of_this_file_left_an_error_behind():
    assert device_errors() == 0
