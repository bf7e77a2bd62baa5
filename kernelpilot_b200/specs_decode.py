"""Contracts of the decode step's operators: what each computes (a float64 PyTorch
reference), how much work one call does and how close an answer must be, in the same
``KernelSpec`` form as ``specs.py``. They stand in a table of their own because they go
past what the reference's harness takes: several outputs, index inputs, caches updated in
place.

* ``qk_norm_rope``, ``qk_norm_rope_backward``: RMS norm of query and key heads, then the
  position rotation, and the gradient of both;
* ``kv_cache_write``, ``kv_cache_read``: rows into a paged key/value cache and out of it
  by slot, as they are or as e4m3 codes with a power-of-two scale per row;
* ``paged_attention``: one new token per sequence against its pages.

``reference`` returns a tuple of float64 tensors (for ``kv_cache_write`` the caches and
scales after the call); ``baseline`` is the same in fp32, rounded to the call's dtypes.
"""

from __future__ import annotations

import math

import torch

from .specs import ALL_DTYPES, KernelSpec, Tolerance, element_size, generator, randn

NORM_EPS = 1e-6
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


# ------------------------------------------------------------------ norm and rotation

def rope_table(max_pos: int, rot: int, device, base: float = 10000.0) -> torch.Tensor:
    """cos and sin of every position's angles, (max_pos, rot) fp32: rot/2 cosines, then
    rot/2 sines. The angles are formed in float64: a far position's angle has lost its
    fraction in fp32."""
    i = torch.arange(rot // 2, device=device, dtype=torch.float64)
    ang = torch.arange(max_pos, device=device, dtype=torch.float64)[:, None] \
        * base ** (-2.0 * i / max(rot, 1))
    return torch.cat([ang.cos(), ang.sin()], dim=1).float()


def _rotate(y, cos, sin, interleaved):
    half = cos.shape[-1]
    r, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, b * c + a * s
    r = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([r, rest], dim=-1)


def _angles(cos_sin, positions, acc):
    rows = cos_sin.to(acc)[positions]
    half = rows.shape[1] // 2
    return rows[:, :half], rows[:, half:]


def _norm_rope(q, k, wq, wk, cos_sin, positions, eps, interleaved, acc):
    cos, sin = _angles(cos_sin, positions, acc)
    out = []
    for x, w in ((q, wq), (k, wk)):
        x, w = x.to(acc), w.to(acc)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
        out.append(_rotate(y, cos, sin, interleaved))
    return tuple(out)


def qk_norm_rope_reference(q, k, q_weight, k_weight, cos_sin, positions, eps=NORM_EPS,
                           interleaved=False):
    return _norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved,
                      torch.float64)


def _norm_rope_backward(gq, gk, q, k, wq, wk, cos_sin, positions, eps, interleaved, acc):
    cos, sin = _angles(cos_sin, positions, acc)
    dx, dw = [], []
    for g, x, w in ((gq, q, wq), (gk, k, wk)):
        x, w = x.to(acc), w.to(acc)
        dy = _rotate(g.to(acc), cos, -sin, interleaved)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        xn, dn = x * r, dy * w
        dx.append(r * (dn - xn * (dn * xn).mean(-1, keepdim=True)))
        dw.append((dy * xn).sum((0, 1)))
    return (*dx, *dw)


def qk_norm_rope_backward_reference(grad_q, grad_k, q, k, q_weight, k_weight, cos_sin,
                                    positions, eps=NORM_EPS, interleaved=False):
    return _norm_rope_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos_sin, positions,
                               eps, interleaved, torch.float64)


def _rope_inputs(shape, dtype, device, seed):
    T, Hq, Hkv, D = shape
    g = generator(device, seed)
    q, k = randn((T, Hq, D), dtype, device, g, 2.0), randn((T, Hkv, D), dtype, device, g, 2.0)
    wq, wk = ((1.0 + 0.2 * torch.randn(D, generator=g, device=device)).to(dtype)
              for _ in range(2))
    rot = D - D % 2
    pos = torch.randint(0, 4096, (T,), generator=g, device=device)
    return q, k, wq, wk, rope_table(4096, rot, device), pos


def _rope_backward_inputs(shape, dtype, device, seed):
    T, Hq, Hkv, D = shape
    g = generator(device, seed + 1000)
    return (randn((T, Hq, D), dtype, device, g), randn((T, Hkv, D), dtype, device, g),
            *_rope_inputs(shape, dtype, device, seed))


def _rope_bytes(streams):
    def count(s, dt):
        T, Hq, Hkv, D = s
        return float(streams * T * (Hq + Hkv) * D * element_size(dt) + T * (4 * D + 8)
                     + 2 * D * element_size(dt))
    return count


_ROPE_SHAPES = [(1, 1, 1, 2), (1, 32, 8, 128), (3, 5, 1, 7), (17, 4, 4, 64), (33, 6, 2, 80),
                (64, 32, 8, 128), (130, 3, 1, 256), (5, 2, 2, 33)]


def _in_fp32(fn):
    def baseline(*inputs):
        dt = inputs[0].dtype
        return tuple(t.to(dt) for t in fn(*inputs, NORM_EPS, False, torch.float32))
    return baseline


# fp32: at most 16 roundings of 2^-24 over values below 16; 16-bit types: half a step
# (2^-9 for bf16) and the fp32 part
_ROPE_TOL = {torch.float32: Tolerance(2e-5, 1e-6), torch.float16: Tolerance(2e-5, 2.0 ** -11),
             torch.bfloat16: Tolerance(2e-5, 2.0 ** -8)}

QK_NORM_ROPE = KernelSpec(
    name="qk_norm_rope",
    description="RMS norm of every query and key head times a weight, then the rotation of "
                "the head's first elements in pairs by the token's position. Outputs have the "
                "input dtype; compute in float32.",
    signature="def kernel_fn(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,"
              " k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor)"
              " -> tuple  # (T, Hq, D), (T, Hkv, D)",
    make_inputs=_rope_inputs,
    reference=qk_norm_rope_reference,
    baseline=_in_fp32(_norm_rope),
    test_shapes=list(_ROPE_SHAPES),
    bench_shapes=[(64, 32, 8, 128), (16384, 32, 8, 128)],
    dtypes=list(ALL_DTYPES),
    flops=lambda s: 7.0 * s[0] * (s[1] + s[2]) * s[3],
    bytes_moved=_rope_bytes(2),
    tolerance=lambda s, dt: _ROPE_TOL[dt],
    shape_names=("T", "Hq", "Hkv", "D"),
)

QK_NORM_ROPE_BACKWARD = KernelSpec(
    name="qk_norm_rope_backward",
    description="Gradient of qk_norm_rope: of q, k and both weights, from the gradients of its "
                "outputs and its inputs. Weight gradients are summed in float32.",
    signature="def kernel_fn(grad_q: torch.Tensor, grad_k: torch.Tensor, q: torch.Tensor,"
              " k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,"
              " cos_sin: torch.Tensor, positions: torch.Tensor)"
              " -> tuple  # dq, dk, dq_weight, dk_weight",
    make_inputs=_rope_backward_inputs,
    reference=qk_norm_rope_backward_reference,
    baseline=_in_fp32(_norm_rope_backward),
    test_shapes=list(_ROPE_SHAPES),
    bench_shapes=[(16384, 32, 8, 128)],
    dtypes=list(ALL_DTYPES),
    flops=lambda s: 16.0 * s[0] * (s[1] + s[2]) * s[3],
    bytes_moved=_rope_bytes(3),
    # the weight gradients sum T * H terms of O(1)
    tolerance=lambda s, dt: Tolerance(2e-5 + 2e-6 * math.sqrt(s[0] * max(s[1], s[2])),
                                      max(1e-6, _ROPE_TOL[dt].rtol)),
    shape_names=("T", "Hq", "Hkv", "D"),
)


# ------------------------------------------------------------------ the paged cache

def e4m3_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of rows over the last dimension: the scale is the smallest power of
    two (2^-126 at least) that brings the largest magnitude to 448 at most, 1 for a row of
    zeros; a row with an infinity or NaN has the scale NaN and codes of zero."""
    x = x.double()
    top = x.abs().amax(-1)
    fine = torch.isfinite(top)
    m, e = torch.frexp(torch.where(fine, top, 0.0))  # top = m 2^e, m in [1/2, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)  # 448 = 7/8 * 2^9
    scale = torch.where(top == 0, 1.0, torch.ldexp(torch.ones_like(top), e))
    # x / scale is exact, also in fp32: rounding to e4m3 is the only one
    codes = torch.where(fine[..., None], x / scale[..., None], 0.0).float().to(E4M3)
    return codes, torch.where(fine, scale, float("nan"))


def _values(cache, scale, pages, offs, acc):
    """Rows of slots (pages, offs): (..., Hkv, D) in `acc`."""
    if scale is None:
        return cache[pages, :, offs].to(acc)
    rows = cache.view(torch.uint8)[pages, :, offs].view(E4M3)
    return rows.to(torch.float32).to(acc) * scale[pages, :, offs].to(acc)[..., None]


def _kv_cache_write(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    page = k_cache.shape[2]
    live = slots >= 0
    p, o = slots[live] // page, slots[live] % page
    out = []
    for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        cache = cache.clone()
        if scale is None:
            cache[p, :, o] = x[live]
            out.append((cache, None))
        else:
            codes, sc = e4m3_rows(x[live])
            cache.view(torch.uint8)[p, :, o] = codes.view(torch.uint8)
            scale = scale.clone()
            scale[p, :, o] = sc.float()
            out.append((cache, scale))
    (kc, ks), (vc, vs) = out
    return (kc, vc) if k_scale is None else (kc, vc, ks, vs)


def kv_cache_write_reference(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    return tuple(t.float().double() for t in _kv_cache_write(k, v, slots, k_cache, v_cache,
                                                             k_scale, v_scale))


def _kv_cache_read(k_cache, v_cache, slots, k_scale, v_scale, acc):
    page = k_cache.shape[2]
    at = slots.clamp(min=0)
    out = []
    for cache, scale in ((k_cache, k_scale), (v_cache, v_scale)):
        rows = _values(cache, scale, at // page, at % page, acc)
        out.append(torch.where((slots < 0)[:, None, None], 0.0, rows))
    return tuple(out)


def kv_cache_read_reference(k_cache, v_cache, slots, k_scale=None, v_scale=None):
    return _kv_cache_read(k_cache, v_cache, slots, k_scale, v_scale, torch.float64)


def _kv_cache_read_baseline(k_cache, v_cache, slots, k_scale=None, v_scale=None):
    dt = k_cache.dtype if k_scale is None else torch.bfloat16
    return tuple(t.to(dt) for t in _kv_cache_read(k_cache, v_cache, slots, k_scale, v_scale,
                                                  torch.float32))


def cache_inputs(pages, heads, page_size, dim, dtype, device, gen, e4m3):
    """(k_cache, v_cache, k_scale, v_scale) full of rows; the scales None unless `e4m3`."""
    rows = [randn((pages, heads, page_size, dim), dtype, device, gen) for _ in range(2)]
    if not e4m3:
        return (*rows, None, None)
    (kc, ks), (vc, vs) = (e4m3_rows(r) for r in rows)
    return kc, vc, ks.float(), vs.float()


def _some_slots(T, page, device, gen):
    pages = -(-T // page) + 2
    return pages, torch.randperm(pages * page, generator=gen, device=device)[:T]


def _write_inputs(shape, dtype, device, seed):
    T, Hkv, D, page, e4m3 = shape
    g = generator(device, seed)
    pages, slots = _some_slots(T, page, device, g)
    kc, vc, ks, vs = cache_inputs(pages, Hkv, page, D, dtype, device, g, e4m3)
    return (randn((T, Hkv, D), dtype, device, g), randn((T, Hkv, D), dtype, device, g), slots,
            kc, vc, ks, vs)


def _read_inputs(shape, dtype, device, seed):
    T, Hkv, D, page, e4m3 = shape
    g = generator(device, seed)
    pages, slots = _some_slots(T, page, device, g)
    kc, vc, ks, vs = cache_inputs(pages, Hkv, page, D, dtype, device, g, e4m3)
    return kc, vc, slots, ks, vs


def _cache_bytes(s, dt):
    T, Hkv, D, _page, e4m3 = s
    held = D + 4 if e4m3 else D * element_size(dt)
    return float(2 * T * Hkv * (D * element_size(dt) + held) + 8 * T)


_CACHE_SHAPES = [(1, 1, 1, 1, 0), (1, 8, 128, 16, 1), (33, 2, 64, 7, 0), (100, 4, 80, 16, 1),
                 (65, 3, 33, 5, 1), (129, 1, 256, 64, 0)]

KV_CACHE_WRITE = KernelSpec(
    name="kv_cache_write",
    description="Rows of keys and values into a paged cache by slot, as they are or as e4m3 "
                "codes with one power-of-two scale per row. Updates the caches in place.",
    signature="def kernel_fn(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,"
              " k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,"
              " v_scale: torch.Tensor) -> None",
    make_inputs=_write_inputs,
    reference=kv_cache_write_reference,
    baseline=_kv_cache_write,
    test_shapes=list(_CACHE_SHAPES),
    bench_shapes=[(64, 8, 128, 16, 1), (32768, 8, 128, 16, 1)],
    dtypes=list(ALL_DTYPES),
    flops=lambda s: 2.0 * s[0] * s[1] * s[2],
    bytes_moved=_cache_bytes,
    tolerance=lambda s, dt: Tolerance(0.0, 0.0),  # one defined rounding: equal bits
    shape_names=("T", "Hkv", "D", "page", "e4m3"),
)

KV_CACHE_READ = KernelSpec(
    name="kv_cache_read",
    description="Rows of keys and values out of a paged cache by slot, e4m3 rows as code times "
                "scale.",
    signature="def kernel_fn(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,"
              " k_scale: torch.Tensor, v_scale: torch.Tensor) -> tuple  # (T, Hkv, D) each",
    make_inputs=_read_inputs,
    reference=kv_cache_read_reference,
    baseline=_kv_cache_read_baseline,
    test_shapes=list(_CACHE_SHAPES),
    bench_shapes=[(5001, 8, 128, 16, 1), (65536, 8, 128, 16, 0)],
    dtypes=list(ALL_DTYPES),
    flops=lambda s: 2.0 * s[0] * s[1] * s[2],
    bytes_moved=_cache_bytes,
    # code * 2^e is exact in fp32, and rounded once to the output dtype
    tolerance=lambda s, dt: Tolerance(0.0, 0.0),
    shape_names=("T", "Hkv", "D", "page", "e4m3"),
)


# ------------------------------------------------------------------ attention

def _paged_attention(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, scale, acc):
    B, Hq, D = q.shape
    Hkv, page = k_cache.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=acc, device=q.device)
    for b, n in enumerate(seq_lens.tolist()):
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        pages = block_table[b].long()[j // page]
        k, v = (_values(c, s, pages, j % page, acc).transpose(0, 1)
                for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        s = q[b].to(acc).view(Hkv, -1, D) @ k.transpose(1, 2) * scale
        out[b] = (torch.softmax(s, dim=-1) @ v).reshape(Hq, D)
    return out


def paged_attention_reference(q, k_cache, v_cache, block_table, seq_lens, k_scale=None,
                              v_scale=None, scale=None):
    return (_paged_attention(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, scale,
                             torch.float64),)


def _paged_attention_baseline(q, *rest):
    return (_paged_attention(q, *rest, None, torch.float32).to(q.dtype),)


def paged_inputs(shape, dtype, device, seed, lens=None):
    """Inputs of ``paged_attention`` for (B, Hq, Hkv, D, max_len, page, e4m3): lengths
    spread over 0..max_len (or the given ones), pages in any order, table entries past a
    sequence's last page -1."""
    B, Hq, Hkv, D, max_len, page, e4m3 = shape
    g = generator(device, seed)
    if lens is None:
        lens = torch.randint(0, max_len + 1, (B,), generator=g, device=device)
        lens[0] = max_len
    lens = torch.as_tensor(lens, device=device).to(torch.int32)
    need = (lens.long() + page - 1) // page
    pages = int(need.sum()) + 2
    order = torch.randperm(pages, generator=g, device=device)
    col = torch.arange(max(1, -(-max_len // page)), device=device)
    at = ((need.cumsum(0) - need)[:, None] + col).clamp(max=pages - 1)
    table = torch.where(col < need[:, None], order[at], -1).to(torch.int32)
    kc, vc, ks, vs = cache_inputs(pages, Hkv, page, D, dtype, device, g, e4m3)
    return randn((B, Hq, D), dtype, device, g), kc, vc, table, lens, ks, vs


def _paged_bytes(s, dt):
    B, Hq, Hkv, D, n, page, e4m3 = s
    row = D + 4 if e4m3 else D * element_size(dt)
    return float(B * (2 * n * Hkv * row + 2 * Hq * D * element_size(dt) + 4 * -(-n // page) + 4))


PAGED_ATTENTION = KernelSpec(
    name="paged_attention",
    description="Attention of one new token per sequence over keys and values in a paged cache "
                "(plain, or e4m3 codes with a scale per row), each sequence of its own length. "
                "Output has q's dtype; empty sequences give zeros.",
    signature="def kernel_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,"
              " block_table: torch.Tensor, seq_lens: torch.Tensor, k_scale: torch.Tensor,"
              " v_scale: torch.Tensor) -> torch.Tensor  # (B, Hq, D)",
    make_inputs=paged_inputs,
    reference=paged_attention_reference,
    baseline=_paged_attention_baseline,
    test_shapes=[(1, 1, 1, 16, 1, 1, 0), (1, 8, 2, 64, 100, 16, 0), (3, 32, 8, 128, 257, 16, 1),
                 (5, 6, 2, 80, 70, 7, 0), (2, 3, 3, 33, 50, 24, 1), (4, 16, 1, 256, 130, 64, 0)],
    bench_shapes=[(1, 32, 8, 128, 1037, 16, 0), (64, 32, 8, 128, 4096, 16, 0),
                  (32, 64, 8, 128, 8192, 64, 1)],
    dtypes=list(ALL_DTYPES),
    flops=lambda s: 4.0 * s[0] * s[1] * s[3] * s[4],
    bytes_moved=_paged_bytes,
    # fp32: a score's error is some 2^-24 times the sum of |q k| (8 at these sizes), and a
    # weight's the same; 16-bit: half a step of the output on top of it
    tolerance=lambda s, dt: Tolerance(2e-5, 2e-6 if dt == torch.float32 else
                                      torch.finfo(dt).eps / 2),
    shape_names=("B", "Hq", "Hkv", "D", "len", "page", "e4m3"),
)


DECODE_SPECS: dict[str, KernelSpec] = {
    s.name: s for s in [QK_NORM_ROPE, QK_NORM_ROPE_BACKWARD, KV_CACHE_WRITE, KV_CACHE_READ,
                        PAGED_ATTENTION]
}
