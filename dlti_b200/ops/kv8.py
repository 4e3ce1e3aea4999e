"""A paged cache of keys and values in 8 bits (csrc/kv8.cu): rows of a step written, attention of single tokens, cached rows laid out in 16 bits.
PyTorch restatements for CPU tensors.

Pages are e4m3 tensors [num_blocks, KV, block_size, hd], with fp32 scales [num_blocks, KV], one for each page and head. A scale is a power of two,
the smallest for which the page's largest finite number is at most 448 scales (2^-120 for a page of zeros). Slots are numbered as those of the
16-bit cache: page * block_size + place in the page, -1 for none.
  * A row at place 0 begins its page: what the page held has no meaning from then on (its bytes stay until they are written).
  * Any other row may raise the scale of its page; all that the page holds is then rounded to the new one. Scales never fall.
  * Infinities are stored as the largest number of their page, 448 scales, and do not raise it; NaN stays NaN.
Rows of one page are neighbours in a call, each slot occurs once (ops/_debug.py checks both). On a GPU rows, pages, rotation tables and accumulators
begin at multiples of 16 bytes."""
from __future__ import annotations

import math

import torch

from . import _debug, _lib
from .elementwise import rope_ref
from .serving import _F, _I, _L, _V

E_LOW, E_HIGH = -120, 120
E4M3 = torch.float8_e4m3fn
TOP = 448.0                      # largest finite e4m3 number


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _cache_fits(k8, v8, k_scale, v_scale, H: int, KV: int, hd: int) -> bool:
    s = k8.shape
    return (len(s) == 4 and s == v8.shape and s[1] == KV and s[3] == hd and s[2] >= 8 and s[2] % 8 == 0 and KV > 0 and H > 0 and H % KV == 0
            and k8.dtype is E4M3 and v8.dtype is E4M3 and k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32
            and k_scale.shape == v_scale.shape == s[:2] and k8.is_contiguous() and v8.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous() and s[0] * s[2] < 1 << 31)


def _check_cache(op: str, k8, v8, k_scale, v_scale, H: int, KV: int, hd: int) -> None:
    if _cache_fits(k8, v8, k_scale, v_scale, H, KV, hd):
        return
    _need(k8.dim() == 4 and k8.shape == v8.shape and k8.shape[1] == KV and k8.shape[3] == hd,
          f"{op}: pages are [num_blocks, {KV}, block_size, {hd}], got {tuple(k8.shape)} and {tuple(v8.shape)}")
    _need(KV > 0 and H > 0 and H % KV == 0, f"{op}: query heads are a multiple of key/value heads, got {H} and {KV}")
    _need(k8.dtype == v8.dtype == E4M3 and k_scale.dtype == v_scale.dtype == torch.float32, f"{op}: pages are float8_e4m3fn with float32 scales")
    _need(k_scale.shape == v_scale.shape == k8.shape[:2], f"{op}: one scale for each page and head")
    _need(k8.shape[2] >= 8 and k8.shape[2] % 8 == 0, f"{op}: block_size is a multiple of 8, got {k8.shape[2]}")
    _need(k8.shape[0] * k8.shape[2] < 1 << 31, f"{op}: slots have 31 bits")
    raise ValueError(f"{op}: pages and scales are contiguous")


def _check_device(op: str, *tensors) -> int:
    """The current device, which every tensor is on."""
    d = torch.cuda.current_device()
    for t in tensors:
        if t.get_device() != d:
            raise ValueError(f"{op}: every tensor is on the current device, cuda:{d}")
    return d


def _check_rows(op: str, x, width: int, written: bool = True) -> None:
    s = x.stride()
    if len(s) != 2 or x.shape[1] != width or s[1] != 1:
        raise ValueError(f"{op}: rows [tokens, {width}] with consecutive columns")
    if s[0] % 8 or x.data_ptr() % 16:
        raise ValueError(f"{op}: rows begin at multiples of 16 bytes")
    if written and s[0] < width and x.shape[0] > 1:
        raise ValueError(f"{op}: rows that are written do not overlap")


def _pages(op: str, k8, v8, unit: int = 16) -> tuple[int, int]:
    """Addresses of the pages, which the kernels read and write in pieces of `unit` bytes."""
    k, v = k8.data_ptr(), v8.data_ptr()
    if (k | v) % unit:
        raise ValueError(f"{op}: pages begin at multiples of {unit} bytes")
    return k, v


def _check_places(op: str, pos, slots, T: int) -> None:
    if not (pos.dtype is torch.int32 and slots.dtype is torch.int64 and pos.shape == slots.shape == (T,) and pos.is_contiguous()
            and slots.is_contiguous()):
        raise ValueError(f"{op}: a position (int32) and a slot (int64) for each row")


_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None
_bound: dict = {}
_SIGNATURES = {
    "dlti_rope_cache8": (_V, _L, _V, _L, _V, _V, _V, _V, _V, _V, _V, _V, _L, _I, _I, _I, _I, _I, _V),
    "dlti_acc_rope_cache8": (_V, _V, _L, _V, _V, _V, _V, _V, _V, _V, _V, _L, _I, _I, _I, _I, _I, _V),
    "dlti_paged_decode8": (_V, _L, _V, _V, _V, _V, _V, _I, _V, _I, _I, _I, _I, _I, _F, _I, _V, _V, _L, _I, _V),
    "dlti_paged_decode8_floats": (_I, _I, _I),
    "dlti_gather_rows8": (_V, _L, _V, _V, _V, _V, _V, _V, _L, _I, _I, _I, _I, _I, _V),
}


def _bind(name: str):
    f = _bound[name] = _lib.fn(name, list(_SIGNATURES[name]), _L if name.endswith("_floats") else _I)
    return f


def _check_slots(op: str, slots, bs: int, num_blocks: int) -> None:
    """Only with the opt-in checks: slots inside the cache, each once, rows of one page next to one another."""
    _debug.check_range(op, "slots", slots, 0, num_blocks * bs, allow=-1)
    s = slots.to("cpu")
    s = s[s >= 0]
    if len(torch.unique(s)) < len(s):
        raise _debug.DltiIndexError(f"{op}: a slot occurs twice")
    page = (slots.to("cpu") // bs).masked_fill(slots.to("cpu") < 0, -1)
    begins = page[torch.cat([torch.ones(min(1, len(page)), dtype=torch.bool), page[1:] != page[:-1]])]
    begins = begins[begins >= 0]
    if len(torch.unique(begins)) < len(begins):
        raise _debug.DltiIndexError(f"{op}: rows of a page are not neighbours")


# ---- rows ---------------------------------------------------------------------------------------------------------------------
def scale_for(largest: torch.Tensor) -> torch.Tensor:
    """Scale of a page whose largest finite number is `largest` (fp32)."""
    m, e = torch.frexp(largest)
    e = torch.where(largest > 0, e - 9 + (m > 0.875).int(), E_LOW).clamp(E_LOW, E_HIGH)
    return torch.ldexp(torch.ones_like(largest), e)


def _write_ref(x, slots, q, scale):
    bs = q.shape[2]
    page, off = slots // bs, slots % bs
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    pages, which = torch.unique(page, return_inverse=True)
    largest = torch.zeros((len(pages), x.shape[1]), device=x.device).scatter_reduce_(0, which[:, None].expand_as(finite), finite, "amax")
    fresh = torch.zeros(len(pages), dtype=torch.bool, device=x.device)
    fresh[which[off == 0]] = True
    old = torch.where(fresh[:, None], 2.0 ** E_LOW, scale[pages])
    new = torch.maximum(old, scale_for(largest))
    held = q[pages].float()
    q[pages] = torch.where(fresh[:, None, None, None], held, held * (old / new)[:, :, None, None]).to(E4M3)
    scale[pages] = new
    q[page, :, off] = (x / new[which][:, :, None]).clamp(-TOP, TOP).to(E4M3)


def rope_cache8_ref(qkv, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale, H, KV, hd, out=None):
    if out is None:
        out = qkv
    else:
        out.copy_(qkv)
    rope_ref(out, pos, cos_t, sin_t, H + KV, hd)
    ok = slots >= 0
    if bool(ok.any()):
        kv = out[ok][:, H * hd:].reshape(-1, 2, KV, hd).float()
        _write_ref(kv[:, 0], slots[ok], k8, k_scale)
        _write_ref(kv[:, 1], slots[ok], v8, v_scale)
    return out


def rope_cache8_(qkv, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale, H, KV, hd, out=None):
    """Rotate q and k of every token row of qkv [T, (H + 2 KV) hd] in place, or from qkv into `out` (qkv itself or apart from it), which then gets v
    too; write rotated k and v of the rows with a slot (int64 [T], -1 = none) to the 8-bit pages. Returns the rotated rows."""
    dst = qkv if out is None else out
    bs = k8.shape[2]
    _check_cache("rope_cache8", k8, v8, k_scale, v_scale, H, KV, hd)
    if _debug.ENABLED:
        _check_slots("rope_cache8", slots, bs, k8.shape[0])
        _debug.check_range("rope_cache8", "positions", pos, 0, cos_t.shape[0])
    T, W = qkv.shape[0], (H + 2 * KV) * hd
    if out is not None:
        _need(dst.shape == qkv.shape and dst.dtype == qkv.dtype, "rope_cache8: out has the shape and type of the rows")
    _check_places("rope_cache8", pos, slots, T)
    if not qkv.is_cuda:
        return rope_cache8_ref(qkv, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale, H, KV, hd, out)
    dev = _check_device("rope_cache8", qkv, dst, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale)
    _check_rows("rope_cache8", qkv, W, out is None)
    if out is not None:
        _check_rows("rope_cache8", dst, W)
    kp, vp = _pages("rope_cache8", k8, v8)
    cp, sp = _tables(cos_t, sin_t, hd)
    f = _bound.get("dlti_rope_cache8") or _bind("dlti_rope_cache8")
    _lib.check(f(qkv.data_ptr(), qkv.stride(0), dst.data_ptr(), dst.stride(0), pos.data_ptr(), cp, sp, slots.data_ptr(),
                 kp, vp, k_scale.data_ptr(), v_scale.data_ptr(), T, H, KV, hd, bs, _lib.dtype_code(qkv.dtype),
                 _stream(dev)), "rope_cache8")
    return dst


def _tables(cos_t, sin_t, hd: int) -> tuple[int, int]:
    if not (cos_t.shape == sin_t.shape and cos_t.shape[1] == hd // 2 and cos_t.dtype is sin_t.dtype is torch.float32 and cos_t.is_contiguous()
            and sin_t.is_contiguous()):
        raise ValueError(f"rotation tables are float32 [positions, {hd // 2}]")
    c, s = cos_t.data_ptr(), sin_t.data_ptr()
    if (c | s) % 16:
        raise ValueError("rotation tables begin at multiples of 16 bytes")
    return c, s


def acc_rope_cache8(acc, dtype, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale, H, KV, hd):
    """Decode path: consume the fp32 qkv accumulator [T, (H + 2 KV) hd] of gemm_skinny_acc (re-zeroing it) and return the 16-bit rows with q and k
    rotated; keys and values also go to the 8-bit pages. Bit-identical to skinny_finish + rope_cache8_."""
    bs = k8.shape[2]
    T, W = acc.shape
    _check_cache("acc_rope_cache8", k8, v8, k_scale, v_scale, H, KV, hd)
    if _debug.ENABLED:
        _check_slots("acc_rope_cache8", slots, bs, k8.shape[0])
        _debug.check_range("acc_rope_cache8", "positions", pos, 0, cos_t.shape[0])
    _need(acc.dtype == torch.float32 and acc.is_contiguous() and W == (H + 2 * KV) * hd, "acc_rope_cache8: a float32 accumulator of whole rows")
    _check_places("acc_rope_cache8", pos, slots, T)
    if not acc.is_cuda:
        out = rope_cache8_ref(acc.to(dtype), pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale, H, KV, hd)
        acc.zero_()
        return out
    dev = _check_device("acc_rope_cache8", acc, pos, cos_t, sin_t, slots, k8, v8, k_scale, v_scale)
    kp, vp = _pages("acc_rope_cache8", k8, v8)
    _need(acc.data_ptr() % 16 == 0, "acc_rope_cache8: the accumulator begins at a multiple of 16 bytes")
    cp, sp = _tables(cos_t, sin_t, hd)
    out = acc.new_empty((T, W), dtype=dtype)
    f = _bound.get("dlti_acc_rope_cache8") or _bind("dlti_acc_rope_cache8")
    _lib.check(f(acc.data_ptr(), out.data_ptr(), W, pos.data_ptr(), cp, sp, slots.data_ptr(), kp, vp,
                 k_scale.data_ptr(), v_scale.data_ptr(), T, H, KV, hd, bs, _lib.dtype_code(dtype), _stream(dev)), "acc_rope_cache8")
    return out


# ---- attention ----------------------------------------------------------------------------------------------------------------
def paged_decode8_ref(q, k8, v8, k_scale, v_scale, block_tables, ctx_lens, H, KV, hd, scale):
    out = torch.zeros(q.shape[0], H * hd, dtype=torch.float32, device=q.device)
    bs = k8.shape[2]
    for b, n in enumerate(ctx_lens.tolist()):
        n = min(n, block_tables.shape[1] * bs)
        if n <= 0:
            continue
        t = block_tables[b, :-(-n // bs)].long()
        k = (k8[t].float() * k_scale[t][..., None, None]).transpose(0, 1).reshape(KV, -1, hd)[:, :n]
        v = (v8[t].float() * v_scale[t][..., None, None]).transpose(0, 1).reshape(KV, -1, hd)[:, :n]
        qq = q[b, :H * hd].float().view(KV, H // KV, hd)
        out[b] = (torch.softmax(qq @ k.transpose(1, 2) * scale, -1) @ v).reshape(H * hd)
    return out.to(q.dtype)


def splits8(ctas: int, reach: int) -> int:
    """CTAs over which contexts of up to `reach` tokens are cut when one each would be `ctas`: one wave of three per SM (a second one costs what it
    should save), 64 tokens at least. Up to 8 are one cluster, more are clusters of one size.

    us of a call alone, from a graph and with a cold L2, 6 of them the launch's, read to 2: 4 rows of up to 30011 tokens with 8 key heads in 6 splits
    72, 8 61, 12 59, 16 (two waves) 72; 32 rows of 4000 tokens with 4 key heads in 1 split 49, 2 39, 3 37, 4 (two waves) 47; 64 rows of up to 1000
    with 4 key heads in 1 split 22, 2 (two waves) 31."""
    n = max(1, min(128, 3 * 148 // max(1, ctas), -(-reach // 64)))
    # 9 .. 15 splits of short contexts: 8, one cluster and no kernel to join two. Measured as above, in 8 / in 12: 4 rows with 8 key heads of 700 tokens
    # 14 / 16, 2000 16 / 18, 4000 20 / 22, 8000 27 / 29, 12000 33 / 35, 16000 41 / 41, 30011 61 / 59; one row with 32 key heads of 4000 18 / 20,
    # 6000 22 / 25, 8000 27 / 27, 16000 41 / 39. So the border could lie up to 16000; between, it costs 2 us at most.
    if n < 16 and reach <= 4096:
        return min(n, 8)
    while n % -(-n // 8):
        n -= 1
    return n


def paged_decode8(q, k8, v8, k_scale, v_scale, block_tables, ctx_lens, H, KV, hd, scale=None, out=None, max_ctx: int | None = None):
    """paged_decode over 8-bit pages. q: [B, >= H hd] (row b = the single new token of sequence b); block_tables int32 [B, *], ctx_lens int32 [B],
    0 = a row of zeros; max_ctx: the longest context that may occur (a context beyond it is read in full). Returns out [B, H hd]: a tensor of its own,
    or the one given, which is the queries' own place or apart from them."""
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    _check_cache("paged_decode8", k8, v8, k_scale, v_scale, H, KV, hd)
    B, W = q.shape
    if W < H * hd:
        raise ValueError("paged_decode8: rows of at least H hd columns")
    if not (block_tables.dtype is torch.int32 and ctx_lens.dtype is torch.int32 and block_tables.dim() == 2 and block_tables.shape[0] == B
            and ctx_lens.shape == (B,) and block_tables.is_contiguous() and ctx_lens.is_contiguous()):
        raise ValueError("paged_decode8: an int32 table and an int32 length for each row")
    if out is not None:
        _need(out.shape == (B, H * hd) and out.dtype == q.dtype and out.stride(1) == 1, "paged_decode8: out is [B, H hd] in q's type")
        _need(B < 2 or out.stride(0) >= H * hd, "paged_decode8: rows that are written do not overlap")
    if _debug.ENABLED:
        _debug.check_paged("paged_decode8", block_tables, ctx_lens, k8.shape[0], k8.shape[2])
    if not q.is_cuda:
        o = paged_decode8_ref(q, k8, v8, k_scale, v_scale, block_tables, ctx_lens, H, KV, hd, scale)
        return o if out is None else out.copy_(o)
    dev = _check_device("paged_decode8", q, k8, v8, k_scale, v_scale, block_tables, ctx_lens)
    ld, unit = q.stride()
    if unit != 1 or ld % 8 or q.data_ptr() % 16:
        raise ValueError("paged_decode8: rows begin at multiples of 16 bytes")
    kp, vp = _pages("paged_decode8", k8, v8)
    bs, width = k8.shape[2], block_tables.shape[1]
    _need(width * bs < 1 << 31, "paged_decode8: contexts have 31 bits")
    if out is None:
        out = q.new_empty((B, H * hd))
    else:
        _check_device("paged_decode8", out)
    splits = splits8(B * KV * -(-(H // KV) // 8), width * bs if max_ctx is None else min(width * bs, max_ctx))
    # a workspace of this call's own: the allocator keeps it for the stream's later work, or inside the graph that captures it
    ws = None
    if splits > 8:
        floats = _bound.get("dlti_paged_decode8_floats") or _bind("dlti_paged_decode8_floats")
        ws = torch.empty(floats(B, H, splits), dtype=torch.float32, device=q.device)
    f = _bound.get("dlti_paged_decode8") or _bind("dlti_paged_decode8")
    _lib.check(f(q.data_ptr(), ld, kp, vp, k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(),
                 width, ctx_lens.data_ptr(), B, bs, H, KV, hd, scale, splits, None if ws is None else ws.data_ptr(),
                 out.data_ptr(), out.stride(0), _lib.dtype_code(q.dtype), _stream(dev)), "paged_decode8")
    return out


# ---- cached rows in 16 bits -----------------------------------------------------------------------------------------------------
def gather_rows8_ref(ext, rows, slots, k8, v8, k_scale, v_scale, H, KV, hd):
    bs = k8.shape[2]
    page, off = slots // bs, slots % bs
    for c, (q, s) in enumerate(((k8, k_scale), (v8, v_scale))):
        ext[rows, (H + c * KV) * hd:(H + (c + 1) * KV) * hd] = (q[page, :, off].float() * s[page][..., None]).flatten(1).to(ext.dtype)
    return ext


def gather_rows8_(ext, rows, slots, k8, v8, k_scale, v_scale, H, KV, hd):
    """Key and value columns of the rows `rows` (int64 [n], each once) of ext [*, (H + 2 KV) hd] from the cached tokens at `slots` (int64 [n]), in
    ext's type. Returns ext; its other rows and columns stay as they are."""
    _check_cache("gather_rows8", k8, v8, k_scale, v_scale, H, KV, hd)
    if not (rows.dim() == 1 and rows.shape == slots.shape and rows.dtype is torch.int64 and slots.dtype is torch.int64 and rows.is_contiguous()
            and slots.is_contiguous()):
        raise ValueError("gather_rows8: an int64 row for each int64 slot")
    if _debug.ENABLED:
        _debug.check_range("gather_rows8", "slots", slots, 0, k8.shape[0] * k8.shape[2])
        _debug.check_range("gather_rows8", "rows", rows, 0, ext.shape[0])
    if not ext.is_cuda:
        return gather_rows8_ref(ext, rows, slots, k8, v8, k_scale, v_scale, H, KV, hd)
    dev = _check_device("gather_rows8", ext, rows, slots, k8, v8, k_scale, v_scale)
    _check_rows("gather_rows8", ext, (H + 2 * KV) * hd)
    kp, vp = _pages("gather_rows8", k8, v8, unit=8)
    f = _bound.get("dlti_gather_rows8") or _bind("dlti_gather_rows8")
    _lib.check(f(ext.data_ptr(), ext.stride(0), rows.data_ptr(), slots.data_ptr(), kp, vp, k_scale.data_ptr(),
                 v_scale.data_ptr(), slots.numel(), H, KV, hd, k8.shape[2], _lib.dtype_code(ext.dtype), _stream(dev)), "gather_rows8")
    return ext
