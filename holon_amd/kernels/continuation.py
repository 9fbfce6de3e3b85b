"""Operations for serving many continuations of a context: the 8-bit paged cache (written, read back, attended over), attention
of a batch whose sequences share a prefix, and the verification of drafted tokens. Methods of `HipKernels`; the contract is in
`holon_amd.kernels.api`.

The smallest of these calls (a step's eight tokens) keep the GPU busy for 3 us, so what a call costs on the host is what it
costs: a tensor is asked for each of its facts once, a message is formatted only where it is raised, and the attention's three
dozen arguments travel packed, as one."""
from __future__ import annotations

import ctypes
import struct

import torch

from .api import AttnRows, SharedPrefix

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_DT = {torch.float32: 0, torch.bfloat16: 1}
_CODES = (torch.float8_e4m3fn, torch.uint8)
_SCALES = (torch.float8_e8m0fnu, torch.uint8)
_INT32 = torch.int32
_HEADS = (64, 128, 256)

SYMBOLS = {
    "holon_kv_write_q8": ([_P, _P, _L, _P, _P, _L, _L, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "holon_qk_norm_rope_write_q8": ([_P, _P, _I, _I, _I, _I, _P, _P, ctypes.c_float, _P, _I, _P, _P, _P, _L, _L, _P, _P, _I, _I, _I, _P], _I),
    "holon_kv_read_q8": ([_P, _P, _P, _P, _L, _L, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "holon_cache_attention_room": ([ctypes.c_char_p], _L),
    "holon_cache_attention": ([ctypes.c_char_p, _P, _P, _P, _P], _I),
    "holon_verify_drafts_room": ([_I, _I, _I], _L),
    "holon_verify_drafts": ([_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
}
# struct HolonCacheAttention (csrc/holon_hip.h): its pointers, its 64-bit sizes, its 32-bit ones
_ATTENTION = struct.Struct("=11Q3q18if")


def _fail(message: str) -> None:
    from .hip import KernelError
    raise KernelError(message)


def _ints(what: str, name: str, t: torch.Tensor, size: int, device: int) -> int:
    """The address of an int32 vector of `size` values."""
    if t.dtype is not _INT32 or t.shape != (size,) or t.get_device() != device or not t.is_contiguous():
        _fail(f"{what} {name}: expected ({size},) int32 on device {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


class ContinuationOps:
    @staticmethod
    def _current() -> int:
        return torch._C._cuda_getDevice()

    @staticmethod
    def _stream_of(device: int) -> int:
        return torch._C._cuda_getCurrentRawStream(device)

    def _place(self, what: str, t: torch.Tensor) -> int:
        """The device that the call runs on: kernels go to the current device's current stream, so the tensors have to be there."""
        device = t.get_device()
        if device < 0:
            _fail(f"{what}: the HIP kernels need a GPU tensor, got one on {t.device}")
        if device != self._current():
            _fail(f"{what}: tensors on {t.device}, but the current device is cuda:{self._current()}")
        return device

    @staticmethod
    def _paged(what: str, pages: torch.Tensor, scales: torch.Tensor | None, page_size: int, device: int) -> tuple:
        """(pages, kv heads, head size, their address, bytes from page to page, the scales' two) of a cache of 8 bits, or (scales
        None) of bfloat16: shapes, types and strides checked."""
        shape = pages.shape
        if len(shape) != 4:
            _fail(f"{what}: pages {tuple(pages.shape)} are no [n, 2, Hkv, P D]")
        (n, two, kv, wide), (step, s1, s2, s3), at = shape, pages.stride(), pages.data_ptr()
        dim = wide // page_size if page_size > 0 else 0
        if page_size % 16 or dim not in _HEADS or dim * page_size != wide:
            _fail(f"{what}: pages {tuple(pages.shape)} of {page_size} tokens hold no heads of 64, 128 or 256 in pages of a multiple of 16")
        if two != 2 or n < 1 or kv < 1 or s3 != 1 or s2 != wide or s1 != kv * wide or (n > 1 and step < 2 * s1) or pages.get_device() != device:
            _fail(f"{what}: pages {tuple(pages.shape)} on {pages.device}, strides {pages.stride()}: [n, 2, Hkv, P D], each in one piece, where the rest is")
        if scales is None:
            if pages.dtype is not torch.bfloat16:
                _fail(f"{what}: a cache of {pages.dtype} (bfloat16, or 8 bits with scales)")
            if (at | 2 * step) % 16:
                _fail(f"{what}: pages have to lie on borders of 16 bytes")
            return n, kv, dim, at, 2 * step, None, 0
        if pages.dtype not in _CODES or scales.dtype not in _SCALES:
            _fail(f"{what}: pages of {pages.dtype} with scales of {scales.dtype} (float8_e4m3fn and float8_e8m0fnu, or uint8 for either)")
        if scales.shape != (n, 2, kv, page_size) or scales.get_device() != device:
            _fail(f"{what}: scales {tuple(scales.shape)} on {scales.device} for pages {tuple(pages.shape)} of {page_size} tokens")
        (gap, t1, t2, t3), to = scales.stride(), scales.data_ptr()
        if t3 != 1 or t2 != page_size or t1 != kv * page_size or (n > 1 and gap < 2 * t1):
            _fail(f"{what}: the scales of a page have to lie in one piece (strides {scales.stride()})")
        if (at | step | to | gap) % 16:
            _fail(f"{what}: pages and scales have to lie on borders of 16 bytes")
        return n, kv, dim, at, step, to, gap

    def _paged_q8(self, what: str, pages: torch.Tensor, scales: torch.Tensor, page_size: int, device: int) -> tuple:
        if scales is None:
            _fail(f"{what}: an 8-bit cache has scales")
        return self._paged(what, pages, scales, page_size, device)

    def check_cache_q8(self, head_dim: int, page_size: int) -> None:
        if head_dim not in _HEADS or page_size <= 0 or page_size % 16:
            _fail(f"8-bit cache: heads of {head_dim} in pages of {page_size} tokens are not served (64, 128 and 256; multiples of 16)")

    def kv_write_q8(self, k, v, pages, scales, write_page, write_off, page_size) -> None:
        what = "kv_write_q8"
        device = self._place(what, k)
        n, kv, dim, at, step, to, gap = self._paged_q8(what, pages, scales, page_size, device)
        shape, dtype = k.shape, k.dtype
        t = shape[0] if shape else -1
        if dtype not in _DT or v.dtype is not dtype or shape != (t, kv, dim) or v.shape != shape or v.get_device() != device:
            _fail(f"{what}: keys {tuple(shape)} {dtype} and values {tuple(v.shape)} {v.dtype} on {v.device} for {kv} heads of {dim}")
        row = kv * dim
        if t > 1:
            row = k.stride(0)
        for one, two, three in (k.stride(), v.stride()):
            if three != 1 or (kv > 1 and two != dim) or (t > 1 and one != row) or row < kv * dim:
                _fail(f"{what}: keys and values are columns of rows as far apart, got strides {k.stride()} and {v.stride()}")
        self._call(self.lib.holon_kv_write_q8, k.data_ptr(), v.data_ptr(), row, at, to, step, gap, _ints(what, "pages", write_page, t, device),
                   _ints(what, "offsets", write_off, t, device), t, kv, dim, page_size, n, _DT[dtype], self._stream_of(device))

    def qk_norm_rope_write_q8(self, qkv, heads, kv_heads, head_dim, q_weight, k_weight, eps, table, positions, pages, scales, write_page,
                              write_off, page_size):
        what = "qk_norm_rope_write_q8"
        device = self._place(what, qkv)
        n, kv, dim, at, step, to, gap = self._paged_q8(what, pages, scales, page_size, device)
        dtype, shape = qkv.dtype, qkv.shape
        if dtype not in _DT or heads < 1 or (kv, dim) != (kv_heads, head_dim) or len(shape) != 2 or shape[1] != (heads + 2 * kv) * dim \
                or not qkv.is_contiguous():
            _fail(f"{what}: a projection {tuple(shape)} {dtype} (strides {qkv.stride()}) of {heads} heads over {kv_heads} of {head_dim}, "
                  f"into a cache of {kv} of {dim}")
        t, weights, turn, where, most = shape[0], [None, None], None, None, 0
        if (q_weight is None) != (k_weight is None):
            _fail(f"{what}: q and k norm weights come together")
        if q_weight is not None:
            for w in (q_weight, k_weight):
                if w.dtype is not dtype or w.shape != (dim,) or not w.is_contiguous() or w.get_device() != device:
                    _fail(f"{what}: a norm weight {tuple(w.shape)} {w.dtype} on {w.device} for heads of {dim} in {dtype}")
            weights = [q_weight.data_ptr(), k_weight.data_ptr()]
        if table is not None:
            if table.dtype is not torch.float32 or table.dim() != 2 or table.shape[1] != dim or table.shape[0] < 1 or not table.is_contiguous() \
                    or table.get_device() != device:
                _fail(f"{what}: a rope table {tuple(table.shape)} {table.dtype} on {table.device} (whole heads of {dim} are turned)")
            turn, most, where = table.data_ptr(), table.shape[0], _ints(what, "positions", positions, t, device)
        q = torch.empty((t, heads, dim), dtype=dtype, device=qkv.device)
        self._call(self.lib.holon_qk_norm_rope_write_q8, qkv.data_ptr(), q.data_ptr(), t, heads, kv, dim, *weights, float(eps), turn, most, where,
                   at, to, step, gap, _ints(what, "pages", write_page, t, device), _ints(what, "offsets", write_off, t, device), page_size, n,
                   _DT[dtype], self._stream_of(device))
        return q

    def kv_read_q8(self, pages, scales, read_page, read_off, page_size, dtype=torch.bfloat16):
        what = "kv_read_q8"
        device = self._place(what, pages)
        n, kv, dim, at, step, to, gap = self._paged_q8(what, pages, scales, page_size, device)
        if dtype not in _DT:
            _fail(f"{what}: into {dtype} (float32 and bfloat16 are served)")
        t = read_page.shape[0] if read_page.dim() == 1 else -1
        rp, ro = _ints(what, "pages", read_page, t, device), _ints(what, "offsets", read_off, t, device)
        k = torch.empty((t, kv, dim), dtype=dtype, device=pages.device)
        v = torch.empty_like(k)
        self._call(self.lib.holon_kv_read_q8, k.data_ptr(), v.data_ptr(), at, to, step, gap, rp, ro, t, kv, dim, page_size, n, _DT[dtype],
                   self._stream_of(device))
        return k, v

    def paged_attention_q8(self, q, pages, scales, table, rows: AttnRows, page_size, scale, window=0, sink=None):
        if scales is None:
            _fail("paged_attention_q8: an 8-bit cache has scales")
        return self._cache_attention("paged_attention_q8", q, pages, scales, table, rows, None, page_size, scale, window, sink)

    def prefix_attention(self, q, pages, table, rows: AttnRows, prefix: SharedPrefix, page_size, scale, scales=None, sink=None):
        return self._cache_attention("prefix_attention", q, pages, scales, table, rows, prefix, page_size, scale, 0, sink)

    def _cache_attention(self, what, q, pages, scales, table, rows, prefix, page_size, scale, window, sink):
        device = self._place(what, q)
        n, kv, dim, at, step, to, gap = self._paged(what, pages, scales, page_size, device)
        dtype, shape = q.dtype, q.shape
        if dtype is not torch.bfloat16 and (scales is None or dtype is not torch.float32):
            _fail(f"{what}: queries of {dtype} (bfloat16; over the 8-bit cache float32 too)")
        if len(shape) != 3:
            _fail(f"{what}: queries {tuple(shape)} are no [T, Hq, D]")
        (t, heads, width), q_at = shape, q.data_ptr()
        if width != dim or heads % kv or heads == 0 or not q.is_contiguous() or q_at % 16:
            _fail(f"{what}: queries {tuple(shape)} (strides {q.stride()}) over {kv} heads of {dim}, contiguous from a border of 16 bytes")
        held = table.shape
        if table.dtype is not _INT32 or len(held) != 2 or not table.is_contiguous() or table.get_device() != device or 0 in held:
            _fail(f"{what}: a block table {tuple(held)} {table.dtype} on {table.device}")
        if not scale > 0:
            _fail(f"{what}: a scale of {scale}")
        slots, n_decode, n_chunk = rows.slots, rows.n_decode, rows.n_chunk
        b = slots.numel()
        sink_at = starts_at = lens_at = decode = chunk = 0
        if sink is not None:
            if sink.dtype is not torch.float32 or sink.shape != (heads,) or not sink.is_contiguous() or sink.get_device() != device:
                _fail(f"{what}: a sink {tuple(sink.shape)} {sink.dtype} for {heads} heads")
            sink_at = sink.data_ptr()
        if n_decode and not (rows.in_order and n_decode == b == t):
            decode = _ints(what, "decode_rows", rows.decode_rows, n_decode, device)
        if n_chunk:
            chunk = _ints(what, "chunk_rows", rows.chunk_rows, n_chunk, device)
        groups = most = longest = 0
        if prefix is not None and prefix.n_groups:
            groups, most, longest = prefix.n_groups, prefix.max_queries, prefix.max_len
            starts_at = _ints(what, "group_start", prefix.group_start, groups + 1, device)
            lens_at = _ints(what, "prefix lens", prefix.lens, groups, device)
        try:
            packed = _ATTENTION.pack(
                at, to or 0, table.data_ptr(), _ints(what, "slots", slots, b, device), _ints(what, "lens", rows.lens, b, device),
                _ints(what, "query_start", rows.query_start, b + 1, device), decode, chunk, starts_at, lens_at, sink_at, step, gap, t,
                n, held[1], held[0], b, n_decode, rows.max_decode_len, n_chunk, rows.max_chunk_query, rows.max_chunk_len, groups, most, longest,
                heads, kv, dim, page_size, int(window), _DT[dtype], scale)
        except (struct.error, OverflowError) as error:
            _fail(f"{what}: sizes, bounds and the window are whole numbers of 32 bits, the scale a float32 ({error})")
        out = torch.empty_like(q)
        room = self.lib.holon_cache_attention_room(packed)
        space = torch.empty((room,), dtype=torch.uint8, device=q.device) if room else None
        self._call(self.lib.holon_cache_attention, packed, q_at, out.data_ptr(), space.data_ptr() if room else None,
                   self._stream_of(device))
        return out

    def verify_drafts(self, logits, drafted, draft_probs, accept, draw, temperature, start, most):
        what = "verify_drafts"
        device = self._place(what, logits)
        shape, f32 = logits.shape, torch.float32
        if logits.dtype is not f32 or len(shape) != 2 or not logits.is_contiguous() or shape[1] == 0:
            _fail(f"{what}: logits {tuple(shape)} {logits.dtype} (contiguous float32 rows)")
        n, vocab = shape
        probs = None
        if draft_probs is not None:
            if draft_probs.dtype is not f32 or draft_probs.shape != shape or not draft_probs.is_contiguous() or draft_probs.get_device() != device:
                _fail(f"{what}: draft probabilities {tuple(draft_probs.shape)} {draft_probs.dtype} for {tuple(shape)} logits")
            probs = draft_probs.data_ptr()
        b = draw.numel()
        for x, size, name in ((accept, n, "accept"), (draw, b, "draw"), (temperature, b, "temperature")):
            if x.dtype is not f32 or x.shape != (size,) or not x.is_contiguous() or x.get_device() != device:
                _fail(f"{what} {name}: expected ({size},) float32 on device {device}, got {tuple(x.shape)} {x.dtype} on {x.device}")
        d, s = _ints(what, "drafted", drafted, n, device), _ints(what, "start", start, b + 1, device)
        if not 0 <= most <= 63:
            _fail(f"{what}: up to {most} drafted tokens a request (at most 63 are served)")
        place = logits.device
        tokens = torch.empty((b, most + 1), dtype=_INT32, device=place)
        accepted = torch.empty((b,), dtype=_INT32, device=place)
        room = torch.empty((self.lib.holon_verify_drafts_room(n, b, vocab),), dtype=torch.uint8, device=place)
        self._call(self.lib.holon_verify_drafts, logits.data_ptr(), d, probs, accept.data_ptr(), draw.data_ptr(), temperature.data_ptr(), s,
                   tokens.data_ptr(), accepted.data_ptr(), room.data_ptr(), n, b, vocab, most, self._stream_of(device))
        return tokens, accepted
