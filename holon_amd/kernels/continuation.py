"""Operations for serving many continuations of a context: the 8-bit paged cache (written, read back, attended over), attention
of a batch whose sequences share a prefix, and the verification of drafted tokens. Methods of `HipKernels`; the contract is in
`holon_amd.kernels.api`."""
from __future__ import annotations

import ctypes

import torch

from .api import AttnRows, SharedPrefix

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_DT = {torch.float32: 0, torch.bfloat16: 1}
_CODES = (torch.float8_e4m3fn, torch.uint8)
_SCALES = (torch.float8_e8m0fnu, torch.uint8)

SYMBOLS = {
    "holon_kv_write_q8": ([_P, _P, _L, _P, _P, _L, _L, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "holon_kv_read_q8": ([_P, _P, _P, _P, _L, _L, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "holon_cache_attention_room": ([_I] * 13 + [_I], _L),
    "holon_cache_attention": ([_P, _P, _P, _P, _L, _L, _I, _P, _I, _I, _P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P, _P, _I, _I, _I,
                               _I, _I, _I, _I, _I, _F, _I, _P, _P, _I, _P], _I),
    "holon_verify_drafts_room": ([_I, _I, _I], _L),
    "holon_verify_drafts": ([_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
}


def _need(ok: bool, message: str) -> None:
    if not ok:
        from .hip import KernelError
        raise KernelError(message)


def _ints(what: str, t: torch.Tensor, size: int, device: torch.device) -> int:
    """The address of an int32 vector of `size` values."""
    if t.dtype != torch.int32 or t.shape != (size,) or t.device != device or not t.is_contiguous():
        _need(False, f"{what}: expected ({size},) int32 on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


class ContinuationOps:
    @staticmethod
    def _place(what: str, t: torch.Tensor) -> torch.device:
        """Kernels run on the current device's current stream: the tensors have to be there."""
        if not t.is_cuda:
            _need(False, f"{what}: the HIP kernels need a GPU tensor, got one on {t.device}")
        if t.device.index != torch.cuda.current_device():
            _need(False, f"{what}: tensors on {t.device}, but the current device is cuda:{torch.cuda.current_device()}")
        return t.device

    @staticmethod
    def _cache8(what: str, pages: torch.Tensor, scales: torch.Tensor, page_size: int, device: torch.device) -> tuple[int, int]:
        """(kv heads, head size) of an 8-bit cache, its shapes, types and strides checked."""
        _need(pages.dtype in _CODES and scales.dtype in _SCALES, f"{what}: pages of {pages.dtype} with scales of {scales.dtype} "
              "(float8_e4m3fn and float8_e8m0fnu, or uint8 for either)")
        _need(pages.dim() == 4 and scales.dim() == 4 and page_size > 0 and pages.shape[3] % page_size == 0
              and scales.shape == (*pages.shape[:3], page_size) and pages.shape[1] == 2 and pages.shape[0] > 0,
              f"{what}: pages {tuple(pages.shape)} and scales {tuple(scales.shape)} are no [n, 2, Hkv, P D] and [n, 2, Hkv, P] at "
              f"pages of {page_size} tokens")
        _need(pages.device == device and scales.device == device, f"{what}: pages on {pages.device}, scales on {scales.device}, the rest on {device}")
        _need(pages[0].is_contiguous() and scales[0].is_contiguous() and pages.stride(0) >= pages[0].numel()
              and scales.stride(0) >= scales[0].numel(), f"{what}: a page has to lie in one piece (strides {pages.stride()}, {scales.stride()})")
        _need((pages.data_ptr() | scales.data_ptr() | pages.stride(0) | scales.stride(0)) % 16 == 0,
              f"{what}: pages and scales have to lie on borders of 16 bytes")
        return pages.shape[2], pages.shape[3] // page_size

    def check_cache_q8(self, head_dim: int, page_size: int) -> None:
        _need(head_dim in (64, 128, 256), f"8-bit cache: head_dim {head_dim} is not served (64, 128 and 256 are)")
        _need(page_size > 0 and page_size % 16 == 0, f"8-bit cache: pages of {page_size} tokens are not served (multiples of 16 are)")

    def kv_write_q8(self, k, v, pages, scales, write_page, write_off, page_size) -> None:
        what = "kv_write_q8"
        device = self._place(what, k)
        kv_heads, head_dim = self._cache8(what, pages, scales, page_size, device)
        self.check_cache_q8(head_dim, page_size)
        t = k.shape[0]
        _need(k.dtype in _DT and v.dtype == k.dtype and k.shape == (t, kv_heads, head_dim) and v.shape == k.shape and v.device == device,
              f"{what}: keys {tuple(k.shape)} {k.dtype} and values {tuple(v.shape)} {v.dtype} for {kv_heads} heads of {head_dim}")
        stride = k.stride(0) if t > 1 else kv_heads * head_dim
        for x in (k, v):
            _need((kv_heads == 1 or x.stride(1) == head_dim) and x.stride(2) == 1 and (t <= 1 or x.stride(0) == stride),
                  f"{what}: keys and values are columns of rows as far apart, got strides {k.stride()} and {v.stride()}")
        wp, wo = _ints(f"{what} pages", write_page, t, device), _ints(f"{what} offsets", write_off, t, device)
        self._call(self.lib.holon_kv_write_q8, k.data_ptr(), v.data_ptr(), stride, pages.data_ptr(), scales.data_ptr(),
                   pages.stride(0), scales.stride(0), wp, wo, t, kv_heads, head_dim, page_size, pages.shape[0], _DT[k.dtype],
                   self._stream())

    def kv_read_q8(self, pages, scales, read_page, read_off, page_size, dtype=torch.bfloat16):
        what = "kv_read_q8"
        device = self._place(what, pages)
        kv_heads, head_dim = self._cache8(what, pages, scales, page_size, device)
        self.check_cache_q8(head_dim, page_size)
        _need(dtype in _DT, f"{what}: into {dtype} (float32 and bfloat16 are served)")
        t = read_page.shape[0] if read_page.dim() == 1 else -1
        rp, ro = _ints(f"{what} pages", read_page, t, device), _ints(f"{what} offsets", read_off, t, device)
        k = torch.empty((t, kv_heads, head_dim), dtype=dtype, device=device)
        v = torch.empty_like(k)
        self._call(self.lib.holon_kv_read_q8, k.data_ptr(), v.data_ptr(), pages.data_ptr(), scales.data_ptr(), pages.stride(0),
                   scales.stride(0), rp, ro, t, kv_heads, head_dim, page_size, pages.shape[0], _DT[dtype], self._stream())
        return k, v

    def paged_attention_q8(self, q, pages, scales, table, rows: AttnRows, page_size, scale, window=0, sink=None):
        what = "paged_attention_q8"
        device = self._place(what, q)
        kv_heads, head_dim = self._cache8(what, pages, scales, page_size, device)
        return self._cache_attention(what, q, pages, scales, table, rows, None, page_size, scale, int(window), sink, kv_heads, head_dim,
                                     device)

    def prefix_attention(self, q, pages, table, rows: AttnRows, prefix: SharedPrefix, page_size, scale, scales=None, sink=None):
        what = "prefix_attention"
        device = self._place(what, q)
        if scales is not None:
            kv_heads, head_dim = self._cache8(what, pages, scales, page_size, device)
        else:
            _need(pages.dtype == torch.bfloat16, f"{what}: a cache of {pages.dtype} (bfloat16, or 8 bits with scales)")
            _need(pages.dim() == 4 and pages.shape[0] > 0 and pages.shape[1] == 2 and page_size > 0 and pages.shape[3] % page_size == 0,
                  f"{what}: pages {tuple(pages.shape)} are no [n, 2, Hkv, P D] at pages of {page_size} tokens")
            _need(pages.device == device and pages[0].is_contiguous() and pages.stride(0) >= pages[0].numel()
                  and (pages.data_ptr() | 2 * pages.stride(0)) % 16 == 0, f"{what}: a page has to lie in one piece, on a border of 16 bytes")
            kv_heads, head_dim = pages.shape[2], pages.shape[3] // page_size
        return self._cache_attention(what, q, pages, scales, table, rows, prefix, page_size, scale, 0, sink, kv_heads, head_dim, device)

    def _cache_attention(self, what, q, pages, scales, table, rows, prefix, page_size, scale, window, sink, kv_heads, head_dim, device):
        self.check_cache_q8(head_dim, page_size)
        _need(q.dtype == torch.bfloat16 or (scales is not None and q.dtype == torch.float32),
              f"{what}: queries of {q.dtype} (bfloat16; over the 8-bit cache float32 too)")
        _need(q.dim() == 3 and q.shape[2] == head_dim and q.shape[1] % kv_heads == 0 and q.shape[1] > 0 and q.is_contiguous()
              and q.data_ptr() % 16 == 0, f"{what}: queries {tuple(q.shape)} (strides {q.stride()}) over {kv_heads} heads of {head_dim}")
        _need(table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous() and table.device == device
              and table.numel() > 0, f"{what}: a block table {tuple(table.shape)} {table.dtype} on {table.device}")
        _need(scale > 0, f"{what}: a scale of {scale}")
        t, heads, _ = q.shape
        b = rows.slots.shape[0]
        slots, lens = _ints(f"{what} slots", rows.slots, b, device), _ints(f"{what} lens", rows.lens, b, device)
        starts = _ints(f"{what} query_start", rows.query_start, b + 1, device)
        n_decode, n_chunk = rows.n_decode, rows.n_chunk
        decode = _ints(f"{what} decode_rows", rows.decode_rows, n_decode, device) if n_decode else None
        chunk = _ints(f"{what} chunk_rows", rows.chunk_rows, n_chunk, device) if n_chunk else None
        if sink is not None:
            _need(sink.dtype == torch.float32 and sink.shape == (heads,) and sink.is_contiguous() and sink.device == device,
                  f"{what}: a sink {tuple(sink.shape)} {sink.dtype} for {heads} heads")
        groups = (None, None, 0, 0, 0)
        if prefix is not None and prefix.n_groups:
            g = prefix.n_groups
            groups = (_ints(f"{what} group_start", prefix.group_start, g + 1, device), _ints(f"{what} prefix lens", prefix.lens, g, device),
                      g, prefix.max_queries, prefix.max_len)
        out = torch.empty_like(q)
        room = self.lib.holon_cache_attention_room(n_decode, rows.max_decode_len, n_chunk, rows.max_chunk_query, rows.max_chunk_len,
                                                   *groups[2:], t, heads, kv_heads, head_dim, window, _DT[q.dtype])
        space = torch.empty((room,), dtype=torch.uint8, device=device) if room else None
        self._call(self.lib.holon_cache_attention, q.data_ptr(), out.data_ptr(), pages.data_ptr(),
                   scales.data_ptr() if scales is not None else None, pages.stride(0) * pages.element_size(),
                   scales.stride(0) if scales is not None else 0, pages.shape[0], table.data_ptr(), table.shape[1], table.shape[0],
                   slots, lens, starts, decode, n_decode, rows.max_decode_len, chunk, n_chunk, rows.max_chunk_query,
                   rows.max_chunk_len, *groups, t, heads, kv_heads, head_dim, page_size, float(scale), window,
                   sink.data_ptr() if sink is not None else None, space.data_ptr() if room else None, _DT[q.dtype], self._stream())
        return out

    def verify_drafts(self, logits, drafted, draft_probs, accept, draw, temperature, start, most):
        what = "verify_drafts"
        device = self._place(what, logits)
        _need(logits.dtype == torch.float32 and logits.dim() == 2 and logits.is_contiguous() and logits.shape[1] > 0,
              f"{what}: logits {tuple(logits.shape)} {logits.dtype} (contiguous float32 rows)")
        n, vocab = logits.shape
        if draft_probs is not None:
            _need(draft_probs.dtype == torch.float32 and draft_probs.shape == logits.shape and draft_probs.is_contiguous()
                  and draft_probs.device == device, f"{what}: draft probabilities {tuple(draft_probs.shape)} {draft_probs.dtype} for {tuple(logits.shape)} logits")
        b = draw.shape[0] if draw.dim() == 1 else -1
        for x, size, name in ((accept, n, "accept"), (draw, b, "draw"), (temperature, b, "temperature")):
            _need(x.dtype == torch.float32 and x.shape == (size,) and x.is_contiguous() and x.device == device,
                  f"{what} {name}: expected ({size},) float32 on {device}, got {tuple(x.shape)} {x.dtype} on {x.device}")
        d, s = _ints(f"{what} drafted", drafted, n, device), _ints(f"{what} start", start, b + 1, device)
        _need(0 <= most <= 63, f"{what}: up to {most} drafted tokens a request (at most 63 are served)")
        tokens = torch.empty((b, most + 1), dtype=torch.int32, device=device)
        accepted = torch.empty((b,), dtype=torch.int32, device=device)
        room = torch.empty((self.lib.holon_verify_drafts_room(n, b, vocab),), dtype=torch.uint8, device=device)
        self._call(self.lib.holon_verify_drafts, logits.data_ptr(), d, draft_probs.data_ptr() if draft_probs is not None else None,
                   accept.data_ptr(), draw.data_ptr(), temperature.data_ptr(), s, tokens.data_ptr(), accepted.data_ptr(),
                   room.data_ptr(), n, b, vocab, most, self._stream())
        return tokens, accepted
