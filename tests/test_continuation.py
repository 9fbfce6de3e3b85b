"""The operators for many continuations of a context: the 8-bit paged cache written, read back and attended over, attention over
prefixes that rows share, the verification of drafted tokens. What is exact is held to equality, attention to a bound that is
derived from the formula's own roundings (`_bound`), the verification's whole numbers to the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from holon_amd.kernels.api import AttnRows, SharedPrefix
from holon_amd.kernels.continuation import ContinuationOps
from holon_amd.kernels.hip import KernelError
from tests.plain.ops import TorchKernels, dequantise_q8, quantise_q8

PLAIN = TorchKernels()
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# -- the format -------------------------------------------------------------------------------------------------------------

def test_a_row_of_the_format():
    """The smallest power of two that brings the largest value to 448 or less; values to half a step of four significant bits."""
    for largest, power in ((448.0, 0), (448.5, 1), (1.0, -8), (1.75, -8), (1.7500001, -7), (0.0, 0), (2.0 ** -140, -126), (3e38, 120)):
        x = torch.zeros(64, dtype=torch.float32)
        x[3] = -largest
        codes, byte = quantise_q8(x)
        assert int(byte) - 127 == power, (largest, int(byte) - 127)
    x = torch.randn(500, 128, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.linspace(-60, 60, 500))[:, None]
    codes, byte = quantise_q8(x)
    held = codes.view(E4M3).double() * torch.exp2(byte.double() - 127)[:, None]
    step = torch.maximum(x.double().abs() * 2.0 ** -4, torch.exp2(byte.double() - 127)[:, None] * 2.0 ** -10)
    assert ((held - x.double()).abs() <= step).all()
    x[7, 5], x[8, 6] = float("nan"), float("inf")
    again, byte2 = quantise_q8(x)
    gone = torch.isnan(again.view(E4M3).float())
    assert gone.sum() == 2 and gone[7, 5] and gone[8, 6]


# -- steps to attend in -----------------------------------------------------------------------------------------------------

def _step(rows, heads, kv, d, page, *, seed=0, shared=(), dtype=torch.bfloat16, q8=True, device="cpu", spare=3, gap=0):
    """rows: (tokens already held, query tokens); shared: (first row, last row, prefix tokens). Pages lie about the pool in any
    order, slots too; what no row holds is NaN."""
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    counts, lens = np.array([n for _, n in rows]), np.array([s + n for s, n in rows])
    need = [-(-int(n) // page) for n in lens]
    wide = max(need + [1]) + 1
    total = sum(need) + spare
    order = list(rng.permutation(total))
    slots = rng.permutation(len(rows) + 2)[: len(rows)]
    table = np.full((len(rows) + 2, wide), total, dtype=np.int64)       # the null page is the last one
    for i, n in enumerate(need):
        table[slots[i], :n] = [order.pop() for _ in range(n)]
    for lo, hi, prefix in shared:
        whole = -(-prefix // page)
        for i in range(lo + 1, hi + 1):
            if prefix % page:                                           # the page in which the prefix ends is copied
                table[slots[i], : whole - 1] = table[slots[lo], : whole - 1]
            else:
                table[slots[i], :whole] = table[slots[lo], :whole]
    n_pages = total + 1
    k = torch.randn(n_pages, kv, page, d, generator=g) * torch.exp(0.6 * torch.randn(n_pages, kv, page, 1, generator=g))
    v = torch.randn(n_pages, kv, d, page, generator=g) * torch.exp(0.6 * torch.randn(n_pages, kv, 1, page, generator=g))
    for lo, hi, prefix in shared:
        if prefix % page:
            at = prefix // page
            for i in range(lo + 1, hi + 1):
                k[table[slots[i], at], :, : prefix % page] = k[table[slots[lo], at], :, : prefix % page]
                v[table[slots[i], at], :, :, : prefix % page] = v[table[slots[lo], at], :, :, : prefix % page]
    held = torch.zeros(n_pages, page, dtype=torch.bool)
    for i, n in enumerate(lens):
        pos = np.arange(n)
        held[table[slots[i], pos // page], pos % page] = True
    k[~held[:, None, :].expand(n_pages, kv, page)] = float("nan")
    v.transpose(2, 3)[~held[:, None, :].expand(n_pages, kv, page)] = float("nan")
    i32 = lambda a: torch.as_tensor(np.asarray(a, dtype=np.int32)).to(device)              # noqa: E731
    dec, chk = np.flatnonzero(counts == 1), np.flatnonzero(counts > 1)
    attn = AttnRows(slots=i32(slots), lens=i32(lens), query_start=i32(np.concatenate([[0], np.cumsum(counts)])), decode_rows=i32(dec),
                    chunk_rows=i32(chk), n_decode=len(dec), n_chunk=len(chk), max_decode_len=int(lens[dec].max()) if len(dec) else 0,
                    max_chunk_query=int(counts[chk].max()) if len(chk) else 0, max_chunk_len=int(lens[chk].max()) if len(chk) else 0, in_order=len(chk) == 0)
    q = (torch.randn(int(counts.sum()), heads, d, generator=g) * 1.5).to(dtype).to(device)
    if q8:
        kc, ke = quantise_q8(k)
        vc, ve = quantise_q8(v.transpose(2, 3))
        pages = torch.stack((kc.reshape(n_pages, kv, -1), vc.transpose(2, 3).reshape(n_pages, kv, -1)), 1)
        scales = torch.stack((ke, ve), 1)
        if gap:                                                         # a page's codes and scales in one piece of a wider row
            both = torch.zeros(n_pages, pages[0].numel() + scales[0].numel() + gap, dtype=torch.uint8)
            both[:, : pages[0].numel()] = pages.reshape(n_pages, -1)
            both[:, pages[0].numel(): pages[0].numel() + scales[0].numel()] = scales.reshape(n_pages, -1)
            both = both.to(device)
            pages = both[:, : pages[0].numel()].view(pages.shape)
            scales = both[:, pages[0].numel(): pages[0].numel() + scales[0].numel()].view(scales.shape)
        pages, scales = pages.to(device).view(E4M3), scales.to(device).view(E8M0)
    else:
        pages, scales = torch.stack((k.reshape(n_pages, kv, -1), v.reshape(n_pages, kv, -1)), 1).to(dtype).to(device), None
    prefix = None
    if shared:
        start = [lo for lo, _, _ in shared] + [shared[-1][1] + 1]
        assert all(shared[i][1] + 1 == shared[i + 1][0] for i in range(len(shared) - 1))
        prefix = SharedPrefix(i32(start), i32([p for _, _, p in shared]), len(shared),
                              int(max(counts[lo: hi + 1].sum() for lo, hi, _ in shared)), max(p for _, _, p in shared))
    return q, pages, scales, i32(table), attn, prefix


def _want(q, pages, scales, table, rows, page, scale, window=0, sink=None):
    """softmax(scale q k^T) v in 64 bits, and beside it sum_j w_j |v_j| and the largest sum_d |q_d k_d| a query meets: what the
    bound is made of. Keys that a query does not see take no part, whatever they hold."""
    d = q.shape[2]
    if scales is not None:
        k, v = dequantise_q8(pages.cpu(), scales.cpu(), page)
    else:
        n, _, hkv, wide = pages.shape
        k, v = pages[:, 0].cpu().float().reshape(n, hkv, page, d), pages[:, 1].cpu().float().reshape(n, hkv, d, page)
    hkv = k.shape[1]
    group = q.shape[1] // hkv
    out, size, dots = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    starts, q = rows.query_start.tolist(), q.double().cpu()
    for b, (slot, n) in enumerate(zip(rows.slots.tolist(), rows.lens.tolist())):
        lo, hi = starts[b], starts[b + 1]
        at = table[slot, : -(-n // page)].long().cpu()
        kk = k[at].transpose(1, 2).reshape(-1, hkv, d)[:n].double()
        vv = v[at].permute(0, 3, 1, 2).reshape(-1, hkv, d)[:n].double()
        for i in range(lo, hi):
            pos = n - (hi - lo) + i - lo
            first = 0 if window == 0 else max(0, pos - window + 1) if window > 0 else max(0, pos) // -window * -window
            if pos < first:
                continue
            for head in range(q.shape[1]):
                ks, vs = kk[first: pos + 1, head // group], vv[first: pos + 1, head // group]
                x = ks @ q[i, head] * scale
                top = x.max()
                e = torch.exp(x - top)
                total = e.sum() + (torch.exp(sink[head].double().cpu() - top) if sink is not None else 0.0)
                out[i, head] = (e / total) @ vs
                size[i, head] = (e / total) @ vs.abs()
                dots[i, head] = (ks.abs() @ q[i, head].abs()).max() * scale
    return out, size, dots


def _bound(want, size, dots, d, keys, dtype):
    """By what a result may be off. A score is a sum of d products in float32 (exact products: off by at most d 2^-24 of the sum
    of their sizes), taken times scale log2(e) (2^-23 more) into exp2 (2^-22 of its result, the instruction's own bound beside the
    rounding of its argument): a weight moves by twice that at most, above and below the fraction's line. Sums over the keys
    are in float32: keys 2^-24. A weight is rounded once to bfloat16 (2^-8), or split in three (2^-24 is left), the result once to its type."""
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    score = dots * (d + 4) * 2.0 ** -24
    return size * (u + 2 * score + 2 * keys * 2.0 ** -24 + 2.0 ** -20) + u * want.abs()


def _check(got, q, pages, scales, table, rows, page, scale, window=0, sink=None):
    want, size, dots = _want(q, pages, scales, table, rows, page, scale, window, sink)
    keys = int(rows.lens.max())
    off, most = (got.double().cpu() - want).abs(), _bound(want, size, dots, q.shape[2], keys, q.dtype)
    assert got.dtype == q.dtype and got.shape == q.shape
    assert torch.isfinite(got).all() and (off <= most).all(), f"up to {(off / most.clamp(min=1e-300)).max().item()} of the bound"


STEPS = [
    # (rows, heads, kv heads, head size, page, window): one key, one page less and more, a tile of 64 less and more, several rows
    ([(0, 1)], 4, 1, 64, 16, 0),
    ([(15, 1), (16, 1), (62, 1), (63, 1), (64, 1), (200, 1)], 8, 2, 128, 16, 0),
    ([(300, 1), (7, 1), (1000, 1)], 5, 1, 128, 32, 0),                       # five heads on one
    ([(700, 1), (31, 1)], 16, 1, 256, 48, 0),                                # pages that no power of two is
    ([(129, 1)] * 3, 20, 1, 64, 64, 0),                                      # more heads a group than a tile has columns
    ([(500, 1), (40, 1)], 8, 2, 128, 16, 50),                                # a window
    ([(500, 1), (40, 1), (130, 1)], 8, 2, 128, 16, -64),                     # chunks
    ([(100, 3), (5, 1), (0, 2), (640, 5)], 8, 2, 128, 16, 0),                # drafted tokens beside decode rows
    ([(90, 7), (0, 33)], 5, 1, 64, 16, 20),
    ([(0, 130), (64, 65), (300, 1), (11, 6)], 8, 4, 128, 32, 0),             # prompts, portions
    ([(100, 70), (0, 40)], 4, 2, 256, 16, 0),
    ([(70, 90)], 14, 2, 128, 16, -32),
    ([(0, 64), (31, 33), (200, 64)], 2, 2, 64, 48, 0),                       # as many columns as the kernel of few takes, and less
    ([(3, 150), (0, 65)], 1, 1, 64, 16, 40),
    ([(2000, 66), (70, 2)], 4, 1, 128, 32, 0),                               # a short portion behind a long context
    ([(40, 1), (33, 2)], 70, 1, 64, 16, 0),                                  # more heads on one than the kernel of few columns takes
]


def test_plain_forms_agree():
    """The twin and the 64-bit definition, and the twin's write with the format."""
    for rows, heads, kv, d, page, window in STEPS[:6]:
        q, pages, scales, table, attn, _ = _step(rows, heads, kv, d, page)
        clean = pages.view(torch.uint8).clone()
        clean[(clean & 0x7f) == 0x7f] = 0
        got = PLAIN.paged_attention_q8(q, clean.view(E4M3), scales, table, attn, page, d ** -0.5, window)
        _check(got, q, pages, scales, table, attn, page, d ** -0.5, window)


# -- what is refused, without a GPU -----------------------------------------------------------------------------------------

class Refusing(ContinuationOps):
    """The checks alone: tensors may lie anywhere, nothing is launched."""

    class lib:
        holon_kv_write_q8 = holon_kv_read_q8 = holon_cache_attention = holon_verify_drafts = holon_qk_norm_rope_write_q8 = None
        holon_cache_attention_room = staticmethod(lambda *a: 0)
        holon_verify_drafts_room = staticmethod(lambda *a: 16)

    def __init__(self):
        self.launched = []

    def _place(self, what, t):
        return -1

    @staticmethod
    def _stream_of(device):
        return 0

    def _call(self, fn, *args):
        self.launched.append(args)


def test_refused_on_the_cpu():
    with pytest.raises(KernelError, match="GPU tensor"):
        ContinuationOps().kv_read_q8(torch.zeros(2, 2, 1, 1024, dtype=torch.uint8), torch.zeros(2, 2, 1, 16, dtype=torch.uint8),
                                     torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 16)


def test_refused_caches_and_rows():
    ops = Refusing()
    q, pages, scales, table, rows, _ = _step([(20, 1), (3, 2)], 4, 2, 64, 16)
    k = torch.randn(5, 2, 64).bfloat16()
    at = torch.zeros(5, dtype=torch.int32)
    ops.kv_write_q8(k, k, pages, scales, at, at, 16)
    ops.kv_write_q8(k.float(), k.float(), pages.view(torch.uint8), scales.view(torch.uint8), at, at, 16)
    wide = torch.randn(5, 384).bfloat16()
    ops.kv_write_q8(wide[:, :128].view(5, 2, 64), wide[:, 128:256].view(5, 2, 64), pages, scales, at, at, 16)
    ops.kv_read_q8(pages, scales, at, at, 16, torch.float32)
    ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1)
    assert len(ops.launched) == 5
    for bad in (lambda: ops.kv_write_q8(k, k.float(), pages, scales, at, at, 16),
                lambda: ops.kv_write_q8(k.half(), k.half(), pages, scales, at, at, 16),
                lambda: ops.kv_write_q8(k[:, :1], k[:, :1], pages, scales, at, at, 16),
                lambda: ops.kv_write_q8(k, wide[:, :128].view(5, 2, 64), pages, scales, at, at, 16),
                lambda: ops.kv_write_q8(k, k, pages, scales, at.long(), at, 16),
                lambda: ops.kv_write_q8(k, k, pages, scales, at[:4], at, 16),
                lambda: ops.kv_write_q8(k, k, pages, scales[:, :, :, :8], at, at, 16),
                lambda: ops.kv_write_q8(k, k, pages.view(torch.int8), scales, at, at, 16),
                lambda: ops.kv_write_q8(k, k, pages, scales, at, at, 8),
                lambda: ops.kv_write_q8(k, k, pages[:, :, :, :512], scales, at, at, 16),
                lambda: ops.kv_read_q8(pages, scales, at, at, 16, torch.float16),
                lambda: ops.kv_read_q8(pages.transpose(1, 2), scales, at, at, 16),
                lambda: ops.paged_attention_q8(q.half(), pages, scales, table, rows, 16, 0.1),
                lambda: ops.paged_attention_q8(q[:, :3], pages, scales, table, rows, 16, 0.1),
                lambda: ops.paged_attention_q8(q.transpose(0, 1), pages, scales, table, rows, 16, 0.1),
                lambda: ops.paged_attention_q8(q, pages, scales, table.long(), rows, 16, 0.1),
                lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.0),
                lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, float("nan")),
                lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1, sink=torch.zeros(3)),
                lambda: ops.prefix_attention(q, pages, table, rows, None, 16, 0.1)):      # 8-bit pages without scales
        with pytest.raises(KernelError):
            bad()
    small = torch.zeros(2, 2, 1, 16 * 96, dtype=torch.uint8), torch.zeros(2, 2, 1, 16, dtype=torch.uint8)
    with pytest.raises(KernelError, match="heads of 64"):
        ops.kv_read_q8(*small, at, at, 16)
    odd = torch.zeros(2, 2, 1, 8 * 64, dtype=torch.uint8), torch.zeros(2, 2, 1, 8, dtype=torch.uint8)
    with pytest.raises(KernelError):
        ops.kv_read_q8(*odd, at, at, 8)
    shifted = torch.zeros(4 * 2048 + 8, dtype=torch.uint8)[8:].view(4, 2, 1, 1024)
    with pytest.raises(KernelError, match="borders of 16"):
        ops.kv_read_q8(shifted, torch.zeros(4, 2, 1, 16, dtype=torch.uint8), at, at, 16)
    assert len(ops.launched) == 5


def test_refused_bounds_past_32_bits():
    ops = Refusing()
    q, pages, scales, table, rows, prefix = _step([(40, 1), (41, 3)], 4, 2, 64, 16, shared=[(0, 1, 32)])
    more = lambda x, **kw: type(x)(**{**vars(x), **kw})                                             # noqa: E731
    ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1, 2 ** 31 - 1)
    for bad in (lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1, 2 ** 31),
                lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1, -2 ** 31 - 1),
                lambda: ops.paged_attention_q8(q, pages, scales, table, rows, 16, 1e39),
                lambda: ops.paged_attention_q8(q, pages, scales, table, more(rows, max_decode_len=2 ** 31), 16, 0.1),
                lambda: ops.paged_attention_q8(q, pages, scales, table, more(rows, max_chunk_query=2 ** 40), 16, 0.1),
                lambda: ops.prefix_attention(q, pages, table, rows, more(prefix, max_len=2 ** 31), 16, 0.1, scales),
                lambda: ops.prefix_attention(q, pages, table, rows, more(prefix, max_queries=2.5), 16, 0.1, scales)):
        with pytest.raises(KernelError, match="32 bits"):
            bad()
    assert len(ops.launched) == 1


def test_refused_caches_without_scales():
    """A bfloat16 cache has pages of the same shape: without scales it is no 8-bit cache."""
    ops, at = Refusing(), torch.zeros(5, dtype=torch.int32)
    k, pages = torch.randn(5, 2, 64).bfloat16(), torch.zeros(3, 2, 2, 1024).bfloat16()
    for bad in (lambda: ops.kv_write_q8(k, k, pages, None, at, at, 16), lambda: ops.kv_read_q8(pages, None, at, at, 16),
                lambda: ops.qk_norm_rope_write_q8(torch.zeros(5, 512).bfloat16(), 4, 2, 64, None, None, 1e-6, None, at, pages, None, at, at, 16)):
        with pytest.raises(KernelError, match="an 8-bit cache has scales"):
            bad()
    assert not ops.launched


def test_refused_projections():
    ops = Refusing()
    at, w, table = torch.zeros(5, dtype=torch.int32), torch.ones(64).bfloat16(), torch.zeros(9, 64)
    pages, scales = torch.zeros(3, 2, 2, 1024, dtype=torch.uint8), torch.zeros(3, 2, 2, 16, dtype=torch.uint8)
    qkv = torch.zeros(5, 512).bfloat16()
    good = dict(qkv=qkv, heads=4, kv_heads=2, head_dim=64, q_weight=w, k_weight=w, eps=1e-6, table=table, positions=at, pages=pages, scales=scales,
                write_page=at, write_off=at, page_size=16)
    ops.qk_norm_rope_write_q8(**good)
    ops.qk_norm_rope_write_q8(**{**good, "q_weight": None, "k_weight": None, "table": None, "positions": None})
    for name, bad in (("qkv", qkv.half()), ("qkv", torch.zeros(512, 5).bfloat16().t()), ("qkv", qkv[:, :448]), ("heads", 3), ("kv_heads", 1),
                      ("head_dim", 128), ("q_weight", None), ("k_weight", w.float()), ("k_weight", w[:32]), ("table", table[:, :32]),
                      ("table", table.bfloat16()), ("table", table[:0]), ("positions", at.long()), ("positions", at[:4]), ("scales", scales[:2]),
                      ("write_page", at[:4]), ("write_off", at.float()), ("page_size", 32)):
        with pytest.raises(KernelError):
            ops.qk_norm_rope_write_q8(**{**good, name: bad})
    assert len(ops.launched) == 2


def test_refused_prefixes():
    ops = Refusing()
    q, pages, _, table, rows, prefix = _step([(40, 1), (41, 1)], 4, 2, 64, 16, shared=[(0, 1, 32)], q8=False)
    ops.prefix_attention(q, pages, table, rows, prefix, 16, 0.1)
    with pytest.raises(KernelError):                                    # the float32 path keeps paged_attention
        ops.prefix_attention(q.float(), pages.float(), table, rows, prefix, 16, 0.1)
    with pytest.raises(KernelError, match="group_start"):
        ops.prefix_attention(q, pages, table, rows, SharedPrefix(prefix.group_start[:1], prefix.lens, 1, 2, 32), 16, 0.1)
    with pytest.raises(KernelError, match="prefix lens"):
        ops.prefix_attention(q, pages, table, rows, SharedPrefix(prefix.group_start, prefix.lens.float(), 1, 2, 32), 16, 0.1)
    assert len(ops.launched) == 1


def test_refused_drafts():
    ops = Refusing()
    n, b = 7, 2
    good = dict(logits=torch.zeros(n, 50), drafted=torch.zeros(n, dtype=torch.int32), draft_probs=torch.zeros(n, 50), accept=torch.zeros(n),
                draw=torch.zeros(b), temperature=torch.ones(b), start=torch.tensor([0, 3, 7], dtype=torch.int32), most=4)
    ops.verify_drafts(**good)
    for name, bad in (("logits", torch.zeros(n, 50).bfloat16()), ("logits", torch.zeros(50, n).t()), ("drafted", torch.zeros(n).long()),
                      ("draft_probs", torch.zeros(n, 49)), ("draft_probs", torch.zeros(n, 50).double()), ("accept", torch.zeros(n - 1)),
                      ("draw", torch.zeros(b + 1)), ("temperature", torch.ones(b).double()), ("start", torch.zeros(b, dtype=torch.int32)),
                      ("most", 64), ("most", -1)):
        with pytest.raises(KernelError):
            ops.verify_drafts(**{**good, name: bad})
    assert len(ops.launched) == 1


# -- the kernels --------------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def hip():
    from holon_amd.kernels import load_hip
    return load_hip()


gpu = pytest.mark.gpu


def _blank(n, kv, page, d, seed, gap=0):
    """A pool full of other bytes: whatever a write leaves alone shows."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = 2 * kv * page * d, 2 * kv * page
    both = torch.randint(0, 256, (n, codes + scales + gap), generator=g, dtype=torch.uint8)
    return both, lambda x: (x[:, :codes].view(n, 2, kv, page * d), x[:, codes: codes + scales].view(n, 2, kv, page))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("t", "kv", "d", "page", "gap"), [(1, 1, 64, 16, 0), (1, 8, 128, 16, 0), (8, 8, 128, 16, 16), (37, 3, 128, 32, 0),
                                                           (100, 2, 256, 16, 0), (33, 1, 64, 48, 32), (513, 4, 128, 64, 0), (16, 2, 256, 32, 0)])
def test_write_and_read_back(hip, t, kv, d, page, gap, dtype):
    """Bytes equal the format's wherever a token goes, and nothing else of the pool changes; what is read back is what they stand for."""
    g = torch.Generator().manual_seed(t + d)
    rows = (torch.randn(t, 3 * kv * d, generator=g) * torch.exp(3 * torch.randn(t, 1, generator=g))).to(dtype)
    rows[0, 0], rows[-1, -1], rows[t // 2, kv * d] = float("nan"), float("inf"), float("-inf")
    rows[t // 3, : kv * d] = 0
    rows[-1, kv * d: 2 * kv * d] = 2.0 ** -133                     # bfloat16's smallest
    k, v = rows[:, kv * d: 2 * kv * d].view(t, kv, d), rows[:, 2 * kv * d:].view(t, kv, d)       # columns of wider rows
    n = t // page + 9
    for run in ("in order", "anywhere", "some nowhere"):
        rng = np.random.default_rng(t)
        if run == "in order":                                     # from the middle of a page on
            order, first = rng.permutation(n), min(5, page - 1)
            at = np.arange(t) + first
            wp, wo = order[at // page], at % page
        else:
            at = rng.permutation(n * page)[:t]
            wp, wo = at // page, at % page
            if run == "some nowhere":
                wp, wo = wp.copy(), wo.copy()
                wp[::3], wo[1::5] = np.where(np.arange(t)[::3] % 2, -1, n), np.where(np.arange(t)[1::5] % 2, -7, page)
        wp, wo = (torch.as_tensor(x.astype(np.int32)) for x in (wp, wo))
        both, views = _blank(n, kv, page, d, t, gap)
        want = both.clone()
        PLAIN.kv_write_q8(k, v, *views(want), wp, wo, page)
        got = both.cuda()
        hip.kv_write_q8(rows.cuda()[:, kv * d: 2 * kv * d].view(t, kv, d), rows.cuda()[:, 2 * kv * d:].view(t, kv, d),
                        *views(got), wp.cuda(), wo.cuda(), page)
        a, b = views(want), views(got.cpu())
        nan = (a[0] & 0x7f) == 0x7f
        assert torch.equal((b[0] & 0x7f) == 0x7f, nan) and torch.equal(a[0][~nan], b[0][~nan]), run
        assert torch.equal(a[1], b[1]) and torch.equal(got.cpu()[:, want.shape[1] - gap:], both[:, want.shape[1] - gap:]), run
        pages, scales = views(got)
        for into in (torch.bfloat16, torch.float32):
            seen = hip.kv_read_q8(pages, scales, wp.cuda(), wo.cuda(), page, into)
            true = PLAIN.kv_read_q8(*views(got.cpu()), wp, wo, page, into)
            for x, y in zip(seen, true):
                assert x.dtype == into and torch.equal(torch.isnan(x.cpu()), torch.isnan(y))
                assert torch.equal(torch.nan_to_num(x.cpu(), 0.0), torch.nan_to_num(y, 0.0)), (run, into)


@gpu
@pytest.mark.parametrize(("d", "page"), [(64, 16), (128, 48), (256, 32)])
@pytest.mark.parametrize("holes", [0.0, 0.02])
def test_stretches_that_begin_and_end_anywhere(hip, d, page, holes):
    """Portions of every length up to 35 from every place of a page on, one behind the other: however a stretch of neighbours meets
    the blocks' borders and those of 16 tokens, exactly its bytes are written, and the same come back."""
    rng = np.random.default_rng(d)
    portions = [(first, n) for first in range(page) for n in rng.permutation(np.arange(1, 36))[:12]]
    n = sum(-(-(first + more) // page) for first, more in portions)
    order, at, wp, wo = rng.permutation(n), 0, [], []
    for first, more in portions:
        place = at * page + first + np.arange(more)
        wp.append(order[place // page])
        wo.append(place % page)
        at += -(-(first + more) // page)
    wp, wo = np.concatenate(wp), np.concatenate(wo)
    wp[rng.random(len(wp)) < holes] = -1
    wp, wo = (torch.as_tensor(x.astype(np.int32)) for x in (wp, wo))
    k, v = torch.randn(2, len(wp), 2, d, generator=torch.Generator().manual_seed(d))
    both, views = _blank(n, 2, page, d, d)
    want, got = both.clone(), both.cuda()
    PLAIN.kv_write_q8(k, v, *views(want), wp, wo, page)
    hip.kv_write_q8(k.cuda(), v.cuda(), *views(got), wp.cuda(), wo.cuda(), page)
    assert torch.equal(got.cpu(), want)
    for x, y in zip(hip.kv_read_q8(*views(got), wp.cuda(), wo.cuda(), page, torch.float32),
                    PLAIN.kv_read_q8(*views(want), wp, wo, page, torch.float32)):
        assert torch.equal(x.cpu(), y)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("t", "heads", "kv", "d", "page", "norm", "turn"),
                         [(1, 1, 1, 64, 16, True, True), (8, 32, 8, 128, 16, True, True), (37, 6, 2, 64, 32, True, True), (100, 4, 2, 256, 16, True, True),
                          (70, 4, 4, 128, 48, False, True), (33, 6, 3, 64, 16, True, False), (50, 5, 1, 256, 16, False, False), (513, 8, 2, 128, 16, True, True)])
def test_projections_normed_turned_and_written(hip, t, heads, kv, d, page, norm, turn, dtype):
    """The merged projection in one kernel. Roundings of `dtype` may fall the other way (a norm's sum is in another order, a rotation's
    products may be fused). The norm's moves a value by eps of itself, which turned is eps of the pair's size |(a, b)| at most (Cauchy),
    the rotation's own by eps more: 2 eps of that size, and 2^-20 for the arithmetic in 32 bits. What the cache holds of a key is off
    by 2^-4 of the value or 2^-10 of its row's power besides, on either side. Values: exactly."""
    g = torch.Generator().manual_seed(t + d)
    qkv = (torch.randn(t, (heads + 2 * kv) * d, generator=g) * torch.exp(torch.randn(t, 1, generator=g))).to(dtype)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)) if norm else (None, None)
    angle = torch.arange(600.0)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    table = torch.cat((angle.cos(), angle.sin()), 1).contiguous() if turn else None
    rng = np.random.default_rng(t)
    n = t // page + 4
    place = rng.permutation(n)[(np.arange(t) + 5) // page] * page + (np.arange(t) + 5) % page
    place[t // 2 + 1: t // 2 + 3] = -1
    wp, wo, pos = (torch.as_tensor(x.astype(np.int32)) for x in (place // page, place % page, rng.integers(0, 600, t)))
    both, views = _blank(n, kv, page, d, t)
    want, got = both.clone(), both.cuda()
    wq = PLAIN.qk_norm_rope_write_q8(qkv, heads, kv, d, qw, kw, 1e-6, table, pos, *views(want), wp, wo, page)
    on = lambda x: None if x is None else x.cuda()                                                  # noqa: E731
    gq = hip.qk_norm_rope_write_q8(on(qkv), heads, kv, d, on(qw), on(kw), 1e-6, on(table), on(pos), *views(got), wp.cuda(), wo.cuda(), page)
    assert gq.dtype == dtype and gq.shape == (t, heads, d)
    gq, wq = gq.double().cpu(), wq.double()
    size = torch.hypot(wq[..., : d // 2], wq[..., d // 2:]).repeat(1, 1, 2)
    off = 2 * torch.finfo(dtype).eps + 2 ** -20
    assert ((gq - wq).abs() <= off * size).all()
    (a, sa), (b, sb) = views(want), views(got.cpu())
    assert torch.equal(a[:, 1], b[:, 1]) and torch.equal(sa[:, 1], sb[:, 1])
    there = torch.zeros(n, page, dtype=torch.bool)
    there[wp[wp >= 0].long(), wo[wp >= 0].long()] = True
    rows = lambda x: x[:, 0].view(n, kv, page, d).transpose(1, 2)                                   # noqa: E731
    assert torch.equal(rows(a)[~there], rows(b)[~there]) and torch.equal(sa[:, 0].transpose(1, 2)[~there], sb[:, 0].transpose(1, 2)[~there])
    x, y = (dequantise_q8(c, s, page)[0].double().transpose(1, 2)[there] for c, s in ((a, sa), (b, sb)))
    power = torch.exp2(torch.maximum(sa[:, 0], sb[:, 0]).double() - 127).transpose(1, 2)[there][..., None]
    size = torch.hypot(x[..., : d // 2], x[..., d // 2:]).repeat(1, 1, 2) * (1 + 2 ** -3) + 2.0 ** -9 * power
    assert ((x - y).abs() <= off * size + 2.0 ** -4 * (1 + 2 ** -3) * (x.abs() + y.abs()) + 2.0 ** -9 * power).all()
    assert (x != y).double().mean() < 0.02              # (2^-20 passes a border between steps of 2^-8 once in 2^11)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attention_over_the_8_bit_cache(hip, step, dtype):
    rows, heads, kv, d, page, window = STEPS[step]
    print(f"step {step} {dtype}", flush=True)
    args = _step(rows, heads, kv, d, page, seed=step, dtype=dtype, device="cuda", gap=16 * (step % 3))[:5]
    q, pages, scales, table, attn = args
    got = hip.paged_attention_q8(q, pages, scales, table, attn, page, d ** -0.5, window)
    _check(got, q, pages, scales, table, attn, page, d ** -0.5, window)
    sink = torch.linspace(-2, 3, heads).cuda()
    got = hip.paged_attention_q8(q, pages, scales, table, attn, page, d ** -0.5, window, sink)
    _check(got, q, pages, scales, table, attn, page, d ** -0.5, window, sink)


@gpu
def test_long_contexts_are_cut_and_joined(hip):
    for rows, heads, kv, d, dtype in (([(5000, 1)], 4, 1, 128, torch.bfloat16), ([(9000, 1), (37, 1)], 2, 1, 64, torch.float32),
                                      ([(6000, 4), (100, 2)], 4, 1, 128, torch.bfloat16), ([(4100, 1)], 2, 1, 256, torch.bfloat16),
                                      # by lengths: one long row among short ones, and rows of no key beside it
                                      ([(9000, 1)] + [(n, 1) for n in (0, 63, 64, 300, 5000, 7, 1200)], 8, 2, 128, torch.bfloat16),
                                      ([(4200, 1), (4500, 1), (1, 1)] * 11, 20, 1, 64, torch.bfloat16), ([(4300, 1), (40, 1), (90, 3)], 2, 1, 256, torch.float32)):
        q, pages, scales, table, attn, _ = _step(rows, heads, kv, d, 16, seed=3, dtype=dtype, device="cuda")
        got = hip.paged_attention_q8(q, pages, scales, table, attn, 16, d ** -0.5)
        _check(got, q, pages, scales, table, attn, 16, d ** -0.5)
        got = hip.paged_attention_q8(q, pages, scales, table, attn, 16, d ** -0.5, 4150)
        _check(got, q, pages, scales, table, attn, 16, d ** -0.5, 4150)


@gpu
@pytest.mark.parametrize(("heads", "kv", "d"), [(71, 1, 64), (130, 2, 128), (66, 1, 256)])
@pytest.mark.parametrize("q8", [True, False])
def test_more_heads_on_one_behind_long_contexts(hip, heads, kv, d, q8):
    """More than 64 heads on one kv head, several decode rows of different lengths, some past 4,096 keys: alone, and beside a portion."""
    for rows in ([(4500, 1), (30, 1), (0, 1)], [(4200, 1), (6, 3), (4097, 1)]):
        print(f"{heads} over {kv} of {d}, {rows}", flush=True)
        q, pages, scales, table, attn, _ = _step(rows, heads, kv, d, 16, seed=heads, q8=q8, device="cuda")
        got = hip.paged_attention_q8(q, pages, scales, table, attn, 16, d ** -0.5) if q8 else hip.prefix_attention(q, pages, table, attn, None, 16, d ** -0.5)
        _check(got, q, pages, scales, table, attn, 16, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("heads", "d"), [(5, 64), (3, 256)])
def test_rows_of_every_kind_are_cut_in_one_call(hip, heads, d, dtype):
    """Decode rows cut by their lengths and rows of a few queries, odd numbers of heads and rows: each kind's partial sums lie on borders."""
    rows = [(5000, 1), (300, 3), (6000, 1), (4100, 5), (7000, 1), (37, 1), (2500, 2)]
    q, pages, scales, table, attn, _ = _step(rows, heads, 1, d, 16, seed=heads, dtype=dtype, device="cuda")
    got = hip.paged_attention_q8(q, pages, scales, table, attn, 16, d ** -0.5)
    _check(got, q, pages, scales, table, attn, 16, d ** -0.5)


BESIDE = [
    # (rows, heads, kv heads, head size, page, window): decode rows of short contexts and long beside portions, rows of a few queries between
    ([(5000, 1), (37, 1), (9000, 1), (10, 1), (200, 70)], 8, 2, 128, 16, 0),
    ([(0, 1), (600, 1), (0, 3), (100, 40), (5, 20)], 8, 2, 64, 16, 0),
    ([(700, 1), (31, 1), (100, 40)], 16, 1, 256, 48, 0),
    ([(4500, 1), (3, 1), (4200, 60)], 4, 1, 64, 32, 0),
    ([(300, 1), (50, 1), (90, 80), (0, 65)], 5, 1, 128, 16, 100),
    ([(3000, 1), (100, 1)] + [(7 * i, 65) for i in range(33)], 32, 8, 64, 16, 0),                # blocks of eight waves
    ([(4300, 1), (1, 1), (2500, 1)] + [(3 * i, 65) for i in range(33)], 32, 8, 128, 16, -64),
    ([(40, 1), (2000, 1), (33, 90)], 20, 1, 128, 16, 0),                                          # more heads on one than a tile has columns
]


@gpu
@pytest.mark.parametrize("case", range(len(BESIDE)))
def test_decode_rows_beside_portions(hip, case):
    """One launch for a step's decode rows and its portions: over codes, and over the bfloat16 cache."""
    rows, heads, kv, d, page, window = BESIDE[case]
    print(f"case {case}", flush=True)
    q, pages, scales, table, attn, _ = _step(rows, heads, kv, d, page, seed=case, device="cuda")
    got = hip.paged_attention_q8(q, pages, scales, table, attn, page, d ** -0.5, window)
    _check(got, q, pages, scales, table, attn, page, d ** -0.5, window)
    assert torch.equal(hip.paged_attention_q8(q, pages, scales, table, attn, page, d ** -0.5, window), got)
    q, pages, _, table, attn, _ = _step(rows, heads, kv, d, page, seed=case, q8=False, device="cuda")
    _check(hip.prefix_attention(q, pages, table, attn, None, page, d ** -0.5), q, pages, None, table, attn, page, d ** -0.5)


@gpu
def test_kinds_of_rows_in_launches_of_their_own(hip):
    """Steps whose decode rows and portions are not joined (heads of 256 over a bfloat16 cache, a long portion): each kind of rows gets
    what it gets alone, and they are joined where that is little."""
    for portion, together in (((8000, 700), False), ((100, 70), True)):
        rows = [(4000, 1), (37, 1), portion, (900, 1)]
        print(rows, flush=True)
        q, pages, _, table, attn, _ = _step(rows, 16, 2, 256, 16, seed=1, q8=False, device="cuda")
        run = lambda q, attn: hip.prefix_attention(q, pages, table, attn, None, 16, 256 ** -0.5)     # noqa: E731
        got, alone = run(q, attn), []
        starts = attn.query_start.tolist()
        for kind in ([0, 1, 3], [2]):
            at = torch.tensor(kind, device="cuda")
            tokens = torch.cat([torch.arange(starts[i], starts[i + 1]) for i in kind]).cuda()
            count = attn.query_start.diff()[at]
            start, order = torch.cat((count[:1] * 0, count.cumsum(0))).int(), torch.arange(len(kind), dtype=torch.int32, device="cuda")
            none, decode = order[:0], len(kind) == 3
            mine = AttnRows(attn.slots[at], attn.lens[at], start, order if decode else none, none if decode else order, 3 * decode, 1 - decode,
                            attn.max_decode_len * decode, attn.max_chunk_query * (1 - decode), attn.max_chunk_len * (1 - decode))
            alone.append((got[tokens], run(q[tokens], mine)))
        assert all(torch.equal(x, y) for x, y in alone) or together
        if together:
            _check(got, q, pages, None, table, attn, 16, 256 ** -0.5)


@gpu
def test_nothing_to_do(hip):
    """Calls of no token, no row, no request: results of their shapes, and nothing is touched."""
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    both, views = _blank(3, 2, 16, 64, 0)
    got = both.cuda()
    pages, scales = views(got)
    k = torch.zeros(0, 2, 64, device="cuda")
    hip.kv_write_q8(k, k, pages, scales, none, none, 16)
    assert all(x.shape == (0, 2, 64) for x in hip.kv_read_q8(pages, scales, none, none, 16))
    q = hip.qk_norm_rope_write_q8(torch.zeros(0, 512, device="cuda"), 4, 2, 64, None, None, 1e-6, None, None, pages, scales, none, none, 16)
    assert q.shape == (0, 4, 64) and torch.equal(got.cpu(), both)
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = AttnRows(none, none, start, none, none, 0, 0, 0, 0, 0)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    assert hip.paged_attention_q8(q, pages, scales, table, rows, 16, 0.1).shape == (0, 4, 64)
    empty = torch.zeros(0, device="cuda")
    tokens, taken = hip.verify_drafts(torch.zeros(0, 9, device="cuda"), none, None, empty, empty, empty, start, 3)
    assert tokens.shape == (0, 4) and taken.shape == (0,)
    one, starts = torch.full((2,), 0.5, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    tokens, taken = hip.verify_drafts(torch.zeros(0, 9, device="cuda"), none, None, empty, one, one, starts, 3)      # requests of no rows
    assert (tokens == -1).all() and (taken == 0).all()


@gpu
def test_pools_past_32_bits(hip):
    """Pages that lie more than 2^32 bytes into the pool, over both caches: written, read and attended over like any others."""
    heads, kv, d, page = 8, 8, 128, 16
    n, t = (1 << 32) // (2 * kv * page * d) + 200, 100
    pages = torch.empty(n, 2, kv, page * d, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, 2, kv, page, dtype=torch.uint8, device="cuda")
    order = torch.tensor([n - 1, 3, n - 7, n - 150, 0, n - 2, n - 90], dtype=torch.int32)
    at = torch.arange(t)
    wp, wo = order[at // page], (at % page).int()
    k, v = torch.randn(2, t, kv, d, generator=torch.Generator().manual_seed(4)).bfloat16()
    hip.kv_write_q8(k.cuda(), v.cuda(), pages, scales, wp.cuda(), wo.cuda(), page)
    small = torch.zeros(7, 2, kv, page * d, dtype=torch.uint8), torch.zeros(7, 2, kv, page, dtype=torch.uint8)
    low = (at // page).int()
    PLAIN.kv_write_q8(k, v, *small, low, wo, page)
    for x, y in zip(hip.kv_read_q8(pages, scales, wp.cuda(), wo.cuda(), page), PLAIN.kv_read_q8(*small, low, wo, page)):
        assert torch.equal(x.cpu(), y)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)                                             # noqa: E731
    q = torch.randn(71, heads, d, generator=torch.Generator().manual_seed(5)).bfloat16()
    rows = AttnRows(i32(0, 0), i32(t, t), i32(0, 1, 71), i32(0), i32(1), 1, 1, t, 70, t)
    there = AttnRows(*(x.cuda() if torch.is_tensor(x) else x for x in (rows.slots, rows.lens, rows.query_start, rows.decode_rows, rows.chunk_rows)),
                     1, 1, t, 70, t)
    got = hip.paged_attention_q8(q.cuda(), pages, scales, order[None].cuda(), there, page, d ** -0.5)
    _check(got, q, *small, i32(*range(7))[None], rows, page, d ** -0.5)
    del pages, scales
    wide = torch.empty(n // 2 + 200, 2, kv, page * d, dtype=torch.bfloat16, device="cuda")
    order = torch.where(order > 9, order - (n - n // 2 - 200), order).int()
    held = [x.bfloat16() for x in dequantise_q8(*small, page)]
    wide[order.long().cuda()] = torch.stack([x.reshape(7, kv, page * d) for x in held], 1).cuda()
    got = hip.prefix_attention(q.cuda(), wide, order[None].cuda(), there, None, page, d ** -0.5)
    _check(got, q, *small, i32(*range(7))[None], rows, page, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_off_every_border(hip, dtype):
    """Keys, values and weights that begin at an odd element: read one by one, to the same bytes."""
    t, kv, d, page = 40, 2, 128, 16
    g = torch.Generator().manual_seed(8)
    rows = torch.randn(t, 1 + 2 * kv * d, generator=g).to(dtype)
    weights = torch.randn(2, 1 + d, generator=g).to(dtype)
    qkv = torch.randn(t, 4 * d, generator=g).to(dtype)
    at = torch.arange(t, dtype=torch.int32)
    wp, wo = (at // page + 1), at % page
    both, views = _blank(5, kv, page, d, 1)
    want, got = both.clone(), both.cuda()
    split = lambda x: (x[:, 1: 1 + kv * d].view(t, kv, d), x[:, 1 + kv * d:].view(t, kv, d))        # noqa: E731
    PLAIN.kv_write_q8(*split(rows), *views(want), wp, wo, page)
    hip.kv_write_q8(*split(rows.cuda()), *views(got), wp.cuda(), wo.cuda(), page)
    assert torch.equal(got.cpu(), want)
    both, views = _blank(5, 1, page, d, 1)
    at, w = at.cuda(), weights.cuda()
    pools = [both.cuda(), both.cuda()]
    outs = [hip.qk_norm_rope_write_q8(qkv.cuda(), 2, 1, d, a, b, 1e-6, None, None, *views(pool), wp.cuda(), wo.cuda(), page)
            for pool, (a, b) in zip(pools, ((w[0, 1:], w[1, 1:]), (w[0, 1:].clone(), w[1, 1:].clone())))]
    assert torch.equal(*outs) and torch.equal(*pools)


@gpu
def test_a_call_gives_the_same_bits_again(hip):
    """Sums have an order that the step's shapes and lengths decide: with other work between, and from another stream."""
    other = torch.cuda.Stream()
    for rows, shared, heads, kv, d, q8 in (([(9000, 1), (30, 1), (700, 1)], (), 8, 2, 128, True), ([(300, 1)] * 20, [(0, 19, 288)], 8, 2, 128, False),
                                           ([(2000, 300), (40, 5)], (), 4, 1, 128, True)):
        q, pages, scales, table, attn, prefix = _step(rows, heads, kv, d, 16, seed=2, shared=shared, q8=q8, device="cuda")
        run = lambda: hip.prefix_attention(q, pages, table, attn, prefix, 16, d ** -0.5, scales)             # noqa: E731
        first = run()
        torch.randn(1 << 22, device="cuda").sort()
        assert torch.equal(run(), first)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            again = run()
        torch.cuda.current_stream().wait_stream(other)
        assert torch.equal(again, first)


@gpu
def test_recorded_and_replayed(hip):
    """Each operation in a graph, replayed on other inputs of the same shapes, with the program's own work between; two graphs do not
    share what they write."""
    from holon_amd.kernels.hip import capture
    steps = [_step([(9000, 1), (30, 1), (700, 1)], 8, 2, 128, 16, seed=s, device="cuda") for s in (1, 2)]
    groups = [_step([(300, 1)] * 6, 8, 2, 128, 16, seed=s, shared=[(0, 5, 288)], q8=False, device="cuda") for s in (1, 2)]
    judged = [{k: x.cuda() if torch.is_tensor(x) else x for k, x in _drafts([4, 4, 4], 9000, s).items()} for s in (1, 2)]
    k, v = torch.randn(40, 2, 128, device="cuda").bfloat16(), torch.randn(40, 2, 128, device="cuda").bfloat16()
    at = torch.randperm(48)[:40]
    wp, wo = (at // 16).int().cuda(), (at % 16).int().cuda()
    pool = lambda: (torch.zeros(4, 2, 2, 2048, dtype=torch.uint8, device="cuda"), torch.ones(4, 2, 2, 16, dtype=torch.uint8, device="cuda"))   # noqa: E731

    def attend(s):
        q, pages, scales, table, attn, _ = s
        return hip.paged_attention_q8(q, pages, scales, table, attn, 16, 128 ** -0.5)

    def prefixed(s):
        q, pages, _, table, attn, prefix = s
        return hip.prefix_attention(q, pages, table, attn, prefix, 16, 128 ** -0.5)

    def written(kv):
        pages, scales = pool()
        hip.kv_write_q8(*kv, pages, scales, wp, wo, 16)
        return torch.stack(hip.kv_read_q8(pages, scales, wp, wo, 16))

    def tensors(x):
        if torch.is_tensor(x):
            return [x]
        if isinstance(x, dict):
            return [t for y in x.values() for t in tensors(y)]
        if isinstance(x, (list, tuple)):
            return [t for y in x for t in tensors(y)]
        return tensors(vars(x)) if hasattr(x, "__dict__") else []

    import copy
    for op, inputs in ((attend, steps), (prefixed, groups), (lambda s: torch.cat([t.flatten() for t in hip.verify_drafts(**s)]), judged),
                       (written, [(k, v), (v, k)])):
        want = [op(s).clone() for s in inputs]
        held = copy.deepcopy(inputs[0])
        op(held)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with capture(graph):
                out = op(held)
            graphs.append((graph, out))
        for turn in (0, 1, 1, 0, 1):
            for to, src in zip(tensors(held), tensors(inputs[turn]), strict=True):
                if to.shape == src.shape:
                    to.copy_(src)
            assert torch.equal(op(held), want[turn])
            for graph, _ in graphs:
                graph.replay()
            torch.randn(1 << 20, device="cuda").sort()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert torch.equal(out, want[turn]), turn
            assert torch.equal(op(held), want[turn])


@gpu
@pytest.mark.parametrize("q8", [True, False])
def test_what_a_query_does_not_see_does_not_reach_it(hip, q8):
    """A value (and a key) that is no number, or infinite, inside a portion: queries in front of it and behind its window get what
    they get without it, those that see it get no finite number."""
    for rows, heads, d, at, window in (([(50, 40)], 4, 128, 70, 0), ([(3, 9)], 5, 64, 6, 0), ([(100, 300)], 2, 128, 250, 0), ([(100, 90)], 4, 128, 130, 24)):
        if window and not q8:
            continue
        for part, value in ((1, float("nan")), (0, float("nan")), (1, float("inf")), (1, float("-inf"))):
            q, pages, scales, table, attn, _ = _step(rows, heads, 1, d, 16, seed=at, device="cuda", q8=q8)
            run = (lambda: hip.paged_attention_q8(q, pages, scales, table, attn, 16, d ** -0.5, window)) if q8 else \
                (lambda: hip.prefix_attention(q, pages, table, attn, None, 16, d ** -0.5))
            clean = run()
            page, off = int(table[attn.slots[0], at // 16]), at % 16
            odd = torch.tensor([0x7f], dtype=torch.uint8, device="cuda").view(E4M3) if q8 else torch.tensor([value], dtype=torch.bfloat16, device="cuda")
            if part == 0:
                pages[page, 0, 0, off * d + 5] = odd[0]
            else:
                pages[page, 1, 0].view(d, 16)[5, off] = odd[0]
            got = run()
            pos = torch.arange(rows[0][0], sum(rows[0]))
            sees = (pos >= at) & ((pos < at + window) if window else torch.ones_like(pos, dtype=torch.bool))
            assert torch.equal(got[~sees], clean[~sees])
            hit = got[sees][:, :, 5] if part == 1 else got[sees]
            if part == 1 and not q8 and value == value:
                assert (hit == value).all()
            else:
                assert torch.isnan(hit).all()
            if part == 1:
                others = [i for i in range(d) if i != 5]
                assert torch.equal(got[:, :, others], clean[:, :, others])


@gpu
def test_rows_that_see_nothing(hip):
    """A row of length 0 and queries that lie before the sequence give zeros; their neighbours are as ever."""
    q, pages, scales, table, attn, _ = _step([(9, 1), (30, 1), (12, 4)], 4, 2, 64, 16, device="cuda")
    attn.lens[0] = 0
    attn.lens[2] = 2                                              # four queries of a sequence of two tokens
    got = hip.paged_attention_q8(q, pages, scales, table, attn, 16, 0.125)
    assert not got[0].any() and not got[2:4].any() and got[4:].any()
    _check(got, q, pages, scales, table, attn, 16, 0.125)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_and_chunks_as_wide_as_there_are(hip, dtype):
    """The widest windows hide nothing, from queries in front of the sequence and their neighbours neither."""
    q, pages, scales, table, attn, _ = _step([(9, 1), (12, 8), (30, 90)], 4, 2, 64, 16, dtype=dtype, device="cuda")
    attn.lens[1], attn.lens[2] = 2, 40                            # eight queries of a sequence of two tokens, 90 of one of 40
    want = hip.paged_attention_q8(q, pages, scales, table, attn, 16, 0.125)
    assert not want[1:7].any() and want[7:9].any() and not want[9:59].any() and want[59:].any()
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, -2 ** 30, 1 - 2 ** 31, -2 ** 31):
        print(window, flush=True)
        assert torch.equal(hip.paged_attention_q8(q, pages, scales, table, attn, 16, 0.125, window), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [[(200, 1)], [(5000, 1), (37, 1), (300, 1)], [(100, 3), (200, 5)], [(70, 90), (20, 1)]])
def test_lengths_past_the_block_table(hip, rows, dtype):
    """A row's walk ends where its table does, whatever its length says: 2^31 - 1 is the table's last key."""
    q, pages, scales, table, attn, _ = _step(rows, 4, 2, 64, 16, seed=1, dtype=dtype, device="cuda")
    pages.view(torch.uint8)[(pages.view(torch.uint8) & 0x7f) == 0x7f] = 0x30          # (the null page's keys are seen here)
    attn.lens[0] = 16 * table.shape[1]
    attn.max_decode_len = 16 * table.shape[1]
    want = hip.paged_attention_q8(q, pages, scales, table, attn, 16, 0.125)
    _check(want, q, pages, scales, table, attn, 16, 0.125)
    for more in (16 * table.shape[1] + 1, 2 ** 31 - 200, 2 ** 31 - 1):
        print(rows, more, flush=True)
        attn.lens[0] = more
        assert torch.equal(hip.paged_attention_q8(q, pages, scales, table, attn, 16, 0.125), want)
    attn.lens[0] = 2 ** 31 - 1
    prefix = SharedPrefix(torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"), 1,
                          rows[0][1], 16 * table.shape[1])
    got = hip.prefix_attention(q, pages, table, attn, prefix, 16, 0.125, scales)
    attn.lens[0] = 16 * table.shape[1]
    _check(got, q, pages, scales, table, attn, 16, 0.125)


@gpu
@pytest.mark.parametrize("q8", [False, True])
def test_groups_of_no_row(hip, q8, monkeypatch):
    """Groups without rows, behind the last row too; and a call of tokens, groups and no row at all, which leaves its result alone."""
    q, pages, scales, table, attn, prefix = _step([(1100, 1)] * 3, 8, 2, 128, 16, shared=[(0, 2, 1056)], q8=q8, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")                              # noqa: E731
    want = hip.prefix_attention(q, pages, table, attn, prefix, 16, 128 ** -0.5, scales)
    more = SharedPrefix(i32(0, 0, 3, 3, 3), i32(1056, 1056, 1056, 16), 4, 3, 1056)
    got = hip.prefix_attention(q, pages, table, attn, more, 16, 128 ** -0.5, scales)
    _check(got, q, pages, scales, table, attn, 16, 128 ** -0.5)
    assert (got.float() - want.float()).abs().max() <= 2 ** -6 * want.float().abs().max()
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: torch.full(t.shape, 7.0, dtype=t.dtype, device=t.device))
    none = AttnRows(i32(), i32(), i32(0), i32(), i32(), 0, 0, 0, 0, 0)
    for shared in (None, SharedPrefix(i32(0, 0), i32(1056), 1, 3, 1056)):
        assert (hip.prefix_attention(q, pages, table, none, shared, 16, 128 ** -0.5, scales) == 7).all()


@gpu
@pytest.mark.parametrize("q8", [False, True])
def test_a_group_of_rows_of_no_key(hip, q8):
    """All of a step's rows are empty, and the bound on their lengths says so."""
    q, pages, scales, table, attn, prefix = _step([(40, 1)] * 3, 4, 2, 64, 16, shared=[(0, 2, 32)], q8=q8, device="cuda")
    attn.lens.zero_()
    attn.max_decode_len = 0
    assert not hip.prefix_attention(q, pages, table, attn, prefix, 16, 0.125, scales).any()


@gpu
@pytest.mark.parametrize("q8", [False, True])
def test_tokens_of_no_row_are_left_alone(hip, q8, monkeypatch):
    """Tokens in front of the first row's and behind the last one's, in every way of cutting a call: what the result held there stays."""
    filled = lambda t, **kw: torch.full(t.shape, 7.0, dtype=t.dtype, device=t.device)              # noqa: E731
    monkeypatch.setattr(torch, "empty_like", filled)
    for rows, shared in (([(300, 1)] * 4, ()), ([(300, 1)] * 4, [(0, 3, 288)]), ([(1100, 1)] * 4, [(0, 3, 1056)]), ([(300, 4)] * 3, [(0, 2, 288)]),
                         ([(6000, 1), (40, 1)], ()), ([(100, 70), (300, 1), (30, 3)], [(0, 1, 96)]), ([(100, 70), (300, 1), (30, 3)], ()),
                         ([(100, 70), (1300, 70)], [(0, 1, 96)])):
        print(rows, shared, q8, flush=True)
        q, pages, scales, table, attn, prefix = _step(rows, 8, 2, 128, 16, seed=1, shared=shared, q8=q8, device="cuda")
        want = hip.prefix_attention(q, pages, table, attn, prefix, 16, 128 ** -0.5, scales)
        _check(want, q, pages, scales, table, attn, 16, 128 ** -0.5)
        wide = torch.cat((q[:1].expand(2, -1, -1), q, q[:1].expand(3, -1, -1)))
        attn.query_start += 2
        attn.in_order = False
        got = hip.prefix_attention(wide, pages, table, attn, prefix, 16, 128 ** -0.5, scales)
        assert torch.equal(got[2:-3], want) and (got[:2] == 7).all() and (got[-3:] == 7).all()


@gpu
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_a_bfloat16_cache_without_a_prefix(hip, step):
    rows, heads, kv, d, page, window = STEPS[step]
    q, pages, _, table, attn, _ = _step(rows, heads, kv, d, page, seed=step, q8=False, device="cuda")
    got = hip.prefix_attention(q, pages, table, attn, None, page, d ** -0.5)
    _check(got, q, pages, None, table, attn, page, d ** -0.5)


SHARED = [
    # (rows, groups, heads, kv heads, head size, page): a prefix of one page, one that ends inside a page, several groups, drafted tokens
    ([(20, 1), (40, 1)], [(0, 1, 16)], 4, 1, 64, 16),
    ([(300, 1), (290, 1), (257, 1), (310, 1)], [(0, 3, 250)], 8, 2, 128, 16),
    ([(100, 1)] * 5 + [(700, 1)] * 3 + [(50, 1)], [(0, 4, 64), (5, 7, 640)], 10, 2, 128, 32),      # and a row in no group
    ([(130, 5), (128, 5), (150, 5)], [(0, 2, 128)], 5, 1, 128, 16),
    ([(64, 1)] * 3 + [(200, 3)] * 2, [(0, 2, 64), (3, 4, 192)], 16, 1, 256, 64),
    ([(129, 70), (128, 2), (500, 1)], [(0, 2, 128)], 4, 2, 64, 16),                                 # a portion in the group
    ([(1000, 1)] * 40, [(0, 39, 992)], 8, 1, 128, 16),                                              # more columns than a block takes
    ([(96, 200), (100, 40)], [(0, 1, 96)], 4, 1, 128, 32),                                          # portions alone
    ([(520, 4)] * 20 + [(17, 3)], [(0, 19, 512)], 6, 2, 64, 16),                                    # and a row in no group
    ([(30, 1), (31, 1)], [(0, 0, 0), (1, 1, 16)], 4, 1, 64, 16),                                    # nothing shared, a row by itself
]


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("step", range(len(SHARED)))
def test_attention_over_a_shared_prefix(hip, step, q8):
    rows, shared, heads, kv, d, page = SHARED[step]
    print(f"step {step} 8-bit {q8}", flush=True)
    q, pages, scales, table, attn, prefix = _step(rows, heads, kv, d, page, seed=step, shared=shared, q8=q8, device="cuda")
    sink = torch.linspace(-2, 3, heads).cuda()
    for s in (None, sink):
        got = hip.prefix_attention(q, pages, table, attn, prefix, page, d ** -0.5, scales, s)
        _check(got, q, pages, scales, table, attn, page, d ** -0.5, 0, s)


@gpu
@pytest.mark.parametrize("step", range(len(SHARED)))
def test_float32_queries_over_a_shared_prefix(hip, step):
    rows, shared, heads, kv, d, page = SHARED[step]
    print(f"step {step}", flush=True)
    q, pages, scales, table, attn, prefix = _step(rows, heads, kv, d, page, seed=step, shared=shared, dtype=torch.float32, device="cuda")
    sink = torch.linspace(-2, 3, heads).cuda()
    for s in (None, sink):
        got = hip.prefix_attention(q, pages, table, attn, prefix, page, d ** -0.5, scales, s)
        _check(got, q, pages, scales, table, attn, page, d ** -0.5, 0, s)


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize(("groups", "queries"), [(63, 1), (64, 1), (65, 1), (140, 1), (70, 3)])
def test_many_groups(hip, groups, queries, q8):
    """More groups than a wave has lanes: a row finds its own, one that is in none finds none."""
    rows, shared = [], []
    for i in range(groups):
        whole = 16 * (1 + i % 3)
        rows += [(whole + j + i % 5, queries) for j in range(2 + i % 3)]
        shared.append((len(rows) - 2 - i % 3, len(rows) - 1, whole))
    rows.append((33, queries))
    q, pages, scales, table, attn, prefix = _step(rows, 4, 4, 64, 16, seed=groups, shared=shared, q8=q8, device="cuda")
    got = hip.prefix_attention(q, pages, table, attn, prefix, 16, 0.125, scales)
    _check(got, q, pages, scales, table, attn, 16, 0.125)


INSIDE = [
    # (rows, groups, lengths instead of theirs, heads, kv heads, head size): rows no longer than the prefix, queries inside it, rows of no key
    ([(300, 1)] * 4, [(0, 3, 288)], {1: 288, 2: 100, 3: 0}, 8, 2, 128),                                # a block a row
    ([(1100, 1)] * 6 + [(40, 1)], [(0, 5, 1056)], {1: 1057, 2: 1056, 3: 1055, 4: 33, 5: 0, 6: 0}, 8, 2, 128),
    ([(300, 5)] * 5, [(0, 4, 288)], {1: 292, 2: 290, 3: 4, 4: 2}, 8, 2, 64),                            # drafted tokens
    ([(1700, 1)] * 40 + [(20, 1)] * 3, [(0, 39, 1680), (40, 42, 16)], {i: 42 * i for i in range(1, 40)}, 10, 1, 128),   # many columns, two groups
    ([(96, 200), (100, 40), (90, 3)], [(0, 2, 80)], {0: 230, 1: 60, 2: 3}, 4, 1, 128),                  # portions
    ([(129, 70), (128, 2), (500, 1), (140, 1)], [(0, 3, 128)], {0: 150, 2: 64, 3: 0}, 4, 2, 256),        # all kinds of rows
    ([(4000, 1)] * 3, [(0, 2, 3984)], {0: 7, 1: 0, 2: 2100}, 4, 1, 64),                                 # none sees the whole prefix
    ([(1300, 1)] * 20, [(0, 19, 1280)], {i: 0 for i in range(20)}, 8, 2, 128),                          # none sees any of it
]


@gpu
@pytest.mark.parametrize(("q8", "dtype"), [(False, torch.bfloat16), (True, torch.bfloat16), (True, torch.float32)])
@pytest.mark.parametrize("step", range(len(INSIDE)))
def test_queries_inside_a_shared_prefix(hip, step, q8, dtype):
    """A query sees the keys up to its own, in the prefix as behind it; what it does not see may hold anything, what nobody sees too."""
    rows, shared, lens, heads, kv, d = INSIDE[step]
    print(f"step {step} 8-bit {q8} {dtype}", flush=True)
    q, pages, scales, table, attn, prefix = _step(rows, heads, kv, d, 16, seed=step, shared=shared, q8=q8, dtype=dtype, device="cuda")
    for i, n in lens.items():
        attn.lens[i] = n
    counts, held = attn.query_start.diff().tolist(), attn.lens.tolist()
    got = hip.prefix_attention(q, pages, table, attn, prefix, 16, d ** -0.5, scales)
    _check(got, q, pages, scales, table, attn, 16, d ** -0.5)
    start = attn.query_start.tolist()
    for i, (n, count) in enumerate(zip(held, counts)):
        assert not got[start[i]: start[i] + max(0, count - n)].any()
    # a value of the first group's prefix that is no number: it reaches those that see it, and changes nothing for the others
    lo, hi, most = shared[0]
    longest = max(held[i] for i in range(lo, hi + 1))
    at = min(most, longest) - 1
    if at < 0:
        return
    if q8:
        pages.view(torch.uint8)[table[attn.slots[lo], at // 16].long(), 1, 0].view(d, 16)[5, at % 16] = 0x7f
    else:
        pages[table[attn.slots[lo], at // 16].long(), 1, 0].view(d, 16)[5, at % 16] = float("nan")
    odd = hip.prefix_attention(q, pages, table, attn, prefix, 16, d ** -0.5, scales)
    for i, (n, count) in enumerate(zip(held, counts)):
        for x in range(count):
            t, sees = start[i] + x, lo <= i <= hi and n - count + x >= at
            mine = odd[t].clone()
            if sees:
                assert torch.isnan(mine[: heads // kv, 5]).all()
                mine[: heads // kv, 5] = got[t, : heads // kv, 5]
            assert torch.equal(mine, got[t]), (i, x)
    if at + 1 < most:                                             # what lies behind the longest row: keys, values and scales of any bytes
        pages.view(torch.uint8)[table[attn.slots[lo], (at + 16) // 16: most // 16].long()] = 0xff
        if q8:
            scales.view(torch.uint8)[table[attn.slots[lo], (at + 16) // 16: most // 16].long()] = 0xff
        assert torch.equal(hip.prefix_attention(q, pages, table, attn, prefix, 16, d ** -0.5, scales).nan_to_num(7.0), odd.nan_to_num(7.0))


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize(("d", "rows"), [(64, [(49300, 8)] * 4), (128, [(49168, 8), (49500, 8), (49169, 8), (49200, 7), (60, 3)])])
def test_a_long_shared_prefix(hip, d, rows, q8):
    """Prefixes long enough for blocks of 256 columns, which eight queries of four rows by eight heads fill."""
    q, pages, scales, table, attn, prefix = _step(rows, 8, 1, d, 16, seed=d, shared=[(0, 3, 49168)], q8=q8, device="cuda")
    got = hip.prefix_attention(q, pages, table, attn, prefix, 16, d ** -0.5, scales)
    _check(got, q, pages, scales, table, attn, 16, d ** -0.5)


def _drafts(counts, vocab, seed, *, probs=True, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    start = [0] + list(np.cumsum(counts))
    n, b = start[-1], len(counts)
    logits = torch.randn(n, vocab, generator=g) * spread
    q = torch.softmax(logits + 0.7 * torch.randn(n, vocab, generator=g), -1)
    return dict(logits=logits, drafted=torch.multinomial(q, 1, generator=g)[:, 0].int() if n else torch.zeros(0, dtype=torch.int32),
                draft_probs=q if probs else None, accept=torch.rand(n, generator=g), draw=torch.rand(b, generator=g),
                temperature=(0.5 + torch.rand(b, generator=g)) * (torch.arange(b) % 4 != 3), start=torch.tensor(start, dtype=torch.int32),
                most=max(list(counts) + [1]) - 1)


def _verify(hip, case):
    want = PLAIN.verify_drafts(**case)
    got = hip.verify_drafts(**{k: x.cuda() if torch.is_tensor(x) else x for k, x in case.items()})
    for x, y in zip(got, want):
        assert x.dtype == torch.int32 and torch.equal(x.cpu(), y), (x.cpu().tolist(), y.tolist())
    return want


@gpu
@pytest.mark.parametrize(("counts", "vocab"), [([1], 7), ([4], 1000), ([5, 3, 1, 5, 2], 4096), ([3] * 9, 4097), ([2, 0, 4], 8190), ([64, 1], 333),
                                               ([4, 4], 50001), ([6], 151936)])
@pytest.mark.parametrize("probs", [True, False])
def test_verify(hip, counts, vocab, probs):
    taken = []
    for seed in range(4):
        taken += _verify(hip, _drafts(counts, vocab, seed, probs=probs))[1].tolist()
    assert not probs or len(counts) < 3 or max(taken) > 0


@gpu
def test_verify_at_the_borders(hip):
    """Numbers of 0 and next to 1, drafts that are none, certain rows, rows without mass, infinite logits and ones that are no number."""
    for seed, probs in ((0, True), (1, False)):
        case = _drafts([4] * 8, 5000, seed, probs=probs)
        case["accept"][::3], case["accept"][1::3] = 0.0, 1.0 - 2.0 ** -24
        case["draw"][::2], case["draw"][1::2] = 0.0, 1.0 - 2.0 ** -24
        _verify(hip, case)
        case["drafted"][::5], case["drafted"][2::7] = -1, 5000
        _verify(hip, case)
        case["logits"][3] = float("-inf")
        case["logits"][5, :4000] = float("-inf")
        case["logits"][9, 17], case["logits"][9, 4900] = float("inf"), float("inf")
        case["logits"][12, ::2] = float("nan")
        case["logits"][14] = float("nan")
        case["logits"][0:4] = 0.0                                  # all alike
        _verify(hip, case)
        case["temperature"][:] = 0
        _verify(hip, case)
        case["temperature"][:] = torch.tensor([1e-30, 1e-3, 0.05, 3e38, float("inf"), 50.0, 1.0, -1.0])
        _verify(hip, case)
    same = _drafts([5] * 4, 3001, 3)
    same["draft_probs"] = torch.softmax(same["logits"], -1)       # drafts from the target itself
    same["temperature"][:] = 1
    assert _verify(hip, same)[1].sum() >= 14


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("probs", [True, False])
def test_a_draft_of_probability_0_is_never_taken(request, device, probs):
    """Tokens that a mask has set to -inf, that are no number, or lie in a row without mass are turned down whatever was drawn against
    them, 0 too and where the draft's own probability is 0; what comes out instead has mass. A draft of probability 0 that the target
    allows is taken. Held to the definition: accept is uniform in [0, 1), so P(accept q < p) = min(1, p / q)."""
    ops = PLAIN if device == "cpu" else request.getfixturevalue("hip")
    vocab, n = 5000, 8
    logits = torch.randn(2 * n, vocab, generator=torch.Generator().manual_seed(3))
    drafted = torch.arange(2 * n, dtype=torch.int32) * 311
    q = torch.full((2 * n, vocab), 1.0 / vocab)
    accept, rows = torch.zeros(2 * n), torch.arange(n) * 2        # request b judges row 2 b
    accept[rows[1]] = accept[rows[4]] = accept[rows[5]] = 0.5
    for b in (0, 1, 2):
        logits[rows[b], drafted[rows[b]]] = float("-inf")
    q[rows[1], drafted[rows[1]]] = q[rows[2], drafted[rows[2]]] = 0.0
    logits[rows[3], drafted[rows[3]]] = float("nan")
    logits[rows[4]], logits[rows[5]] = float("-inf"), float("nan")                       # no mass at all
    q[rows[6], drafted[rows[6]]] = 0.0                                                   # rows 6, 7: allowed, and drawn against with 0
    case = dict(logits=logits, drafted=drafted, draft_probs=q if probs else None, accept=accept, draw=torch.rand(n, generator=torch.Generator().manual_seed(4)),
                temperature=torch.ones(n), start=torch.arange(0, 2 * n + 1, 2, dtype=torch.int32), most=1)
    tokens, taken = (x.cpu().tolist() for x in ops.verify_drafts(**{k: x.to(device) if torch.is_tensor(x) else x for k, x in case.items()}))
    assert taken == [0] * 6 + [1, 1]
    for b in range(4):
        assert tokens[b][0] != int(drafted[rows[b]]) and logits[rows[b], tokens[b][0]] > float("-inf") and tokens[b][1] == -1
    assert tokens[4] == tokens[5] == [0, -1]
    assert [tokens[b][0] for b in (6, 7)] == drafted[rows[6:]].tolist()


@gpu
@pytest.mark.parametrize("probs", [True, False])
def test_verify_where_little_is_left(hip, probs):
    """A draft that holds all but some 2^-20 of a row and is turned down all the same: what is left lies in pieces of its own, beside the
    draft in its piece, or nowhere in that piece; drawn from its first value (0) and its last. Whatever the draft's weight is rounded to,
    its piece has no mass without it."""
    vocab = 3 * 4096 + 7
    others = ([], [0, 4095], [4100, 4200], [4096, 8191, 8192, vocab - 1], [vocab - 2], [1, 12290])
    logits = torch.full((2 * 2 * len(others), vocab), float("-inf"))
    drafted = torch.full((len(logits),), 4100 + 57, dtype=torch.int32)
    for i, places in enumerate(others):
        for row in range(4 * i, 4 * i + 4):
            logits[row, drafted[row]] = 0.0
            logits[row, places] = -14.0 - torch.arange(float(len(places)))
            if not places:
                logits[row, 9] = -15.0
    q = torch.zeros_like(logits)
    q[torch.arange(len(logits)), drafted.long()] = 1.0
    start = torch.arange(0, len(logits) + 1, 2, dtype=torch.int32)
    case = dict(logits=logits, drafted=drafted, draft_probs=q if probs else None, accept=torch.full((len(logits),), 1.0 - 2.0 ** -24),
                draw=torch.tensor([0.0, 1.0 - 2.0 ** -24] * len(others)), temperature=torch.ones(2 * len(others)), start=start, most=1)
    want = _verify(hip, case)
    assert (want[1] == 0).all() and (want[0][:, 0] != drafted[0]).all()


@gpu
@pytest.mark.parametrize("vocab", [262145, 262208, 600001])
@pytest.mark.parametrize("probs", [True, False])
def test_verify_over_many_pieces(hip, vocab, probs):
    """Vocabularies of more than 64 pieces of 4,096: tokens drawn from the first of them, from behind 64 and from the very last, and rows
    whose largest logit lies there."""
    for seed, draw in ((0, (0.0, 0.5, 0.999, 1.0 - 2.0 ** -24)), (1, (0.97, 0.3, 1.0 - 2.0 ** -24, 0.9))):
        case = _drafts([3, 1, 2, 3], vocab, seed, probs=probs, spread=1.0)
        case["draw"][:] = torch.tensor(draw)
        _verify(hip, case)
        case["logits"][:, 64 * 4096:] += 30.0                      # all that matters lies behind 64 pieces
        case["temperature"][2] = 0.0
        want = _verify(hip, case)[0][case["draw"] > 0]               # (a number of 0 draws the first token of any mass)
        assert ((want >= 64 * 4096) | (want == -1)).all()
        case["logits"][:, : vocab - 2] = float("-inf")
        assert set(_verify(hip, case)[0].flatten().tolist()) <= {-1, vocab - 2, vocab - 1}


@gpu
def test_verify_keeps_the_targets_law(hip):
    """Whatever the drafts come from, the first token is distributed as p: frequencies over many numbers within five standard errors."""
    vocab, n = 11, 30000
    g = torch.Generator().manual_seed(5)
    logits, other = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g) * 1.5
    p, q = torch.softmax(logits.double(), -1), torch.softmax(other, -1)
    drafted = torch.zeros(2 * n, dtype=torch.int32)
    drafted[::2] = torch.multinomial(q, n, replacement=True, generator=g).int()
    tokens, _ = hip.verify_drafts(logits.expand(2 * n, -1).contiguous().cuda(), drafted.cuda(), q.expand(2 * n, -1).contiguous().cuda(),
                                  torch.rand(2 * n, generator=g).cuda(), torch.rand(n, generator=g).cuda(), torch.ones(n).cuda(),
                                  torch.arange(0, 2 * n + 1, 2, dtype=torch.int32).cuda(), 1)
    seen = torch.bincount(tokens[:, 0].cpu().long(), minlength=vocab).double() / n
    assert ((seen - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all()


def _answers(ops, device):
    """Six answers to one prompt of 40 tokens, three drafted tokens checked a step: written into the 8-bit cache, attended to over the
    prefix that all share, judged, and what was taken written over what was not. Keys, values and queries are tables' rows."""
    heads, kv, d, page, vocab, batch, drafts = 4, 2, 64, 16, 300, 6, 3
    g = torch.Generator().manual_seed(9)
    keys, values = torch.randn(2, vocab, kv, d, generator=g)
    queries, head = torch.randn(vocab, heads, d, generator=g), torch.randn(heads * d, vocab, generator=g).double() * 0.08
    i32 = lambda x: torch.as_tensor(np.asarray(x, dtype=np.int32)).to(device)                       # noqa: E731
    prompt = torch.randint(0, vocab, (40,), generator=g)
    table = np.array([[0, 1] + [2 + 4 * b + i for i in range(4)] for b in range(batch)])
    pages = torch.zeros(2 + 4 * batch, 2, kv, page * d, dtype=torch.uint8, device=device)
    scales = torch.zeros(2 + 4 * batch, 2, kv, page, dtype=torch.uint8, device=device)

    def write(tokens, rows, places):
        page_of, off = table[rows, places // page], places % page
        ops.kv_write_q8(keys[tokens].to(device), values[tokens].to(device), pages, scales, i32(page_of), i32(off), page)

    for b in range(batch):                                    # the first two pages once, the eight tokens behind them into each row's third
        lo = 0 if b == 0 else 32
        write(prompt[lo:], np.full(40 - lo, b), np.arange(lo, 40))
    held, last, out = np.full(batch, 40), torch.randint(0, vocab, (batch,), generator=g), [[] for _ in range(batch)]
    for _ in range(6):
        q = torch.softmax(torch.randn(batch * (drafts + 1), vocab, generator=g), -1)
        drafted = torch.multinomial(q, 1, generator=g)[:, 0].int()
        fed = torch.cat((last[:, None], drafted.view(batch, -1)[:, :drafts]), 1).flatten().long()
        rows = np.repeat(np.arange(batch), drafts + 1)
        write(fed, rows, held[rows] + np.tile(np.arange(drafts + 1), batch))
        starts = np.arange(batch + 1) * (drafts + 1)
        attn = AttnRows(i32(range(batch)), i32(held + drafts + 1), i32(starts), i32([]), i32(range(batch)), 0, batch, 0, drafts + 1,
                        int(held.max()) + drafts + 1)
        shared = SharedPrefix(i32([0, batch]), i32([32]), 1, batch * (drafts + 1), 32)
        seen = ops.prefix_attention(queries[fed].to(device), pages, i32(table), attn, shared, page, 1.5 * d ** -0.5, scales)
        logits = (seen.cpu().double().view(len(fed), -1) @ head).float()
        accept, draw = torch.rand(len(fed), generator=g), torch.rand(batch, generator=g)
        tokens, taken = ops.verify_drafts(logits.to(device), drafted.to(device), q.to(device), accept.to(device), draw.to(device),
                                          torch.full((batch,), 0.9, device=device), i32(starts), drafts)
        tokens, taken = tokens.cpu(), taken.cpu().numpy()
        for b in range(batch):
            out[b] += tokens[b, : taken[b] + 1].tolist()
        last, held = tokens[torch.arange(batch), taken].long(), held + taken + 1
    return out, pages.cpu(), scales.cpu()


@gpu
def test_answers_to_one_prompt(hip):
    """The operations one after the other, against the twins: the same tokens, the same cache."""
    want, got = _answers(PLAIN, "cpu"), _answers(hip, "cuda")
    assert want[0] == got[0] and torch.equal(want[1], got[1]) and torch.equal(want[2], got[2])
    assert 6 * 6 + 3 < sum(map(len, want[0])) < 6 * 6 * 4                    # drafts were taken, and turned down
