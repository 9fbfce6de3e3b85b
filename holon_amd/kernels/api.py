"""The kernel contract: every device operation the parts call, with shapes, dtypes and in-place rules.

`holon_amd.kernels.hip.HipKernels` is the only implementation the product has (hand-written gfx950 HIP, loaded from
the in-tree library; it fails loudly when the library is missing). A plain twin with the same methods lives under
`tests/` and is handed to the engine only by tests. The shapes follow the reference's op contracts
(std/holon_std/ops/kernels.py:1-45, std/holon_std/mixers/gqa/kernels.py:1-52), with this engine's cache layout.

Conventions: T tokens in the step, B rows (requests in the step), Hq/Hkv heads, D head_dim, P page size. Activations
and weights are `dtype` (bfloat16 or float32) unless stated; index tensors are int32. Norms, softmax, rotation angles
and every sum are computed in float32 and rounded once to `dtype`.

Cache layout of one page of one site, `pages[page]` = `[2, Hkv, P * D]`: keys as rows `[P, D]` (token-major),
values as columns `[D, P]` (transposed inside the page, so that a matrix-core operand of the value product is one
contiguous 16-byte load). Block table row `slot` lists the page of token positions `i*P .. i*P+P-1` at index i.
"""
from __future__ import annotations

import dataclasses
from typing import Protocol

import torch


@dataclasses.dataclass
class AttnRows:
    """The rows of a step, as attention sees them. Row b reads block table row `slots[b]`, holds `lens[b]` tokens
    including this step's, and owns query tokens `query_start[b]:query_start[b+1]`, the last of its sequence
    ("bottom-right causal": query i of the row sits at position lens[b] - n_query[b] + i). Rows with one query token
    are listed in `decode_rows`, the others in `chunk_rows` (row indices, int32, device). `in_order` says that the
    step is decode rows alone, listed as they lie (a kernel then need not read the lists)."""

    slots: torch.Tensor                  # [B] int32
    lens: torch.Tensor                   # [B] int32
    query_start: torch.Tensor            # [B+1] int32
    decode_rows: torch.Tensor            # [n_decode] int32
    chunk_rows: torch.Tensor             # [n_chunk] int32
    n_decode: int
    n_chunk: int
    max_decode_len: int                  # host bounds for launch shapes
    max_chunk_query: int
    max_chunk_len: int
    in_order: bool = False               # every row is a decode row, and decode_rows[i] = query_start[i] = i


@dataclasses.dataclass
class SharedPrefix:
    """Rows of a step that begin with the same tokens: group g is rows group_start[g] .. group_start[g + 1] - 1 (neighbours; a
    row may be in none), whose first lens[g] tokens are the same ones in the same cache pages. A row may be shorter than that, or
    begin with queries inside it: they see the prefix up to themselves. The block table of a group's first row names all of its pages."""

    group_start: torch.Tensor            # [G+1] int32, rising
    lens: torch.Tensor                   # [G] int32
    n_groups: int
    max_queries: int                     # host bounds for launch shapes: the most query tokens of a group's rows together,
    max_len: int                         # and the longest prefix


class Kernels(Protocol):
    name: str

    def embedding(self, ids: torch.Tensor, table: torch.Tensor,
                  take: tuple[torch.Tensor, torch.Tensor] | None = None, want_stats: bool = False):
        """ids [T] int32, table [V, H] -> [T, H] (rows of the table). `take` = (take_slot [T] int32, last_token [S]
        int32): token t is last_token[take_slot[t]] where take_slot[t] >= 0 (a token the previous step drew and left
        on the device), ids[t] otherwise. With `want_stats` -> (rows, row statistics or None): see `row_sumsq`."""

    def row_sumsq(self, x: torch.Tensor) -> torch.Tensor:
        """Row statistics of x [M <= 16, H]: float32 [parts, 16] whose column m sums to the sum of squares of row m
        (here parts = 1). A kernel that writes rows may leave the same thing in several parts (`linear_add`); a
        product with a folded norm (`linear(..., row_scale=)`) adds the parts in a fixed order."""

    def folds_norm(self, rows: int, weight: torch.Tensor, tiled: torch.Tensor | None) -> bool:
        """Whether `linear(x, weight, tiled=tiled, row_scale=...)` serves `rows` rows."""

    def rmsnorm(self, x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
        """x [..., dim] contiguous -> a new tensor; x is not modified."""

    def add_rmsnorm(self, x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
        """residual += x in place (sum rounded to dtype), returns rmsnorm(residual) as a new tensor. `x` may be what
        `linear_parts` returned, float32 [S, *residual.shape]: what is added is then the parts' sum in order, rounded
        to the residual's dtype first (the product that `linear` would have returned)."""

    def linear(self, x: torch.Tensor, weight: torch.Tensor, out_dtype: torch.dtype | None = None,
               tiled: torch.Tensor | None = None, row_scale: tuple[torch.Tensor, float] | None = None) -> torch.Tensor:
        """x [T, K] @ weight [N, K].T -> [T, N], float32 accumulation, rounded to x's dtype; with another `out_dtype`
        that rounded product is then cast (the reference's `F.linear(...).float()`, std/holon_std/ops/units.py:348): one
        rule for every number of rows. `tiled`: what `tile_weight(weight)` returned, if anything.
        `row_scale` = (row statistics of x, eps): an RMSNorm folded into the product. `tiled` is then
        `tile_weight(weight, norm_weight)`, x the un-normed rows, and row m of the float32 sums is scaled by
        rsqrt(mean(x[m]^2) + eps) before it is rounded: norm(x) W^T with the rounding of the normed activations
        moved to the folded weights."""

    def tile_weight(self, weight: torch.Tensor, scale: torch.Tensor | None = None) -> torch.Tensor | None:
        """Once per weight after loading: a copy in the layout steps of few rows stream fastest, or None. With
        `scale` [K] the copy holds weight * scale[None, :] (rounded): a norm's weight folded in."""

    def serves_rows(self, rows: int, weight: torch.Tensor, tiled: torch.Tensor | None, gated: bool = False) -> bool:
        """Whether `linear` (gated: `linear_silu_mul`) reads `tiled` for a step of `rows` rows beyond the few-row
        kernels' (17 to 64): a caller whose tiled copy has a norm folded in then passes rows normed without the
        norm's weight."""
        return False

    def linear_parts(self, x: torch.Tensor, weight: torch.Tensor, tiled: torch.Tensor | None) -> torch.Tensor | None:
        """linear(x, weight) as float32 sums over S shares of K, [S, T, N], for a reader that adds them up itself
        (`add_rmsnorm`; `sum_parts` for anyone else): their sum in order, rounded to x's dtype, is the product. None
        when this step is not served that way (then nothing was done); a kernel set serves it only where that is
        faster than `linear` even with the reader's extra reads."""
        return None

    def sum_parts(self, parts: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """float32 [S, ...] -> [...] in `dtype`: the parts added up in order, rounded once."""

    def linear_add(self, x: torch.Tensor, weight: torch.Tensor, tiled: torch.Tensor | None, residual: torch.Tensor,
                   want_stats: bool = False) -> "bool | torch.Tensor":
        """residual += linear(x, weight) in place in one kernel: the product rounded to dtype, then the sum rounded,
        as the add of `add_rmsnorm` does. False when not fused for this shape; then nothing was done. Otherwise
        True, or with `want_stats` the row statistics of the residual rows as they now are, when the kernel can
        leave them."""

    def linear_silu_mul(self, x: torch.Tensor, weight: torch.Tensor, tiled: torch.Tensor | None = None,
                        row_scale: tuple[torch.Tensor, float] | None = None) -> torch.Tensor | None:
        """silu_mul(linear(x, weight)) fused, with the composition's roundings; None when not fused for this shape.
        `row_scale` as in `linear`."""

    def linear_glu(self, x: torch.Tensor, weight: torch.Tensor, act: int) -> torch.Tensor | None:
        """`linear_silu_mul` (`act` 0) or `linear_gelu_mul` (1) for steps of more than 128 rows over the weight as it is; None where the
        composition is to be taken. (A kernel set without it: the operation registered in `parts/ffn.py`, which never serves.)"""

    def silu_mul(self, gate_up: torch.Tensor) -> torch.Tensor:
        """gate_up [T, 2I] (gate columns first) -> [T, I] = round(silu(gate)) * up."""

    def rope(self, x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor) -> None:
        """Rotate the first table.shape[1] dims of x [T, heads, D] in place, half-split pairing; table
        [max_positions, rotary_dim] float32 = cos of the rotary_dim/2 angles, then their sin."""

    def kv_write(self, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, write_page: torch.Tensor,
                 write_off: torch.Tensor, page_size: int) -> None:
        """k, v [T, Hkv, D] into the cache layout at (write_page[t], write_off[t])."""

    def qk_norm_rope_write(self, qkv: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                           q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float,
                           table: torch.Tensor | None, positions: torch.Tensor, pages: torch.Tensor | None,
                           write_page: torch.Tensor | None, write_off: torch.Tensor | None, page_size: int
                           ) -> torch.Tensor:
        """The fused form of per-head rmsnorm (if weights), rope (if table) and kv_write (if pages) on the merged
        projection qkv [T, (Hq + 2 Hkv) D]: q and k heads are normed and rounded, rotated and rounded; k and v go to
        the cache; returns q' [T, Hq, D], a new tensor. Same roundings as the three ops one after the other."""

    def check_attention(self, head_dim: int, page_size: int, dtype: torch.dtype) -> None:
        """Raise, with a message that names the limit, when no attention kernel serves this head size, page size and
        dtype. Mixers call it when they are built, so that a model is refused before it takes a request."""

    def attention_on_cores(self, head_dim: int, page_size: int, dtype: torch.dtype) -> bool:
        """Whether `paged_attention` runs on the matrix cores at this head size, page size and dtype (there it also
        takes a sink)."""
        return False

    def paged_attention(self, q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, rows: AttnRows,
                        page_size: int, scale: float, window: int, sink: torch.Tensor | None = None,
                        softcap: float = 0.0, dist: tuple[torch.Tensor, torch.Tensor] | None = None,
                        keep_first: int = 0, value_share: int = 1, head_gate: torch.Tensor | None = None
                        ) -> torch.Tensor:
        """softmax(q k^T * scale) v per row over its cached tokens, causal; with window W > 0 a query at position p
        sees keys p-W+1 .. p, with -W < 0 the keys of its own chunk of W positions (from p - p mod W). q [T, Hq, D] ->
        [T, Hq, D]. This step's keys are already in the cache. `sink` [Hq]
        float32: exp(sink[h] - max) is added to the softmax's denominator (it has no key and no value). Where
        `attention_on_cores` says so it also takes changed scores: `softcap` > 0: s <- softcap tanh(s / softcap);
        `dist` = (r1 [Hq], r2 [Hq]) float32: s <- s - r1 ln(1 + r2 (p - j)) for the key at position j; `keep_first`:
        under a window, keys 0 .. keep_first - 1 stay visible. `value_share` s > 1 (there as well): `pages` is
        [n, Hkv + Hkv / s, P * D], Hkv planes of keys and then Hkv / s of values, and key head h reads value head
        h // s (several score maps over one set of values). `head_gate` [T, Hq] (there as well; columns of wider rows
        will do): head h's result of token t is multiplied by sigmoid(head_gate[t, h]) before it is rounded."""

    def check_cache_q8(self, head_dim: int, page_size: int) -> None:
        """Raise, with a message that names the limit, when no 8-bit cache of this head size and page size is served."""

    def kv_write_q8(self, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, write_page: torch.Tensor,
                    write_off: torch.Tensor, page_size: int) -> None:
        """k, v [T, Hkv, D] into an 8-bit cache at (write_page[t], write_off[t]): pages [n, 2, Hkv, P * D] float8_e4m3fn in the
        cache layout above, scales [n, 2, Hkv, P] float8_e8m0fnu (either may be a uint8 view; pages may lie apart, each in one
        piece). A (token, head) row is held as round(x / 2^e) and the byte of 2^e, e the smallest power of two, at least -126,
        that brings its largest finite value to 448 or less (a row of zeros: 0); a value that is not finite is held as NaN.
        k and v may be columns of wider rows (equally far apart). A token whose place lies outside the pool or the page is not
        written. Two tokens of one place: their bytes mix (the padding rows of a captured step share the null page)."""

    def qk_norm_rope_write_q8(self, qkv: torch.Tensor, heads: int, kv_heads: int, head_dim: int, q_weight: torch.Tensor | None,
                              k_weight: torch.Tensor | None, eps: float, table: torch.Tensor | None, positions: torch.Tensor,
                              pages: torch.Tensor, scales: torch.Tensor, write_page: torch.Tensor, write_off: torch.Tensor,
                              page_size: int) -> torch.Tensor:
        """`qk_norm_rope_write` with keys and values into an 8-bit cache (`kv_write_q8`), the roundings of the two one after the
        other; the whole head is rotated or none of it. A position outside the table takes its first or its last row."""

    def kv_read_q8(self, pages: torch.Tensor, scales: torch.Tensor, read_page: torch.Tensor, read_off: torch.Tensor, page_size: int,
                   dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """What the places (read_page[t], read_off[t]) of an 8-bit cache stand for: (k, v), new tensors [T, Hkv, D], code * 2^e
        in `dtype` (bfloat16 holds it exactly). Zeros for a place outside the pool or the page."""

    def paged_attention_q8(self, q: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, rows: AttnRows,
                           page_size: int, scale: float, window: int = 0, sink: torch.Tensor | None = None) -> torch.Tensor:
        """`paged_attention` over an 8-bit cache (see `kv_write_q8`): the softmax and its sums in float32 over the values that the
        cache stands for. q [T, Hq, D] bfloat16 or float32 -> a new tensor of its type; heads of 64, 128 and 256, pages of a
        multiple of 16 tokens; `scale` > 0. A query that sees no key gets zeros; what a query does not see, finite or not, does
        not reach it. Tokens of no row are not written. A page or slot number out of range is not followed, a length past the end
        of its block table's row is taken as that."""

    def prefix_attention(self, q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, rows: AttnRows, prefix: SharedPrefix,
                         page_size: int, scale: float, scales: torch.Tensor | None = None, sink: torch.Tensor | None = None
                         ) -> torch.Tensor:
        """`paged_attention` (window 0) of a batch whose rows share their first tokens by groups: a group's prefix is read once for
        all of its rows' queries (through its first row's block table), each row's further keys by itself, and the two are joined.
        pages bfloat16, or with `scales` an 8-bit cache. Sizes, types and masks as in `paged_attention_q8`."""

    def qkv_attention(self, qkv: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                      q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float,
                      rope_table: torch.Tensor | None, positions: torch.Tensor, pages: torch.Tensor | None,
                      table: torch.Tensor, write_page: torch.Tensor, write_off: torch.Tensor, rows: AttnRows,
                      page_size: int, scale: float, window: int, writes: bool = True) -> torch.Tensor:
        """`paged_attention(qk_norm_rope_write(qkv, ...), pages, table, rows, ...)` as one operation, with that
        composition's roundings; a kernel set may run it in fewer kernels (a step of decode rows alone). `writes`
        False: the keys and values are not stored (a run that reads another run's cache)."""

    def argmax(self, logits: torch.Tensor) -> torch.Tensor:
        """logits [R, V] float32 -> [R] int32, the first maximal index of each row."""

    def store_tokens(self, last_token: torch.Tensor, slots: torch.Tensor, tokens: torch.Tensor) -> None:
        """last_token[slots[r]] = tokens[r] (all int32, slots distinct): drawn tokens kept on the device by slot."""

    def logprobs(self, logits: torch.Tensor, tokens: torch.Tensor, k: int
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """log_softmax of the raw logits [R, V]: (the log-probability of tokens[r] [R], the k largest ids [R, k] int32,
        their log-probabilities [R, k]); k <= 32; ties go to the lower id."""

    def sample(self, logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor,
               min_p: torch.Tensor, seeds: torch.Tensor, positions: torch.Tensor,
               slots: torch.Tensor | None = None) -> torch.Tensor:
        """One token per row [R] int32. temperature/top_p/min_p float32, top_k int32, seeds int64: [R], row r's own;
        or, with `slots` [R] int32, tables [S] of which row r reads entry slots[r]. positions [R] int32 or int64 (the
        position of the token being drawn). Rows with temperature 0 take the argmax; the others draw by inverse CDF
        at the hashed uniform of (seed, position): in vocabulary order when the row has no filter (top_k 0, top_p 1,
        min_p 0), else in sorted order (scaled logit descending, equal ones by index)."""

    def verify_drafts(self, logits: torch.Tensor, drafted: torch.Tensor, draft_probs: torch.Tensor | None, accept: torch.Tensor,
                      draw: torch.Tensor, temperature: torch.Tensor, start: torch.Tensor, most: int
                      ) -> tuple[torch.Tensor, torch.Tensor]:
        """Drafted tokens judged against the target's probabilities from given random numbers. Request b (of B) owns rows start[b]
        .. start[b + 1] - 1 (start [B+1] int32) of logits [N, V] float32: row i judges drafted[i] ([N] int32), the last row none.
        p = softmax(logits / temperature[b]), q = draft_probs[i] ([N, V] float32; None: the drafts were certain). Row i takes its
        draft x when accept[i] q(x) < p(x) (never one of probability 0); behind the drafts taken one more token is drawn: from
        max(p - q, 0) where a draft was turned down (where that leaves nothing: from p), from p otherwise: the first whose running
        sum exceeds draw[b] times the whole. accept [N] and draw [B] float32 lie in [0, 1). Temperature 0 (or less): p is the first
        largest logit. A drafted id outside the vocabulary is no draft: the row draws from p. Sums and exponentials in 64 bits; a
        logit that is NaN has no mass; a row without any gives token 0. -> (tokens [B, most + 1] int32: those taken, the drawn
        one, then -1; how many were taken [B] int32); a request of no rows gets -1 and 0, of its rows only the first most + 1 (at
        most 64) count."""

    def scatter_rows(self, dst: torch.Tensor, idx: torch.Tensor, src: torch.Tensor) -> None:
        """dst[idx[r]] = src[r] for int32 rows: dst [N, W], idx [n], src n * W values."""
