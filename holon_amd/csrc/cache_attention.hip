// Paged causal attention over the 8-bit cache (cache_q8.h), and over a bfloat16 cache where rows share their first pages.
//
// softmax(scale q k^T) v on v_mfma_f32_16x16x32_bf16, online and in float32 as in attention_mfma.hip. A row's queries and the
// heads of a group are one list of columns, column f = (query f / G, head f % G), so that tiles of 16 are full whatever G is.
//
// Codes enter the matrix cores as bfloat16, which holds code * 2^e exactly: a key's power goes into the conversion of its
// codes, a value's power into its probability (p 2^e, exact too), so that neither costs an instruction a code. A float32
// query, and the probabilities behind it, are split into three bfloat16 numbers (8 + 8 + 8 bits of mantissa): the products with
// codes are then exact to 2^-24 of the larger operand.
#include <algorithm>
#include <type_traits>

#include "cache_q8.h"
#include "holon_hip.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct CacheArgs {
  const void* q;               // [T, Hq, D]
  void* out;                   // [T, Hq, D]
  const uint8_t* pages;        // codes, or bfloat16 values; a page's first byte, pages `page_stride` bytes apart
  const uint8_t* scales;
  int64_t page_stride, scale_stride;
  int num_pages;
  const int32_t* table;        // [slots, table_stride]
  int table_stride, n_slots;
  const int32_t* slots;        // [B]
  const int32_t* lens;         // [B]
  const int32_t* qstart;       // [B + 1]
  const int32_t* row_ids;      // the rows of this launch (null: they are decode rows alone, in order)
  int n_tokens;
  int heads, kv_heads, page_size;
  uint32_t page_magic;         // see page_index
  float scale_log2;            // scale * log2(e)
  int window;                  // see first_seen
  const float* sink;           // [Hq], nullable
  float* part_o;               // partial results of (token, head) cells, `parts` each: [cells, parts, D] and [cells, parts, 2]
  float* part_ml;
  int parts, part_first;       // this launch's come from `part_first` on
  int cell_queries;            // > 0: cell (row in row_ids) * cell_queries + query; 0: the token
  int splits;                  // over which waves a row's keys are cut
  int budget, n_rows;          // budget > 0: blocks a kv head has for its n_rows <= 64 decode rows together, see RowShares;
  int2* row_parts;             // then [n_rows]: the first of a row's parts, and how many it has
  // rows that share their first tokens: group g is rows group_start[g] .. group_start[g + 1] - 1 and shares group_lens[g] of them
  const int32_t* group_start;
  const int32_t* group_lens;
  int n_groups;
  int rows;                    // B. (Here, where the struct ended in a gap: eight more bytes of it took the merge of 64 rows from 8 to 13 us.)
};

// The page that a position lies in: position / page_size, by a product (a division is forty vector instructions, also where every
// lane asks the same, and a stage of 32 keys asks four times). With magic = ceil(2^32 / P), the high half of position * magic is the
// quotient while position * (magic P - 2^32) < 2^32, which the host checks of a whole table row (a P that is a power of two: always).
__device__ __forceinline__ int page_index(const CacheArgs& a, int pos) { return (int)__umulhi((uint32_t)pos, a.page_magic); }

// What is out of range is not followed: the pool's last page, the table's last row.
__device__ __forceinline__ int64_t page_at(const CacheArgs& a, int32_t page) {
  return (int64_t)min((uint32_t)page, (uint32_t)(a.num_pages - 1));
}
__device__ __forceinline__ const int32_t* table_at(const CacheArgs& a, int32_t slot) {
  return a.table + (int64_t)min((uint32_t)slot, (uint32_t)(a.n_slots - 1)) * a.table_stride;
}

// A row's length, as far as its block table goes (so that every walk ends: a table's row holds fewer than 2^31 - 256 keys).
__device__ __forceinline__ int length_of(const CacheArgs& a, int row) { return min(a.lens[row], a.table_stride * a.page_size); }

// The keys a row shares with its group (0: it is in none), by the lanes of a wave side by side.
__device__ __forceinline__ int shared_keys(const CacheArgs& a, int row) {
  if (a.n_groups == 0) return 0;
  int before = 0;
  for (int at = 0; at <= a.n_groups; at += WAVE) {
    const int j = at + (int)(threadIdx.x % WAVE);
    before += __popcll(__ballot(j <= a.n_groups && a.group_start[min(j, a.n_groups)] <= row));
  }
  return before >= 1 && before <= a.n_groups ? max(a.group_lens[before - 1], 0) : 0;
}

__device__ __forceinline__ int wave_least(int v) {
  v = min(v, lane_xor<32>(v));
  v = min(v, lane_xor<16>(v));
  v = min(v, lane_xor<8>(v));
  v = min(v, lane_xor<4>(v));
  v = min(v, lane_xor<2>(v));
  return min(v, lane_xor<1>(v));
}

// Whose queries a block takes, and which keys: queries qs .. qs + nq - 1 against keys from .. n - 1 of a row, the last of them at
// position n - 1; or all queries of a group's rows (up to row `end`) against the prefix of n keys. Those see it whole but where a row is
// no longer than the prefix, or begins with queries inside it: `lowest` is the smallest position of a group's query, n no more than the
// largest and one. (Lengths and starts of 64 rows are loaded together, beside the group's own: no chain of loads gets longer.)
struct Job {
  int row, slot, qs, nq, n, from, end, lowest;             // slot: the block table's row
  __device__ __forceinline__ bool apart() const { return lowest < n - 1; }      // (of a group) some query does not see all n keys
};
__device__ __forceinline__ Job job_of(const CacheArgs& a, int by_group, int at) {
  Job j;
  j.end = j.lowest = 0;
  if (by_group) {
    j.row = a.group_start[at];
    j.end = a.group_start[at + 1];
    j.qs = a.qstart[j.row];
    j.n = a.group_lens[at];
    j.slot = a.slots[min(j.row, a.rows - 1)];              // (asked for with the rest: the walk's chain of loads begins at it)
    j.nq = j.end > j.row && j.n > 0 ? a.qstart[j.end] - j.qs : 0;
    j.from = 0;
    int low = 0x7fffffff, high = -1;
    for (int at64 = j.row; at64 < j.end; at64 += WAVE) {
      const int r = min(at64 + (int)(threadIdx.x % WAVE), j.end - 1), n = length_of(a, r), queries = a.qstart[r + 1] - a.qstart[r];
      low = min(low, queries > 0 ? n - queries : low);
      high = max(high, queries > 0 ? n - 1 : high);
    }
    j.lowest = __builtin_amdgcn_readfirstlane(wave_least(low));
    j.n = min(j.n, 1 - __builtin_amdgcn_readfirstlane(wave_least(-high)));
  } else {
    const bool in_order = a.row_ids == nullptr;            // rows of one query, one a token, from the first on
    j.row = in_order ? at : a.row_ids[at];
    j.qs = in_order ? at : a.qstart[j.row];
    j.nq = in_order ? 1 : a.qstart[j.row + 1] - j.qs;
    j.n = length_of(a, j.row);
    j.slot = a.slots[j.row];
    j.from = shared_keys(a, j.row);
  }
  return j;
}

// The position of a token of a group's rows: its row is the last that begins at it or in front of it.
__device__ __forceinline__ int position_in_group(const CacheArgs& a, const Job& j, int token) {
  int row = j.row, end = j.end;
  while (end - row > 1) {
    const int mid = row + (end - row) / 2;
    if (a.qstart[mid] <= token) row = mid;
    else end = mid;
  }
  return length_of(a, row) - (a.qstart[row + 1] - token);
}

// Decode rows of different lengths: as many blocks for each as its keys are of all rows' keys, so that blocks have about the same to
// do whatever the lengths are. With `units` the blocks of 64 keys that a row sees, a block takes `per` of them and a row
// ceil(units / per) blocks (one at least), per the least, as far as eight steps find it, for which all rows' blocks are within the
// budget. Every wave works it out for itself, lane r row r, and has what it needs of the row then.
struct RowShares {
  int row, n, slot;            // lane r: row r of the launch
  int per, blocks, upto;       // a block's units; lane r: row r's blocks, and those of all rows up to it
  __device__ __forceinline__ explicit RowShares(const CacheArgs& a) {
    const int r = threadIdx.x % WAVE, here = min(r, a.n_rows - 1);
    row = a.row_ids == nullptr ? here : a.row_ids[here];
    n = length_of(a, row);
    slot = a.slots[row];
    const int units = r < a.n_rows && n > 0 ? (n - 1) / 64 - max(0, first_seen(n - 1, a.window)) / 64 + 1 : 0;
    // (A sum past 2^24 is rounded; one step makes `per` large enough then: never more than budget + n_rows blocks, the launch's.)
    per = max(1, (int)ceilf(wave_sum((float)units) / (float)a.budget));
    for (int step = 0; step < 8; ++step) {
      blocks = r < a.n_rows ? max(1, (units + per - 1) / per) : 0;
      if (wave_sum((float)blocks) <= (float)a.budget) break;
      per += 1 + per / 16;
    }
    upto = blocks;
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
      const int before = __shfl_up(upto, o, WAVE);
      if (r >= o) upto += before;
    }
  }
};

// Sixteen codes as 16 bfloat16 values times `power`, in order.
__device__ __forceinline__ void widen(const u32x4_t& w, float power, bf16x8_t& lo, bf16x8_t& hi) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], power, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], power, true);
    lo[4 * i] = a[0]; lo[4 * i + 1] = a[1]; lo[4 * i + 2] = b[0]; lo[4 * i + 3] = b[1];
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i + 2], power, false);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i + 2], power, true);
    hi[4 * i] = c[0]; hi[4 * i + 1] = c[1]; hi[4 * i + 2] = d[0]; hi[4 * i + 3] = d[1];
  }
}

// x as the sum of PARTS bfloat16 numbers: its rounding, and the rounding of what is left.
template <int PARTS>
__device__ __forceinline__ void split(float x, __bf16 (&to)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    to[i] = (__bf16)x;
    x -= (float)to[i];
  }
}

// Whether a bfloat16 pair or a word of codes holds what is not finite.
template <bool Q8> __device__ __forceinline__ bool not_finite(uint32_t w) {
  if constexpr (Q8) return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
  else return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// A wave's tiles of 16 columns and where their sums stand.
template <int D, int NT>
struct Tiles {
  f32x4_t o[NT][D / 16];       // O^T: dims 16 ds + 4 g + r of column c
  float m[NT], l[NT];          // the largest score so far (in units of log2), this lane's share of the sum
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds) o[t][ds] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// What a column is: a token's head.
struct Column {
  bool valid;
  int token, head, pos;
};
__device__ __forceinline__ Column column_of(const CacheArgs& a, int f, int hk, int group, int qs, int nq, int n) {
  const int qi = f / group, hi = f - qi * group;
  Column r;
  r.token = qs + qi;
  r.valid = qi < nq && (uint32_t)r.token < (uint32_t)a.n_tokens;
  r.head = hk * group + hi;
  r.pos = r.valid ? n - nq + qi : -1;
  return r;
}

// Rows of few queries: every wave has keys of its own, read from the cache straight into the operands' registers.
//   S^T = K Q^T: A = 16 keys x 32 dims. A block of KB keys is cut into four runs of KB / 4, run g for lane group g: row i of
//   the j-th product is key KB/4 * (i / 4) + 4 j + i % 4, so that lane group g ends up with the scores of its run, in order.
//   O^T = V^T P^T: A = 16 dims x 32 keys straight from the transposed values (a run is one 16-byte load), B = the probabilities.
// Codes: KB = 64, and a lane's 16-byte load of a key is 16 dims, its first 8 the operand of one product and its last 8 of the
// next; the queries lie the same way. bfloat16: KB = 32.
// Memory bounds it behind long contexts, a chain of loads (length and slot, table, keys, values) behind short ones. 32 heads over 8 of
// 128: 8 rows of up to 32,768 keys of 8 bits 74 us and the merge 7 (4.9 TB/s), 64 of 4,096 102 with it (5.3), of bfloat16 180 (5.9); one
// row of 300 7.8.
// Waves a block at most: eight where a lane needs no more than 256 registers.
constexpr int most_waves(int D, bool f32, int NT) { return D == 256 || f32 || NT > 1 ? 4 : 8; }

// Whether a wave may take two tiles of columns: what they hold then fits its registers.
constexpr bool two_tiles(int D, bool f32) { return D <= 128 && !f32; }

// `at`: which tiles of columns and which share of the keys; `red`: (waves - 1) * NT * (16 D + 32) numbers of LDS.
template <int D, bool Q8, typename QT, int NT>
__device__ __forceinline__ void rows_block(const CacheArgs& a, int by_group, int max_query, int at, int hk, int ri, float* red) {
  constexpr int PARTS = std::is_same<QT, float>::value ? 3 : 1;
  constexpr int KB = Q8 ? 64 : 32, RUN = KB / 4, SCORES = KB / 16, PV = KB / 32;
  constexpr int KLOADS = Q8 ? D / 64 : D / 32;             // 16-byte loads of a key's share
  constexpr int PART = 16 * D + 32;                        // [waves - 1][NT][16 D values, 16 maxima, 16 sums]
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, waves = blockDim.x / WAVE;
  const int g = lane / 16, c = lane % 16;
  const int group = a.heads / a.kv_heads, P = a.page_size;
  const int out_splits = a.budget ? a.budget + a.n_rows : a.splits / waves;
  const int tile0 = at / out_splits * NT;
  int piece = at % out_splits, pieces = a.parts, per = 0;
  const int nth = piece;
  Job job;
  if (a.budget) {
    const RowShares shares(a);
    const uint64_t rows_to_go = __ballot(shares.upto > nth);
    if (rows_to_go == 0) return;                           // (the same for the whole block)
    ri = __ffsll((unsigned long long)rows_to_go) - 1;
    pieces = __builtin_amdgcn_readlane(shares.blocks, ri);
    piece = nth - (__builtin_amdgcn_readlane(shares.upto, ri) - pieces);
    per = shares.per;
    job.row = __builtin_amdgcn_readlane(shares.row, ri);
    job.n = __builtin_amdgcn_readlane(shares.n, ri);
    job.slot = __builtin_amdgcn_readlane(shares.slot, ri);
    job.qs = a.row_ids == nullptr ? job.row : a.qstart[job.row];
    job.nq = a.row_ids == nullptr ? 1 : a.qstart[job.row + 1] - job.qs;
    job.from = job.end = job.lowest = 0;
    if (piece == 0 && tile0 == 0 && hk == 0 && threadIdx.x == 0) a.row_parts[ri] = int2{nth, pieces};      // (for the merge)
  } else {
    job = job_of(a, by_group, ri);
  }
  const int qs = job.qs, nq = job.nq, n = job.n, from = job.from;
  const bool apart = by_group && job.apart();
  if (tile0 * 16 >= nq * group || (!by_group && nq > max_query)) return;      // (the same for the whole block)
  Column col[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    col[t] = column_of(a, (tile0 + t) * 16 + c, hk, group, qs, nq, n);
    if (by_group && col[t].valid) col[t].pos = apart ? position_in_group(a, job, col[t].token) : n - 1;
  }
  // the tiles' first and last positions (of a group's queries: all tiles')
  const int pos_first = by_group ? min(job.lowest, n - 1) : n - nq + tile0 * 16 / group;
  const int pos_last = by_group ? n - 1 : n - nq + min((tile0 + NT) * 16 - 1, nq * group - 1) / group;
  const int first = max(from, first_seen(pos_first, a.window)), whole_from = max(from, first_seen(pos_last, a.window));
  // a wave's keys: an equal share of the row's, or of its block's
  const int base = a.budget ? first / 64 * 64 : first / KB * KB;
  const int share = a.budget ? (per * 64 + waves * KB - 1) / (waves * KB) * KB
                             : max(KB, ((pos_last - base + a.splits) / a.splits + KB - 1) / KB * KB);
  const int key_lo = base + (a.budget ? piece * per * 64 + wave * share : (piece * waves + wave) * share);
  const int key_hi = min(min(pos_last, key_lo + share - 1), a.budget ? base + (piece + 1) * per * 64 - 1 : 0x7fffffff);
  int from_here[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) from_here[t] = max(from, first_seen(col[t].pos, a.window));

  Tiles<D, NT> tl;
  tl.clear();
  if (key_lo <= key_hi) {
    const int32_t* trow = table_at(a, job.slot);
    const int max_page = a.table_stride - 1;
    const int bytes = Q8 ? 1 : 2;
    const int64_t plane = (int64_t)P * D * bytes;
    const int krun = RUN * (c / 4);                        // this lane's keys: krun + c % 4 + 4 j; its values: RUN g ..
    // Everything that a block of keys needs is asked for while the block before it is multiplied, the table's entries a block
    // earlier still: a wave's loads come back in order, so none may wait for one asked for just now.
    struct Keys {
      u32x4_t raw[SCORES][KLOADS], power;
    };
    const auto look = [&](int kb, int32_t& ek, int32_t& ev) {
      ek = trow[min(page_index(a, kb + krun), max_page)];
      ev = trow[min(page_index(a, kb + RUN * g), max_page)];
    };
    const auto load_keys = [&](int kb, int32_t ek, Keys& to) {
      const int at = kb + krun - page_index(a, kb + krun) * P;
      const int64_t page = page_at(a, ek);
      const uint8_t* p = a.pages + page * a.page_stride + hk * plane + (int64_t)(at + c % 4) * D * bytes + 16 * g;
#pragma unroll
      for (int j = 0; j < SCORES; ++j)
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) to.raw[j][i] = *reinterpret_cast<const u32x4_t*>(p + 4 * j * D * bytes + 64 * i);
      if constexpr (Q8) to.power = *reinterpret_cast<const u32x4_t*>(a.scales + page * a.scale_stride + (int64_t)hk * P + at);
    };
    int32_t ek, ev, ek_next, ev_next;
    Keys keys;
    look(key_lo, ek, ev);
    look(key_lo + KB, ek_next, ev_next);
    bf16x8_t qf[NT][PARTS][D / 32];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const QT* qp = (const QT*)a.q + ((int64_t)col[t].token * a.heads + col[t].head) * D;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        const int d0 = Q8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
        if constexpr (PARTS == 1) {
          u32x4_t x = {0, 0, 0, 0};
          if (col[t].valid) x = *reinterpret_cast<const u32x4_t*>(qp + d0);
          qf[t][0][ks] = __builtin_bit_cast(bf16x8_t, x);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            f32x4_t x = {0.f, 0.f, 0.f, 0.f};
            if (col[t].valid) x = *reinterpret_cast<const f32x4_t*>(qp + d0 + i);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              __bf16 p[PARTS];
              split<PARTS>(x[r], p);
#pragma unroll
              for (int s = 0; s < PARTS; ++s) qf[t][s][ks][i + r] = p[s];
            }
          }
        }
      }
    }
    load_keys(key_lo, ek, keys);
    for (int kb = key_lo; kb <= key_hi; kb += KB) {
      const int vk = kb + RUN * g;
      u32x4_t vraw[D / 16], vs4 = {};
      {
        const int at = vk - page_index(a, vk) * P;
        const int64_t page = page_at(a, ev);
        const uint8_t* p = a.pages + page * a.page_stride + (a.kv_heads + hk) * plane + ((int64_t)c * P + at) * bytes;
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds) vraw[ds] = *reinterpret_cast<const u32x4_t*>(p + (int64_t)ds * 16 * P * bytes);
        if constexpr (Q8) vs4 = *reinterpret_cast<const u32x4_t*>(a.scales + page * a.scale_stride + (int64_t)(a.kv_heads + hk) * P + at);
      }
      Keys next;
      if (kb + KB <= key_hi) {
        load_keys(kb + KB, ek_next, next);
        ev = ev_next;
        if (kb + 2 * KB <= key_hi) look(kb + 2 * KB, ek_next, ev_next);
      }
      const bool whole = kb >= whole_from && kb + KB - 1 <= min(pos_first, key_hi);
      f32x4_t sc[NT][SCORES];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < SCORES; ++j) sc[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < SCORES; ++j) {
        const float power = Q8 ? q8_power((keys.power[j] >> (8 * (c % 4))) & 0xffu) : 1.f;
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) {
          bf16x8_t f[Q8 ? 2 : 1];
          if constexpr (Q8) widen(keys.raw[j][i], power, f[0], f[1]);
          else f[0] = __builtin_bit_cast(bf16x8_t, keys.raw[j][i]);
#pragma unroll
          for (int u = 0; u < (Q8 ? 2 : 1); ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int s = 0; s < PARTS; ++s)
                sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[u], qf[t][s][Q8 ? 2 * i + u : i], sc[t][j], 0, 0, 0);
        }
      }
      // What lies outside the keys that the tiles' last query sees is not the row's, or not kept: no value, no scale of it
      // may reach a sum, not even times zero.
      if (!whole) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t keep = 0, keep_scale = 0;
#pragma unroll
          for (int e = 0; e < (Q8 ? 4 : 2); ++e) {
            const int key = vk + (Q8 ? 4 : 2) * w + e;
            const bool in = key >= first && key <= key_hi;
            keep |= in ? (Q8 ? 0xffu << (8 * e) : 0xffffu << (16 * e)) : 0u;
          }
          keep_scale = keep;
          if constexpr (Q8) vs4[w] &= keep_scale;
#pragma unroll
          for (int ds = 0; ds < D / 16; ++ds) vraw[ds][w] &= keep;
        }
      }
      bf16x8_t pb[NT][PV][PARTS];
      float alpha[NT];
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sv[RUN];
#pragma unroll
        for (int i = 0; i < RUN; ++i) sv[i] = sc[t][i / 4][i % 4];
        if (!whole) {
#pragma unroll
          for (int i = 0; i < RUN; ++i) {
            const int key = vk + i;
            if (!(key <= col[t].pos && key >= from_here[t] && key <= key_hi)) sv[i] = -INFINITY;
          }
        }
        float mx = sv[0];
#pragma unroll
        for (int i = 1; i < RUN; ++i) mx = fmaxf(mx, sv[i]);
        mx = xor_max<16>(mx);
        mx = xor_max<32>(mx);
        const float top = mx * a.scale_log2;
        const bool move = __any(top > tl.m[t]);
        const float m_new = move ? fmaxf(tl.m[t], top) : tl.m[t], m_use = m_new == -INFINITY ? 0.f : m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          float p = __builtin_amdgcn_exp2f(fmaf(sv[i], a.scale_log2, -m_use));
          sum += p;
          if constexpr (Q8) p *= q8_power((vs4[i / 4] >> (8 * (i % 4))) & 0xffu);
          __bf16 pp[PARTS];
          split<PARTS>(p, pp);
#pragma unroll
          for (int s = 0; s < PARTS; ++s) pb[t][i / 8][s][i % 8] = pp[s];
        }
        alpha[t] = move ? __builtin_amdgcn_exp2f(tl.m[t] - m_use) : 1.f;
        moved |= move;
        tl.m[t] = m_new;
        tl.l[t] = tl.l[t] * alpha[t] + sum;
      }
      if (moved) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int ds = 0; ds < D / 16; ++ds) tl.o[t][ds] *= alpha[t];
      }
      // Where queries of the tiles see different keys, a value that is not finite reaches those alone that see it: it leaves
      // the product (zero times it is no number) and sets their sums by itself.
      if (!whole && nq > 1 && (!by_group || apart)) {
        bool odd = false;
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds)
#pragma unroll
          for (int w = 0; w < 4; ++w) odd |= not_finite<Q8>(vraw[ds][w]);
        if (__any(odd)) {
#pragma unroll
          for (int ds = 0; ds < D / 16; ++ds) {
            uint32_t up[4 * PV], down[4 * PV];             // bfloat16 ones where the value is +inf or NaN, -inf or NaN
            constexpr int EACH = Q8 ? 4 : 2;
#pragma unroll
            for (int i = 0; i < 4 * PV; ++i) up[i] = down[i] = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
              for (int e = 0; e < EACH; ++e) {
                const int shift = (Q8 ? 8 : 16) * e, i = EACH * w + e;
                const uint32_t v = vraw[ds][w] >> shift & (Q8 ? 0xffu : 0xffffu), size = v & (Q8 ? 0x7fu : 0x7fffu);
                const bool gone = size >= (Q8 ? 0x7fu : 0x7f80u), nan = Q8 || size > 0x7f80u;
                if (gone) {
                  vraw[ds][w] &= ~((Q8 ? 0xffu : 0xffffu) << shift);
                  if (nan || !(v & 0x8000u)) up[i / 2] |= 0x3f80u << (16 * (i % 2));
                  if (nan || (v & 0x8000u)) down[i / 2] |= 0x3f80u << (16 * (i % 2));
                }
              }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              f32x4_t ups = {0.f, 0.f, 0.f, 0.f}, downs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int u = 0; u < PV; ++u) {
                const u32x4_t a0 = {up[4 * u], up[4 * u + 1], up[4 * u + 2], up[4 * u + 3]};
                const u32x4_t a1 = {down[4 * u], down[4 * u + 1], down[4 * u + 2], down[4 * u + 3]};
                ups = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a0), pb[t][u][0], ups, 0, 0, 0);
                downs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a1), pb[t][u][0], downs, 0, 0, 0);
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                if (ups[r] > 0.f) tl.o[t][ds][r] += INFINITY;
                if (downs[r] > 0.f) tl.o[t][ds][r] -= INFINITY;
              }
            }
          }
        }
      }
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds) {
        bf16x8_t f[PV];
        if constexpr (Q8) widen(vraw[ds], 1.f, f[0], f[1]);
        else f[0] = __builtin_bit_cast(bf16x8_t, vraw[ds]);
#pragma unroll
        for (int u = 0; u < PV; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int s = 0; s < PARTS; ++s)
              tl.o[t][ds] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[u], pb[t][u][s], tl.o[t][ds], 0, 0, 0);
      }
      keys = next;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) tl.l[t] = xor_sum<32>(xor_sum<16>(tl.l[t]));
  if (waves > 1) {                                         // the block's partial sums, added up in wave order by wave 0
    if (wave > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float* mine = red + (int64_t)((wave - 1) * NT + t) * PART;
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds) *reinterpret_cast<f32x4_t*>(mine + (ds * WAVE + lane) * 4) = tl.o[t][ds];
        if (g == 0) { mine[16 * D + c] = tl.m[t]; mine[16 * D + 16 + c] = tl.l[t]; }
      }
    }
    __syncthreads();
    if (wave > 0) return;
    for (int w = 1; w < waves; ++w) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float* theirs = red + (int64_t)((w - 1) * NT + t) * PART;
        const float mw = theirs[16 * D + c], lw = theirs[16 * D + 16 + c];
        const float m_new = fmaxf(tl.m[t], mw), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float mine = __builtin_amdgcn_exp2f(tl.m[t] - m_use), other = __builtin_amdgcn_exp2f(mw - m_use);
        tl.l[t] = tl.l[t] * mine + lw * other;
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds)
          tl.o[t][ds] = tl.o[t][ds] * mine + *reinterpret_cast<const f32x4_t*>(theirs + (ds * WAVE + lane) * 4) * other;
        tl.m[t] = m_new;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (!col[t].valid) continue;
    if (pieces == 1) {
      float l = tl.l[t];
      if (a.sink != nullptr && tl.m[t] != -INFINITY) l += exp2f(a.sink[col[t].head] * 1.4426950408889634f - tl.m[t]);
      const float inv = l == 0.f ? 0.f : 1.0f / l;         // (a NaN stays one)
      QT* op = (QT*)a.out + ((int64_t)col[t].token * a.heads + col[t].head) * D + 4 * g;
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds)
#pragma unroll
        for (int r = 0; r < 4; ++r) op[16 * ds + r] = Elem<QT>::store(tl.o[t][ds][r] * inv);
    } else {
      const int64_t place = a.cell_queries > 0 ? (int64_t)ri * a.cell_queries + (col[t].token - qs) : col[t].token;
      const int64_t cell = a.budget ? (int64_t)nth * a.heads + col[t].head : (place * a.heads + col[t].head) * a.parts + a.part_first + piece;
      float* po = a.part_o + cell * D + 4 * g;
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds) *reinterpret_cast<f32x4_t*>(po + 16 * ds) = tl.o[t][ds];
      if (g == 0) { a.part_ml[2 * cell] = tl.m[t]; a.part_ml[2 * cell + 1] = tl.l[t]; }
      if (a.part_first > 0 && from == 0 && piece == 0) {   // no prefix: its parts are another launch's, which leaves this row out
        const int64_t none = (place * a.heads + col[t].head) * a.parts;
        for (int i = g; i < a.part_first; i += 4) { a.part_ml[2 * (none + i)] = -INFINITY; a.part_ml[2 * (none + i) + 1] = 0.f; }
      }
    }
  }
}

// Many columns over the same keys: a portion's queries, or all queries of a group's rows over their prefix. A block of four waves
// takes 128 columns, a wave 32 on v_mfma_f32_32x32x16_bf16, and walks the keys in stages of 32, which its threads bring into LDS
// as bfloat16 (codes are widened once a block, not once a wave): three buffers, the stage after the next on its way in registers.
//   S^T (32 keys x 32 columns): A = 32 keys x 16 dims: lane (h, c) reads row c of the stage's keys, dims 8 h .. + 7 of 16. Row
//     8 i + 4 h + r holds key 16 (i / 2) + 8 h + 4 (i % 2) + r, so that a lane's 16 scores are, in order, those of keys 8 h .. + 7
//     of the stage's first 16 and of its last: the B operands of
//   O^T (32 dims x 32 columns) += V^T P^T: A = 32 dims x 16 keys, the values transposed as in the pages.
// Rows of LDS are swizzled by pieces of 16 bytes, so that 16 lanes that read one piece of 16 rows touch every bank once.
// A wave's own chain bounds it, scores, softmax, products, with two waves a SIMD: 32 heads over 8 of 128, 2,048 tokens behind 6,144 335
// us over codes and 296 over bfloat16 (0.72, 0.81 PFLOP/s), 4,096 behind 28,672 0.83 and 0.94. The next stage's scores beside this one's
// softmax would need more registers than there are (spilled: 498 us), and a second stage ahead in registers brings nothing (407).
constexpr float SLACK = 8.f;   // see where it is used

template <int D, bool Q8, int WAVES>
struct Stage {
  static constexpr int K_BYTES = 32 * D * 2, BYTES = 2 * K_BYTES, THREADS = WAVES * WAVE;
  static constexpr int HALF = Q8 ? 2 * D : 4 * D;          // 16-byte loads of keys in all, and as many of values behind them
  static constexpr int N = (2 * HALF + THREADS - 1) / THREADS;      // of a thread
  // A load reads one half of the stage, 16 keys of one page, the same one for all lanes of its wave; where a thread has four loads and
  // more, which half is known here, else a wave's loads share theirs.
  static constexpr bool ONE_HALF = HALF / 2 % THREADS != 0;
  u32x4_t w[N];
  uint32_t ks[N];                                          // a key's scale; in 16 threads of each half's, a value's

  static __device__ __forceinline__ int row_of(int key) { return 8 * (2 * (key / 16) + key % 8 / 4) + 4 * (key % 16 / 8) + key % 4; }
  static __device__ __forceinline__ int swizzle(int row) { return D == 64 ? row / 2 % 8 : row % 16; }
  static __device__ __forceinline__ int half_of(int i) {
    return ONE_HALF ? __builtin_amdgcn_readfirstlane((threadIdx.x + THREADS * i) % HALF / (HALF / 2)) : THREADS * i % HALF / (HALF / 2);
  }

  // The table's entries of the stage at kb that a wave needs.
  static __device__ __forceinline__ void look(const CacheArgs& a, const int32_t* trow, int kb, int32_t (&e)[2]) {
    const int last = a.table_stride - 1;
    if constexpr (ONE_HALF) {
      e[0] = trow[min(page_index(a, kb + 16 * half_of(0)), last)];
    } else {
      e[0] = trow[min(page_index(a, kb), last)];
      e[1] = trow[min(page_index(a, kb + 16), last)];
    }
  }
  // Asks for it: what a lane adds to its load's base is the same for every stage.
  __device__ __forceinline__ void load(const CacheArgs& a, int hk, int kb, const int32_t (&e)[2]) {
    constexpr int B = Q8 ? 1 : 2;
    const uint32_t P = a.page_size, plane = P * D * B;
    const uint8_t* keys[2];
    const uint8_t* values[2];
    const uint8_t* powers[2];
#pragma unroll
    for (int x = 0; x < (ONE_HALF ? 1 : 2); ++x) {
      const int from = kb + 16 * (ONE_HALF ? half_of(0) : x);
      const uint32_t off = from - page_index(a, from) * P;
      const uint64_t page = min((uint32_t)__builtin_amdgcn_readfirstlane(e[x]), (uint32_t)(a.num_pages - 1));
      const uint8_t* base = a.pages + page * (uint32_t)a.page_stride;
      keys[x] = base + (hk * plane + off * (D * B));
      values[x] = base + ((a.kv_heads + hk) * plane + off * B);
      if constexpr (Q8) powers[x] = a.scales + page * (uint32_t)a.scale_stride + (hk * P + off);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = threadIdx.x + THREADS * i, x = ONE_HALF ? 0 : half_of(i);
      if (2 * HALF % THREADS != 0 && idx >= 2 * HALF) break;
      if (idx < HALF) {
        constexpr int CH = D * B / 16;
        const uint32_t key = idx / CH % 16;
        w[i] = *reinterpret_cast<const u32x4_t*>(keys[x] + (key * (D * B) + idx % CH * 16));
        if constexpr (Q8) ks[i] = powers[x][key];
      } else {
        const uint32_t v = idx - HALF, dim = v % D, piece = v / D;
        w[i] = *reinterpret_cast<const u32x4_t*>(values[x] + (dim * (P * B) + piece % B * 16));
        if constexpr (Q8) {
          if (dim < 16) ks[i] = powers[x][a.kv_heads * P + dim];
        }
      }
    }
  }
  // Puts it into LDS. Values of keys outside [lo, hi] are cleared (they are not the row's). `watch`: so are values that are not
  // finite, and `up` and `down` (a word a dim, a bit a key) say where those were that are +inf or NaN, -inf or NaN; the
  // answer is whether there were any.
  __device__ __forceinline__ bool store(unsigned char* lds, float* powers, uint8_t* up, uint8_t* down, int kb, int lo, int hi, bool watch) {
    const int tid = threadIdx.x;
    const bool edge = kb < lo || kb + 31 > hi;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + THREADS * i;
      if (2 * HALF % THREADS != 0 && idx >= 2 * HALF) break;
      if (idx < HALF) {
        constexpr int CH = D * (Q8 ? 1 : 2) / 16;
        const int row = row_of(idx / CH), ch = idx % CH;
        unsigned char* to = lds + row * (2 * D);
        if constexpr (Q8) {
          bf16x8_t x, y;
          widen(w[i], q8_power(ks[i]), x, y);
          *reinterpret_cast<bf16x8_t*>(to + 16 * ((2 * ch) ^ swizzle(row))) = x;
          *reinterpret_cast<bf16x8_t*>(to + 16 * ((2 * ch + 1) ^ swizzle(row))) = y;
        } else {
          *reinterpret_cast<u32x4_t*>(to + 16 * (ch ^ swizzle(row))) = w[i];
        }
      } else {
        const int v = idx - HALF, dim = v % D, piece = v / D;
        if (edge) {
          const int key = kb + piece * (Q8 ? 16 : 8);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t keep = 0;
#pragma unroll
            for (int e = 0; e < (Q8 ? 4 : 2); ++e) {
              const int k = key + (Q8 ? 4 : 2) * x + e;
              keep |= k >= lo && k <= hi ? (Q8 ? 0xffu << (8 * e) : 0xffffu << (16 * e)) : 0u;
            }
            w[i][x] &= keep;
          }
        }
        if (watch) {
          uint32_t ups = 0, downs = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int e = 0; e < (Q8 ? 4 : 2); ++e) {
              const int shift = (Q8 ? 8 : 16) * e, k = (Q8 ? 4 : 2) * x + e;
              const uint32_t v = w[i][x] >> shift & (Q8 ? 0xffu : 0xffffu), size = v & (Q8 ? 0x7fu : 0x7fffu);
              if (size < (Q8 ? 0x7fu : 0x7f80u)) continue;
              w[i][x] &= ~((Q8 ? 0xffu : 0xffffu) << shift);
              if (Q8 || size > 0x7f80u || !(v & 0x8000u)) ups |= 1u << k;
              if (Q8 || size > 0x7f80u || (v & 0x8000u)) downs |= 1u << k;
            }
          odd |= (ups | downs) != 0;
          if constexpr (Q8) {
            *reinterpret_cast<uint16_t*>(up + 4 * dim + 2 * piece) = (uint16_t)ups;
            *reinterpret_cast<uint16_t*>(down + 4 * dim + 2 * piece) = (uint16_t)downs;
          } else {
            up[4 * dim + piece] = (uint8_t)ups;
            down[4 * dim + piece] = (uint8_t)downs;
          }
        }
        const int half = Q8 ? piece : piece / 2;
        unsigned char* to = lds + K_BYTES + half * (K_BYTES / 2) + dim * 32;
        const int turn = dim / 8 % 2;
        if constexpr (Q8) {
          bf16x8_t x, y;
          if (dim < 16) {                                  // (key `dim` of the half: its power)
            const int key = kb + 16 * piece + dim;
            powers[16 * piece + dim] = key >= lo && key <= hi ? q8_power(ks[i]) : 0.f;
          }
          widen(w[i], 1.f, x, y);
          *reinterpret_cast<bf16x8_t*>(to + 16 * turn) = x;
          *reinterpret_cast<bf16x8_t*>(to + 16 * (1 ^ turn)) = y;
        } else {
          *reinterpret_cast<u32x4_t*>(to + 16 * (piece % 2 ^ turn)) = w[i];
        }
      }
    }
    return odd;
  }
  static __device__ __forceinline__ bf16x8_t key(const unsigned char* lds, int ds) {
    const int lane = threadIdx.x % WAVE, h = lane / 32, c = lane % 32;
    return *reinterpret_cast<const bf16x8_t*>(lds + c * (2 * D) + 16 * ((2 * ds + h) ^ swizzle(c)));
  }
  static __device__ __forceinline__ bf16x8_t value(const unsigned char* lds, int db, int half) {
    const int lane = threadIdx.x % WAVE, h = lane / 32, c = lane % 32;
    return *reinterpret_cast<const bf16x8_t*>(lds + K_BYTES + half * (K_BYTES / 2) + (32 * db + c) * 32 + 16 * (h ^ (c / 8 % 2)));
  }
};

template <int D, bool Q8, int WAVES>
struct TilesLds {
  __attribute__((aligned(1024))) unsigned char stage[3][Stage<D, Q8, WAVES>::BYTES];
  __attribute__((aligned(16))) float powers[3][32];
  uint32_t ups[3][D], downs[3][D];
  int odd_stage[3];                                        // the key of a stage with values that are not finite
};

// `at`: which columns (of `blocks` / a.splits tiles of them) and which share of the keys.
template <int D, bool Q8, int WAVES>
__device__ __forceinline__ void tiles_block(const CacheArgs& a, int by_group, int less_than, int folded, int at, int blocks, int hk, int ri,
                                            TilesLds<D, Q8, WAVES>& sh) {
  using S = Stage<D, Q8, WAVES>;
  constexpr int COLUMNS = 32 * WAVES;
  auto& lds = sh.stage;
  auto& powers = sh.powers;
  auto& ups = sh.ups;
  auto& downs = sh.downs;
  auto& odd_stage = sh.odd_stage;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE, h = lane / 32, c = lane % 32;
  const int piece = at % a.splits, group = a.heads / a.kv_heads;
  // The last columns' walks are the longest: they begin. Where all blocks run at once, two a compute unit, the second half begins
  // with the shortest, so that the two that share a unit have about the same to do together.
  const int tiles = blocks / a.splits, nth = at / a.splits;
  const int tile = folded && nth >= (tiles + 1) / 2 ? nth - (tiles + 1) / 2 : tiles - 1 - nth;
  const Job job = job_of(a, by_group, ri);
  const int qs = job.qs, nq = job.nq, n = job.n, from = job.from;
  const int columns = nq * group;
  if (tile * COLUMNS >= columns || (!by_group && nq <= less_than)) return;
  const int f0 = tile * COLUMNS + 32 * wave, f = f0 + c;
  Column col = column_of(a, f, hk, group, qs, nq, n);
  const int behind = n - nq;                               // the first query's position
  const int pos_first = by_group ? min(job.lowest, n - 1) : behind + tile * COLUMNS / group;
  const int pos_last = by_group ? n - 1 : behind + min(tile * COLUMNS + COLUMNS - 1, columns - 1) / group;
  if (by_group && col.valid) col.pos = job.apart() ? position_in_group(a, job, col.token) : n - 1;
  const int tile_first = by_group ? pos_first : behind + f0 / group;
  const int tile_last = f0 >= columns ? -1 : by_group ? n - 1 : behind + min(f0 + 31, columns - 1) / group;
  const int first = max(from, first_seen(pos_first, a.window)), whole_from = max(from, first_seen(tile_last, a.window));
  const int from_here = max(from, first_seen(col.pos, a.window));
  const int base = first / 32 * 32;
  const int share = max(32, ((pos_last - base + a.splits) / a.splits + 31) / 32 * 32);
  const int lo = max(base + piece * share, first), hi = min(pos_last, base + piece * share + share - 1);

  f32x16_t o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (lo <= hi) {
    bf16x8_t qf[D / 16];
    const bf16_t* qp = (const bf16_t*)a.q + ((int64_t)col.token * a.heads + col.head) * D + 8 * h;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) {
      u32x4_t x = {0, 0, 0, 0};
      if (col.valid) x = *reinterpret_cast<const u32x4_t*>(qp + 16 * ds);
      qf[ds] = __builtin_bit_cast(bf16x8_t, x);
    }
    const int32_t* trow = table_at(a, job.slot);
    // queries of the block see different keys from here on, or up to here
    const int seen_last = first_seen(pos_last, a.window), seen_tile = a.window ? first_seen(tile_first, a.window) : 0;
    const auto differs = [&](int kb) { return kb + 31 > pos_first || kb < seen_last; };
    const int kb_first = lo / 32 * 32;
    const auto store = [&](S& s, int kb, int buf) {
      if (s.store(lds[buf], powers[buf], (uint8_t*)ups[buf], (uint8_t*)downs[buf], kb, lo, hi, differs(kb))) odd_stage[buf] = kb;
    };
    if (threadIdx.x < 3) odd_stage[threadIdx.x] = -1;
    S coming;
    int32_t e[2];
    {
      S first_stage;
      S::look(a, trow, kb_first, e);
      first_stage.load(a, hk, kb_first, e);
      if (kb_first + 32 <= hi) {
        S::look(a, trow, kb_first + 32, e);
        coming.load(a, hk, kb_first + 32, e);
      }
      if (kb_first + 64 <= hi) S::look(a, trow, kb_first + 64, e);
      lds_barrier();
      store(first_stage, kb_first, 0);
      if (kb_first + 32 <= hi) store(coming, kb_first + 32, 1);
    }
    lds_barrier();
    int buf = 0;
    for (int kb = kb_first; kb <= hi; kb += 32) {
      if (kb + 64 <= hi) {
        coming.load(a, hk, kb + 64, e);
        if (kb + 96 <= hi) S::look(a, trow, kb + 96, e);
      }
      const unsigned char* st = lds[buf];
      if (kb <= tile_last && kb + 31 >= seen_tile) {
        f32x16_t sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
        constexpr int AT_ONCE = D / 16 < 8 ? D / 16 : 8;
#pragma unroll
        for (int d0 = 0; d0 < D / 16; d0 += AT_ONCE) {
          bf16x8_t kf[AT_ONCE];
#pragma unroll
          for (int ds = 0; ds < AT_ONCE; ++ds) kf[ds] = S::key(st, d0 + ds);
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int ds = 0; ds < AT_ONCE; ++ds) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ds], qf[d0 + ds], sc, 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        // the values are asked for before the softmax that their products wait for
        bf16x8_t vf[D / 32][2];
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          vf[db][0] = S::value(st, db, 0);
          vf[db][1] = S::value(st, db, 1);
        }
        // score 8 t + i of this lane: key kb + 16 t + 8 h + i
        const bool whole = kb >= max(lo, whole_from) && kb + 31 <= min(hi, tile_first);
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = kb + 16 * (i / 8) + 8 * h + i % 8;
            if (!(key <= col.pos && key >= from_here && key <= hi)) sc[i] = -INFINITY;
          }
        }
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
        mx = xor_max<32>(mx);
        // The sums stand under a maximum that may lag behind by SLACK: weights up to 2^SLACK lose nothing in float32, and what was summed
        // is rescaled (64 products a lane) in a few stages, not wherever any of 32 columns meets a new largest score. What it costs: the
        // largest weight is then no 1 that rounds to itself, so that results are up to 1.4 times as far from 64 bits as float32 rounded
        // once, not 1.1 times (rounded weights are 0.0016 off on average, as a rounded result is); 2,048 tokens behind 6,144 387 -> 347
        // us over codes, 361 -> 331 over bfloat16. Sums of the rounded weights bring nothing of it back.
        const float top = mx * a.scale_log2;
        const bool move = __any(top > m + SLACK);
        const float m_new = move ? fmaxf(m, top) : m, m_use = m_new == -INFINITY ? 0.f : m_new;
        bf16x8_t pb[2];
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4_t pw[2];
          if constexpr (Q8) {
            pw[0] = *reinterpret_cast<const f32x4_t*>(&powers[buf][16 * t + 8 * h]);
            pw[1] = *reinterpret_cast<const f32x4_t*>(&powers[buf][16 * t + 8 * h + 4]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float p = __builtin_amdgcn_exp2f(fmaf(sc[8 * t + i], a.scale_log2, -m_use));
            sum += p;
            if constexpr (Q8) p *= pw[i / 4][i % 4];
            pb[t][i] = (__bf16)p;
          }
        }
        if (move) {
          const float alpha = __builtin_amdgcn_exp2f(m - m_use);
          l *= alpha;
#pragma unroll
          for (int db = 0; db < D / 32; ++db) o[db] *= alpha;
          m = m_new;
        }
        l += sum;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db][0], pb[0], o[db], 0, 0, 0);
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db][1], pb[1], o[db], 0, 0, 0);
        }
        if (odd_stage[buf] == kb) {                        // values that are not finite: to the columns that see them alone
          uint32_t seen = 0;                               // a bit a key
#pragma unroll
          for (int i = 0; i < 16; ++i) seen |= (float)pb[i / 8][i % 8] > 0.f ? 1u << (16 * (i / 8) + 8 * h + i % 8) : 0u;
          seen |= lane_xor<32>(seen);
#pragma unroll
          for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int dim = 32 * db + 8 * (i / 4) + 4 * h + i % 4;
              if (seen & ups[buf][dim]) o[db][i] += INFINITY;
              if (seen & downs[buf][dim]) o[db][i] -= INFINITY;
            }
        }
      }
      if (kb + 64 <= hi) store(coming, kb + 64, buf == 0 ? 2 : buf - 1);      // the buffer that was read a stage ago
      lds_barrier();
      buf = buf == 2 ? 0 : buf + 1;
    }
  }
  l = xor_sum<32>(l);
  if (!col.valid) return;
  if (a.parts == 1) {
    if (a.sink != nullptr && m != -INFINITY) l += exp2f(a.sink[col.head] * 1.4426950408889634f - m);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    bf16_t* op = (bf16_t*)a.out + ((int64_t)col.token * a.heads + col.head) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ushort4 w;
        w.x = float_to_bf16(o[db][4 * i + 0] * inv);
        w.y = float_to_bf16(o[db][4 * i + 1] * inv);
        w.z = float_to_bf16(o[db][4 * i + 2] * inv);
        w.w = float_to_bf16(o[db][4 * i + 3] * inv);
        *reinterpret_cast<ushort4*>(op + 32 * db + 8 * i) = w;
      }
  } else {
    const int64_t place = a.cell_queries > 0 ? (int64_t)ri * a.cell_queries + (col.token - qs) : col.token;
    const int64_t cell = (place * a.heads + col.head) * a.parts + a.part_first + piece;
    float* po = a.part_o + cell * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4_t*>(po + 32 * db + 8 * i) = f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
    if (h == 0) { a.part_ml[2 * cell] = m; a.part_ml[2 * cell + 1] = l; }
    if (a.part_first > 0 && from == 0 && piece == 0) {     // (as in the kernel above)
      const int64_t none = (place * a.heads + col.head) * a.parts;
      for (int i = h; i < a.part_first; i += 2) { a.part_ml[2 * (none + i)] = -INFINITY; a.part_ml[2 * (none + i) + 1] = 0.f; }
    }
  }
}

template <int D, bool Q8, typename QT, int NT>
__global__ void __launch_bounds__(WAVE * most_waves(D, std::is_same<QT, float>::value, NT)) cache_rows_kernel(CacheArgs a, int by_group,
                                                                                                             int max_query) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  rows_block<D, Q8, QT, NT>(a, by_group, max_query, blockIdx.x, blockIdx.y, blockIdx.z, red);
}

template <int D, bool Q8, int WAVES>
__global__ void __launch_bounds__(WAVES * WAVE, D == 256 || WAVES == 8 ? 1 : 2) cache_tiles_kernel(CacheArgs a, int by_group, int less_than,
                                                                                                   int folded) {
  __shared__ TilesLds<D, Q8, WAVES> sh;
  tiles_block<D, Q8, WAVES>(a, by_group, less_than, folded, blockIdx.y, gridDim.y, blockIdx.x, blockIdx.z, sh);
}

// Two kinds of work in one launch, blocks of the first kind first: the groups' prefixes and the rows' own keys, neither of which fills the
// GPU by itself for long (the first are few long walks, the second many short ones); or a portion's tiles and the decode rows of the
// step, which take the compute units that the shorter walks of the portion leave.
// 64 rows of 32 heads over 8 of 128, up to 512 keys of their own behind one prefix of up to 16,384, bfloat16: 52 us, in two launches 44 + 24.
template <int D, bool Q8, bool TILES, int WAVES>
__global__ void __launch_bounds__(WAVES* WAVE, D == 256 || WAVES == 8 ? 1 : 2)
    cache_both_kernel(CacheArgs p, CacheArgs r, int by_group, int less_than, int folded, int first_blocks, int jobs, int row_blocks, int max_query) {
  using Tiles = TilesLds<D, Q8, WAVES>;
  constexpr size_t ROWS = (WAVES - 1) * (16 * D + 32) * sizeof(float);
  __shared__ __attribute__((aligned(1024))) unsigned char mem[TILES && sizeof(Tiles) > ROWS ? sizeof(Tiles) : ROWS];
  const int hk = blockIdx.x % p.kv_heads, at = blockIdx.x / p.kv_heads;
  if (at < first_blocks * jobs) {
    if constexpr (TILES)
      tiles_block<D, Q8, WAVES>(p, by_group, less_than, folded, at % first_blocks, first_blocks, hk, at / first_blocks, *reinterpret_cast<Tiles*>(mem));
    else rows_block<D, Q8, bf16_t, 1>(p, by_group, 0, at % first_blocks, hk, at / first_blocks, reinterpret_cast<float*>(mem));
  } else {
    const int x = at - first_blocks * jobs;
    rows_block<D, Q8, bf16_t, 1>(r, 0, max_query, x % row_blocks, hk, x / row_blocks, reinterpret_cast<float*>(mem));
  }
}

// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over a cell's parts, in their order: D / 4 threads a (token, head). 5 to 8 us, of
// which the launch and the chain of two loads are 4.
template <int D, typename QT>
__global__ void __launch_bounds__(256) cache_merge_kernel(CacheArgs a, int max_query, int less_than, int64_t cells) {
  constexpr int LANES = D / 4;
  const int64_t at = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int d0 = 4 * (threadIdx.x % LANES);
  const int head = (int)(at % a.heads);
  int64_t token = at / a.heads, place = token, apart = 1;  // its parts lie `apart` cells from one another
  int parts = a.parts;
  if (at >= cells) return;
  // (cells by token: of no row's tokens a kernel left anything; what they hold is read beside the rows' bounds, and not written)
  const bool nobodys = !a.budget && a.cell_queries == 0 && (token < a.qstart[0] || token >= a.qstart[a.rows]);
  if (a.budget) {
    const int2 mine = a.row_parts[token];
    parts = mine.y;
    place = mine.x;
    apart = a.heads;
    if (parts <= 1) return;                                // (one block: it has written the result)
  }
  if (a.cell_queries > 0) {                                // cells by row and query
    const int ri = (int)(token / max_query), qi = (int)(token % max_query);
    const bool in_order = a.row_ids == nullptr;
    const int row = in_order ? ri : a.row_ids[ri];
    const int qs = in_order ? ri : a.qstart[row], nq = in_order ? 1 : a.qstart[row + 1] - qs;
    if (qi >= nq || nq > max_query || nq <= less_than) return;      // (a row of more queries, or of fewer, is another kernel's)
    token = qs + qi;
  }
  if (token < 0 || token >= a.n_tokens) return;
  const int64_t first = a.budget ? place * a.heads + head : (place * a.heads + head) * a.parts;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
  const float* po = a.part_o + first * D + d0;
  float big = -INFINITY;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) big = fmaxf(big, ml[i * apart].x);
  float l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float2 x = ml[i * apart];
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(po + i * apart * D);
    const float w = x.y != 0.f ? __builtin_amdgcn_exp2f(x.x - big) : 0.f;      // (a sum of 0: it saw no key, and left nothing else)
    l += x.y != 0.f ? w * x.y : 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] += x.y != 0.f ? w * v[r] : 0.f;
  }
  if (a.sink != nullptr && big != -INFINITY) l += exp2f(a.sink[head] * 1.4426950408889634f - big);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (nobodys) return;
  QT* op = (QT*)a.out + (token * a.heads + head) * D + d0;
  if constexpr (std::is_same<QT, float>::value) {
    *reinterpret_cast<f32x4_t*>(op) = o * inv;
  } else {
    ushort4 w;
    w.x = float_to_bf16(o[0] * inv); w.y = float_to_bf16(o[1] * inv); w.z = float_to_bf16(o[2] * inv); w.w = float_to_bf16(o[3] * inv);
    *reinterpret_cast<ushort4*>(op) = w;
  }
}

// How the keys of a launch are cut: `splits` shares, `waves` of them a block of the kernel of few columns (their sums meet in
// LDS), so that parts() partial results a cell are left.
struct Cut {
  int splits = 1, waves = 1, two = 0;      // two: two tiles of columns a wave
  int tiles = 0;                           // > 0: the kernel of many columns, so many blocks of them
  int budget = 0;                          // > 0: blocks a kv head for decode rows by their lengths
  int parts() const { return tiles ? splits : splits / waves; }
};

struct Launch {
  hipStream_t stream;
  int q8, dtype;
};

template <int D, bool Q8, typename QT>
void launch_size(const CacheArgs& a, const Cut& c, int jobs, int by_group, int most, int less_than, hipStream_t s) {
  constexpr bool F32 = std::is_same<QT, float>::value;
  if constexpr (!F32) {
    if (c.tiles) {
      const dim3 grid(a.kv_heads, c.tiles * c.splits, jobs);
      if constexpr (D <= 128) {
        if (c.waves == 8) {
          cache_tiles_kernel<D, Q8, 8><<<grid, 512, 0, s>>>(a, by_group, less_than, 0);
          return;
        }
      }
      cache_tiles_kernel<D, Q8, 4><<<grid, 256, 0, s>>>(a, by_group, less_than, (int64_t)grid.x * grid.y * grid.z <= 512);
      return;
    }
  }
  const int nt = 1 + c.two, tiles = (int)(((int64_t)most * (a.heads / a.kv_heads) + 16 * nt - 1) / (16 * nt));
  const size_t lds = (size_t)(c.waves - 1) * nt * (16 * D + 32) * sizeof(float);
  dim3 grid(tiles * (c.splits / c.waves), a.kv_heads, jobs);
  if (c.budget) grid = dim3(tiles * (c.budget + jobs), a.kv_heads, 1);
  if constexpr (two_tiles(D, F32)) {
    if (c.two) {
      cache_rows_kernel<D, Q8, QT, 2><<<grid, c.waves * WAVE, lds, s>>>(a, by_group, most);
      return;
    }
  }
  cache_rows_kernel<D, Q8, QT, 1><<<grid, c.waves * WAVE, lds, s>>>(a, by_group, most);
}
template <int D>
void launch_kind(const CacheArgs& a, const Launch& w, const Cut& c, int jobs, int by_group, int most, int less_than) {
  if (!w.q8) launch_size<D, false, bf16_t>(a, c, jobs, by_group, most, less_than, w.stream);
  else if (w.dtype == HOLON_BF16) launch_size<D, true, bf16_t>(a, c, jobs, by_group, most, less_than, w.stream);
  else launch_size<D, true, float>(a, c, jobs, by_group, most, less_than, w.stream);
}
// Two kinds of work in one launch: `jobs` groups (or rows) of up to `columns` columns, cut by `first`, and then n_rows rows of up to `most`
// queries that leave `own` parts each (r.budget: as many blocks in all as that says).
template <int D>
void launch_both(const CacheArgs& p, const CacheArgs& r, const Launch& w, const Cut& first, int by_group, int less_than, int jobs, int64_t columns,
                 int n_rows, int most, int own) {
  const int first_blocks = (first.tiles ? first.tiles : (int)((columns + 15) / 16)) * first.parts();
  const int row_tiles = (int)(((int64_t)most * (r.heads / r.kv_heads) + 15) / 16);
  const int row_blocks = row_tiles * (r.budget ? r.budget + n_rows : own), row_jobs = r.budget ? 1 : n_rows;
  const dim3 grid((unsigned)(p.kv_heads * ((int64_t)first_blocks * jobs + (int64_t)row_blocks * row_jobs)));
  const int folded = !by_group && (int64_t)p.kv_heads * first_blocks * jobs <= 512;
  const auto go = [&](auto q8, auto tiles, auto waves) {
    constexpr int WAVES = decltype(waves)::value;
    cache_both_kernel<D, decltype(q8)::value, decltype(tiles)::value, WAVES><<<grid, WAVES * WAVE, 0, w.stream>>>(
        p, r, by_group, less_than, folded, first_blocks, jobs, row_blocks, most);
  };
  const auto kind = [&](auto q8) {
    const std::integral_constant<int, 4> four;
    if constexpr (D <= 128) {
      if (!first.tiles) return go(q8, std::false_type{}, four);
      if (first.waves == 8) return go(q8, std::true_type{}, std::integral_constant<int, 8>{});
    }
    go(q8, std::true_type{}, four);
  };
  if (w.q8) kind(std::true_type{});
  else kind(std::false_type{});
}
template <int D>
void launch_merge(const CacheArgs& a, const Launch& w, int max_query, int less_than, int64_t cells) {
  const unsigned blocks = (unsigned)((cells + 256 / (D / 4) - 1) / (256 / (D / 4)));
  if (w.dtype == HOLON_BF16) cache_merge_kernel<D, bf16_t><<<blocks, 256, 0, w.stream>>>(a, max_query, less_than, cells);
  else cache_merge_kernel<D, float><<<blocks, 256, 0, w.stream>>>(a, max_query, less_than, cells);
}

// Rows whose columns (queries times the heads of a group) are at most this many take the kernel of few columns, which reads the keys
// once for every 32 of them.
constexpr int FEW_COLUMNS = 64;

// `jobs` rows of up to `queries` queries, or groups (0: all see all keys), up to `columns` columns in all over up to `span` keys.
Cut cut_keys(int jobs, int64_t columns, int64_t span, int64_t queries, int kv_heads, int head_dim, int value_bytes, bool f32) {
  Cut r;
  const int64_t units = std::max<int64_t>(1, (int64_t)jobs * kv_heads);
  span = std::max<int64_t>(span, 1);
  columns = std::max<int64_t>(columns, 1);
  if (columns > FEW_COLUMNS && !f32) {
    // Blocks of 256 columns (a stage is brought in once for twice the columns; one block a compute unit) where there are about two for every
    // unit; where there is one, if the first ones' walks are not much shorter than the last ones'; where there is one and a part, if what
    // is left behind the first round is short. 32 heads over 8 of 128, us over codes (over bfloat16), 128 columns | 256: 4,096 tokens
    // behind 28,672 2,669 | 2,456 (2,499 | 2,183), a whole prompt of 8,192 724 | 708 (674 | 630); 2,048, one block a unit, behind 2,048 155 | 173
    // (141 | 153), 6,144 327 | 334 (301 | 295), 28,672 1,321 | 1,227 (1,212 | 1,075), a whole prompt of 2,048 83 | 92 (73 | 82); of 40 heads, 1.25
    // blocks a unit, behind 2,048 243 | 224 (225 | 198), 4,096 371 | 384 (340 | 339), 28,672 2,158 | 2,337 (1,999 | 2,075). Heads of 64: over
    // codes 4,096 behind 28,672 1,936 | 1,734, 2,048 behind 6,144 235 | 235, a whole prompt of 8,192 532 | 495; over bfloat16, whose stages cost
    // no widening, 1,585 | 1,678, 213 | 228, 385 | 477: not there.
    const int64_t wide = units * ((columns + 255) / 256);
    const bool pays = wide >= 448 || (wide >= 256 && wide <= 288 && 4 * queries <= span) ||
                      (wide > 288 && 4 * queries <= 3 * span && 2 * span <= 5 * queries);
    r.waves = head_dim <= 128 && (head_dim > 64 || value_bytes == 1) && pays ? 8 : 4;
    r.tiles = (int)((columns + 32 * r.waves - 1) / (32 * r.waves));
    const int64_t want = std::max<int64_t>(1, 2048 / r.waves / (units * r.tiles));      // two waves a SIMD
    r.splits = (int)std::min<int64_t>(std::min<int64_t>(want, 32), std::max<int64_t>(1, (span + 127) / 128));
    return r;
  }
  r.two = columns > 16 && two_tiles(head_dim, f32);
  const int64_t pairs = units * ((columns + 16 * (1 + r.two) - 1) / (16 * (1 + r.two)));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(64, 2048 / std::max<int64_t>(1, pairs)));
  const int64_t per = std::max<int64_t>(64, ((span + want - 1) / want + 63) / 64 * 64);
  const int64_t shares = std::max<int64_t>(1, (span + per - 1) / per);
  const int64_t blocks = pairs <= 16 ? 256 : 512;
  const int cap = most_waves(head_dim, f32, 1 + r.two);
  // A block's waves take all of a row's keys, and no merge follows, where a wave has 16 KB of keys at most. One block | several and
  // the merge, us in a graph, where the merge's own launch costs least: 32 heads over 8 of 128, 8 bits, 4 rows of 600 / 1,000 / 1,500 keys
  // 10.6 / 11.6 / 15.2 | 8.8 / 9.2 / 11.1, 16 rows 10.8 / 12.8 / 17.4 | 11.3 / 13.1 / 17.0; 16 over 8 of 64, 4 rows of 1,000 / 2,000 / 3,000 7.4 /
  // 10.7 / 13.4 | 8.3 / 8.9 / 9.1. A call that is not recorded spends 4 us on the second launch.
  const bool one = span * head_dim * value_bytes <= (int64_t)16384 * cap;
  const int64_t outer = one ? 1 : std::min(shares, std::max<int64_t>(1, (blocks + pairs - 1) / pairs));
  r.waves = (int)std::min<int64_t>(cap, (shares + outer - 1) / outer);
  r.splits = one ? r.waves : (int)((shares + r.waves - 1) / r.waves) * r.waves;
  return r;
}
int64_t seen_span(int64_t len, int64_t queries, int window) {
  if (window > 0) return std::min<int64_t>(len, window + queries + 63);
  if (window < 0) return std::min<int64_t>(len, -(int64_t)window + 63);
  return len;
}

// What one call runs: the decode rows, the rows of a few queries, those of many, the groups' prefixes.
struct Plan {
  Cut decode, few, many, shared;
  int few_query = 0;                       // rows of up to so many queries are among the few
  bool any_decode, any_few, any_many, any_shared, by_token, together = false, beside = false;
  int parts = 1;                           // of a cell, where cells go by token
  int64_t decode_cells = 0, few_cells = 0, many_cells = 0;
};
Plan plan_of(int n_decode, int max_decode_len, int n_chunk, int max_chunk_query, int max_chunk_len, int n_groups, int max_group_query,
             int max_group_len, int64_t n_tokens, int heads, int kv_heads, int head_dim, int window, int value_bytes, bool f32) {
  Plan p;
  const int group = heads / kv_heads;
  p.any_shared = n_groups > 0 && max_group_query > 0 && max_group_len > 0;
  // Decode rows that one block each serves read their prefix themselves, from L2, while the GPU has room for all blocks and a row's keys
  // are 192 KB at most: one launch for two. Two (the groups' and the rows', the merge) | one, four rows, us in a graph, where the merge's own
  // launch costs least (not recorded, two take 15 us at least); keys behind | us: 32 heads over 8 of 128, codes 256 9.6 | 7.3, 768 10.6 | 10.5,
  // 1,536 11.9 | 15.8, float32 queries 256 17 | 9, 1,536 18 | 21, bfloat16 256 10.9 | 8.1, 768 11.9 | 13.3; 16 over 8 of 64, codes 256 8.2 | 5.7,
  // 1,536 10.3 | 10.2, 2,560 10.2 | 13.3, float32 queries 1,536 16 | 14, bfloat16 1,024 10.1 | 9.7, 1,536 11.0 | 11.8; 16 over 2 of 256, codes
  // 256 18.2 | 10.4, 512 15.6 | 14.3, 768 17.3 | 17.9, float32 queries 512 20 | 19, 768 22 | 24, bfloat16 384 17.7 | 15.4, 512 16.5 | 18.3.
  const int64_t alone = 192 * 1024;
  const bool one_each = p.any_shared && n_chunk == 0 && group <= 16 && (int64_t)n_decode * kv_heads <= 256 &&
                        (int64_t)max_decode_len * head_dim * value_bytes <= alone;
  if (one_each) p.any_shared = false;
  const int own_decode = p.any_shared ? std::max(max_decode_len - max_group_len, 64) : max_decode_len;
  const int own_chunk = p.any_shared ? std::max(max_chunk_len - max_group_len, 64) : max_chunk_len;
  const int few = f32 ? max_chunk_query : std::min(max_chunk_query, std::max(1, FEW_COLUMNS / group));
  p.few_query = few;
  p.any_decode = n_decode > 0;
  p.any_few = n_chunk > 0 && few > 1;
  p.any_many = n_chunk > 0 && max_chunk_query > few;
  if (p.any_many && n_chunk == 1) p.any_few = false;       // (the one row is as long as the longest)
  p.decode = cut_keys(n_decode, group, seen_span(own_decode, 1, window), 1, kv_heads, head_dim, value_bytes, f32);
  if (one_each) p.decode.splits = p.decode.waves = std::max(1, (int)std::min<int64_t>(most_waves(head_dim, f32, 1), ((int64_t)max_decode_len + 63) / 64));
  p.few = cut_keys(n_chunk, (int64_t)few * group, seen_span(own_chunk, few, window), few, kv_heads, head_dim, value_bytes, f32);
  p.many = cut_keys(n_chunk, std::max<int64_t>((int64_t)max_chunk_query * group, FEW_COLUMNS + 1), seen_span(own_chunk, max_chunk_query, window),
                    max_chunk_query, kv_heads, head_dim, value_bytes, f32);
  p.by_token = p.any_shared;
  if (p.by_token) {
    p.shared = cut_keys(n_groups, (int64_t)max_group_query * group, max_group_len, 0, kv_heads, head_dim, value_bytes, f32);
    // every cell has the prefix's parts and then as many of its row's own whichever kernel made them
    int own = p.any_decode ? p.decode.parts() : p.any_few ? p.few.parts() : p.many.parts();
    // one launch for both where there is one kind of rows, of few columns
    const Cut& rows = p.any_decode ? p.decode : p.few;
    p.together = p.any_decode != p.any_few && !p.any_many && head_dim <= 128 && !f32 && !rows.tiles;
    if (p.together) {
      const int64_t units = (int64_t)n_groups * kv_heads;
      if (p.shared.tiles) {                                // one block a compute unit, the rows' blocks beside them
        // Blocks of 256 columns, if they are full, over long prefixes. 128 columns | 256, us, 64 rows of 32 heads over 8 of 128 with 256 keys of
        // their own, bfloat16: behind 16,384 50 | 60, 32,768 77 | 78, 49,152 106 | 100, 65,536 136 | 120, 131,072 249 | 205; of heads of 64
        // 38 | 43, 57 | 57, 76 | 71, 96 | 85, 174 | 144, over codes 40 | 45, 61 | 58, 81 | 73, 103 | 87, 190 | 144.
        const int64_t columns = (int64_t)max_group_query * group;
        p.shared.waves = max_group_len >= 49152 && (columns + 255) / 256 * 2 == (columns + 127) / 128 ? 8 : 4;
        p.shared.tiles = (int)((columns + 32 * p.shared.waves - 1) / (32 * p.shared.waves));
        const int64_t want = std::max<int64_t>(1, (p.shared.waves == 8 ? 256 : 384) / (units * p.shared.tiles));
        p.shared.splits = (int)std::min<int64_t>(std::min<int64_t>(want, 32), std::max<int64_t>(1, (max_group_len + 127) / 128));
      } else {
        const int64_t tiles = ((int64_t)max_group_query * group + 15) / 16;
        const int64_t want = std::max<int64_t>(1, 256 / (units * tiles)), shares = std::max(1, (max_group_len + 63) / 64);
        p.shared.two = 0;
        p.shared.waves = 4;
        p.shared.splits = 4 * (int)std::min<int64_t>(std::min<int64_t>(want, 32), (shares + 3) / 4);
      }
      const int64_t jobs = (p.any_decode ? n_decode : n_chunk) * (int64_t)kv_heads;
      const int64_t span = p.any_decode ? own_decode : own_chunk;
      own = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(16, 512 / jobs), (span + 255) / 256));
    }
    for (Cut* cut : {&p.decode, &p.few, &p.many}) cut->splits = cut->tiles ? own : own * cut->waves;
    p.parts = p.shared.parts() + own;
    p.decode_cells = (int64_t)n_tokens * heads * p.parts;
  } else {
    // Rows of long contexts are cut by their lengths. In equal numbers of shares | by lengths, us in a graph, 32 heads over 8 of 128, 8
    // bits: 32,768 and seven of 500 keys 40 | 29, 32,768 and fifteen of 500 67 | 31, 16,384 and 47 of 700 83 | 33, eight of 11,000 to 32,768 80 |
    // 79; all alike, eight of 32,768 109 | 112, 32 of 4,096 51 | 51; where rows are short, 900 to 4,096, 12 | 16.
    // A portion's blocks and the decode rows in one launch, but where the decode rows are most of a long step (their blocks then run at a
    // portion's occupancy). Two | one, us in a graph, over codes: 32 heads over 8 of 128, a portion of 512 behind 28,672 and 16 of 4,096
    // 372 | 352, a whole prompt of 2,048 and as many 111 | 88, 128 and one of 300 18 | 11; 128 behind 8,000 and 64 of 4,096 154 | 158, 16 over 8 of
    // 64, 32 of 16,384 133 | 140. No line in a step's bytes and operations is sooner there: 0.3% from the best on average over 264 steps, 5%
    // at most. Over bfloat16 (32 over 8 of 128, then of 64): 512 behind 28,672 and 16 of 4,096 378 | 352, 249 | 226; 128 behind 8,000 and 64 of
    // 4,096 235 | 241, 130 | 138, behind 2,000 220 | 226, 119 | 138. At heads of 256 (16 over 2) the joined kernel's tiles are slower: 2,048
    // behind 28,672 and eight of 1,000 1,531 | 1,614, a whole prompt of 2,048 and 16 of 4,096 146 | 126. By this rule 0.3 and 0.5% from the best
    // on average over 216 and 48 steps, 9% at most; always joined 1.0 and 2.5%, 19%.
    const double keys = 2.0 * value_bytes * n_decode * kv_heads * head_dim * seen_span(max_decode_len, 1, window);       // bytes
    const double work = 4.0 * n_chunk * max_chunk_query * heads * head_dim *                                             // operations
                        std::min(seen_span(max_chunk_len, max_chunk_query, window), std::max((int64_t)max_chunk_len - max_chunk_query / 2, (int64_t)1));
    const bool pays = value_bytes == 1 || (head_dim < 256 ? keys <= std::max(3e8, work / 15) : keys <= 1.5e8 && work <= 4e10);
    p.beside = p.any_decode && p.any_many && group <= 16 && !f32 && pays;
    if (p.beside) {                                        // (in blocks of the portion's size)
      p.decode.splits = p.decode.parts() * p.many.waves;
      p.decode.waves = p.many.waves;
    }
    // (Rows of few columns alone: the kernel of many cuts all rows into the same number of shares.)
    if (p.any_decode && !p.decode.tiles && p.decode.parts() > 1 && n_decode > 1 && n_decode <= 64 &&
        seen_span(max_decode_len, 1, window) > 4096)
      p.decode.budget = p.decode.parts() * n_decode;
    if (p.any_decode && p.decode.parts() > 1)
      p.decode_cells = p.decode.budget ? (int64_t)(p.decode.budget + n_decode) * heads : (int64_t)n_decode * heads * p.decode.parts();
    if (p.any_few && p.few.parts() > 1) p.few_cells = (int64_t)n_chunk * few * heads * p.few.parts();
    if (p.any_many && p.many.parts() > 1) p.many_cells = (int64_t)n_chunk * max_chunk_query * heads * p.many.parts();
  }
  return p;
}

// Floats of scratch for the partial sums of so many cells (and, where rows are cut by their lengths, `listed` rows' shares): whole
// pieces of 16 bytes, so that what follows begins on a border for its vectors.
int64_t room_of(int64_t cells, int head_dim, int listed) { return (cells * (head_dim + 2) + 2 * (int64_t)listed + 3) / 4 * 4; }

}  // namespace

static Plan plan_of(const HolonCacheAttention& c) {
  return plan_of(c.n_decode, c.max_decode_len, c.n_chunk, c.max_chunk_query, c.max_chunk_len, c.n_groups, c.max_group_query, c.max_group_len,
                 c.tokens, c.heads, c.kv_heads, c.head_dim, c.window, c.scales != nullptr ? 1 : 2, c.dtype == HOLON_F32);
}

extern "C" int64_t holon_cache_attention_room(const HolonCacheAttention* call) {
  const HolonCacheAttention& c = *call;
  if (c.kv_heads <= 0 || c.heads < c.kv_heads) return 0;   // (refused by the call that follows)
  const Plan p = plan_of(c);
  return (room_of(p.decode_cells, c.head_dim, p.decode.budget ? c.n_decode : 0) + room_of(p.few_cells, c.head_dim, 0) +
          room_of(p.many_cells, c.head_dim, 0)) * (int64_t)sizeof(float);
}

extern "C" int holon_cache_attention(const HolonCacheAttention* call, const void* q, void* out, void* room, void* stream) {
  const HolonCacheAttention& c = *call;
  const int head_dim = c.head_dim, heads = c.heads, dtype = c.dtype;
  const bool q8 = c.scales != nullptr;
  HOLON_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "attention: heads of %d (64, 128 and 256 are served)", head_dim);
  HOLON_CHECK(c.page_size > 0 && c.page_size % 16 == 0, "attention: pages of %d tokens (multiples of 16 are served)", c.page_size);
  HOLON_CHECK(dtype == HOLON_BF16 || (q8 && dtype == HOLON_F32), "attention: queries of another type than the cache serves");
  HOLON_CHECK(heads > 0 && c.kv_heads > 0 && c.kv_heads <= 65535 && heads % c.kv_heads == 0, "attention: %d heads over %d", heads, c.kv_heads);
  HOLON_CHECK(c.n_decode >= 0 && c.n_chunk >= 0 && c.n_decode <= 65535 && c.n_chunk <= 65535 && c.max_chunk_query <= 65535 && c.tokens >= 0 &&
                  c.tokens <= 0x7fffffff && c.n_groups <= 65535 && c.max_decode_len >= 0 && c.max_chunk_len >= 0 && c.max_group_query >= 0 &&
                  c.max_group_len >= 0 && c.num_pages > 0 && c.n_slots > 0 && c.table_stride > 0 && c.n_groups >= 0 &&
                  (c.n_chunk == 0 || c.max_chunk_query > 0), "attention: bad sizes");
  HOLON_CHECK(c.scale > 0.f, "attention: a scale of %g", (double)c.scale);
  HOLON_CHECK(c.page_stride % 16 == 0 && c.scale_stride % 16 == 0, "attention: pages lie on no borders of 16 bytes");
  // (positions are 32-bit numbers; and see page_index)
  const uint64_t magic = ((1ull << 32) + c.page_size - 1) / c.page_size, excess = magic * c.page_size - (1ull << 32);
  HOLON_CHECK((int64_t)c.table_stride * c.page_size < (1ll << 31) - 256 && ((uint64_t)c.table_stride * c.page_size + 256) * excess < (1ull << 32),
              "attention: a table row of %d pages of %d tokens is too long", c.table_stride, c.page_size);
  HOLON_CHECK(c.page_stride < (1ll << 32) && c.scale_stride < (1ll << 32), "attention: pages lie too far apart");
  if (c.tokens == 0 || c.rows <= 0) return 0;              // (tokens of no row are left alone)
  CacheArgs a{};
  a.q = q; a.out = out; a.pages = (const uint8_t*)c.pages; a.scales = (const uint8_t*)c.scales;
  a.page_stride = c.page_stride; a.scale_stride = c.scale_stride; a.num_pages = c.num_pages;
  a.table = c.table; a.table_stride = c.table_stride; a.n_slots = c.n_slots;
  a.slots = c.slots; a.lens = c.lens; a.qstart = c.qstart; a.rows = c.rows; a.n_tokens = (int)c.tokens;
  a.heads = heads; a.kv_heads = c.kv_heads; a.page_size = c.page_size;
  a.page_magic = (uint32_t)magic;
  a.scale_log2 = c.scale * 1.4426950408889634f; a.sink = c.sink;
  // (a query may lie up to 65,534 positions in front of the sequence, and what it sees begins a window before that: see first_seen)
  a.window = std::min(std::max(c.window, -0x7fffffff), 0x7fffffff - 0x10000);
  const Plan p = plan_of(c);
  float* at = (float*)room;
  const Launch w{(hipStream_t)stream, q8, dtype};
  const auto launch = [&](const Cut& cut, int jobs, int by_group, int most, int less_than) {
    a.splits = cut.splits;
    if (head_dim == 64) launch_kind<64>(a, w, cut, jobs, by_group, most, less_than);
    else if (head_dim == 128) launch_kind<128>(a, w, cut, jobs, by_group, most, less_than);
    else launch_kind<256>(a, w, cut, jobs, by_group, most, less_than);
  };
  const auto merge = [&](int max_query, int less_than, int64_t cells) {
    if (head_dim == 64) launch_merge<64>(a, w, max_query, less_than, cells);
    else if (head_dim == 128) launch_merge<128>(a, w, max_query, less_than, cells);
    else launch_merge<256>(a, w, max_query, less_than, cells);
  };
  if (p.by_token) {
    a.group_start = c.group_start; a.group_lens = c.group_lens; a.n_groups = c.n_groups;
    a.parts = p.parts; a.part_o = at; a.part_ml = at + p.decode_cells * head_dim;
    if (p.together) {
      CacheArgs r = a;
      const int own = p.parts - p.shared.parts(), n_rows = p.any_decode ? c.n_decode : c.n_chunk, most = p.any_decode ? 1 : p.few_query;
      a.splits = p.shared.splits;
      r.row_ids = p.any_decode ? c.decode_rows : c.chunk_rows;
      r.splits = own * p.shared.waves;
      r.part_first = p.shared.parts();
      const int64_t columns = (int64_t)c.max_group_query * (heads / c.kv_heads);
      if (head_dim == 64) launch_both<64>(a, r, w, p.shared, 1, 0, c.n_groups, columns, n_rows, most, own);
      else launch_both<128>(a, r, w, p.shared, 1, 0, c.n_groups, columns, n_rows, most, own);
      merge(1, 0, c.tokens * heads);
      HOLON_LAUNCH_OK();
      return 0;
    }
    launch(p.shared, c.n_groups, 1, c.max_group_query, 0);
    a.part_first = p.shared.parts();
  }
  const auto set = [&](const Cut& cut, const int32_t* ids, int n_rows, int most, int64_t cells) {
    a.row_ids = ids;
    a.budget = cut.budget;
    a.n_rows = n_rows;
    a.splits = cut.splits;
    if (p.by_token) return;
    a.parts = cut.parts(); a.cell_queries = most;
    a.part_o = at; a.part_ml = at + cells * head_dim;
    a.row_parts = (int2*)(at + cells * (head_dim + 2));
    at += room_of(cells, head_dim, cut.budget ? n_rows : 0);
  };
  const auto join = [&](int n_rows, int most, int less_than) {
    if (!p.by_token && a.parts > 1) merge(most, less_than, (int64_t)n_rows * most * heads);
  };
  const auto serve = [&](bool any, const Cut& cut, const int32_t* ids, int n_rows, int most, int less_than, int64_t cells) {
    if (!any) return;
    set(cut, ids, n_rows, most, cells);
    launch(cut, n_rows, 0, most, less_than);
    join(n_rows, most, less_than);
  };
  const int many_from = p.any_few ? p.few_query : 0;       // rows of up to so many queries are not among the many
  serve(p.any_few, p.few, c.chunk_rows, c.n_chunk, p.few_query, 0, p.few_cells);
  if (p.beside) {
    set(p.decode, c.decode_rows, c.n_decode, 1, p.decode_cells);
    const CacheArgs rows = a;
    set(p.many, c.chunk_rows, c.n_chunk, c.max_chunk_query, p.many_cells);
    const CacheArgs tiles = a;
    const int64_t columns = (int64_t)c.max_chunk_query * (heads / c.kv_heads);
    const int own = p.decode.parts();
    if (head_dim == 64) launch_both<64>(tiles, rows, w, p.many, 0, many_from, c.n_chunk, columns, c.n_decode, 1, own);
    else if (head_dim == 128) launch_both<128>(tiles, rows, w, p.many, 0, many_from, c.n_chunk, columns, c.n_decode, 1, own);
    else launch_both<256>(tiles, rows, w, p.many, 0, many_from, c.n_chunk, columns, c.n_decode, 1, own);
    a = rows;
    join(c.n_decode, 1, 0);
    a = tiles;
    join(c.n_chunk, c.max_chunk_query, many_from);
  } else {
    serve(p.any_decode, p.decode, c.decode_rows, c.n_decode, 1, 0, p.decode_cells);
    serve(p.any_many, p.many, c.chunk_rows, c.n_chunk, c.max_chunk_query, many_from, p.many_cells);
  }
  if (p.by_token) merge(1, 0, c.tokens * heads);
  HOLON_LAUNCH_OK();
  return 0;
}
