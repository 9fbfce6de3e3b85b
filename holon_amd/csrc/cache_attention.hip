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
  const int32_t* row_ids;      // the rows of this launch
  int n_tokens;
  int heads, kv_heads, page_size;
  float scale_log2;            // scale * log2(e)
  int window;                  // see first_seen
  const float* sink;           // [Hq], nullable
  float* part_o;               // partial results of (token, head) cells, `parts` each: [cells, parts, D] and [cells, parts, 2]
  float* part_ml;
  int parts, part_first;       // this launch's come from `part_first` on
  int cell_queries;            // > 0: cell (row in row_ids) * cell_queries + query; 0: the token
  int splits;                  // over which waves a row's keys are cut
  // rows that share their first tokens: group g is rows group_start[g] .. group_start[g + 1] - 1 and shares group_lens[g] of them
  const int32_t* group_start;
  const int32_t* group_lens;
  int n_groups;
};

// What is out of range is not followed: the pool's last page, the table's last row.
__device__ __forceinline__ int64_t page_at(const CacheArgs& a, int32_t page) {
  return (int64_t)min((uint32_t)page, (uint32_t)(a.num_pages - 1));
}
__device__ __forceinline__ const int32_t* table_row(const CacheArgs& a, int row) {
  return a.table + (int64_t)min((uint32_t)a.slots[row], (uint32_t)(a.n_slots - 1)) * a.table_stride;
}

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
// Waves a block at most: eight where a lane needs no more than 256 registers.
constexpr int most_waves(int D, bool f32, int NT) { return D == 256 || f32 || NT > 1 ? 4 : 8; }

// Whether a wave may take two tiles of columns: what they hold then fits its registers.
constexpr bool two_tiles(int D, bool f32) { return D <= 128 && !f32; }

template <int D, bool Q8, typename QT, int NT>
__global__ void __launch_bounds__(WAVE * most_waves(D, std::is_same<QT, float>::value, NT)) cache_rows_kernel(CacheArgs a) {
  constexpr int PARTS = std::is_same<QT, float>::value ? 3 : 1;
  constexpr int KB = Q8 ? 64 : 32, RUN = KB / 4, SCORES = KB / 16, PV = KB / 32;
  constexpr int KLOADS = Q8 ? D / 64 : D / 32;             // 16-byte loads of a key's share
  constexpr int PART = 16 * D + 32;
  extern __shared__ __attribute__((aligned(16))) float red[];   // [waves - 1][NT][16 D values, 16 maxima, 16 sums]
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, waves = blockDim.x / WAVE;
  const int g = lane / 16, c = lane % 16;
  const int ri = blockIdx.z, hk = blockIdx.y, row = a.row_ids[ri];
  const int group = a.heads / a.kv_heads, P = a.page_size;
  const int out_splits = a.splits / waves;
  const int tile0 = blockIdx.x / out_splits * NT, piece = blockIdx.x % out_splits;
  const int qs = a.qstart[row], nq = a.qstart[row + 1] - qs, n = a.lens[row];
  if (tile0 * 16 >= nq * group) return;                    // (the same for the whole block: a shorter row's)
  Column col[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) col[t] = column_of(a, (tile0 + t) * 16 + c, hk, group, qs, nq, n);
  const int pos_first = n - nq + tile0 * 16 / group;                               // the tiles' first and last positions
  const int pos_last = n - nq + min((tile0 + NT) * 16 - 1, nq * group - 1) / group;
  const int from = max(shared_keys(a, row), 0);
  const int first = max(from, first_seen(pos_first, a.window)), whole_from = max(from, first_seen(pos_last, a.window));
  const int base = first / KB * KB;
  const int share = max(KB, ((pos_last - base + a.splits) / a.splits + KB - 1) / KB * KB);
  const int key_lo = base + (piece * waves + wave) * share;
  const int key_hi = min(pos_last, key_lo + share - 1);
  int from_here[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) from_here[t] = max(from, first_seen(col[t].pos, a.window));

  Tiles<D, NT> tl;
  tl.clear();
  if (n > 0 && nq > 0 && key_lo <= key_hi) {
    const int32_t* trow = table_row(a, row);
    const int max_page = a.table_stride - 1;
    bf16x8_t qf[NT][PARTS][D / 32];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const QT* qp = (const QT*)a.q + ((int64_t)col[t].token * a.heads + col[t].head) * D;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        const int d0 = Q8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          __bf16 p[PARTS];
          const float x = col[t].valid ? Elem<QT>::load(qp[d0 + i]) : 0.f;
          split<PARTS>(x, p);
#pragma unroll
          for (int s = 0; s < PARTS; ++s) qf[t][s][ks][i] = p[s];
        }
      }
    }
    const int bytes = Q8 ? 1 : 2;
    const int64_t plane = (int64_t)P * D * bytes;
    const uint8_t* kplane = a.pages + hk * plane;
    const uint8_t* vplane = a.pages + (a.kv_heads + hk) * plane;
    const uint8_t* ksplane = Q8 ? a.scales + (int64_t)hk * P : nullptr;
    const uint8_t* vsplane = Q8 ? a.scales + (int64_t)(a.kv_heads + hk) * P : nullptr;
    const int krun = RUN * (c / 4);                        // this lane's keys: krun + c % 4 + 4 j; its values: RUN g ..
    for (int kb = key_lo; kb <= key_hi; kb += KB) {
      const int kk = kb + krun, vk = kb + RUN * g;
      const int64_t kpage = page_at(a, trow[min(kk / P, max_page)]), vpage = page_at(a, trow[min(vk / P, max_page)]);
      u32x4_t kraw[SCORES][KLOADS], vraw[D / 16], ks4 = {}, vs4 = {};
      if constexpr (Q8) {
        ks4 = *reinterpret_cast<const u32x4_t*>(ksplane + kpage * a.scale_stride + kk % P);
        vs4 = *reinterpret_cast<const u32x4_t*>(vsplane + vpage * a.scale_stride + vk % P);
      }
      const uint8_t* kp = kplane + kpage * a.page_stride + (int64_t)(kk % P + c % 4) * D * bytes + 16 * g;
#pragma unroll
      for (int j = 0; j < SCORES; ++j)
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) kraw[j][i] = *reinterpret_cast<const u32x4_t*>(kp + (int64_t)4 * j * D * bytes + 64 * i);
      const uint8_t* vp = vplane + vpage * a.page_stride + ((int64_t)c * P + vk % P) * bytes;
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds) vraw[ds] = *reinterpret_cast<const u32x4_t*>(vp + (int64_t)ds * 16 * P * bytes);

      const bool whole = kb >= whole_from && kb + KB - 1 <= min(pos_first, key_hi);
      f32x4_t sc[NT][SCORES];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < SCORES; ++j) sc[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < SCORES; ++j) {
        const float power = Q8 ? q8_power((ks4[j] >> (8 * (c % 4))) & 0xffu) : 1.f;
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) {
          bf16x8_t f[Q8 ? 2 : 1];
          if constexpr (Q8) widen(kraw[j][i], power, f[0], f[1]);
          else f[0] = __builtin_bit_cast(bf16x8_t, kraw[j][i]);
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
        const float m_new = fmaxf(tl.m[t], mx * a.scale_log2);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
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
        alpha[t] = __builtin_amdgcn_exp2f(tl.m[t] - m_use);
        moved |= m_new != tl.m[t];
        tl.m[t] = m_new;
        tl.l[t] = tl.l[t] * alpha[t] + sum;
      }
      if (__any(moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int ds = 0; ds < D / 16; ++ds) tl.o[t][ds] *= alpha[t];
      }
      // Where queries of the tiles see different keys, a value that is not finite reaches those alone that see it: it leaves
      // the product (zero times it is no number) and sets their sums by itself.
      if (!whole && nq > 1) {
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
    if (a.parts == 1) {
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
      const int64_t cell = (place * a.heads + col[t].head) * a.parts + a.part_first + piece;
      float* po = a.part_o + cell * D + 4 * g;
#pragma unroll
      for (int ds = 0; ds < D / 16; ++ds) *reinterpret_cast<f32x4_t*>(po + 16 * ds) = tl.o[t][ds];
      if (g == 0) { a.part_ml[2 * cell] = tl.m[t]; a.part_ml[2 * cell + 1] = tl.l[t]; }
    }
  }
}

// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over a cell's parts, in their order: a block of D / 4 threads a
// (token, head).
template <int D, typename QT>
__global__ void __launch_bounds__(D / 4) cache_merge_kernel(CacheArgs a) {
  const int ri = blockIdx.z, qi = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
  const int row = a.row_ids[ri], qs = a.qstart[row], nq = a.qstart[row + 1] - qs, token = qs + qi;
  if (qi >= nq || (uint32_t)token >= (uint32_t)a.n_tokens) return;
  const int64_t place = a.cell_queries > 0 ? (int64_t)ri * a.cell_queries + qi : token;
  const int64_t cell = (place * a.heads + head) * a.parts;
  float big = -INFINITY;
  bool odd = false;
  for (int i = 0; i < a.parts; ++i) {
    big = fmaxf(big, a.part_ml[2 * (cell + i)]);
    odd |= !(a.part_ml[2 * (cell + i) + 1] >= 0.f);        // a sum that is no number
  }
  float l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < a.parts; ++i) {
    const float m = a.part_ml[2 * (cell + i)];
    if (m == -INFINITY && !odd) continue;                  // it saw no key
    const float w = __builtin_amdgcn_exp2f(m - big);
    l += w * a.part_ml[2 * (cell + i) + 1];
    o += w * *reinterpret_cast<const f32x4_t*>(a.part_o + (cell + i) * D + 4 * tid);
  }
  if (a.sink != nullptr && big != -INFINITY) l += exp2f(a.sink[head] * 1.4426950408889634f - big);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  QT* op = (QT*)a.out + ((int64_t)token * a.heads + head) * D + 4 * tid;
#pragma unroll
  for (int r = 0; r < 4; ++r) op[r] = Elem<QT>::store(o[r] * inv);
}

template <int D, bool Q8, typename QT, int NT>
void launch_rows(const CacheArgs& a, int n_rows, int max_query, int waves, hipStream_t s) {
  const int tiles = ((int64_t)max_query * (a.heads / a.kv_heads) + 16 * NT - 1) / (16 * NT);
  const size_t lds = (size_t)(waves - 1) * NT * (16 * D + 32) * sizeof(float);
  cache_rows_kernel<D, Q8, QT, NT><<<dim3(tiles * (a.splits / waves), a.kv_heads, n_rows), waves * WAVE, lds, s>>>(a);
}

template <int D, bool Q8, typename QT>
void launch_rows_tiles(const CacheArgs& a, int n_rows, int max_query, int waves, int two, hipStream_t s) {
  if constexpr (two_tiles(D, std::is_same<QT, float>::value)) {
    if (two) return launch_rows<D, Q8, QT, 2>(a, n_rows, max_query, waves, s);
  }
  launch_rows<D, Q8, QT, 1>(a, n_rows, max_query, waves, s);
}
template <int D>
void launch_rows_kind(const CacheArgs& a, int q8, int dtype, int n_rows, int max_query, int waves, int two, hipStream_t s) {
  if (!q8) launch_rows_tiles<D, false, bf16_t>(a, n_rows, max_query, waves, two, s);
  else if (dtype == HOLON_BF16) launch_rows_tiles<D, true, bf16_t>(a, n_rows, max_query, waves, two, s);
  else launch_rows_tiles<D, true, float>(a, n_rows, max_query, waves, two, s);
}

}  // namespace

namespace {

// How the keys of a launch's rows are cut over waves: `splits` shares, `waves` of them a block (their sums meet in LDS), so that
// splits / waves parts a cell are left for the merge.
struct Cut {
  int splits, waves, two;      // two: two tiles of columns a wave
  int parts() const { return splits / waves; }
};
Cut cut_rows(int n_rows, int max_query, int64_t span, int heads, int kv_heads, int head_dim, int window, bool f32) {
  Cut r;
  const int64_t columns = (int64_t)max_query * (heads / kv_heads);
  r.two = columns > 16 && two_tiles(head_dim, f32);
  const int64_t pairs = std::max<int64_t>(1, n_rows * kv_heads * ((columns + 16 * (1 + r.two) - 1) / (16 * (1 + r.two))));
  if (window > 0) span = std::min<int64_t>(span, window + max_query + 63);
  if (window < 0) span = std::min<int64_t>(span, -(int64_t)window + 63);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(64, 2048 / pairs));
  const int64_t per = std::max<int64_t>(64, ((span + want - 1) / want + 63) / 64 * 64);
  const int64_t shares = std::max<int64_t>(1, (span + per - 1) / per);
  const int64_t blocks = pairs <= 16 ? 256 : 512;
  const int cap = most_waves(head_dim, f32, 1 + r.two);
  const int64_t outer = std::min(shares, std::max<int64_t>(1, (blocks + pairs - 1) / pairs));
  r.waves = (int)std::min<int64_t>(cap, (shares + outer - 1) / outer);
  r.splits = (int)((shares + r.waves - 1) / r.waves) * r.waves;
  return r;
}

// What one call runs.
struct Plan {
  Cut decode, chunk;
  int64_t decode_cells, chunk_cells;      // of partial results
};
Plan plan_of(int n_decode, int max_decode_len, int n_chunk, int max_chunk_query, int max_chunk_len, int heads, int kv_heads,
             int head_dim, int window, bool f32) {
  Plan p;
  p.decode = cut_rows(n_decode, 1, max_decode_len, heads, kv_heads, head_dim, window, f32);
  p.chunk = cut_rows(n_chunk, max_chunk_query, max_chunk_len, heads, kv_heads, head_dim, window, f32);
  p.decode_cells = p.decode.parts() > 1 ? (int64_t)n_decode * heads * p.decode.parts() : 0;
  p.chunk_cells = p.chunk.parts() > 1 ? (int64_t)n_chunk * max_chunk_query * heads * p.chunk.parts() : 0;
  return p;
}

}  // namespace

extern "C" int64_t holon_cache_attention_room(int n_decode, int max_decode_len, int n_chunk, int max_chunk_query, int max_chunk_len,
                                              int n_groups, int max_group_query, int max_group_len, int n_tokens, int heads,
                                              int kv_heads, int head_dim, int window, int dtype) {
  const Plan p = plan_of(n_decode, max_decode_len, n_chunk, max_chunk_query, max_chunk_len, heads, kv_heads, head_dim, window,
                         dtype == HOLON_F32);
  return (p.decode_cells + p.chunk_cells) * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int holon_cache_attention(const void* q, void* out, const void* pages, const void* scales, int64_t page_stride,
                                     int64_t scale_stride, int num_pages, const int32_t* table, int table_stride, int n_slots,
                                     const int32_t* slots, const int32_t* lens, const int32_t* qstart, const int32_t* decode_rows,
                                     int n_decode, int max_decode_len, const int32_t* chunk_rows, int n_chunk, int max_chunk_query,
                                     int max_chunk_len, const int32_t* group_start, const int32_t* group_lens, int n_groups,
                                     int max_group_query, int max_group_len, int n_tokens, int heads, int kv_heads, int head_dim,
                                     int page_size, float scale, int window, const float* sink, void* room, int dtype, void* stream) {
  const bool q8 = scales != nullptr;
  HOLON_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "attention: heads of %d (64, 128 and 256 are served)", head_dim);
  HOLON_CHECK(page_size > 0 && page_size % 16 == 0, "attention: pages of %d tokens (multiples of 16 are served)", page_size);
  HOLON_CHECK(dtype == HOLON_BF16 || (q8 && dtype == HOLON_F32), "attention: queries of another type than the cache serves");
  HOLON_CHECK(heads > 0 && kv_heads > 0 && kv_heads <= 65535 && heads % kv_heads == 0, "attention: %d heads over %d", heads, kv_heads);
  HOLON_CHECK(n_decode >= 0 && n_chunk >= 0 && n_decode <= 65535 && n_chunk <= 65535 && max_chunk_query <= 65535 && n_tokens >= 0 &&
                  num_pages > 0 && n_slots > 0 && table_stride > 0 && n_groups >= 0, "attention: bad sizes");
  HOLON_CHECK(scale > 0.f, "attention: a scale of %g", (double)scale);
  HOLON_CHECK(page_stride % 16 == 0 && scale_stride % 16 == 0, "attention: pages lie on no borders of 16 bytes");
  CacheArgs a{};
  a.q = q; a.out = out; a.pages = (const uint8_t*)pages; a.scales = (const uint8_t*)scales;
  a.page_stride = page_stride; a.scale_stride = scale_stride; a.num_pages = num_pages;
  a.table = table; a.table_stride = table_stride; a.n_slots = n_slots;
  a.slots = slots; a.lens = lens; a.qstart = qstart; a.n_tokens = n_tokens;
  a.heads = heads; a.kv_heads = kv_heads; a.page_size = page_size;
  a.scale_log2 = scale * 1.4426950408889634f; a.window = window; a.sink = sink;
  const Plan p = plan_of(n_decode, max_decode_len, n_chunk, max_chunk_query, max_chunk_len, heads, kv_heads, head_dim, window,
                         dtype == HOLON_F32);
  float* at = (float*)room;
  hipStream_t s = (hipStream_t)stream;
  const auto serve = [&](const int32_t* ids, int n_rows, int max_query, const Cut& c, int64_t cells) {
    if (n_rows == 0 || max_query == 0) return;
    a.row_ids = ids;
    a.splits = c.splits; a.parts = c.parts(); a.part_first = 0; a.cell_queries = max_query;
    a.part_o = at; a.part_ml = at + cells * head_dim;
    at += cells * (head_dim + 2);
    if (head_dim == 64) launch_rows_kind<64>(a, q8, dtype, n_rows, max_query, c.waves, c.two, s);
    else if (head_dim == 128) launch_rows_kind<128>(a, q8, dtype, n_rows, max_query, c.waves, c.two, s);
    else launch_rows_kind<256>(a, q8, dtype, n_rows, max_query, c.waves, c.two, s);
    if (a.parts > 1) {
      const dim3 grid(heads, max_query, n_rows);
      const auto merge = [&](auto size) {
        constexpr int D = decltype(size)::value;
        if (dtype == HOLON_BF16) cache_merge_kernel<D, bf16_t><<<grid, D / 4, 0, s>>>(a);
        else cache_merge_kernel<D, float><<<grid, D / 4, 0, s>>>(a);
      };
      if (head_dim == 64) merge(std::integral_constant<int, 64>{});
      else if (head_dim == 128) merge(std::integral_constant<int, 128>{});
      else merge(std::integral_constant<int, 256>{});
    }
  };
  serve(decode_rows, n_decode, 1, p.decode, p.decode_cells);
  serve(chunk_rows, n_chunk, max_chunk_query, p.chunk, p.chunk_cells);
  HOLON_LAUNCH_OK();
  return 0;
}
