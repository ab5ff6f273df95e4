// Attention over the paged K/V cache for the tokens of one step: single tokens, a run of tokens, or a tree of drafts.
//
// Row (b, i, h) sees the keys j < lens[b] and the drafted keys lens[b] + t with t <= i (no mask) or mask[b, i, t]:
//   s_j = sm_scale * ks_j * (q . k8_j),   p_j = exp(s_j - m),   o = sum_j p_j vs_j v8_j / sum_j p_j
//
// One pass over the keys with a running maximum.  The row scale of V goes into the exponent, so that the products with
// V take weights of at most 1 (2^8 with the lazy maximum below) that fp16 holds to 2^-11 whatever the scales are:
//   t_j = log2(e) s_j + log2(vs_j),   m' = max t_j,   p'_j = 2^(t_j - m'),   O = sum p'_j v8_j,   l = sum p'_j / vs_j
//   o = O / l,   lse = ln 2 (m' + log2 l)
// A row of V that is all zeros has no such logarithm: it counts in m' with -100 and in l with its plain weight, and its
// p', whatever it is, meets zero codes.  (Scales of V rows may lie up to 2^100 apart; the weight of a row further below
// the others is lost from l.)
// m' moves only when it is exceeded by more than 8, as in the dense kernel, and O is rescaled only then.
// Both products run on fp16 operands with fp32 accumulators: int8 and e4m3 codes are exact in fp16, bf16 queries are
// scaled by a power of two of their row (what is below 2^-24 of the row's largest value is rounded).  l and m' are fp32.
//
// The query rows of a kv head (T tokens of H / Hkv heads) are cut into row tiles, the keys into tiles of 64.  All
// (sequence, kv head, row tile, key tile) of a call form one list that the CTAs share evenly, whatever the lengths are: a
// CTA walks a contiguous stretch of it with one load pipeline.  A row tile that falls to several CTAs is joined from
// their partial (O, l, m') by a second small kernel, in the order of the keys.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/sage_b200.h"
#include "sage_internal.h"
#include "sage_paged.cuh"
#include "sage_ptx.cuh"

namespace sage {

constexpr int kTileKeys = 64;
constexpr int kStages = 3;
constexpr int kThreads = 128;
constexpr int kMinTiles = 2;               // tiles a CTA takes at the least
constexpr float kZeroLog = -100.0f;        // log2 of a zero V scale in the running maximum

struct PagedAttnArgs {
  PagedArgs p;
  const void* q;
  Strides3 q_st;
  void* out;
  Strides3 out_st;
  float* lse;          // [B, H, T] or null
  const int* counts;
  const uint8_t* mask;
  int64_t mask_b, mask_i;
  int B, T, H, group;  // group = H / Hkv
  int row_tiles;       // row tiles of one kv head
  int ctas;            // CTAs that share the list
  float scale;         // sm_scale * log2(e)
  float* part_o;       // [2 * ctas][rows of a tile][D]
  float2* part_ml;     // [2 * ctas][rows of a tile]
};

// Context length and fresh tokens of sequence b; returns its key tiles (0 where no row has anything to see).
__device__ __forceinline__ int sequence(const PagedAttnArgs& a, int b, int& len, int& fresh) {
  len = a.p.lens[b];
  fresh = a.counts != nullptr ? a.counts[b] : a.T;
  if (len < 0 || fresh < 0 || fresh > a.T || (int64_t)len + fresh > ((int64_t)a.p.max_pages << a.p.page_shift)) {
    raise_invalid(a.p);
    len = fresh = 0;
  }
  return fresh > 0 ? (len + fresh + kTileKeys - 1) / kTileKeys : 0;
}

// Sum over the CTA's threads before this one; `total` receives the sum over all.
__device__ __forceinline__ int64_t scan_before(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  total = 0;
  int64_t before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

// The list's length: key tiles over all sequences, kv heads and row tiles.
__device__ __forceinline__ int64_t list_length(const PagedAttnArgs& a, int64_t* warp_sums) {
  int64_t mine = 0;
  int len, fresh;
  for (int b = threadIdx.x; b < a.B; b += kThreads) mine += sequence(a, b, len, fresh);
  int64_t total;
  scan_before(mine, warp_sums, total);
  return total * (a.p.Hkv * a.row_tiles);
}

__device__ __forceinline__ int sharers(const PagedAttnArgs& a, int64_t list) {
  return (int)min((int64_t)a.ctas, (list + kMinTiles - 1) / kMinTiles);
}

// Where the list's element x lies: sequence b and the element's number within the sequence.
__device__ __forceinline__ void find(const PagedAttnArgs& a, int64_t x, int64_t* warp_sums, int64_t* found, int& b,
                                     int64_t& within) {
  int64_t carry = 0;
  int len, fresh;
  const int per = a.p.Hkv * a.row_tiles;
  for (int base = 0; base < a.B; base += kThreads) {
    const int mine = base + threadIdx.x;
    const int64_t v = mine < a.B ? (int64_t)sequence(a, mine, len, fresh) * per : 0;
    int64_t total;
    const int64_t at = carry + scan_before(v, warp_sums, total);
    if (x >= at && x < at + v) found[0] = mine, found[1] = x - at;
    carry += total;
    if (x < carry) break;
  }
  __syncthreads();
  b = (int)found[0];
  within = found[1];
}

// A place in the list.
struct Cursor {
  int b, unit, tile;        // sequence, kv head * row_tiles + row tile, key tile
  int tiles, len, fresh;    // of the sequence
};

__device__ __forceinline__ void advance(const PagedAttnArgs& a, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.unit < a.p.Hkv * a.row_tiles) return;
  c.unit = 0;
  do {
    ++c.b;
    c.tiles = c.b < a.B ? sequence(a, c.b, c.len, c.fresh) : 1;
  } while (c.tiles == 0);
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four int8 codes -> two fp16 pairs, exactly: 0x6400 + u is the fp16 number 1024 + u, and u = code + 128.
__device__ __forceinline__ void int8_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
  uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), off), q = __hsub2(*reinterpret_cast<__half2*>(&y), off);
  lo = *reinterpret_cast<const uint32_t*>(&p);
  hi = *reinterpret_cast<const uint32_t*>(&q);
}

// Two weights -> an fp16 pair, the largest finite number for what is above it (only weights of zero rows are).
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two e4m3 codes -> an fp16 pair (exact).
__device__ __forceinline__ uint32_t e4m3_to_f16(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

// Shared-memory tiles.  A warp works on groups of 16 keys; lane (n = lane / 4, c = lane % 4) owns keys 4c .. 4c + 3 of a
// group in the products with V, which is what the accumulator layout of the first product leaves it with when column n
// of its tile j stands for key 4 (n / 2) + 2 j + n % 2.  K rows lie in order; lane c reads the 16-byte chunks c, c + 4,
// ... of row n.  V rows lie transposed within the group (key 4c + k at slot 4k + c); lane n reads the d channels that it
// holds as columns, D / 8 consecutive ones (256: two runs of 16).  Chunks are permuted so that the eight lanes of a
// 16-byte shared load (sixteen of an 8-byte one) touch different banks (96: up to two-way conflicts are left).
template <int D>
struct Tile {
  static constexpr int CH = D / 16;                       // 16-byte chunks of a row
  static constexpr int kBytes = kTileKeys * D;
  static constexpr int kStage = 2 * kBytes + 2 * kTileKeys * 4;
  __device__ static int k_at(int row, int ch) { return row * D + ((D % 128 == 0 ? ch ^ ((row & 1) << 2) : ch) << 4); }
  __device__ static int v_at(int row, int ch) {
    const int c = (row >> 2) & 3, slot = (row & ~15) | ((row & 3) << 2) | c;
    return slot * D + ((D % 128 == 0 ? ch ^ (c << 1) : D == 64 ? ch ^ (c & 2) : ch) << 4);
  }
};

template <int D>
constexpr int smem_bytes() {
  return kStages * Tile<D>::kStage + 2 * kTileKeys * 16;
}

// First row of the d channels behind column n of the output tile t.
template <int D>
__device__ __forceinline__ int channel(int n, int t) {
  return D == 256 ? (n + 8 * (t / 16)) * 16 + t % 16 : n * (D / 8) + t;
}

// WM row tiles of 16 rows, each with 4 / WM warps that share its keys.
template <typename T, int D, int WM>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int WK = 4 / WM, CH = Tile<D>::CH, NS = D / 16, NT = D / 8, ROWS = 16 * WM;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t warp_sums[kThreads / 32], found[2];
  unsigned char* stages = smem;
  float4* params = reinterpret_cast<float4*>(smem + kStages * Tile<D>::kStage);          // [2][64]
  __shared__ float2 join_ml[4 * 16];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, n = lane / 4, c = lane % 4;
  const int wm = warp % WM, wk = warp / WM;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int64_t list = list_length(a, warp_sums);
  const int share = sharers(a, list);
  if ((int)blockIdx.x >= share) return;
  const int64_t first = (int64_t)blockIdx.x * list / share, end = (int64_t)(blockIdx.x + 1) * list / share;
  Cursor now;
  {
    int64_t within;
    find(a, first, warp_sums, found, now.b, within);
    now.tiles = sequence(a, now.b, now.len, now.fresh);
    now.unit = (int)(within / now.tiles);
    now.tile = (int)(within - (int64_t)now.unit * now.tiles);
  }
  Cursor ahead = now;
  int64_t to_load = end - first, to_do = end - first;

  // lane g < 4: cache row of the first key of group g of the tile to be loaded next, or -1
  auto lookup = [&](const Cursor& t) -> int64_t {
    const int64_t at = (int64_t)t.tile * kTileKeys + lane * 16;
    return lane < 4 && at < t.len + t.fresh ? paged_row(a.p, t.b, t.unit / a.row_tiles, at) : -1;
  };
  int64_t base = lookup(ahead);
  int load_slot = 0;
  auto load = [&]() {
    if (to_load > 0) {
      const uint32_t dst = smem_u32(stages) + load_slot * Tile<D>::kStage;
      const int total = ahead.len + ahead.fresh, key0 = ahead.tile * kTileKeys;
#pragma unroll
      for (int i = 0; i < kTileKeys * CH / kThreads; ++i) {
        const int id = tid + i * kThreads, row = id / CH, ch = id % CH;
        const int64_t from = __shfl_sync(0xffffffffu, base, row / 16);
        const bool ok = from >= 0 && key0 + row < total;
        const int64_t off = ok ? (from + row % 16) * D + ch * 16 : 0;
        copy_async16(dst + Tile<D>::k_at(row, ch), a.p.k8 + off, ok);
        copy_async16(dst + Tile<D>::kBytes + Tile<D>::v_at(row, ch), a.p.v8 + off, ok);
      }
      const int row = tid % kTileKeys;   // a thread below 64 loads both scales of a key and prepares them itself
      const int64_t from = __shfl_sync(0xffffffffu, base, row / 16);
      const bool ok = from >= 0 && key0 + row < total;
      const int64_t off = ok ? from + row % 16 : 0;
      if (tid < kTileKeys) {
        copy_async4(dst + 2 * Tile<D>::kBytes + row * 4, a.p.ks + off, ok);
        copy_async4(dst + 2 * Tile<D>::kBytes + (kTileKeys + row) * 4, a.p.vs + off, ok);
      }
      load_slot = load_slot + 1 == kStages ? 0 : load_slot + 1;
      if (--to_load > 0) {
        advance(a, ahead);
        base = lookup(ahead);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load();

  uint32_t qf[NS][4];
  float o[NT][4], m[2], l[2], row_scale[2];
  int token[2], head[2];
  bool fresh_unit = true;
  int slot = 0, parity = 0;
  int segment = 0;                    // 0 for the first row tile that this CTA works on
  int first_tile = now.tile;          // of the row tile, by this CTA
  for (; to_do > 0; --to_do) {
    if (fresh_unit) {
      fresh_unit = false;
      first_tile = now.tile;
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
      m[0] = m[1] = -3.402823466e38f;
      l[0] = l[1] = 0.0f;
      const int row0 = now.unit % a.row_tiles * ROWS + wm * 16 + n;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        token[r] = (row0 + 8 * r) / a.group;
        head[r] = now.unit / a.row_tiles * a.group + (row0 + 8 * r) % a.group;
        const bool live = token[r] < now.fresh;
        const T* src = static_cast<const T*>(a.q) + now.b * a.q_st.b + token[r] * a.q_st.s + head[r] * a.q_st.h;
        // channels of step s: four consecutive ones, as a word of four codes holds them
        uint2 w[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const int d = D % 64 == 0 ? (c + 4 * (s / 4)) * 16 + s % 4 * 4 : (c + 4 * (s / 2)) * 8 + s % 2 * 4;
          w[s] = live ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
        }
        row_scale[r] = 1.0f;
        if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
          for (int s = 0; s < NS; ++s) qf[s][r] = w[s].x, qf[s][2 + r] = w[s].y;
        } else {
          uint32_t top = 0;
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, (e < 2 ? w[s].x : w[s].y) >> (16 * (e & 1)) & 0x7fffu);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // 2^e with e the exponent of the row's largest value (zero, infinite and NaN rows: 1; tiny ones: 2^-100)
          const int e = top == 0 || top >= 0x7f80u ? 127 : max((int)(top >> 7), 27);
          row_scale[r] = __int_as_float(e << 23);
          const float inverse = __int_as_float((254 - e) << 23);
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            qf[s][r] = pack2(__uint_as_float(w[s].x << 16) * inverse, __uint_as_float(w[s].x & 0xffff0000u) * inverse,
                             __half());
            qf[s][2 + r] = pack2(__uint_as_float(w[s].y << 16) * inverse,
                                 __uint_as_float(w[s].y & 0xffff0000u) * inverse, __half());
          }
        }
      }
    }

    copy_wait<kStages - 2>();
    unsigned char* stage = stages + slot * Tile<D>::kStage;
    const int key0 = now.tile * kTileKeys, total = now.len + now.fresh;
    const bool drafts = key0 + kTileKeys > now.len;   // the tile holds keys that some rows do not see
    if (drafts) {
      // a NaN code in a drafted row that its reader does not see must not reach it through 0 * NaN
#pragma unroll
      for (int i = 0; i < kTileKeys * CH / kThreads; ++i) {
        const int id = tid + i * kThreads, row = id / CH, ch = id % CH;
        if (key0 + row >= now.len) {
          uint4* at = reinterpret_cast<uint4*>(stage + Tile<D>::kBytes + Tile<D>::v_at(row, ch));
          uint4 v = *at;
          v.x &= ~__vcmpeq4(v.x & 0x7f7f7f7fu, 0x7f7f7f7fu);
          v.y &= ~__vcmpeq4(v.y & 0x7f7f7f7fu, 0x7f7f7f7fu);
          v.z &= ~__vcmpeq4(v.z & 0x7f7f7f7fu, 0x7f7f7f7fu);
          v.w &= ~__vcmpeq4(v.w & 0x7f7f7f7fu, 0x7f7f7f7fu);
          *at = v;
        }
      }
    }
    bool zeros = false;
    if (tid < kTileKeys) {
      // what the rows need of a key: factor of its score, log2 of its V scale, the inverse of that scale, and what the
      // exponent of a zero row gains over its part in the maximum
      const float* scales = reinterpret_cast<const float*>(stage + 2 * Tile<D>::kBytes);
      const float vs = scales[kTileKeys + tid];
      zeros = vs == 0.0f && key0 + tid < total;
      params[parity * kTileKeys + tid] =
          key0 + tid >= total ? make_float4(0.0f, -INFINITY, 0.0f, 0.0f)
          : zeros             ? make_float4(scales[tid] * a.scale, kZeroLog, 1.0f, -kZeroLog)
                              : make_float4(scales[tid] * a.scale, __log2f(vs), __fdividef(1.0f, vs), 0.0f);
    }
    const bool special = __syncthreads_or(drafts || zeros);
    load();

#pragma unroll 1
    for (int g = wk; g < 4; g += WK) {
      float s[2][4] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = g * 16 + 4 * (n / 2) + 2 * j + n % 2;
        uint32_t kw[NS];
        if constexpr (D % 64 == 0) {
#pragma unroll
          for (int i = 0; i < NS / 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(stage + Tile<D>::k_at(row, c + 4 * i));
            kw[4 * i] = v.x, kw[4 * i + 1] = v.y, kw[4 * i + 2] = v.z, kw[4 * i + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < NS / 2; ++i) {
            const uint2 v = *reinterpret_cast<const uint2*>(stage + row * D + (c + 4 * i) * 8);
            kw[2 * i] = v.x, kw[2 * i + 1] = v.y;
          }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          uint32_t b0, b1;
          int8_to_f16(kw[i], b0, b1);
          mma_f16(s[j], qf[i], b0, b1);
        }
      }
      // s[j][2 r + e]: row n + 8 r, key 4c + 2j + e of the group
      float4 key[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) key[k] = params[parity * kTileKeys + g * 16 + 4 * c + k];
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[j][2 * r + e];
            const float4& y = key[2 * j + e];
            x = fmaf(x * row_scale[r], y.x, y.y);
            if (drafts) {
              const int t = key0 + g * 16 + 4 * c + 2 * j + e - now.len;
              const bool seen = t < 0 || (t < now.fresh && token[r] < now.fresh &&
                                          (a.mask != nullptr ? a.mask[now.b * a.mask_b + token[r] * a.mask_i + t] != 0
                                                             : t <= token[r]));
              if (!seen) x = -INFINITY;
            }
            top[r] = fmaxf(top[r], x);
          }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
        float keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float next = top[r] > m[r] + 8.0f ? top[r] : m[r];
          keep[r] = next == m[r] ? 1.0f : fast_exp2(m[r] - next);
          m[r] = next;
          l[r] *= keep[r];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][0] *= keep[0], o[t][1] *= keep[0], o[t][2] *= keep[1], o[t][3] *= keep[1];
      }
      uint32_t pf[4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float p[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = s[j][2 * r + e];
            p[e] = fast_exp2(special ? x - m[r] + key[2 * j + e].w : x - m[r]);
            // an unseen key's inverse scale may be NaN
            if (!special || x != -INFINITY) l[r] = fmaf(p[e], key[2 * j + e].z, l[r]);
          }
          pf[2 * j + r] = pack_weights(p[0], p[1]);
        }
      const unsigned char* vt = stage + Tile<D>::kBytes;
#pragma unroll
      for (int i = 0; i < NT / 4; ++i) {   // four output tiles at a time: a word of four channels of each of four keys
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = g * 16 + 4 * c + k;
          const int byte = D == 256 ? n * 16 + i % 4 * 4 + i / 4 * 128 : n * (D / 8) + i * 4;
          w[k] = *reinterpret_cast<const uint32_t*>(vt + Tile<D>::v_at(row, byte / 16) + byte % 16);
        }
        const uint32_t x01 = __byte_perm(w[0], w[1], 0x5140), y01 = __byte_perm(w[0], w[1], 0x7362);
        const uint32_t x23 = __byte_perm(w[2], w[3], 0x5140), y23 = __byte_perm(w[2], w[3], 0x7362);
        mma_f16(o[4 * i], pf, e4m3_to_f16((uint16_t)x01), e4m3_to_f16((uint16_t)x23));
        mma_f16(o[4 * i + 1], pf, e4m3_to_f16((uint16_t)(x01 >> 16)), e4m3_to_f16((uint16_t)(x23 >> 16)));
        mma_f16(o[4 * i + 2], pf, e4m3_to_f16((uint16_t)y01), e4m3_to_f16((uint16_t)y23));
        mma_f16(o[4 * i + 3], pf, e4m3_to_f16((uint16_t)(y01 >> 16)), e4m3_to_f16((uint16_t)(y23 >> 16)));
      }
    }
    slot = slot + 1 == kStages ? 0 : slot + 1;
    parity ^= 1;

    const bool last_tile = now.tile + 1 == now.tiles;
    if (last_tile || to_do == 1) {
      // the row tile ends here, or this CTA's part of it does
      const bool whole = last_tile && first_tile == 0;
      const int64_t part = (2 * (int64_t)blockIdx.x + (segment > 0)) * ROWS;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      float factor[2] = {1.0f, 1.0f};
      if constexpr (WK > 1) {
        // the warps of a row tile join in their order, through the stage that they have just read
        static_assert(WM == 4 || ROWS * (D + 4) * 4 <= Tile<D>::kStage, "a joined row tile must fit a stage");
        float* join_o = reinterpret_cast<float*>(stage);   // [ROWS][D + 4]
        if (c == 0) join_ml[warp * 16 + n] = make_float2(m[0], l[0]), join_ml[warp * 16 + n + 8] = make_float2(m[1], l[1]);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = -3.402823466e38f, sum = 0.0f;
#pragma unroll
          for (int w = 0; w < WK; ++w) top = fmaxf(top, join_ml[(w * WM + wm) * 16 + n + 8 * r].x);
#pragma unroll
          for (int w = 0; w < WK; ++w) {
            const float2 x = join_ml[(w * WM + wm) * 16 + n + 8 * r];
            sum += fast_exp2(x.x - top) * x.y;
          }
          factor[r] = fast_exp2(m[r] - top);
          m[r] = top, l[r] = sum;
        }
#pragma unroll 1
        for (int w = 0; w < WK; ++w) {
          if (w == wk) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                float* at = join_o + (wm * 16 + n + 8 * (x / 2)) * (D + 4) + channel<D>(2 * c + x % 2, t);
                const float y = o[t][x] * factor[x / 2];
                o[t][x] = w == 0 ? y : *at + y;
                if (w < WK - 1) *at = o[t][x];
              }
          }
          __syncthreads();
        }
      }
      if (wk == WK - 1) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = now.unit % a.row_tiles * ROWS + wm * 16 + n + 8 * r;
          if (row >= a.T * a.group) continue;
          const bool live = token[r] < now.fresh;
          if (whole) {
            T* dst = static_cast<T*>(a.out) + now.b * a.out_st.b + token[r] * a.out_st.s + head[r] * a.out_st.h;
            const float inverse = !live || l[r] == 0.0f ? 0.0f : 1.0f / l[r];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < NT; t += 4)
                *reinterpret_cast<uint2*>(dst + channel<D>(2 * c + e, t)) =
                    live ? make_uint2(pack2(o[t][2 * r + e] * inverse, o[t + 1][2 * r + e] * inverse, T()),
                                      pack2(o[t + 2][2 * r + e] * inverse, o[t + 3][2 * r + e] * inverse, T()))
                         : make_uint2(0, 0);
            if (a.lse != nullptr && c == 0)
              a.lse[((int64_t)now.b * a.H + head[r]) * a.T + token[r]] =
                  !live || l[r] == 0.0f ? -INFINITY : (m[r] + log2f(l[r])) * 0.69314718055994531f;
          } else {
            const int64_t at = part + wm * 16 + n + 8 * r;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < NT; t += 4)
                *reinterpret_cast<float4*>(a.part_o + at * D + channel<D>(2 * c + e, t)) = make_float4(
                    o[t][2 * r + e], o[t + 1][2 * r + e], o[t + 2][2 * r + e], o[t + 3][2 * r + e]);
            if (c == 0) a.part_ml[at] = make_float2(m[r], l[r]);
          }
        }
      }
      ++segment;
      fresh_unit = true;
    }
    if (to_do > 1) advance(a, now);
  }
  copy_wait<0>();
}

// Joins the partial rows of the row tiles that fell to several CTAs, and writes the rows that see nothing at all.  A warp
// takes a row; the CTAs of a row tile are joined in the order of its keys.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const PagedAttnArgs a, int tile_rows, int blocks_per_unit) {
  __shared__ int64_t warp_sums[kThreads / 32];
  const int64_t id = blockIdx.x / blocks_per_unit;
  const int per = a.p.Hkv * a.row_tiles, b = (int)(id / per), unit = (int)(id - (int64_t)b * per);
  int len, fresh;
  const int tiles = sequence(a, b, len, fresh);
  int64_t mine = 0, before = 0;
  {
    int x, y;
    for (int s = threadIdx.x; s < a.B; s += kThreads) {
      const int t = sequence(a, s, x, y);
      mine += t;
      if (s < b) before += t;
    }
  }
  int64_t list, start;
  scan_before(mine, warp_sums, list);
  scan_before(before, warp_sums, start);
  list *= per;
  start = start * per + (int64_t)unit * tiles;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int c0 = 0, c1 = 0, slot = 0;
  if (tiles > 0) {
    const int share = sharers(a, list);
    c0 = (int)(((start + 1) * share - 1) / list);
    c1 = (int)(((start + tiles) * share - 1) / list);
    if (c0 == c1) return;                                       // the CTA wrote the rows itself
    slot = (int64_t)c0 * list / share < start ? 1 : 0;          // not the first row tile of CTA c0
  }
  const int lane = threadIdx.x % 32;
  for (int row = blockIdx.x % blocks_per_unit * (kThreads / 32) + threadIdx.x / 32; row < tile_rows;
       row += blocks_per_unit * (kThreads / 32)) {
    const int r = unit % a.row_tiles * tile_rows + row;
    if (r >= a.T * a.group) break;
    const int token = r / a.group, head = unit / a.row_tiles * a.group + r % a.group;
    const bool live = tiles > 0 && token < fresh;
    float top = -3.402823466e38f, sum = 0.0f, o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.0f;
    if (live) {
      for (int x = c0 + lane; x <= c1; x += 32)
        top = fmaxf(top, a.part_ml[(2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows + row].x);
#pragma unroll
      for (int x = 16; x > 0; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
#pragma unroll 4
      for (int x = c0; x <= c1; ++x) {
        const int64_t at = (2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows + row;
        const float2 ml = a.part_ml[at];
        const float f = fast_exp2(ml.x - top);
        sum = fmaf(f, ml.y, sum);
#pragma unroll
        for (int i = 0; i < D / 32; i += D % 64 ? 1 : 2) {
          if constexpr (D % 64 == 0) {
            const float2 v = *reinterpret_cast<const float2*>(a.part_o + at * D + i * 32 + lane * 2);
            o[i] = fmaf(f, v.x, o[i]), o[i + 1] = fmaf(f, v.y, o[i + 1]);
          } else {
            o[i] = fmaf(f, a.part_o[at * D + i * 32 + lane], o[i]);
          }
        }
      }
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* dst = static_cast<T*>(a.out) + b * a.out_st.b + token * a.out_st.s + head * a.out_st.h;
#pragma unroll
    for (int i = 0; i < D / 32; i += D % 64 ? 1 : 2) {
      if constexpr (D % 64 == 0)
        *reinterpret_cast<uint32_t*>(dst + i * 32 + lane * 2) = pack2(o[i] * inverse, o[i + 1] * inverse, T());
      else
        dst[i * 32 + lane] = T(o[i] * inverse);
    }
    if (a.lse != nullptr && lane == 0)
      a.lse[((int64_t)b * a.H + head) * a.T + token] =
          sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
  }
}

// Row tiles of 16, 32 or 64 rows: the smallest that holds the rows of a kv head, 64 at the most.
static int row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

static int shared_ctas(int D) { return sm_count() * (D == 256 ? 2 : 3); }

template <typename T, int D, int WM>
static int launch_paged_attn(const PagedAttnArgs& a, cudaStream_t st) {
  constexpr int kSmem = smem_bytes<D>();
  static std::atomic<uint64_t> prepared{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(prepared.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(paged_attn_kernel<T, D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess && dev < 64) prepared.fetch_or(uint64_t(1) << dev);
  }
  if (e == cudaSuccess) {
    paged_attn_kernel<T, D, WM><<<a.ctas, kThreads, kSmem, st>>>(a);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    const int rows = std::min(16 * WM, a.T * a.group);
    const int blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.B * a.p.Hkv * a.row_tiles * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D>, a, 16 * WM, blocks);
  }
  if (e == cudaSuccess) return SAGE_OK;
  set_error("paged attention: %s", cudaGetErrorString(e));
  return SAGE_ERR_LAUNCH;
}

}  // namespace sage

using namespace sage;

extern "C" size_t sage_paged_attention_workspace_bytes(int B, int T, int H, int Hkv, int D) {
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || sage_qk_row_bytes(D) == 0) return 0;
  const int64_t rows = (int64_t)T * (H / Hkv);
  const size_t slots = (size_t)2 * shared_ctas(D) * 16 * row_warps(rows > 64 ? 64 : (int)rows);
  return slots * (D * sizeof(float) + sizeof(float2));
}

extern "C" int sage_paged_attention(const void* q, int dtype, int B, int T, int H, int Hkv, int D, int64_t qsb,
                                    int64_t qss, int64_t qsh, const int8_t* k8, const float* ks, const uint8_t* v8,
                                    const float* vs, int num_pages, int page_size, const int32_t* page_table,
                                    int64_t table_stride, int max_pages, const int32_t* lens, const int32_t* counts,
                                    const uint8_t* mask, int64_t mask_b, int64_t mask_i, double sm_scale, void* out,
                                    int64_t osb, int64_t oss, int64_t osh, float* lse, void* workspace,
                                    size_t workspace_bytes, int* status, void* stream) {
  NvtxRange nvtx("sage_paged_attention");
  set_error("%s", "");
  int rc = check_rows(dtype, B, T, H, D);
  if (rc == SAGE_OK && (Hkv <= 0 || H % Hkv != 0)) {
    set_error("heads %d must be a multiple of kv heads %d", H, Hkv);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK) rc = check_rows_pointer(q, qsb, qss, qsh, "q");
  if (rc == SAGE_OK) rc = check_rows_pointer(out, osb, oss, osh, "out");
  PagedAttnArgs a{};
  if (rc == SAGE_OK)
    rc = paged_args(&a.p, const_cast<int8_t*>(k8), const_cast<float*>(ks), const_cast<uint8_t*>(v8),
                    const_cast<float*>(vs), num_pages, page_size, Hkv, D, page_table, table_stride, max_pages, lens,
                    status);
  if (rc == SAGE_OK && (int64_t)max_pages * page_size > (int64_t)INT_MAX - T - kTileKeys) {
    set_error("%d pages of %d keys: positions must fit 32 bits", max_pages, page_size);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK && (int64_t)B * T * H > INT_MAX / 64) {
    set_error("%d sequences of %d tokens and %d heads are too many for one call", B, T, H);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  const size_t need = rc == SAGE_OK ? sage_paged_attention_workspace_bytes(B, T, H, Hkv, D) : 0;
  if (rc == SAGE_OK && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u))) {
    set_error("workspace of %zu bytes (16-byte aligned) required, got %zu", need, workspace_bytes);
    rc = SAGE_ERR_INVALID;
  }
  if (rc != SAGE_OK) return rc;
  a.q = q, a.q_st = {qsb, qss, qsh};
  a.out = out, a.out_st = {osb, oss, osh};
  a.lse = lse, a.counts = counts;
  a.mask = mask, a.mask_b = mask_b, a.mask_i = mask_i;
  a.B = B, a.T = T, a.H = H, a.group = H / Hkv;
  const int rows = T * a.group, wm = row_warps(rows);
  a.row_tiles = (rows + 16 * wm - 1) / (16 * wm);
  a.ctas = shared_ctas(D);
  a.scale = (float)((sm_scale > 0.0 ? sm_scale : 1.0 / std::sqrt((double)D)) * 1.4426950408889634);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * a.ctas * 16 * wm * D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    constexpr int kD = decltype(d)::value;
    if (dtype == SAGE_BF16)
      return wm == 1 ? launch_paged_attn<__nv_bfloat16, kD, 1>(a, st)
                     : wm == 2 ? launch_paged_attn<__nv_bfloat16, kD, 2>(a, st) : launch_paged_attn<__nv_bfloat16, kD, 4>(a, st);
    return wm == 1 ? launch_paged_attn<__half, kD, 1>(a, st)
                   : wm == 2 ? launch_paged_attn<__half, kD, 2>(a, st) : launch_paged_attn<__half, kD, 4>(a, st);
  });
}
