// Shared by the two kernels of paged attention (sage_paged_attn.cu for few query rows of a kv head, sage_paged_wide.cu for
// many): the list of work, the places in it, the tiles that TMA writes, and small device helpers.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/sage_b200.h"
#include "sage_internal.h"
#include "sage_paged.cuh"
#include "sage_ptx.cuh"

namespace sage {

constexpr int kTileKeys = 64;
constexpr int kMinTiles = 2;               // tiles a CTA takes at the least
constexpr float kLowest = -3.402823466e38f;   // of a reference: nothing seen yet
constexpr float kLazy = 8.0f;              // log2 of what may exceed a reference before it moves
constexpr float kHigh = 8.0f;              // log2 of a row's largest weight when its reference is placed
constexpr float kMostWeight = 32768.0f;    // a weight above it moves a reference
constexpr float kMostLog = 15.0f;          // its log2
constexpr float kMostSum = 256.0f;         // a mean of plain weights above it moves a reference
// Bounds of the references' ratio, log2.  From -110 up the sum of 64 numbers 2^(x - t) stays below 2^125; the lower bound binds
// where every V row so far is zero (their weights are 0) and for V scales below 2^-102, whose weights then lie up to 2^7 lower in
// fp16.  Up to 64 the weights down to 2^-62 of the largest are normal numbers.  120 is beyond all that append writes.
constexpr float kLeastRatio = -110.0f, kTameRatio = 64.0f, kMostRatio = 120.0f;

// What is known of a query row beside its O: the reference of its scores, the sum of its weights, the reference of its
// scores with the V scale in them (all three in the units of 2^x).
struct alignas(16) RowState {
  float m, l, t;
};

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
  RowState* part_state;   // [2 * ctas][rows of a tile]
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
template <int THREADS>
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
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

__device__ __forceinline__ int sharers(const PagedAttnArgs& a, int64_t list) {
  return (int)min((int64_t)a.ctas, (list + kMinTiles - 1) / kMinTiles);
}

// A place in the list.
struct Cursor {
  int b, unit, tile;        // sequence, kv head * row_tiles + row tile, key tile
  int tiles, len, fresh;    // of the sequence
};

// The CTA's stretch of the list: its first place, and its length (0: none; the call then returns at once, for all threads).
// Ends with a barrier of the CTA.
template <int THREADS>
__device__ __forceinline__ int64_t locate(const PagedAttnArgs& a, int64_t* warp_sums, int64_t* found, Cursor& now) {
  const int per = a.p.Hkv * a.row_tiles;
  int len, fresh;
  int64_t mine = 0, total;
  for (int b = threadIdx.x; b < a.B; b += THREADS) mine += sequence(a, b, len, fresh);
  int64_t at = scan_before<THREADS>(mine, warp_sums, total) * per;   // one sequence a thread: where it begins
  const int64_t list = total * per;
  const int share = sharers(a, list);
  if ((int)blockIdx.x >= share) return 0;
  const int64_t first = (int64_t)blockIdx.x * list / share, end = (int64_t)(blockIdx.x + 1) * list / share;
  if (a.B <= THREADS) {
    if (first >= at && first < at + mine * per) found[0] = threadIdx.x, found[1] = first - at;
  } else {
    int64_t carry = 0;
    for (int base = 0; base < a.B; base += THREADS) {
      const int b = base + threadIdx.x;
      const int64_t v = b < a.B ? (int64_t)sequence(a, b, len, fresh) * per : 0;
      at = carry + scan_before<THREADS>(v, warp_sums, total);
      if (first >= at && first < at + v) found[0] = b, found[1] = first - at;
      carry += total;
      if (first < carry) break;
    }
  }
  __syncthreads();
  now.b = (int)found[0];
  now.tiles = sequence(a, now.b, now.len, now.fresh);
  now.unit = (int)((uint32_t)found[1] / (uint32_t)now.tiles);   // below tiles * per, checked to fit 32 bits
  now.tile = (int)(found[1] - (int64_t)now.unit * now.tiles);
  return end - first;
}

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

// 2-D tile load: rows `y` ... of a [rows, bytes] tensor, bytes from `x` on.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait for a phase of a stage barrier.  Unlike mbar_wait it does not give up on an error that stands in the
// status word: a bad page of one sequence leaves the others' work as it is.
__device__ __forceinline__ bool wait_stage(uint64_t* bar, uint32_t parity, volatile int* given_up, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 63u) != 0) continue;
    if (*given_up != 0) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      *given_up = 1;
      *const_cast<volatile int*>(status) = kStatusTimeout;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What the online softmax knows of a query row: t, the reference of its scores with the V scale in them (m'); l, the sum of
// 2^(x - m); and ratio = 2^(t - m), where m is the reference of the scores themselves.  A ratio at which 2^(x - t) may leave the
// range of fp32 is negative: what is multiplied by it fails a comparison of bits().  Sign and exponent of the ratio, which has no
// fraction, share a word with the exponent of the power of two that a bf16 row was divided by: a register a row less, 161 -> 156
// us for one token of 16 long sequences.
struct Softmax {
  float t, l;
  uint32_t word;

  __device__ __forceinline__ void clear() { t = kLowest, l = 0.0f, word = 0x3f800000u; }
  __device__ __forceinline__ void set_row_exponent(int e) { word = (word & 0xff800000u) | (uint32_t)e; }
  __device__ __forceinline__ float row_scale() const { return __uint_as_float(word << 23); }
  __device__ __forceinline__ float ratio() const { return __uint_as_float(word & 0xff800000u); }
  __device__ __forceinline__ float exponent() const { return (float)((int)(word >> 23 & 255u) - 127); }
  __device__ __forceinline__ float m() const { return t - exponent(); }
  __device__ __forceinline__ float v_unit() const { return fabsf(ratio()); }                                        // 2^(t - m)
  __device__ __forceinline__ float score_unit() const { return __int_as_float((254 << 23) - __float_as_int(v_unit())); }   // 2^(m - t)
  // Whether a score x, or the same with the V scale in it, exceeds its reference by more than they wait for.
  __device__ __forceinline__ bool exceeded(float x, float with_v) const { return x > m() + kLazy || with_v > t + kMostLog; }
  // Moves the references to the largest of either, rescales l, and returns the factor of O.
  __device__ __forceinline__ float move(float top, float top_v) {
    const float before = m(), old = exponent();
    const float next = fmaxf(before, ceilf(top)), step = before - next;
    const float now = fminf(fmaxf(fmaxf(old + step, ceilf(top_v) - kHigh - next), kLeastRatio), kMostRatio);
    t = next + now;
    word = (word & 0xffu) | (uint32_t)((int)now + 127) << 23 | (now > kTameRatio ? 0x80000000u : 0u);
    l *= fast_exp2(step);
    return fast_exp2(step + (old - now));
  }
  __device__ __forceinline__ RowState state() const { return RowState{m(), l, t}; }
};

// The exponent (biased) of a power of two near the largest value of a bf16 row, whose bits without the sign are `top`: with it
// the row is divided before it becomes fp16.  Zero, infinite and NaN rows: 1; tiny ones: 2^-100; the largest: 2^126, the last
// one whose inverse is normal (the row is then below 4).
__device__ __forceinline__ int row_exponent(uint32_t top) {
  return top == 0 || top >= 0x7f80u ? 127 : min(max((int)(top >> 7), 27), 253);
}

// As a bit pattern a positive float orders as it does as a number, with NaN and every negative one above.
__device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }

// Two weights -> an fp16 pair, the largest finite number for what is above it.
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Transposes an 8 x 8 tile of 16-bit values across the warp (row lane / 4, columns 2 (lane % 4) and the next).
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Shared-memory tiles, as TMA writes them: 64 rows of K, 64 rows of V, of 128 swizzled bytes (D 256: two such halves), 64
// swizzled bytes (D 64) or 96 plain ones.  A warp works on groups of 16 keys; lane (n = lane / 4, c = lane % 4) takes the
// scores of the keys in slots n and n + 8 for the columns 2c and 2c + 1, and after the transposition the weights of the
// keys in slots 2c, 2c + 1, 2c + 8, 2c + 9 for column n.  slot_key() and first_channel() are chosen so that the lanes of one
// phase of a shared load touch different banks (D 64 and 96: two-way conflicts are left in V).
template <int D>
struct Tile {
  static constexpr bool kWide = D % 128 == 0;
  static constexpr int kBox = kWide ? 128 : D;            // bytes of a row in a box
  static constexpr int kHalves = D / kBox;
  static constexpr int kBytes = kTileKeys * D;            // of K, and of V
  static constexpr int kStage = 2 * kBytes;
  // where byte x of row `row` lies
  __device__ static int at(int row, int x) {
    if constexpr (kWide) return x / 128 * (kTileKeys * 128) + row * 128 + ((x % 128) ^ ((row & 7) << 4));
    if constexpr (D == 64) return row * 64 + (x ^ ((row >> 1 & 3) << 4));
    return row * D + x;
  }
  __device__ static int slot_key(int slot) { return kWide ? (slot & 8) | (slot & 7) >> 1 | (slot & 1) << 2 : slot; }
  // first of the D / 8 channels (D 256: of either half) whose output lane row n holds
  __device__ static int first_channel(int n) { return kWide ? ((n >> 1) | (n & 1) << 2) * 16 : n * (D / 8); }
  // channel of row n + 8 e of the output tile t
  __device__ static int channel(int n, int t, int e) { return first_channel(n) + (kWide ? t / 8 * 128 + t % 8 * 2 : t * 2) + e; }
};

// The producer warp's part: loads `todo` tiles from `now` on into a ring of raw stages (K rows, V rows) and their scales
// (64 of K, 64 of V a stage); a lane per page of the tile.
template <int D>
__device__ __forceinline__ void load_tiles(const PagedAttnArgs& a, const CUtensorMap* k_map, const CUtensorMap* v_map,
                                           Cursor now, int64_t todo, unsigned char* stages, float* scales,
                                           uint64_t* full, uint64_t* empty, int count, volatile int* given_up) {
  using S = Tile<D>;
  const int lane = threadIdx.x % 32;
  const int box_rows = min(kTileKeys, 1 << a.p.page_shift), boxes = kTileKeys / box_rows;
  auto lookup = [&](const Cursor& t) -> int64_t {   // cache row of the lane's first key, or -1
    const int64_t at = (int64_t)t.tile * kTileKeys + lane * box_rows;
    return lane < boxes && at < t.len + t.fresh ? paged_row(a.p, t.b, t.unit / a.row_tiles, at) : -1;
  };
  int64_t row = lookup(now);
  int slot = 0;
  uint32_t phase = 0;
  for (; todo > 0; --todo) {
    if (!wait_stage(empty + slot, phase ^ 1, given_up, a.p.status)) break;
    const int there = __popc(__ballot_sync(0xffffffffu, row >= 0));
    const uint32_t bar = smem_u32(full + slot);
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(there * box_rows * (2 * D + 8))
                   : "memory");
    __syncwarp();
    if (row >= 0) {
      const uint32_t k = smem_u32(stages + slot * S::kStage) + lane * box_rows * S::kBox;
      const uint32_t scale = smem_u32(scales + slot * 2 * kTileKeys + lane * box_rows);
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) {
        tma_load_2d(k + h * (kTileKeys * 128), k_map, bar, h * 128, (int)row);
        tma_load_2d(k + S::kBytes + h * (kTileKeys * 128), v_map, bar, h * 128, (int)row);
      }
      bulk_load(scale, a.p.ks + row, box_rows * 4, bar);
      bulk_load(scale + kTileKeys * 4, a.p.vs + row, box_rows * 4, bar);
    }
    if (todo > 1) {
      advance(a, now);
      row = lookup(now);
    }
    if (++slot == count) slot = 0, phase ^= 1;
  }
  if (*given_up != 0)   // leave no copy in flight behind
    for (int s = 0; s < count; ++s) mbar_drain(full + s, s < slot ? phase : phase ^ 1);
}

// SMs of the current device (148 without one), asked for once per device.
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Launch that may begin while the stream's kernel before it ends (its blocks are placed and set themselves up); the kernel
// waits with griddepcontrol.wait before it touches global memory.
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The codes as [rows, D] bytes; a box is the rows of a page that a tile of keys takes, 128 bytes of each (or all of them).
template <int D>
inline bool code_map(CUtensorMap* map, const void* base, uint64_t rows, int page_size) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the CUDA driver");
    return false;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)D, rows}, strides[1] = {(cuuint64_t)D};
  const cuuint32_t box[2] = {(cuuint32_t)Tile<D>::kBox, (cuuint32_t)std::min(page_size, kTileKeys)}, steps[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE,
                        Tile<D>::kWide ? CU_TENSOR_MAP_SWIZZLE_128B
                                       : D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return true;
  set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
  return false;
}

// The kernel for many rows: its CTAs, the rows of its row tiles, and its launch (the join follows by the caller).
int wide_ctas();
int wide_rows(int D);
int launch_paged_wide(const PagedAttnArgs& a, int dtype, cudaStream_t st);

}  // namespace sage
