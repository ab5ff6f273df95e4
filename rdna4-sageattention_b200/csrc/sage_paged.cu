// The paged K/V cache: rows quantised as they are written, read back, and moved when drafted tokens are dropped.
//
// A row (one token of one kv head) is stored on its own, so the cache grows by single tokens:
//   K: int8 codes round(127 x / a), scale a / 127;   V: e4m3 codes of 448 x / a, scale a / 448;   a = max |x|.
// Both roundings are to nearest, ties away from zero.  For 16-bit x the quotient is a ratio of small integers: it is a
// tie exactly, or at least 2^-16 (relative, e4m3) resp. 2^-(12 + d) (absolute, int8, for a quotient below 2^(8 - d)) away
// from one.  The product with 127 / a resp. 448 / a is off by less than 2^-21 (the reciprocal by 2^-23, three roundings by
// 2^-24), so pushed outwards by 2^-21 it falls on the right side of every border, and no division per element is needed.
// Rows with an infinity or NaN store scale NaN and codes 0; rows with a < 2^-100 store zeros.
//
// Measured on B200, 8 kv heads, D 128: append of 4 x 8190 tokens (ragged, 25 us at the measured copy rate) 39 us, bound by its
// instructions; read of 8 x 32760 positions 240 us, 98 % of that rate (with 16 channels a thread, two stores half a line
// apart, 304); keep of 12 rows of 256 sequences 6 us, a chain of dependent loads.
#include "../../include/sage_b200.h"
#include "sage_internal.h"
#include "sage_paged.cuh"
#include "sage_ptx.cuh"

namespace sage {

int paged_args(PagedArgs* out, const sage_paged_kv& kv) {
  int shift = 4;
  while (shift < 8 && (1 << shift) < kv.page_size) ++shift;
  if ((1 << shift) != kv.page_size) {
    set_error("page_size %d (a power of two from 16 to 256 required)", kv.page_size);
    return SAGE_ERR_UNSUPPORTED;
  }
  if (kv.num_pages <= 0 || kv.Hkv <= 0 || kv.max_pages <= 0) {
    set_error("empty cache (num_pages=%d Hkv=%d max_pages=%d)", kv.num_pages, kv.Hkv, kv.max_pages);
    return SAGE_ERR_UNSUPPORTED;
  }
  for (const void* p : {(const void*)kv.k8, (const void*)kv.ks, (const void*)kv.v8, (const void*)kv.vs})
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u)) {
      set_error("cache buffers k8, ks, v8 and vs must be 16-byte aligned");
      return SAGE_ERR_INVALID;
    }
  if (kv.page_table == nullptr || kv.lens == nullptr) {
    set_error("page_table and lens must be device arrays");
    return SAGE_ERR_INVALID;
  }
  int* word = kv.status != nullptr ? kv.status : default_status_word();
  if (word == nullptr) {
    set_error("no status word on this device");
    return SAGE_ERR_LAUNCH;
  }
  *out = PagedArgs{kv.k8, kv.ks, kv.v8, kv.vs, kv.num_pages, shift, kv.Hkv, kv.D, kv.page_table, kv.table_stride,
                   kv.max_pages, kv.lens, word};
  return SAGE_OK;
}

constexpr float kTiny = 0x1p-100f;
constexpr float kOutwards = 1.0f + 0x1p-21f;

template <typename T>
constexpr uint32_t kInfBits = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;

__device__ __forceinline__ float from_bits(uint32_t bits, __nv_bfloat16) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float from_bits(uint32_t bits, __half) { return __half2float(__ushort_as_half((uint16_t)bits)); }

struct AppendArgs {
  PagedArgs p;
  const void* x[2];   // K, V
  Strides3 st[2];
  const int* counts;
  int S;
};

// A group of LPR lanes (a power of two, D / 8 of them with data) holds kTokens consecutive tokens of one head of K and of V,
// 8 channels a lane.  The rows are loaded before their places in the cache are looked up: the chain of dependent loads
// (length, page, row) would otherwise leave the memory idle (one token a lane, looked up first: 55 us for 4 x 8190
// tokens of 8 heads, D 128).
constexpr int kTokens = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  constexpr int LPR = D == 64 ? 8 : D == 256 ? 32 : 16;
  const int lane = threadIdx.x % LPR;
  const uint32_t id = blockIdx.x * (256u / LPR) + threadIdx.x / LPR, run = id / a.p.Hkv;
  const int h = (int)(id - run * a.p.Hkv), s0 = (int)run * kTokens, b = blockIdx.y;
  uint4 x[2][kTokens];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const T* src = static_cast<const T*>(a.x[w]) + b * a.st[w].b + s0 * a.st[w].s + h * a.st[w].h + lane * 8;
#pragma unroll
    for (int r = 0; r < kTokens; ++r)
      x[w][r] = s0 + r < a.S && lane * 8 < D ? *reinterpret_cast<const uint4*>(src + r * a.st[w].s)
                                             : make_uint4(0, 0, 0, 0);
  }
  const int len = a.p.lens[b];
  int n = a.counts != nullptr ? a.counts[b] : a.S;
  if (n < 0 || n > a.S || len < 0) {   // none of the sequence's tokens: some would land in its context
    raise_invalid(a.p);
    n = 0;
  }
#pragma unroll
  for (int r = 0; r < kTokens; ++r) {
    const bool live = s0 + r < n;
    const int64_t dst = live ? paged_row(a.p, b, h, (int64_t)len + s0 + r) : -1;
    // The largest magnitudes of the K row (low half) and of the V row, as 16-bit patterns: without the sign they order as
    // the numbers do, with infinity and NaN above every finite one.
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint4 v = x[w][r];
      const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                  __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
      top |= max(m & 0xffffu, m >> 16) << (16 * w);
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o /= 2) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float y[8];
      unpack8(x[w][r], y, T());
      const uint32_t bits = w == 0 ? top & 0xffffu : top >> 16;
      const bool finite = bits < kInfBits<T>;
      const float amax = from_bits(bits, T());
      const bool kept = finite && amax >= kTiny;
      const float most = w == 0 ? 127.0f : 448.0f;
      float inverse;   // of amax / 4, which is normal for every amax that is kept
      asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(kept ? amax * 0.25f : 1.0f));
      const float mul = inverse * (most * 0.25f) * kOutwards;
      uint32_t code[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* z = y + 4 * i;
        if (w == 0) {   // 1.5 * 2^23 + x rounds x to a whole number, whose low byte is the code
          const uint32_t lo = __byte_perm(__float_as_uint(fmaf(z[0], mul, kMagicF)), __float_as_uint(fmaf(z[1], mul, kMagicF)), 0x0040);
          const uint32_t hi = __byte_perm(__float_as_uint(fmaf(z[2], mul, kMagicF)), __float_as_uint(fmaf(z[3], mul, kMagicF)), 0x0040);
          code[i] = __byte_perm(lo, hi, 0x5410);
        } else {
          code[i] = __byte_perm(pack_e4m3x2(z[0] * mul, z[1] * mul), pack_e4m3x2(z[2] * mul, z[3] * mul), 0x5410);
        }
      }
      if (dst >= 0 && lane * 8 < D) {
        uint8_t* to = w == 0 ? reinterpret_cast<uint8_t*>(a.p.k8) : a.p.v8;
        *reinterpret_cast<uint2*>(to + dst * D + lane * 8) = kept ? make_uint2(code[0], code[1]) : make_uint2(0, 0);
        // The quotient a / most, rounded once: the product in 64 bits is off by 2^-52 of it, and with an 11-bit a the quotient lies
        // on a border between two floats or at least 2^-32 of itself away from it (a division here: 41 us for 39).
        if (lane == 0) {
          const float scale = (float)((double)amax * (1.0 / most));
          (w == 0 ? a.p.ks : a.p.vs)[dst] = kept ? scale : finite ? 0.0f : __uint_as_float(0x7fc00000u);
        }
      }
    }
  }
}

struct ReadArgs {
  PagedArgs p;
  void* out[2];
  Strides3 st[2];
  int S;
};

// A thread reads 8 codes of kRun consecutive tokens (a run never leaves its page) of K and of V, all of them under way at
// once, and writes 8 channels of each, so that a warp's stores are whole lines.
constexpr int kRun = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  constexpr int LPR = D / 8;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x, row = id / LPR;   // run of tokens and head of the sequence
  const int c = (int)(id % LPR) * 8, b = blockIdx.y;
  const int run = (int)(row / a.p.Hkv), h = (int)(row - run * (uint32_t)a.p.Hkv), s0 = run * kRun;
  if (s0 >= a.S) return;
  const int n = a.p.lens[b];
  if (n < 0 || n > (int64_t)a.p.max_pages << a.p.page_shift) raise_invalid(a.p);
  const int64_t src = s0 < n ? paged_row(a.p, b, h, s0) : -1;
  uint2 code[2][kRun];
  float4 scale[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint8_t* from = w == 0 ? reinterpret_cast<const uint8_t*>(a.p.k8) : a.p.v8;
    const float* scales = w == 0 ? a.p.ks : a.p.vs;
#pragma unroll
    for (int r = 0; r < kRun; ++r)
      code[w][r] = src >= 0 && s0 + r < min(n, a.S) ? *reinterpret_cast<const uint2*>(from + (src + r) * D + c)
                                                    : make_uint2(0, 0);
    scale[w] = src >= 0 ? make_float4(scales[src], scales[src + 1], scales[src + 2], scales[src + 3])
                        : make_float4(0, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < kRun; ++r) {
    if (s0 + r >= a.S) break;
    const bool held = src >= 0 && s0 + r < n;   // what lies behind may be anything, a NaN scale too
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float f = !held ? 0.0f : r == 0 ? scale[w].x : r == 1 ? scale[w].y : r == 2 ? scale[w].z : scale[w].w;
      const uint32_t q[2] = {code[w][r].x, code[w][r].y};
      float x[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t lo, hi;
        if (w == 0)
          int8_to_f16(q[i], lo, hi);
        else
          lo = e4m3_to_f16((uint16_t)q[i]), hi = e4m3_to_f16((uint16_t)(q[i] >> 16));
        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[4 * i] = u.x * f, x[4 * i + 1] = u.y * f, x[4 * i + 2] = v.x * f, x[4 * i + 3] = v.y * f;
      }
      store8(static_cast<T*>(a.out[w]) + b * a.st[w].b + (s0 + r) * a.st[w].s + h * a.st[w].h + c, x);
    }
  }
}

struct KeepArgs {
  PagedArgs p;
  const int* keep;
  int64_t keep_stride;
  const int* counts;
  int N;
};

// One CTA per (sequence, head).  Kept rows move to the front in chunks, in order: a chunk is read before any of it is
// written, and since keep is strictly increasing (keep[i] >= i) no later chunk reads a row that an earlier one wrote.
template <int D>
__global__ void __launch_bounds__(256) keep_kernel(const KeepArgs a) {
  constexpr int LPR = D / 16, ROWS = 256 / (2 * LPR);   // lanes per row of one tensor; rows of a chunk
  const int b = blockIdx.x / a.p.Hkv, h = blockIdx.x % a.p.Hkv;
  const int n = a.counts != nullptr ? a.counts[b] : a.N;
  const int* keep = a.keep + b * a.keep_stride;
  const int64_t base = a.p.lens[b];
  bool bad = n < 0 || n > a.N || base < 0;
  if (!bad)
    for (int i = threadIdx.x; i < n; i += 256) bad |= keep[i] < 0 || (i > 0 && keep[i] <= keep[i - 1]);
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_invalid(a.p);
    return;
  }
  const int r = threadIdx.x / (2 * LPR), w = threadIdx.x / LPR % 2, lane = threadIdx.x % LPR;
  uint8_t* codes = w == 0 ? reinterpret_cast<uint8_t*>(a.p.k8) : a.p.v8;
  float* scales = w == 0 ? a.p.ks : a.p.vs;
  for (int i0 = 0; i0 < n; i0 += ROWS) {
    const int i = i0 + r;
    int64_t src = -1, dst = -1;
    if (r < ROWS && i < n) {
      src = paged_row(a.p, b, h, base + keep[i]);
      dst = paged_row(a.p, b, h, base + i);
    }
    const bool move = src >= 0 && dst >= 0 && src != dst;
    uint4 c = make_uint4(0, 0, 0, 0);
    float scale = 0.0f;
    if (move) {
      c = *reinterpret_cast<const uint4*>(codes + src * D + lane * 16);
      scale = scales[src];
    }
    __syncthreads();
    if (move) {
      *reinterpret_cast<uint4*>(codes + dst * D + lane * 16) = c;
      if (lane == 0) scales[dst] = scale;
    }
  }
}

}  // namespace sage

using namespace sage;

extern "C" {

// The arguments that append and read share, checked.
static int rows_args(PagedArgs* p, const sage_paged_rows_args* args, const char* what) {
  set_error("%s", "");
  if (args == nullptr) {
    set_error("%s: no arguments", what);
    return SAGE_ERR_INVALID;
  }
  int rc = check_rows(args->dtype, args->kv.B, args->S, args->kv.Hkv, args->kv.D);
  if (rc == SAGE_OK) rc = check_rows_pointer(args->k, args->k_st, "k");
  if (rc == SAGE_OK) rc = check_rows_pointer(args->v, args->v_st, "v");
  return rc == SAGE_OK ? paged_args(p, args->kv) : rc;
}

int sage_paged_append(const sage_paged_rows_args* args, void* stream) {
  NvtxRange nvtx("sage_paged_append");
  AppendArgs a{};
  const int rc = rows_args(&a.p, args, "append");
  if (rc != SAGE_OK) return rc;
  const int B = args->kv.B, S = args->S, Hkv = args->kv.Hkv, D = args->kv.D, dtype = args->dtype;
  a.x[0] = args->k, a.x[1] = args->v;
  a.st[0] = strides3(args->k_st), a.st[1] = strides3(args->v_st);
  a.counts = args->kv.counts;
  a.S = S;
  const int per_block = 256 / (D == 64 ? 8 : D == 256 ? 32 : 16);
  const int64_t blocks = ((int64_t)((S + kTokens - 1) / kTokens) * Hkv + per_block - 1) / per_block;
  if (blocks > (1 << 23) || B > 65535) {   // 32-bit thread numbers, grid limit
    set_error("append: %d sequences of %d tokens and %d heads are too many for one call", B, S, Hkv);
    return SAGE_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)blocks, (unsigned)B);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    if (dtype == SAGE_BF16)
      append_kernel<__nv_bfloat16, decltype(d)::value><<<grid, 256, 0, st>>>(a);
    else
      append_kernel<__half, decltype(d)::value><<<grid, 256, 0, st>>>(a);
    return launch_result("append");
  });
}

int sage_paged_read(const sage_paged_rows_args* args, void* stream) {
  NvtxRange nvtx("sage_paged_read");
  ReadArgs a{};
  const int rc = rows_args(&a.p, args, "read");
  if (rc != SAGE_OK) return rc;
  const int B = args->kv.B, S = args->S, Hkv = args->kv.Hkv, D = args->kv.D, dtype = args->dtype;
  a.out[0] = args->k, a.out[1] = args->v;
  a.st[0] = strides3(args->k_st), a.st[1] = strides3(args->v_st);
  a.S = S;
  const int64_t blocks = ((int64_t)((S + kRun - 1) / kRun) * Hkv * (D / 8) + 255) / 256;
  if (blocks > (1 << 23) || B > 65535) {   // 32-bit thread numbers, grid limit
    set_error("read: %d sequences of %d tokens and %d heads are too many for one call", B, S, Hkv);
    return SAGE_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)blocks, (unsigned)B);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    if (dtype == SAGE_BF16)
      read_kernel<__nv_bfloat16, decltype(d)::value><<<grid, 256, 0, st>>>(a);
    else
      read_kernel<__half, decltype(d)::value><<<grid, 256, 0, st>>>(a);
    return launch_result("read");
  });
}

int sage_paged_keep(const sage_paged_keep_args* args, void* stream) {
  NvtxRange nvtx("sage_paged_keep");
  set_error("%s", "");
  if (args == nullptr || args->keep == nullptr) {
    set_error("keep must be a device array");
    return SAGE_ERR_INVALID;
  }
  const int B = args->kv.B, N = args->N, Hkv = args->kv.Hkv, D = args->kv.D;
  int rc = check_rows(SAGE_BF16, B, N, Hkv, D);
  KeepArgs a{};
  if (rc == SAGE_OK) rc = paged_args(&a.p, args->kv);
  if (rc == SAGE_OK && (int64_t)B * Hkv > INT_MAX) {
    set_error("keep: %d sequences of %d heads are too many for one call", B, Hkv);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc != SAGE_OK) return rc;
  a.keep = args->keep, a.keep_stride = args->keep_stride, a.counts = args->kv.counts, a.N = N;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    keep_kernel<decltype(d)::value><<<B * Hkv, 256, 0, st>>>(a);
    return launch_result("keep");
  });
}

}  // extern "C"
