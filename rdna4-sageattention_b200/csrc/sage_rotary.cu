// Rotary positions for q and k, forward and gradient.
//
// Pair (x1, x2) of channels with frequency w_i at position p, a = p * w_i:
//   y1 = m * (x1 cos a - x2 sin a),   y2 = m * (x2 cos a + x1 sin a);   the gradient is the same with -a.
// Half layout pairs channel i with i + R/2, interleaved layout 2i with 2i + 1 (i < R/2); channels past R are copied.
//
// The angle is reduced in integers: a frequency is held in turns (w / 2 pi) as a 64-bit fixed-point fraction, so the
// fraction of a turn at position p is the low 64 bits of p * turns, exact for any position (a product in 32-bit
// floats is off by 0.06 radians at p = 10^6).  Its upper 32 bits go to sincospi.
//
// Bound by memory: 4 x 8192 tokens of 40 heads, D 128, take 114 us on B200, 5.9 TB/s or 90 % of the measured copy rate (with
// one head under way at a time 245 us).
#include <algorithm>

#include "../../include/sage_b200.h"
#include "sage_internal.h"
#include "sage_ptx.cuh"
#include "sage_rows.cuh"

namespace sage {

struct RotaryArgs {
  const void* in[2];   // q, k
  void* out[2];
  Strides3 in_st[2], out_st[2];
  int heads[2];
  int S, D, R;
  int64_t tokens;      // B * S
  const void* positions;
  int pos64;
  int64_t pos_b, pos_s;
  const uint64_t* turns;
  float magnitude;     // factor of both cosine and sine
  float sine_sign;     // -1 in the gradient
};

// One thread holds two runs of 8 channels (8 pairs in all) of one token and walks over the heads, so each sine is computed
// once for all of its heads; kBatch heads are loaded before the first is turned.  Half layout: the runs are the partners
// of one another; interleaved: each holds four pairs.  Neighbouring threads hold neighbouring runs.
constexpr int kBatch = 4;

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  const uint32_t units = a.D / 16;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const uint32_t u = id % units, token = id / units;
  if (token >= (uint32_t)a.tokens) return;
  const uint32_t b = token / a.S, s = token - b * a.S;
  // first channel of either run, and whether it is turned
  int c0, c1;
  bool turned, turned1;
  if (INTERLEAVED) {
    c0 = u * 8, c1 = a.D / 2 + u * 8;
    turned = c0 < a.R, turned1 = c1 < a.R;
  } else {
    const int v = (int)u - a.R / 16;   // past the turned runs
    turned = turned1 = v < 0;
    c0 = turned ? u * 8 : a.R + v * 8, c1 = turned ? a.R / 2 + u * 8 : a.R + (a.D - a.R) / 2 + v * 8;
  }
  const T* src[2];
  T* dst[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    src[w] = static_cast<const T*>(a.in[w]) + b * a.in_st[w].b + s * a.in_st[w].s;
    dst[w] = static_cast<T*>(a.out[w]) + b * a.out_st[w].b + s * a.out_st[w].s;
  }
  const int total = a.heads[0] + a.heads[1], step = gridDim.y * kBatch;
  float cs[8], sn[8];
  for (int h0 = blockIdx.y * kBatch; h0 < total; h0 += step) {
    uint4 x[kBatch][2];
    int64_t at[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i, w = h >= a.heads[0], hh = h - (w ? a.heads[0] : 0);
      at[i] = hh * a.out_st[w].h;
      if (h < total) {
        const T* p = src[w] + hh * a.in_st[w].h;
        x[i][0] = *reinterpret_cast<const uint4*>(p + c0);
        x[i][1] = *reinterpret_cast<const uint4*>(p + c1);
      }
    }
    if (h0 == (int)blockIdx.y * kBatch && turned) {   // beside the first loads
      const int64_t place = b * a.pos_b + s * a.pos_s;
      const uint64_t pos = a.pos64 ? (uint64_t) static_cast<const int64_t*>(a.positions)[place]
                                   : (uint64_t)(int64_t) static_cast<const int*>(a.positions)[place];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int pair = !INTERLEAVED ? u * 8 + e : (e < 4 ? c0 : c1) / 2 + e % 4;
        if (INTERLEAVED && e >= 4 && !turned1) break;
        const uint64_t turn = pos * a.turns[pair];
        const int half_turns = (int)(uint32_t)((turn + 0x80000000ull) >> 32);   // units of 2^-31 half turns
        sincospif((float)half_turns * 0x1p-31f, &sn[e], &cs[e]);
        cs[e] *= a.magnitude;
        sn[e] *= a.magnitude * a.sine_sign;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i;
      if (h >= total) break;
      T* p = dst[h >= a.heads[0]] + at[i];
      if (turned) {
        float y[2][8];
        unpack8(x[i][0], y[0], T());
        unpack8(x[i][1], y[1], T());
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (INTERLEAVED && e >= 4 && !turned1) break;
          float& p1 = INTERLEAVED ? y[e / 4][2 * e % 8] : y[0][e];
          float& p2 = INTERLEAVED ? y[e / 4][2 * e % 8 + 1] : y[1][e];
          const float x1 = p1, x2 = p2;
          p1 = x1 * cs[e] - x2 * sn[e];
          p2 = x2 * cs[e] + x1 * sn[e];
        }
        store8(p + c0, y[0]);
        if (turned1)
          store8(p + c1, y[1]);
        else
          *reinterpret_cast<uint4*>(p + c1) = x[i][1];
      } else {
        *reinterpret_cast<uint4*>(p + c0) = x[i][0];
        *reinterpret_cast<uint4*>(p + c1) = x[i][1];
      }
    }
  }
}

}  // namespace sage

using namespace sage;

extern "C" int sage_rotary(const sage_rotary_args* args, void* stream) {
  NvtxRange nvtx("sage_rotary");
  set_error("%s", "");
  if (args == nullptr) {
    set_error("rotary: no arguments");
    return SAGE_ERR_INVALID;
  }
  const sage_rotary_args& x = *args;
  const int dtype = x.dtype, B = x.B, S = x.S, H = x.H, Hkv = x.Hkv, D = x.D, R = x.R;
  const bool interleaved = x.interleaved != 0;
  int rc = check_rows(dtype, B, S, H, D);
  if (rc != SAGE_OK) return rc;
  if (R < 16 || R > D || R % 16 != 0 || Hkv < 0 || (x.position_bits != 32 && x.position_bits != 64)) {
    set_error("rotary: rotary_dim %d (a multiple of 16 up to head_dim %d), kv heads %d, %d-bit positions", R, D, Hkv,
              x.position_bits);
    return SAGE_ERR_UNSUPPORTED;
  }
  if (x.positions == nullptr || x.turns == nullptr) {
    set_error("rotary: positions and turns must be device arrays");
    return SAGE_ERR_INVALID;
  }
  rc = check_rows_pointer(x.q, x.q_st, "q");
  if (rc == SAGE_OK) rc = check_rows_pointer(x.q_out, x.q_out_st, "q_out");
  if (rc == SAGE_OK && Hkv > 0) rc = check_rows_pointer(x.k, x.k_st, "k");
  if (rc == SAGE_OK && Hkv > 0) rc = check_rows_pointer(x.k_out, x.k_out_st, "k_out");
  if (rc != SAGE_OK) return rc;
  RotaryArgs a{};
  a.in[0] = x.q, a.in[1] = x.k, a.out[0] = x.q_out, a.out[1] = x.k_out;
  a.in_st[0] = strides3(x.q_st), a.in_st[1] = strides3(x.k_st);
  a.out_st[0] = strides3(x.q_out_st), a.out_st[1] = strides3(x.k_out_st);
  a.heads[0] = H, a.heads[1] = Hkv;
  a.S = S, a.D = D, a.R = R;
  a.tokens = (int64_t)B * S;
  a.positions = x.positions, a.pos64 = x.position_bits == 64, a.pos_b = x.position_st[0], a.pos_s = x.position_st[1];
  a.turns = x.turns;
  a.magnitude = x.magnitude;
  a.sine_sign = x.backward ? -1.0f : 1.0f;
  const int64_t blocks = (a.tokens * (D / 16) + 255) / 256;
  if (blocks > (1 << 23)) {   // 32-bit thread numbers
    set_error("rotary: %lld tokens are too many for one call", (long long)a.tokens);
    return SAGE_ERR_UNSUPPORTED;
  }
  // few tokens: their heads are shared by several threads, so that the GPU is filled
  const int batches = (H + Hkv + kBatch - 1) / kBatch;
  const int64_t share = blocks >= 2048 ? 1 : (2048 + blocks - 1) / blocks;
  const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(batches, share));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SAGE_BF16)
    interleaved ? rotary_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(a)
                : rotary_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(a);
  else
    interleaved ? rotary_kernel<__half, true><<<grid, 256, 0, st>>>(a)
                : rotary_kernel<__half, false><<<grid, 256, 0, st>>>(a);
  return launch_result("rotary");
}
