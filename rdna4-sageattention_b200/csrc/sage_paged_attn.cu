// Attention over the paged K/V cache for the tokens of one step: single tokens, a run of tokens, or a tree of drafts.
//
// Row (b, i, h) sees the keys j < lens[b] and the drafted keys lens[b] + t with t <= i (no mask) or mask[b, i, t]:
//   s_j = sm_scale * ks_j * (q . k8_j),   p_j = exp(s_j - m),   o = sum_j p_j vs_j v8_j / sum_j p_j
// One pass over the keys with a running maximum m and sum.
#include <cmath>

#include "../../include/sage_b200.h"
#include "sage_internal.h"
#include "sage_paged.cuh"
#include "sage_ptx.cuh"

namespace sage {

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
  int B, T, H;
  float scale;         // sm_scale * log2(e)
};

__device__ __forceinline__ bool sees(const PagedAttnArgs& a, int b, int i, int t) {
  return t < 0 || (a.mask != nullptr ? a.mask[b * a.mask_b + i * a.mask_i + t] != 0 : t <= i);
}

// One CTA per row; its four warps take every fourth key and join at the end.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int C = D / 32;   // channels of a lane
  __shared__ float part[4][D + 2];
  const int h = blockIdx.x % a.H, i = blockIdx.x / a.H % a.T, b = blockIdx.x / a.H / a.T;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int len = a.p.lens[b], fresh = a.counts != nullptr ? a.counts[b] : a.T;
  const bool bad = len < 0 || fresh < 0 || fresh > a.T ||
                   (int64_t)len + fresh > ((int64_t)a.p.max_pages << a.p.page_shift);
  if (bad && threadIdx.x == 0) raise_invalid(a.p);
  const int keys = bad || i >= fresh ? 0 : len + fresh;
  float q[C], o[C], m = -INFINITY, l = 0.0f;
  const T* src = static_cast<const T*>(a.q) + b * a.q_st.b + i * a.q_st.s + h * a.q_st.h;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    q[c] = (float)src[lane * C + c] * a.scale;
    o[c] = 0.0f;
  }
  for (int j = warp; j < keys; j += 4) {
    if (!sees(a, b, i, j - len)) continue;
    const int64_t row = paged_row(a.p, b, h / (a.H / a.p.Hkv), j);
    if (row < 0) continue;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += q[c] * (float)a.p.k8[row * D + lane * C + c];
#pragma unroll
    for (int x = 16; x > 0; x /= 2) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.p.ks[row];
    const float top = fmaxf(m, s), keep = m == top ? 1.0f : exp2f(m - top), p = exp2f(s - top), vs = a.p.vs[row];
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const __nv_fp8_storage_t code = a.p.v8[row * D + lane * C + c];
      o[c] = o[c] * keep + p * vs * __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) part[warp][lane * C + c] = o[c];
  if (lane == 0) part[warp][D] = m, part[warp][D + 1] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][D]);
  float factor[4];
  for (int w = 0; w < 4; ++w) {
    factor[w] = part[w][D + 1] == 0.0f ? 0.0f : exp2f(part[w][D] - top);
    sum += factor[w] * part[w][D + 1];
  }
  T* dst = static_cast<T*>(a.out) + b * a.out_st.b + i * a.out_st.s + h * a.out_st.h;
  for (int c = threadIdx.x; c < D; c += 128) {
    float x = 0.0f;
    for (int w = 0; w < 4; ++w) x += factor[w] * part[w][c];
    dst[c] = T(sum == 0.0f ? 0.0f : x / sum);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[((int64_t)b * a.H + h) * a.T + i] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace sage

using namespace sage;

extern "C" size_t sage_paged_attention_workspace_bytes(int B, int T, int H, int Hkv, int D) {
  (void)B, (void)T, (void)H, (void)Hkv, (void)D;
  return 0;
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
  if (rc == SAGE_OK && (int64_t)max_pages * page_size > (int64_t)INT_MAX - T) {
    set_error("%d pages of %d keys: positions must fit 32 bits", max_pages, page_size);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK && (int64_t)B * T * H > INT_MAX) {
    set_error("%d sequences of %d tokens and %d heads are too many for one call", B, T, H);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  const size_t need = sage_paged_attention_workspace_bytes(B, T, H, Hkv, D);
  if (rc == SAGE_OK && need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("workspace of %zu bytes (16-byte aligned) required, got %zu", need, workspace_bytes);
    rc = SAGE_ERR_INVALID;
  }
  if (rc != SAGE_OK) return rc;
  a.q = q, a.q_st = {qsb, qss, qsh};
  a.out = out, a.out_st = {osb, oss, osh};
  a.lse = lse, a.counts = counts;
  a.mask = mask, a.mask_b = mask_b, a.mask_i = mask_i;
  a.B = B, a.T = T, a.H = H;
  a.scale = (float)((sm_scale > 0.0 ? sm_scale : 1.0 / std::sqrt((double)D)) * 1.4426950408889634);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    if (dtype == SAGE_BF16)
      paged_attn_kernel<__nv_bfloat16, decltype(d)::value><<<B * T * H, 128, 0, st>>>(a);
    else
      paged_attn_kernel<__half, decltype(d)::value><<<B * T * H, 128, 0, st>>>(a);
    return launch_result("paged attention");
  });
}
