// Attention of a batch whose requests share long prefixes (16 query heads, 8 KV heads,
// head dim 128; query head h reads KV head h / 2).
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / 2]) v[j, h / 2]
//
// over the visible keys j of row t's request: its group's prefix rows, then its own
// cached rows, then its new rows, read in place from three sources. With `causal`, row
// x of a request with q rows and n keys sees keys j <= n - q + x. A row without a
// visible key gives zeros.
#pragma once
#include "attention.cuh"
#include "prefix_plan.cuh"

namespace dspark {
namespace prefix {

struct Source {
  const void* k;
  const void* v;
  long long off;     // row offset added to the plan's rows
  long long rows;
};

struct Params {
  const void* q;     // [total_q, 16, 128]
  void* out;
  const int* plan;
  int check, total_q, grid, slots;
  Source src[3];     // prefix, own, new
  float scale, scale_log2;
};

// Partial rows of one MMA tile: [128][128] fp32 (normalised), then 128 log2-sum-exp2.
constexpr size_t kSlotFloats = 128 * kHeadDim;
inline size_t workspace_bytes(int slots) { return static_cast<size_t>(slots) * (kSlotFloats + 128) * sizeof(float); }

__device__ __forceinline__ bool plan_ok(const Params& p) {
  return p.plan[kHMagic] == kPlanMagic && p.plan[kHCheck] == p.check && p.plan[kHTotalQ] == p.total_q;
}

template <typename T>
__device__ __forceinline__ void store_out(T* dst, float v);
template <>
__device__ __forceinline__ void store_out<float>(float* dst, float v) { *dst = v; }
template <>
__device__ __forceinline__ void store_out<__nv_bfloat16>(__nv_bfloat16* dst, float v) { *dst = __float2bfloat16_rn(v); }

__device__ __forceinline__ float load_in(const float* p) { return *p; }
__device__ __forceinline__ float load_in(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// CUDA-core kernel: one CTA per (request, block of 8 query rows, KV head); its 16 MMA
// rows (2 heads x 8 query rows) walk the request's keys 32 at a time with an online
// softmax, products and sums in fp32.
constexpr int kSimpleThreads = 128;
constexpr int kSimpleKeys = 32;

template <typename T>
__global__ void __launch_bounds__(kSimpleThreads) prefix_simple_kernel(const Params p) {
  __shared__ float sq[16][kHeadDim];
  __shared__ float sk[kSimpleKeys][kHeadDim + 1];
  __shared__ float sv[kSimpleKeys][kHeadDim];
  __shared__ float sp[16][kSimpleKeys];
  const int tid = threadIdx.x;
  if (!plan_ok(p)) {
    if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  const int* rec = p.plan + p.plan[kHRequestsAt] + static_cast<size_t>(blockIdx.x) * kRequestWords;
  const int h = blockIdx.z;
  const int q0 = rec[kRQ0], nq = rec[kRNq], r0 = blockIdx.y * kQBlock;
  if (r0 >= nq) return;
  const int len[3] = {rec[kRPrefixLen], rec[kROwnLen], rec[kRNewLen]};
  const int start[3] = {rec[kRPrefixRow], rec[kROwnRow], rec[kRNewRow]};
  const int keys = len[0] + len[1] + len[2];
  const int rows = min(kQBlock, nq - r0);
  const bool causal = p.plan[kHCausal] != 0;
  const int vis = causal ? keys - nq + r0 + rows : keys;      // keys the block's last row sees
  const T* qg = static_cast<const T*>(p.q);
  T* og = static_cast<T*>(p.out);
  for (int u = tid; u < 16 * kHeadDim; u += kSimpleThreads) {
    const int m = u / kHeadDim, d = u % kHeadDim, r = m & 7, row = q0 + r0 + r;
    sq[m][d] = r < rows && row < p.total_q
                   ? load_in(qg + (static_cast<size_t>(row) * kQHeads + 2 * h + (m >> 3)) * kHeadDim + d)
                   : 0.f;
  }
  const int m = tid >> 3, kq = tid & 7, r = m & 7;
  float mrow = -INFINITY, lrow = 0.f;
  float acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  const int row_vis = causal ? keys - nq + r0 + r + 1 : keys;
  for (int kb0 = 0; kb0 < vis; kb0 += kSimpleKeys) {
    __syncthreads();
    for (int u = tid; u < kSimpleKeys * kHeadDim; u += kSimpleThreads) {
      const int n = u / kHeadDim, d = u % kHeadDim, j = kb0 + n;
      float kv = 0.f, vv = 0.f;
      if (j < vis) {
        const int s = j < len[0] ? 0 : (j < len[0] + len[1] ? 1 : 2);
        const int at = s == 0 ? j : (s == 1 ? j - len[0] : j - len[0] - len[1]);
        const Source& src = p.src[s];
        const long long row = src.off + start[s] + at;
        if (row >= 0 && row < src.rows) {
          const size_t off = (static_cast<size_t>(row) * kKVHeads + h) * kHeadDim + d;
          kv = load_in(static_cast<const T*>(src.k) + off);
          vv = load_in(static_cast<const T*>(src.v) + off);
        } else {
          atomicOr(&g_device_status, kStatusBadArgument);
        }
      }
      sk[n][d] = kv;
      sv[n][d] = vv;
    }
    __syncthreads();
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = kq * 4 + i, j = kb0 + n;
      float dot = 0.f;
      for (int d = 0; d < kHeadDim; ++d) dot = fmaf(sq[m][d], sk[n][d], dot);
      s[i] = j < row_vis && j < vis ? dot * p.scale : -INFINITY;
    }
    float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(mrow, mx);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = expf(mrow - mu);
    float ps = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = expf(s[i] - mu);
      sp[m][kq * 4 + i] = e;
      ps += e;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    lrow = lrow * alpha + ps;
    mrow = mn;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] *= alpha;
    for (int n = 0; n < kSimpleKeys; ++n) {
      const float pn = sp[m][n];
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = fmaf(pn, sv[n][kq * 16 + i], acc[i]);
    }
  }
  const int row = q0 + r0 + r;
  if (r < rows && row < p.total_q) {
    const float inv = lrow > 0.f ? 1.f / lrow : 0.f;
    T* dst = og + (static_cast<size_t>(row) * kQHeads + 2 * h + (m >> 3)) * kHeadDim + kq * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) store_out(dst + i, acc[i] * inv);
  }
}

}  // namespace prefix
}  // namespace dspark
