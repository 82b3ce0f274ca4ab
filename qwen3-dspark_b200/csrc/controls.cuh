// Logits controls: repetition / frequency / presence penalties, biases and grammar masks.
//
// Row j of request i's chunk x_0 .. x_j (x_0 is in the request's counts already):
//   c    = count_i[v] + #{1 <= k <= j : x_k = v},   seen = prompt_i[v] or c > 0
//   z    = logit;  z = z > 0 ? z / rep : z * rep        where seen
//   z    = (z - freq * c) - pres                        where c > 0
//   z    = z + bias_i[v];   z = mask_value              where the row's mask bit v is 0
// Every step is one rounded fp32 operation (no contraction), so the values are those of
// the same steps in torch float32. A forbidden entry is selected, never added to, so
// infinities and NaN there do not spread.
//
// A request's tables (counts 2 bytes, prompt bits 1/8 byte per token) are read once per
// vocabulary chunk and serve all rows of its chunk: one CTA owns (request, 2048 tokens),
// keeps the chunk's counts and biases in registers and walks the rows, adding each row's
// proposal to the count of the thread that owns it.
#pragma once
#include "accept.cuh"

namespace dspark {
namespace controls {

constexpr int kThreads = 256;
constexpr int kPer = 8;                        // tokens per thread
constexpr int kChunk = kThreads * kPer;
constexpr int kRowBatch = 16;                  // argmax rows reduced per barrier
constexpr int kMaxCount = 32767;               // counts saturate here

struct Params {
  const void* logits;
  long long ld;
  int rows, vocab;
  const int* cu_q;              // [R+1], or null: row i belongs to request i
  const long long* tokens;      // [rows] chunk tokens, or null: no proposals
  const int* slots;             // [R] table row of each request
  int num_requests;
  const short* counts;          // [num_slots] rows of ld_counts
  long long ld_counts;
  const uint32_t* prompt_bits;  // [num_slots] rows of ld_bits words
  long long ld_bits;
  const float* penalties;       // [num_slots, 3]: repetition, frequency, presence
  int num_slots;
  const int* bias_ids;          // [num_slots, max_bias], or null
  const float* bias_values;
  const int* bias_len;
  int max_bias;
  const uint32_t* masks;        // [num_masks] rows of ld_mask words, or null
  long long ld_mask;
  int num_masks;
  const int* mask_index;        // [rows], -1: no mask
  float mask_value;
  void* out;
  long long ld_out;
  int in_place;
  unsigned long long* part;     // argmax: [rows][chunks] packed maxima
  int* pred;
  int chunks;
};

// First row and row count of request r; false when the offsets are out of range.
__device__ __forceinline__ bool request_rows(const Params& p, int r, int& q0, int& nq) {
  q0 = p.cu_q ? p.cu_q[r] : r;
  const int q1 = p.cu_q ? p.cu_q[r + 1] : r + 1;
  nq = q1 - q0;
  return q0 >= 0 && nq >= 0 && q1 <= p.rows;
}

// Order-preserving key of a candidate: NaN above numbers, -0 equal to +0, then the
// lowest index. 0 is no candidate.
__device__ __forceinline__ unsigned long long arg_key(float z, int v) {
  uint32_t u = __float_as_uint(z + 0.f);
  u = z != z ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
}

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) {
  return a > b ? a : b;
}

template <typename T>
__device__ __forceinline__ void put(T* dst, float z);
template <>
__device__ __forceinline__ void put<float>(float* dst, float z) { *dst = z; }
template <>
__device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* dst, float z) { *dst = __float2bfloat16_rn(z); }

// kVec: rows of every table start on 16-byte boundaries and a thread owns 8 consecutive
// tokens (16-byte accesses); otherwise its tokens lie 256 apart, so that the element
// accesses of a warp stay contiguous whatever the row's alignment.
template <typename TIn, typename TOut, bool kArgmax, bool kVec>
__global__ void __launch_bounds__(kThreads) control_kernel(const Params p) {
  __shared__ int s_id[kThreads];
  __shared__ float s_val[kThreads];
  __shared__ int s_warp[kThreads / 32];
  __shared__ unsigned long long s_best[kRowBatch][kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int base = chunk * kChunk;
  int q0, nq;
  const int slot = p.slots[r];
  if (!request_rows(p, r, q0, nq) || slot < 0 || slot >= p.num_slots) {
    if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  auto index = [&](int e) { return kVec ? base + tid * kPer + e : base + e * kThreads + tid; };

  int c[kPer];
  uint32_t prompt = 0;
  {
    const short* cr = p.counts + static_cast<long long>(slot) * p.ld_counts;
    const uint32_t* br = p.prompt_bits + static_cast<long long>(slot) * p.ld_bits;
    if (kVec && index(kPer - 1) < p.vocab) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(cr + index(0)));
      const short* s = reinterpret_cast<const short*>(&raw);
#pragma unroll
      for (int e = 0; e < kPer; ++e) c[e] = s[e];
      prompt = (br[index(0) >> 5] >> (index(0) & 31)) & 0xffu;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int v = index(e);
        c[e] = v < p.vocab ? cr[v] : 0;
        if (v < p.vocab) prompt |= ((br[v >> 5] >> (v & 31)) & 1u) << e;
      }
    }
  }
  const float rep = p.penalties[3 * slot], freq = p.penalties[3 * slot + 1], pres = p.penalties[3 * slot + 2];

  // biases of the chunk, added in list order whatever the number of entries per token
  float bias[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) bias[e] = 0.f;
  const int nb = p.bias_ids ? min(max(p.bias_len[slot], 0), p.max_bias) : 0;
  for (int b0 = 0; b0 < nb; b0 += kThreads) {
    const int b = b0 + tid;
    const int id = b < nb ? p.bias_ids[static_cast<long long>(slot) * p.max_bias + b] : -1;
    const bool in = id >= base && id < base + kChunk;
    const unsigned ballot = __ballot_sync(0xffffffffu, in);
    if (lane == 0) s_warp[warp] = __popc(ballot);
    __syncthreads();
    int at = __popc(ballot & ((1u << lane) - 1)), n = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += s_warp[w];
      n += s_warp[w];
    }
    if (in) {
      s_id[at] = id;
      s_val[at] = p.bias_values[static_cast<long long>(slot) * p.max_bias + b];
    }
    __syncthreads();
    for (int k = 0; k < n; ++k) {
      const int x = s_id[k] - base;
      const int owner = kVec ? x / kPer : x % kThreads, el = kVec ? x % kPer : x / kThreads;
      if (owner == tid) {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (e == el) bias[e] = __fadd_rn(bias[e], s_val[k]);
      }
    }
    __syncthreads();
  }

  const TIn* lg = static_cast<const TIn*>(p.logits);
  for (int j = 0; j < nq; ++j) {
    const int row = q0 + j;
    if (j > 0 && p.tokens) {
      const long long x = p.tokens[row];
      if (x >= base && x < base + kChunk && x < p.vocab) {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (index(e) == static_cast<int>(x)) c[e] = min(c[e] + 1, kMaxCount);
      } else if ((x < 0 || x >= p.vocab) && chunk == 0 && tid == 0) {
        atomicOr(&g_device_status, kStatusBadArgument);
      }
    }
    uint32_t allow = 0xffu;
    if (p.masks) {
      const int mi = p.mask_index[row];
      if (mi >= p.num_masks) {
        if (chunk == 0 && tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
      } else if (mi >= 0) {
        const uint32_t* mr = p.masks + static_cast<long long>(mi) * p.ld_mask;
        if (kVec) {
          allow = index(0) < p.vocab ? (__ldg(mr + (index(0) >> 5)) >> (index(0) & 31)) & 0xffu : 0u;
        } else {
          allow = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int v = index(e);
            if (v < p.vocab) allow |= ((__ldg(mr + (v >> 5)) >> (v & 31)) & 1u) << e;
          }
        }
      }
    }
    const TIn* lr = lg + static_cast<long long>(row) * p.ld;
    float z[kPer];
    const bool whole = kVec && index(kPer - 1) < p.vocab;
    if (allow == 0) {
      // nothing of this thread's tokens is allowed: their logits are not read
    } else if (whole) {
      if (sizeof(TIn) == 2) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(lr + index(0)));
        const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&raw);
#pragma unroll
        for (int e = 0; e < kPer; ++e) z[e] = __bfloat162float(x[e]);
      } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(lr + index(0)));
        const uint4 b = __ldg(reinterpret_cast<const uint4*>(lr + index(0)) + 1);
        const float* x = reinterpret_cast<const float*>(&a);
        const float* y = reinterpret_cast<const float*>(&b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[e] = x[e];
          z[e + 4] = y[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) z[e] = index(e) < p.vocab ? to_f32(lr[index(e)]) : 0.f;
    }
    unsigned long long best = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      float y = z[e];
      if (((prompt >> e) & 1u) || c[e] > 0) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      if (c[e] > 0) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(c[e]))), pres);
      if (nb > 0) y = __fadd_rn(y, bias[e]);
      const bool ok = (allow >> e) & 1u;
      z[e] = ok ? y : p.mask_value;
      if (kArgmax && ok && index(e) < p.vocab) best = max_u64(best, arg_key(y, index(e)));
    }
    if (kArgmax) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) best = max_u64(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (lane == 0) s_best[j % kRowBatch][warp] = best;
      if (j % kRowBatch == kRowBatch - 1 || j + 1 == nq) {
        const int j0 = j - j % kRowBatch;
        __syncthreads();
        if (tid <= j - j0) {
          unsigned long long m = 0;
          for (int w = 0; w < kThreads / 32; ++w) m = max_u64(m, s_best[tid][w]);
          p.part[static_cast<long long>(q0 + j0 + tid) * p.chunks + chunk] = m;
        }
        __syncthreads();
      }
      continue;
    }
    TOut* orow = static_cast<TOut*>(p.out) + static_cast<long long>(row) * p.ld_out;
    if (whole) {
      uint4 w[sizeof(TOut) / 2];
      TOut* t = reinterpret_cast<TOut*>(w);
#pragma unroll
      for (int e = 0; e < kPer; ++e) put(t + e, z[e]);
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(TOut) / 2); ++k) reinterpret_cast<uint4*>(orow + index(0))[k] = w[k];
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (index(e) < p.vocab) put(orow + index(e), z[e]);
    }
  }
}

// One warp per row: the maximum over the row's chunks. A row whose mask allows nothing
// gets -1 and sets the status bit.
__global__ void __launch_bounds__(128) control_argmax_finish_kernel(const Params p) {
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int q0, nq;
  if (!request_rows(p, r, q0, nq)) return;
  const int slot = p.slots[r];
  const bool ok = slot >= 0 && slot < p.num_slots;
  for (int j = warp; j < nq; j += 4) {
    unsigned long long best = 0;
    if (ok)
      for (int k = lane; k < p.chunks; k += 32)
        best = max_u64(best, p.part[static_cast<long long>(q0 + j) * p.chunks + k]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max_u64(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) {
      p.pred[q0 + j] = best == 0 ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
      if (best == 0 && ok) atomicOr(&g_device_status, kStatusEmptyMask);
    }
  }
}

// Adds tokens to the tables: counts[slot][token] += 1 (saturating), or the prompt bit.
// Request i's tokens are tokens[cu[i] .. cu[i + 1]), cut to n[i] where n is not null.
struct TokenParams {
  const long long* tokens;
  const int* cu;
  const int* n;
  const int* slots;
  int num_tokens, num_slots, vocab;
  short* counts;
  long long ld_counts;
  uint32_t* prompt_bits;
  long long ld_bits;
};

__global__ void __launch_bounds__(256) control_tokens_kernel(const TokenParams p) {
  const int r = blockIdx.x, slot = p.slots[r];
  const int a = p.cu[r], b = p.cu[r + 1];
  if (a < 0 || b < a || b > p.num_tokens || slot < 0 || slot >= p.num_slots) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  const int n = p.n ? min(max(p.n[r], 0), b - a) : b - a;
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const long long t = p.tokens[a + k];
    if (t < 0 || t >= p.vocab) {
      atomicOr(&g_device_status, kStatusBadArgument);
      continue;
    }
    if (p.counts) {
      // a 16-bit counter inside its 32-bit word; the counters saturate
      const size_t at = static_cast<size_t>(slot) * p.ld_counts + static_cast<size_t>(t);
      unsigned int* word = reinterpret_cast<unsigned int*>(p.counts) + (at >> 1);
      const int shift = static_cast<int>(at & 1) * 16;
      unsigned int old = *word;
      while (true) {
        if (((old >> shift) & 0xffffu) >= static_cast<unsigned>(kMaxCount)) break;
        const unsigned int got = atomicCAS(word, old, old + (1u << shift));
        if (got == old) break;
        old = got;
      }
    } else {
      atomicOr(p.prompt_bits + static_cast<size_t>(slot) * p.ld_bits + (t >> 5), 1u << (t & 31));
    }
  }
}

}  // namespace controls
}  // namespace dspark
