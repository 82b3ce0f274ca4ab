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
// One CTA owns (request, 4096 tokens) and serves all rows of the request's chunk, so the
// request's tables (counts 2 bytes, prompt bits 1/8 byte per token) are read once. Few tokens
// are seen or biased: they go into a list in shared memory first. Then the rows stream
// through untouched - bf16 stays packed, masks are applied to pairs, maxima are packed - and
// a second pass over the list computes the penalised values and stores them over, or
// compares them. 896 rows (7 of each of 128 requests) x 151936 bf16 tokens with masks and
// biases take 129 us (2.5 TB/s of the 325 MB), 260 rows to float32 62 us (4.1 TB/s). The start
// of the CTAs, the list pass and the instructions per row bound it beside DRAM: one row a
// request takes 54 us and each further one 12.5; without masks and lists 37 us and 8.1, which
// is 4.8 TB/s of a row's 38.9 MB. With the penalties inside the streaming pass (per token, or in
// loops over set bits) the 896 rows took 252 and 165 us. Four CTAs an SM leave a thread 64
// registers: the forms that read float32 or unaligned rows spill 12 to 96 bytes.
#pragma once
#include "accept.cuh"

namespace dspark {
namespace controls {

constexpr int kThreads = 256;
constexpr int kPer = 16;                       // tokens per thread: two runs of 8
constexpr int kChunk = kThreads * kPer;
constexpr int kRun = kThreads * 8;             // tokens between a thread's two runs
constexpr int kStage = 2 * kThreads;           // biases of a chunk summed up at a time
constexpr int kRowBatch = 16;                  // rows whose indices are staged at a time
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

// Order-preserving key of a number: NaN above all, -0 equal to +0; never 0.
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);
  return z != z ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) {
  return a > b ? a : b;
}

// a / b rounded to nearest, from r = 1 / b rounded to nearest: q = a r, corrected by its
// residual, q + (a - q b) r (P. Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", 1990), as long as nothing over- or underflows; __fdiv_rn
// otherwise. A penalised warp is bound by its instructions, and this takes four.
// Markstein's theorem asks for a q within an ulp, whose residual is exact. Here q is off by up
// to 1.5 ulp and a residual may lose its last bit, so the correction is right to 2^-23 of
// itself, and the result to 1.5 * 2^-23 ulp before the last rounding. With 24-bit integers for
// the mantissas a quotient lies c / (2 B) ulp from a midpoint, c = 1, 2, ..: only c <= 6 could
// round the wrong way. All 93 million pairs with c <= 16 were enumerated (by the inverse of B
// modulo 2^24 and 2^25) and computed on the host: every one rounds as the division does.
constexpr float kDivLow = 1e-20f, kDivHigh = 1e20f;
__device__ __forceinline__ float divide(float a, float b, float r, bool b_safe) {
  if (b_safe && a > kDivLow && a < kDivHigh) {
    const float q = __fmul_rn(a, r);
    return __fmaf_rn(__fmaf_rn(-q, b, a), r, q);
  }
  return __fdiv_rn(a, b);
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 32 bytes in one access (sm_100), 32-byte aligned.
__device__ __forceinline__ void load_f32x8(const float* p, float (&z)[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(z[0]), "=f"(z[1]), "=f"(z[2]), "=f"(z[3]), "=f"(z[4]), "=f"(z[5]), "=f"(z[6]), "=f"(z[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store_f32x8(float* p, const float (&z)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(z[0]), "f"(z[1]), "f"(z[2]),
               "f"(z[3]), "f"(z[4]), "f"(z[5]), "f"(z[6]), "f"(z[7])
               : "memory");
}

// Masks of packed pairs from a bit per token: `spread_bits` puts the bits of tokens 2 k and
// 2 k + 1 at 2 k and 2 k + 16; shifted to the top bits of bytes 0 and 2, prmt replicates them
// over the halves.
__device__ __forceinline__ uint32_t spread_bits(uint32_t allow) { return (allow & 0x5555u) | ((allow & 0xaaaau) << 15); }
__device__ __forceinline__ uint32_t pair_mask(uint32_t spread, int k) {
  const uint32_t t = 2 * k <= 7 ? spread << (7 - 2 * k) : spread >> (2 * k - 7);
  uint32_t m;
  asm("prmt.b32 %0, %1, 0, 0xAA88;" : "=r"(m) : "r"(t));
  return m;
}

__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 0xffff in each half whose values are equal.
__device__ __forceinline__ uint32_t equal_bf16x2(uint32_t a, uint32_t b) {
  return __heq2_mask(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
}

__device__ __forceinline__ float bf16_half(uint32_t w, int high) {
  return __uint_as_float(high ? w & 0xffff0000u : w << 16);
}

// List entry: token - base (12 bits), in the prompt, has a bias.
constexpr uint32_t kEntryPrompt = 1u << 12, kEntryBias = 1u << 13;

// kVec: every row starts on a boundary of the vector accesses and a thread owns two runs of
// 8 consecutive tokens; otherwise its tokens lie 256 apart, so that the element accesses of
// a warp stay contiguous whatever the row's alignment.
template <typename TIn, typename TOut, bool kArgmax, bool kVec>
__global__ void __launch_bounds__(kThreads, 4) control_kernel(const Params p) {
  __shared__ uint16_t s_list[kChunk];
  __shared__ __align__(16) uint16_t s_counts[kChunk];
  __shared__ float s_bias[kChunk];               // of biased tokens (the rest is not written)
  __shared__ int s_id[kStage];
  __shared__ float s_val[kStage];
  __shared__ int s_count[kThreads / 32];
  __shared__ unsigned long long s_best[kRowBatch][kThreads / 32], s_list_best[kRowBatch];
  __shared__ uint32_t s_top[kRowBatch];
  __shared__ int s_mask[kRowBatch], s_token[kRowBatch];
  __shared__ int s_n;
  __shared__ uint32_t s_proposals;               // rows whose proposal lies in this chunk
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // chunks in order, so that the first ones (low token ids are the frequent ones: long lists)
  // do not start last
  const int r = blockIdx.x % p.num_requests, chunk = blockIdx.x / p.num_requests;
  const int base = chunk * kChunk;
  int q0, nq;
  const int slot = p.slots[r];
  if (!request_rows(p, r, q0, nq) || slot < 0 || slot >= p.num_slots) {
    if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  // token of bit e, less base
  auto rel = [&](int e) { return kVec ? (e >> 3) * kRun + tid * 8 + (e & 7) : e * kThreads + tid; };
  auto index = [&](int e) { return base + rel(e); };
  auto owner = [&](int x) { return kVec ? (x % kRun) >> 3 : x % kThreads; };
  auto bit_of = [&](int x) { return kVec ? (x / kRun) * 8 + (x & 7) : x / kThreads; };
  const bool whole0 = kVec && index(7) < p.vocab, whole1 = kVec && index(15) < p.vocab;
  auto whole = [&](int o) { return o == 0 ? whole0 : whole1; };
  uint32_t inside = 0xffffu;                     // tokens of the vocabulary
  if (!(whole0 && whole1)) {
    inside = 0;
#pragma unroll 1
    for (int e = 0; e < kPer; ++e) inside |= static_cast<uint32_t>(index(e) < p.vocab) << e;
  }
  // The request's tables, on their way while the rows' indices and the biases are staged.
  const short* cr = p.counts + static_cast<long long>(slot) * p.ld_counts;
  const uint32_t* br = p.prompt_bits + static_cast<long long>(slot) * p.ld_bits;
  uint32_t cw[8], prompt = 0, used = 0;          // counts in pairs; bit e: in the prompt, emitted
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    if (whole(o)) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(cr + index(8 * o)));
      cw[4 * o] = raw.x;
      cw[4 * o + 1] = raw.y;
      cw[4 * o + 2] = raw.z;
      cw[4 * o + 3] = raw.w;
      prompt |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint8_t*>(br) + (index(8 * o) >> 3))) << (8 * o);
    } else {
#pragma unroll
      for (int e = 8 * o; e < 8 * o + 8; e += 2) {
        uint32_t lo = 0, hi = 0;
        if (index(e) < p.vocab) {
          lo = static_cast<uint16_t>(cr[index(e)]);
          prompt |= ((br[index(e) >> 5] >> (index(e) & 31)) & 1u) << e;
        }
        if (index(e + 1) < p.vocab) {
          hi = static_cast<uint16_t>(cr[index(e + 1)]);
          prompt |= ((br[index(e + 1) >> 5] >> (index(e + 1) & 31)) & 1u) << (e + 1);
        }
        cw[e >> 1] = lo | (hi << 16);
      }
    }
  }
  const float rep = p.penalties[3 * slot], freq = p.penalties[3 * slot + 1], pres = p.penalties[3 * slot + 2];
  const float inv_rep = __frcp_rn(rep);
  const bool rep_safe = rep > 1e-10f && rep < 1e10f;
  const TIn* lg = static_cast<const TIn*>(p.logits);
  constexpr bool kPacked = kVec && sizeof(TIn) == 2;

  uint32_t changed = 0;                          // bit e: token e is in the list

  int j0 = 0, batch = 0;
  auto stage = [&]() {
    // the batch's mask rows (-1: none) and proposals (-1: none in this chunk)
    batch = min(kRowBatch, nq - j0);
    __syncthreads();
    if (tid == 0) {
      s_proposals = 0;
      if (j0 == 0) s_n = 0;
    }
    if (tid < batch) {
      const int row = q0 + j0 + tid;
      int mi = p.masks ? p.mask_index[row] : -1, x = -1;
      if (mi < -1 || mi >= p.num_masks) mi = -2;
      if (j0 + tid > 0 && p.tokens) {
        const long long t = p.tokens[row];
        if (t < 0 || t >= p.vocab)
          x = -2;
        else if (t >= base && t < base + kChunk)
          x = static_cast<int>(t) - base;
      }
      if (chunk == 0 && (mi == -2 || x == -2)) atomicOr(&g_device_status, kStatusBadArgument);
      s_mask[tid] = mi;
      s_token[tid] = x;
      s_top[tid] = 0;
      s_list_best[tid] = 0;
    }
    __syncthreads();
  };
  const bool masked = p.masks != nullptr;
  auto allowed = [&](int j) -> uint32_t {
    if (j >= batch) return 0u;
    const int mi = masked ? s_mask[j] : -1;
    if (mi < 0) return inside;
    const uint32_t* mr = p.masks + static_cast<long long>(mi) * p.ld_mask;
    uint32_t m = 0;
    if (kVec) {
      // the byte of tokens index(8 o) .. + 7 (little endian words)
      const uint8_t* mb = reinterpret_cast<const uint8_t*>(mr) + (base >> 3) + tid;
      if (whole0 || index(0) < p.vocab) m = __ldg(mb);
      if (whole1 || index(8) < p.vocab) m |= static_cast<uint32_t>(__ldg(mb + kRun / 8)) << 8;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int v = index(e);
        if (v < p.vocab) m |= ((__ldg(mr + (v >> 5)) >> (v & 31)) & 1u) << e;
      }
    }
    return m & inside;
  };
  // whether the streaming pass needs run o's logits
  auto wanted = [&](int o, uint32_t allow) {
    const uint32_t a = (allow >> (8 * o)) & 0xffu, all = (inside >> (8 * o)) & 0xffu;
    return a != 0 && (kArgmax || !(p.in_place && a == all));
  };
  // packed: word 4 o + k holds tokens 8 o + 2 k and + 1; otherwise one token a word
  constexpr int kWords = kPacked ? 8 : 16;
  auto fetch = [&](int j, uint32_t allow, uint32_t (&w)[kWords], bool all = false) {
    if (j >= batch) return;
    const TIn* lr = lg + static_cast<long long>(q0 + j0 + j) * p.ld;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      if (!all && !wanted(o, allow)) continue;
      if constexpr (kPacked) {
        if (whole(o)) {
          const uint4 v = *reinterpret_cast<const uint4*>(lr + index(8 * o));
          w[4 * o] = v.x;
          w[4 * o + 1] = v.y;
          w[4 * o + 2] = v.z;
          w[4 * o + 3] = v.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t lo = 0, hi = 0;
            if (index(8 * o + 2 * k) < p.vocab) lo = __bfloat16_as_ushort(lr[index(8 * o + 2 * k)]);
            if (index(8 * o + 2 * k + 1) < p.vocab) hi = __bfloat16_as_ushort(lr[index(8 * o + 2 * k + 1)]);
            w[4 * o + k] = lo | (hi << 16);
          }
        }
      } else {
        if (kVec && whole(o)) {
          float z[8];
          load_f32x8(reinterpret_cast<const float*>(lr) + index(8 * o), z);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[8 * o + e] = __float_as_uint(z[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[8 * o + e] = index(8 * o + e) < p.vocab ? __float_as_uint(to_f32(lr[index(8 * o + e)])) : 0u;
        }
      }
    }
  };
  uint32_t next[kWords];
  // row 0 is on its way with the tables, read whole before its mask is there
  batch = min(kRowBatch, nq);
  fetch(0, inside, next, !p.in_place || p.masks);
  stage();
  // The chunk's biases, compacted in list order; each thread sums its own tokens' entries up, in
  // that order, so a list of any length is read once.
  uint32_t biased = 0;
  int staged = 0;
  const int nb = p.bias_ids ? min(max(p.bias_len[slot], 0), p.max_bias) : 0;
  const int* list_id = p.bias_ids + static_cast<long long>(slot) * p.max_bias;
  const float* list_val = p.bias_values + static_cast<long long>(slot) * p.max_bias;
  auto sum_up = [&]() {
    __syncthreads();
    for (int k = 0; k < staged; ++k) {
      const int x = s_id[k] - base;
      if (owner(x) != tid) continue;
      const uint32_t bit = 1u << bit_of(x);
      s_bias[x] = __fadd_rn((biased & bit) ? s_bias[x] : 0.f, s_val[k]);
      biased |= bit;
    }
    staged = 0;
  };
  for (int b0 = 0; b0 < nb; b0 += kThreads) {
    if (staged > kStage - kThreads) sum_up();
    const int b = b0 + tid;
    const int id = b < nb ? list_id[b] : -1;
    const bool in = id >= base && id < base + kChunk && id < p.vocab;
    const unsigned ballot = __ballot_sync(0xffffffffu, in);
    __syncthreads();
    if (lane == 0) s_count[warp] = __popc(ballot);
    __syncthreads();
    int at = staged + __popc(ballot & ((1u << lane) - 1));
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += s_count[w];
      staged += s_count[w];
    }
    if (in) {
      s_id[at] = id;
      s_val[at] = list_val[b];
    }
  }
  if (staged > 0) sum_up();
  // Counts into shared memory (a thread's own tokens, which only it will change), tokens that
  // were seen or have a bias into the list (in any order).
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    used |= static_cast<uint32_t>(static_cast<short>(cw[k] & 0xffffu) > 0) << (2 * k);
    used |= static_cast<uint32_t>(static_cast<int>(cw[k]) >> 16 > 0) << (2 * k + 1);
  }
  if (kVec) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
      *reinterpret_cast<uint4*>(&s_counts[rel(8 * o)]) = make_uint4(cw[4 * o], cw[4 * o + 1], cw[4 * o + 2], cw[4 * o + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) s_counts[rel(e)] = static_cast<uint16_t>(cw[e >> 1] >> (16 * (e & 1)));
  }
  changed = prompt | used | biased;
  if (__any_sync(0xffffffffu, changed != 0)) {
    int at = __popc(changed);                    // the warp's entries lie behind one another
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    int first = 0;
    if (lane == 31) first = atomicAdd(&s_n, at);
    at += __shfl_sync(0xffffffffu, first, 31) - __popc(changed);
#pragma unroll 1
    for (uint32_t m = changed; m != 0; m &= m - 1, ++at) {
      const int e = __ffs(m) - 1;
      s_list[at] = static_cast<uint16_t>(static_cast<uint32_t>(rel(e)) | (((prompt >> e) & 1u) * kEntryPrompt) |
                                         (((biased >> e) & 1u) * kEntryBias));
    }
  }

  for (; j0 < nq; j0 += kRowBatch) {
    if (j0 > 0) {
      stage();
      fetch(0, inside, next, !p.in_place || p.masks);
    }
    // Pipelined by rows: while row j is decided, row j + 1's logits and row j + 2's mask words
    // are in flight.
    uint32_t allow = allowed(0), allow1 = allowed(1);
    // proposals join the list (not seen until their row)
    for (int j = 0; j < batch; ++j) {
      const int x = s_token[j];
      if (x < 0 || owner(x) != tid) continue;
      atomicOr(&s_proposals, 1u << j);
      if (!((changed >> bit_of(x)) & 1u)) {
        changed |= 1u << bit_of(x);
        s_list[atomicAdd(&s_n, 1)] = static_cast<uint16_t>(x);
      }
    }
    const uint32_t plain = inside & ~changed;    // tokens the streaming pass decides by itself
#pragma unroll 1
    for (int j = 0; j < batch; ++j) {
      uint32_t w[kWords];
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = next[k];
      fetch(j + 1, allow1, next);
      const uint32_t allow2 = allowed(j + 2);
      if constexpr (kArgmax) {
        const uint32_t keep = allow & plain;
        if (!__any_sync(0xffffffffu, keep != 0)) {
          if (lane == 0) s_best[j][warp] = 0;
        } else {
          float top;
          if constexpr (kPacked) {
            if (keep != 0xffffu) {
              const uint32_t spread = spread_bits(keep);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t m = pair_mask(spread, k);
                w[k] = (w[k] & m) | (0xff80ff80u & ~m);
              }
            }
            uint32_t t = max_nan_bf16x2(w[0], w[1]);
#pragma unroll
            for (int k = 2; k < 8; ++k) t = max_nan_bf16x2(t, w[k]);
            top = max_nan(bf16_half(t, 0), bf16_half(t, 1));
          } else {
            top = -INFINITY;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              w[e] = ((keep >> e) & 1u) ? w[e] : 0xff800000u;
              top = max_nan(top, __uint_as_float(w[e]));
            }
          }
          const uint32_t key = keep ? order_key(top) : 0u;
          const uint32_t best = __reduce_max_sync(0xffffffffu, key);
          // a warp below the row's maximum so far has nothing to add (a stale read is lower)
          const uint32_t so_far = *reinterpret_cast<volatile uint32_t*>(&s_top[j]);
          unsigned long long mine = 0;
          if (__any_sync(0xffffffffu, best >= so_far)) {
            uint32_t at = 0xffffffffu;
            if (key == best && keep) {
              if (top == -INFINITY) {              // left-out tokens look the same: the first kept one
                at = static_cast<uint32_t>(index(__ffs(keep) - 1));
              } else if (kPacked && top == top) {
                // bit k of each half: the pair's low or high token has the maximum
                const uint32_t t2 = pack_bf16x2(top, top);
                uint32_t hit = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) hit |= equal_bf16x2(w[k % kWords], t2) & (0x00010001u << k);
                const uint32_t lo = hit & 0xffffu, hi = hit >> 16;
                at = static_cast<uint32_t>(index(min(lo ? 2 * (__ffs(lo) - 1) : kPer, hi ? 2 * (__ffs(hi) - 1) + 1 : kPer)));
              } else {
#pragma unroll
                for (int e = kPer - 1; e >= 0; --e) {
                  const float y = kPacked ? bf16_half(w[(e >> 1) % kWords], e & 1) : __uint_as_float(w[e % kWords]);
                  if (y == top || (top != top && y != y)) at = static_cast<uint32_t>(index(e));
                }
              }
            }
            at = __reduce_min_sync(0xffffffffu, at);
            mine = (static_cast<unsigned long long>(best) << 32) | (0xffffffffu - at);
            if (lane == 0) atomicMax(&s_top[j], best);
          }
          if (lane == 0) s_best[j][warp] = mine;
        }
      } else {
        TOut* orow = static_cast<TOut*>(p.out) + static_cast<long long>(q0 + j0 + j) * p.ld_out;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t a = (allow >> (8 * o)) & 0xffu, all = (inside >> (8 * o)) & 0xffu;
          if (all == 0 || (p.in_place && a == all)) continue;      // in place, nothing forbidden: as it is
          if constexpr (kPacked && sizeof(TOut) == 2) {
            const uint32_t hidden = pack_bf16x2(p.mask_value, p.mask_value);
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t m = a == 0xffu ? 0xffffffffu : pair_mask(spread_bits(a), k);
              v[k] = (w[(4 * o + k) % kWords] & m) | (hidden & ~m);
            }
            if (whole(o)) {
              *reinterpret_cast<uint4*>(orow + index(8 * o)) = make_uint4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (index(8 * o + e) < p.vocab)
                  orow[index(8 * o + e)] = __ushort_as_bfloat16(static_cast<unsigned short>(v[e >> 1] >> (16 * (e & 1))));
            }
          } else {
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = kPacked ? bf16_half(w[(4 * o + (e >> 1)) % kWords], e & 1)
                                      : __uint_as_float(w[(8 * o + e) % kWords]);
              z[e] = ((a >> e) & 1u) ? y : p.mask_value;
            }
            if (sizeof(TOut) == 4 && whole(o)) {
              store_f32x8(reinterpret_cast<float*>(orow) + index(8 * o), z);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (index(8 * o + e) < p.vocab) {
                  if constexpr (sizeof(TOut) == 4)
                    orow[index(8 * o + e)] = z[e];
                  else
                    orow[index(8 * o + e)] = __float2bfloat16_rn(z[e]);
                }
            }
          }
        }
      }
      allow = allow1;
      allow1 = allow2;
    }
    __syncthreads();                             // the list is complete, the streamed stores are done
    const int n = s_n;
    const uint32_t proposals = s_proposals;
    constexpr int kAhead = 4;                    // entries of a lane whose loads are in flight together
    // A warp takes a row, or a slice of one: where there are fewer rows than warps, and of a
    // long list, so that rows that are no multiple of the warps leave none idle (24 requests x
    // 5 float32 rows x 50257: 33.0 us with a warp a row, 29.0 with slices).
    constexpr int kWarps = kThreads / 32;
    const int slices = max(kWarps / min(batch, kWarps), min(kWarps, (n + kAhead * 32 - 1) / (kAhead * 32)));
    for (int job = warp; job < batch * slices; job += kThreads / 32) {
      const int slice = job / batch, j = job - slice * batch;
      const TIn* lr = lg + static_cast<long long>(q0 + j0 + j) * p.ld + base;
      const int mi = s_mask[j];
      const uint32_t* mr = mi >= 0 ? p.masks + static_cast<long long>(mi) * p.ld_mask + (base >> 5) : nullptr;
      const uint32_t before = proposals & ((2u << j) - 1u);   // rows up to this one with proposals here
      uint32_t best = 0, best_at = 0;
#pragma unroll 1
      for (int i0 = slice * 32 + lane; i0 - lane < n; i0 += kAhead * 32 * slices) {
        uint32_t entry[kAhead], word[kAhead];
        float value[kAhead];
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
          const int i = i0 + h * 32 * slices;
          entry[h] = i < n ? s_list[i] : 0xffffu;
          const int x = static_cast<int>(entry[h] & 0xfffu);
          word[h] = 0;
          value[h] = 0.f;
          if (i < n) {
            word[h] = mr ? __ldg(mr + (x >> 5)) : 0xffffffffu;
            value[h] = to_f32(lr[x]);
          }
        }
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
          const int x = static_cast<int>(entry[h] & 0xfffu);
          if (!((word[h] >> (x & 31)) & 1u)) continue;        // forbidden, or past the list
          int count = max(static_cast<int>(static_cast<short>(s_counts[x])), 0);
          for (uint32_t m = before; m != 0; m &= m - 1) count += s_token[__ffs(m) - 1] == x;
          count = min(count, kMaxCount);
          float y = value[h];
          if (count > 0 || (entry[h] & kEntryPrompt))
            y = y > 0.f ? divide(y, rep, inv_rep, rep_safe) : __fmul_rn(y, rep);
          if (count > 0) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(count))), pres);
          if (entry[h] & kEntryBias) y = __fadd_rn(y, s_bias[x]);
          if constexpr (kArgmax) {
            const uint32_t key = order_key(y), at = static_cast<uint32_t>(base + x);
            if (key > best || (key == best && at < best_at)) {
              best = key;
              best_at = at;
            }
          } else {
            TOut* orow = static_cast<TOut*>(p.out) + static_cast<long long>(q0 + j0 + j) * p.ld_out + base;
            if constexpr (sizeof(TOut) == 4)
              orow[x] = y;
            else
              orow[x] = __float2bfloat16_rn(y);
          }
        }
      }
      if constexpr (kArgmax) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        if (top != 0) {
          const uint32_t at = __reduce_min_sync(0xffffffffu, best == top ? best_at : 0xffffffffu);
          if (lane == 0)
            atomicMax(&s_list_best[j], (static_cast<unsigned long long>(top) << 32) | (0xffffffffu - at));
        }
      }
    }
    __syncthreads();
    if (kArgmax && tid < batch) {
      unsigned long long m = s_list_best[tid];
      for (int w = 0; w < kThreads / 32; ++w) m = max_u64(m, s_best[tid][w]);
      p.part[static_cast<long long>(q0 + j0 + tid) * p.chunks + chunk] = m;
    }
    if (j0 + kRowBatch < nq && proposals) {
      // the next batch counts this one's proposals (each by the thread that owns its token)
      for (int j = 0; j < batch; ++j) {
        const int x = s_token[j];
        if (x >= 0 && owner(x) == tid)
          s_counts[x] = static_cast<uint16_t>(min(max(static_cast<int>(static_cast<short>(s_counts[x])), 0) + 1, kMaxCount));
      }
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

// Sets the status bit where a row's mask allows no token of the vocabulary: a warp per row,
// 16 words a lane in flight, done at the first word with a bit.
__global__ void __launch_bounds__(256) control_masks_kernel(const uint32_t* masks, long long ld_mask, int num_masks,
                                                            const int* mask_index, int rows, int vocab,
                                                            const int* cu_q) {
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q0 = cu_q ? cu_q[r] : r, q1 = cu_q ? cu_q[r + 1] : r + 1;
  if (q0 < 0 || q1 < q0 || q1 > rows) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  const int words = (vocab + 31) / 32;
  const uint32_t last = 0xffffffffu >> (31 - ((vocab - 1) & 31));
  for (int j = q0 + warp; j < q1; j += 8) {
    const int mi = mask_index[j];
    if (mi < 0 || mi >= num_masks) continue;     // no mask, or refused by the controls
    const uint32_t* m = masks + static_cast<long long>(mi) * ld_mask;
    bool any = false;
    for (int w0 = 0; w0 < words && !any; w0 += 512) {
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int w = w0 + 32 * k + lane;
        if (w < words) bits |= __ldg(m + w) & (w == words - 1 ? last : 0xffffffffu);
      }
      any = __any_sync(0xffffffffu, bits != 0);
    }
    if (!any && lane == 0) atomicOr(&g_device_status, kStatusEmptyMask);
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
  for (int k = blockIdx.y * blockDim.x + threadIdx.x; k < n; k += gridDim.y * blockDim.x) {
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
