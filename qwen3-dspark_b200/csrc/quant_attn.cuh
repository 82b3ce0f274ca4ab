// Attention over the paged 8-bit cache on the tensor cores, bf16 queries and new rows.
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / 2]) v[j, h / 2]
//
// over the tokens of row t's request: its pages (k = ks code, v = vs code, one scale per page
// and KV head), its open tail rows, and its new rows up to t itself.
//
// An item is up to 8 query rows of a request: with the 2 query heads of a KV head they are the
// 16 rows of an m16n8k16 MMA (row m = 8 * head + row, so that both rows of a thread end at the
// same key). Its keys are cut into units of equal bytes, 32 unquantised rows or one page, the
// rows first. A plan (one small launch per batch, reused by every layer) numbers the units of
// all items and gives every CTA an equal contiguous range; warp h of a CTA computes KV head h
// of its range on its own. A page's 16 KB of a head come by bulk copies of 4 KB (half of the
// dims of K, half of the dims of V) into the warp's own ring of 7 stages, so no warp ever
// waits for another one. Items cut by ranges leave fp32 partial rows that a dependent launch
// merges.
//
// Codes become halves in registers (int8: the byte under the exponent of 1024, minus 1152;
// e4m3: one conversion), both exactly. So does Q: bf16 has 8 significant bits, a half 11, and
// each query row is scaled by the power of two that takes its largest value to 2^14, so that
// only values below 2^-38 of it lose bits; the scale is undone in the scores. Probabilities are
// rounded to halves relative to 2^7 of the running maximum (2^-11 of each; below 2^-31 of
// the maximum they vanish), their sum is of the unrounded ones. The V scale multiplies a page's
// product when it is added to the float32 accumulator.
#pragma once
#include "quant.cuh"

namespace dspark {
namespace quant {

constexpr int kStagesA = 7, kStageA = 4096;
constexpr int kWarpRing = kStagesA * kStageA;
constexpr int kAttnThreadsQ = kKVHeads * 32;
constexpr size_t kAttnSmemQ = 1024 + static_cast<size_t>(kKVHeads) * kWarpRing + kKVHeads * kStagesA * 8;
constexpr int kRowUnit = 32;                                // unquantised keys of a unit

// ---------------------------------------------------------------------------
// Plan: int32 words [head | CTA ranges | merges | items].
constexpr int kPlanMagicQ = 0x51a77e11;
enum PlanWord { kQMagic = 0, kQGrid, kQItems, kQRequests, kQRows, kQHeadWords = 8 };
constexpr int kCtaWords = 4;                                // first item, its first unit, last item, its end unit
constexpr int kMergeWords = 4;                              // item (-1: none), last contributor, slot of the first
constexpr int kItemWordsQ = 8;
// item: first global row | rows | row in the request | request | row units | pages | start | cost
__host__ __device__ constexpr int plan_cta_at() { return kQHeadWords; }
__host__ __device__ constexpr int plan_merge_at(int grid) { return kQHeadWords + grid * kCtaWords; }
__host__ __device__ constexpr int plan_items_at(int grid) { return kQHeadWords + grid * (kCtaWords + kMergeWords); }
__host__ __device__ inline long long plan_words(int grid, long long requests, long long rows) {
  return plan_items_at(grid) + kItemWordsQ * (rows / kQBlock + requests);
}

// Units' worth of a new item (its queries, a partial row) and the least range of a CTA.
constexpr int kItemCost = 1, kMinUnits = 2;

struct PlanParams {
  const int* cu_q;
  const int* ctx;
  int requests, rows, width, grid;
  int* plan;
};

constexpr int kPlanThreads = 1024;
__device__ __forceinline__ int row_units(int ctx, int q_len, int r0) {
  return (ctx % kPage + min(r0 + kQBlock, q_len) + kRowUnit - 1) / kRowUnit;
}

// One CTA. Requests whose lengths do not fit the batch have no items (the status is set).
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  __shared__ long long s_cost[32];
  __shared__ int s_items[32];
  __shared__ long long carry_cost;
  __shared__ int carry_items;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* items = p.plan + plan_items_at(p.grid);
  if (tid == 0) {
    carry_cost = 0;
    carry_items = 0;
  }
  __syncthreads();
  for (int base = 0; base < p.requests; base += kPlanThreads) {
    const int i = base + tid;
    int q0 = 0, q_len = 0, ctx = 0, n = 0;
    long long cost = 0;
    if (i < p.requests) {
      q0 = p.cu_q[i];
      q_len = p.cu_q[i + 1] - q0;
      ctx = p.ctx[i];
      if (q0 >= 0 && q_len >= 0 && q0 <= p.rows - q_len && ctx >= 0 && ctx / kPage <= p.width) {
        n = (q_len + kQBlock - 1) / kQBlock;
        for (int x = 0; x < n; ++x) cost += kItemCost + ctx / kPage + row_units(ctx, q_len, x * kQBlock);
      } else {
        atomicOr(&g_device_status, kStatusBadArgument);
      }
    }
    // exclusive scans of the costs and item counts
    long long c = cost;
    int m = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long cu = __shfl_up_sync(0xffffffffu, c, o);
      const int mu = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) {
        c += cu;
        m += mu;
      }
    }
    if (lane == 31) {
      s_cost[warp] = c;
      s_items[warp] = m;
    }
    __syncthreads();
    if (warp == 0) {
      long long wc = s_cost[lane];
      int wm = s_items[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long cu = __shfl_up_sync(0xffffffffu, wc, o);
        const int mu = __shfl_up_sync(0xffffffffu, wm, o);
        if (lane >= o) {
          wc += cu;
          wm += mu;
        }
      }
      s_cost[lane] = wc;
      s_items[lane] = wm;
    }
    __syncthreads();
    long long at = carry_cost + (warp > 0 ? s_cost[warp - 1] : 0) + c - cost;
    int idx = carry_items + (warp > 0 ? s_items[warp - 1] : 0) + m - n;
    for (int x = 0; x < n; ++x, ++idx) {
      const int ru = row_units(ctx, q_len, x * kQBlock), full = ctx / kPage, total = kItemCost + full + ru;
      int4* w = reinterpret_cast<int4*>(items + static_cast<size_t>(idx) * kItemWordsQ);
      w[0] = make_int4(q0 + x * kQBlock, min(kQBlock, q_len - x * kQBlock), x * kQBlock, i);
      w[1] = make_int4(ru, full, static_cast<int>(at), total);
      at += total;
    }
    __syncthreads();
    if (tid == 0) {
      carry_cost += s_cost[31];
      carry_items += s_items[31];
    }
    __syncthreads();
  }
  const int count = carry_items;
  long long total = carry_cost;
  if (total >= (1ll << 31)) {                                // (the starts are 32-bit words)
    if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
    total = 0;
  }
  const long long want = total / kMinUnits;
  const int ranges = total == 0 ? 0 : static_cast<int>(want < 1 ? 1 : (want < p.grid ? want : p.grid));
  // position in the costs -> (item, unit); the cost of an item comes before its first unit
  auto find = [&](long long pos, int& item, int& unit) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (items[static_cast<size_t>(mid) * kItemWordsQ + 6] <= pos) lo = mid; else hi = mid - 1;
    }
    const long long u = pos - items[static_cast<size_t>(lo) * kItemWordsQ + 6] - kItemCost;
    item = lo;
    unit = u > 0 ? static_cast<int>(u) : 0;
  };
  int4* ctas = reinterpret_cast<int4*>(p.plan + plan_cta_at());
  int4* merges = reinterpret_cast<int4*>(p.plan + plan_merge_at(p.grid));
  for (int c = tid; c < p.grid; c += kPlanThreads) {
    int4 range = make_int4(0, 0, -1, 0), merge = make_int4(-1, 0, 0, 0);
    if (c < ranges) {
      int i0, u0, i1, u1;
      find(total * c / ranges, i0, u0);
      const long long end = total * (c + 1) / ranges;
      if (c + 1 == ranges) {
        i1 = count;
        u1 = 0;
      } else {
        find(end, i1, u1);
      }
      if (u1 == 0) {                                         // ends with the item before
        --i1;
        u1 = items[static_cast<size_t>(i1) * kItemWordsQ + 4] + items[static_cast<size_t>(i1) * kItemWordsQ + 5];
      } else if (i1 > i0 || u0 == 0) {                       // the first of the last item's contributors
        const long long stop = items[static_cast<size_t>(i1) * kItemWordsQ + 6] +
                               static_cast<long long>(items[static_cast<size_t>(i1) * kItemWordsQ + 7]);
        // the last range k with floor(total k / ranges) < stop
        const int last = static_cast<int>(min(static_cast<long long>(ranges - 1), (stop * ranges - 1) / total));
        merge = make_int4(i1, last, i1 > i0 ? 1 : 0, 0);
      }
      if (i1 >= i0) range = make_int4(i0, u0, i1, u1);
    }
    ctas[c] = range;
    merges[c] = merge;
  }
  if (tid == 0) {
    p.plan[kQGrid] = p.grid;
    p.plan[kQItems] = count;
    p.plan[kQRequests] = p.requests;
    p.plan[kQRows] = p.rows;
    p.plan[kQMagic] = kPlanMagicQ;
  }
}

// ---------------------------------------------------------------------------
struct AttnParamsQ {
  const __nv_bfloat16* q;
  const __nv_bfloat16* new_k;
  const __nv_bfloat16* new_v;
  __nv_bfloat16* out;
  Cache cache;
  Batch batch;
  const int* plan;
  int grid;
  float scale_log2;
  float* part;               // [grid][2][8][16 * 128 + 32]
};
// Partial rows of one (CTA, slot, head): 16 x 128 float32, then (maximum, sum) per row.
constexpr int kPartFloats = 16 * kHeadDim + 32;
__host__ __device__ inline size_t part_index(int cta, int slot, int head) {
  return ((static_cast<size_t>(cta) * 2 + slot) * kKVHeads + head) * kPartFloats;
}
inline size_t attn_workspace(int grid) { return part_index(grid, 0, 0) * sizeof(float); }

struct ItemQ {
  int q0, rows, r0, request, row_units, pages;
};
__device__ __forceinline__ ItemQ load_item_q(const AttnParamsQ& p, int idx) {
  const int4* w = reinterpret_cast<const int4*>(p.plan + plan_items_at(p.grid) + static_cast<size_t>(idx) * kItemWordsQ);
  const int4 a = __ldg(w), b = __ldg(w + 1);
  return ItemQ{a.x, a.y, a.z, a.w, b.x, b.y};
}

// D(16x8 f32) += A(16x16 f16, row) * B(16x8 f16, col)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 4 codes of a word as two pairs of halves.
template <int kCode>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (kCode == kInt8) {
    w ^= 0x80808080u;                                        // code + 128
    const __half2 bias = __floats2half2_rn(-1152.f, -1152.f);
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);   // 1024 + that
    __half2 x = __hadd2(*reinterpret_cast<__half2*>(&a), bias), y = __hadd2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    lo = e4m3x2_to_f16x2(w & 0xffffu);
    hi = e4m3x2_to_f16x2(w >> 16);
  }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// The state of a warp's 16 rows: thread (g, c) = (lane / 4, lane % 4) holds rows g (query head
// 2 h) and g + 8 (head 2 h + 1) of the same query row. Column n of output tile (j, r) is dim
// 64 j + 16 (n / 2) + 2 r + n % 2, so a thread's columns of a half j are 16 consecutive dims.
constexpr float kNoMaxQ = -3.402823466e38f;
constexpr float kLift = 7.f, kSlack = 15.f;                 // p = 2^(s - m), m between max - 15 and max - 7
struct RowsQ {
  float o[2][8][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][r][e] = 0.f;
    m[0] = m[1] = kNoMaxQ;
    l[0] = l[1] = 0.f;
  }
  // Raises m where the new maxima need it, and rescales what was added up relative to the old.
  // Rarely: only past kSlack. The result does not depend on m.
  __device__ __forceinline__ void raise(float mx0, float mx1) {
    const bool up0 = mx0 > m[0] + kSlack, up1 = mx1 > m[1] + kSlack;
    if (!__any_sync(0xffffffffu, up0 || up1)) return;
    const float n0 = up0 ? mx0 - kLift : m[0], n1 = up1 ? mx1 - kLift : m[1];
    const float a0 = up0 ? ex2(m[0] - n0) : 1.f, a1 = up1 ? ex2(m[1] - n1) : 1.f;
    m[0] = n0;
    m[1] = n1;
    l[0] *= a0;
    l[1] *= a1;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        o[j][r][0] *= a0;
        o[j][r][1] *= a0;
        o[j][r][2] *= a1;
        o[j][r][3] *= a1;
      }
  }
};

// 16 unquantised keys from key t0 of the item: scores, probabilities and their product with V.
// qa: bf16 A fragments, k-step (j, w) = dims 64 j + 16 c + 4 w .. + 3. Keys are read straight
// into B fragments: lane n reads key n's 32 bytes of each half; V is transposed 8 x 8 at a time
// in registers.
struct RowSource {
  const __nv_bfloat16 *tk, *tv, *nk, *nv;                   // tail and new rows of this head
  int tail, count;                                          // tail rows; keys in all
};
__device__ __forceinline__ bool not_finite(uint32_t w) {    // either bf16 of a word
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ void row_step(RowsQ& st, const uint32_t (&qa)[32], const RowSource& src, int t0, int limit,
                                         int diagonal, float f) {
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
  uint32_t kw[2][2][8], vw[2][2][8];                        // [keys 8 u + n][half][word]
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = t0 + 8 * u + n;
    const bool in = t < src.count, old = t < src.tail;
    const size_t at = static_cast<size_t>(old ? t : t - src.tail) * kRowElems + 16 * c;
    const uint4* k = reinterpret_cast<const uint4*>((old ? src.tk : src.nk) + (in ? at : 0));
    const uint4* v = reinterpret_cast<const uint4*>((old ? src.tv : src.nv) + (in ? at : 0));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        const uint4 a = in ? k[8 * j + x] : zero, b = in ? v[8 * j + x] : zero;
        kw[u][j][4 * x] = a.x;
        kw[u][j][4 * x + 1] = a.y;
        kw[u][j][4 * x + 2] = a.z;
        kw[u][j][4 * x + 3] = a.w;
        vw[u][j][4 * x] = b.x;
        vw[u][j][4 * x + 1] = b.y;
        vw[u][j][4 * x + 2] = b.z;
        vw[u][j][4 * x + 3] = b.w;
      }
    }
  }
  float s[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t(&a)[4] = *reinterpret_cast<const uint32_t(*)[4]>(&qa[16 * j + 4 * w]);
        mma_bf16(s[u], a, kw[u][j][2 * w], kw[u][j][2 * w + 1]);
      }
  }
  // keys 8 u + 2 c + e of the step; a row sees those below `limit`
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool see = t0 + 8 * u + 2 * c + e < limit;
      s[u][e] = see ? s[u][e] * f : -INFINITY;
      s[u][2 + e] = see ? s[u][2 + e] * f : -INFINITY;
    }
  st.raise(quad_max(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]))),
           quad_max(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]))));
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[u][e] = ex2(s[u][e] - st.m[e >> 1]);
      st.l[e >> 1] += s[u][e];
    }
  const uint32_t pa[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]), pack_bf16x2(s[1][0], s[1][1]),
                          pack_bf16x2(s[1][2], s[1][3])};
  // On the diagonal a key's V must not reach the rows before it, not even as 0 * infinity:
  // what is not finite there is taken out of the product and added to the rows that see it.
  if (t0 + 16 > diagonal) {
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = 0; w < 8; ++w) bad = bad || not_finite(vw[u][j][w]);
    if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            uint32_t x = vw[u][j][w];
            if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
            if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
            vw[u][j][w] = x;
          }
#pragma unroll 1
      for (int t = t0; t < min(min(t0 + 16, src.count), limit); ++t) {
        const bool old = t < src.tail;
        const __nv_bfloat16* v = (old ? src.tv : src.nv) + static_cast<size_t>(old ? t : t - src.tail) * kRowElems + 16 * c;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(v + 64 * j + 2 * r);
            const float a = (x & 0x7f80u) == 0x7f80u ? __uint_as_float(x << 16) : 0.f;
            const float b = (x & 0x7f800000u) == 0x7f800000u ? __uint_as_float(x & 0xffff0000u) : 0.f;
            st.o[j][r][0] += a;
            st.o[j][r][1] += b;
            st.o[j][r][2] += a;
            st.o[j][r][3] += b;
          }
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 8; ++r) mma_bf16(st.o[j][r], pa, movm(vw[0][j][r]), movm(vw[1][j][r]));
}

// A warp's ring: 4 KB stages, filled in the order K low, K high, V low, V high of page after page.
struct RingQ {
  uint32_t base, bars;
  int stage = 0;
  uint32_t parity = 0;                                       // of the stage's next use
  __device__ __forceinline__ uint32_t addr() const { return base + stage * kStageA; }
  __device__ __forceinline__ uint32_t bar() const { return bars + 8 * stage; }
  __device__ __forceinline__ void next() {
    if (++stage == kStagesA) {
      stage = 0;
      parity ^= 1;
    }
  }
};

template <int kCode>
__global__ void __launch_bounds__(kAttnThreadsQ, 1) quant_attn_kernel(const AttnParamsQ p) {
  extern __shared__ uint8_t smem_q[];
  const int h = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
  const uint32_t sbase = (smem_u32(smem_q) + 1023u) & ~1023u;
  RingQ fill, use;
  fill.base = use.base = sbase + h * kWarpRing;
  fill.bars = use.bars = sbase + kKVHeads * kWarpRing + h * kStagesA * 8;
  if (lane == 0) {
    for (int s = 0; s < kStagesA; ++s) mbar_init(use.bars + 8 * s, 1);
    fence_barrier_init();
  }
  __syncwarp();
  asm volatile("griddepcontrol.launch_dependents;");
  if (p.plan[kQMagic] != kPlanMagicQ || p.plan[kQGrid] != p.grid || p.plan[kQRequests] != p.batch.requests ||
      p.plan[kQRows] != p.batch.rows) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  const int4 range = __ldg(reinterpret_cast<const int4*>(p.plan + plan_cta_at()) + blockIdx.x);
  const uint8_t* key = p.cache.key + static_cast<size_t>(h) * kHeadBytes;
  const uint8_t* value = p.cache.value + static_cast<size_t>(h) * kHeadBytes;
  bool alive = true;                                         // no wait ran out
  RowsQ st;
#pragma unroll 1
  for (int idx = range.x; idx <= range.z && alive; ++idx) {
    const ItemQ it = load_item_q(p, idx);
    const Request req = load_request(p.batch, p.cache, it.request);
    const int units = it.row_units + it.pages;
    const int ub = idx == range.x ? range.y : 0, ue = idx == range.z ? range.w : units;
    // what a stale plan says of another batch is not followed
    if (!req.ok || it.pages != req.ctx / kPage || it.q0 != req.q0 + it.r0 || it.r0 + it.rows > req.q_len ||
        it.row_units != row_units(req.ctx, req.q_len, it.r0)) {
      if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
      continue;
    }
    // pages [pb, pe) of the request; lane l knows the id of page chunk + l
    const int pb = max(ub - it.row_units, 0), pe = max(ue - it.row_units, 0);
    int chunk = pb, id = -1;
    float ks = 0.f, vs = 0.f;
    auto load_ids = [&](int first) {
      chunk = first;
      id = first + lane < pe ? __ldg(req.table + first + lane) : 0;
      const bool good = id >= 0 && id < p.cache.pages;
      if (!good) {
        atomicOr(&g_device_status, kStatusBadArgument);
        id = -1;
      }
      const size_t at = static_cast<size_t>(good ? id : 0) * kKVHeads + h;
      ks = good ? __ldg(p.cache.key_scale + at) : 0.f;
      vs = good ? __ldg(p.cache.value_scale + at) : 0.f;
    };
    // copies of the stages are issued one by one: piece x of page fp
    int fp = pb, piece = 0, ahead = 0;                       // ahead: stages filled and not yet used
    auto fill_one = [&]() {
      const int pid = __shfl_sync(0xffffffffu, id, fp - chunk);
      if (pid >= 0) {
        if (lane == 0) {
          mbar_arrive_expect_tx(fill.bar(), kStageA);
          bulk_load(fill.addr(), (piece < 2 ? key : value) + static_cast<size_t>(pid) * kPageBytes + (piece & 1) * kStageA,
                    kStageA, fill.bar());
        }
        fill.next();
        ++ahead;
      } else {
        piece = 3;                                           // (a page that is not there is left out)
      }
      if (++piece == 4) {
        piece = 0;
        ++fp;
      }
    };
    if (pb < pe) {
      load_ids(pb);
      while (ahead < kStagesA && fp < min(pe, chunk + 32)) fill_one();
    }
    // Q: k-step (j, w) of row n holds dims 64 j + 16 c + 4 w .. + 3, words 2 w and 2 w + 1
    uint32_t qa[32];
    {
      const __nv_bfloat16* q = p.q + (static_cast<size_t>(it.q0 + min(n, it.rows - 1)) * kQHeads + 2 * h) * kHeadDim + 16 * c;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint4 w = *reinterpret_cast<const uint4*>(q + x * kHeadDim + 64 * j + 8 * y);
            qa[16 * j + 8 * y + x] = w.x;
            qa[16 * j + 8 * y + 2 + x] = w.y;
            qa[16 * j + 8 * y + 4 + x] = w.z;
            qa[16 * j + 8 * y + 6 + x] = w.w;
          }
    }
    st.clear();
    if (ub < it.row_units) {
      const int tail = req.ctx % kPage;
      const size_t tail_at = tail_row(req.slot, req.ctx - tail) * kRowElems + h * kHeadDim;
      const size_t new_at = static_cast<size_t>(req.q0) * kRowElems + h * kHeadDim;
      const RowSource src{static_cast<const __nv_bfloat16*>(p.cache.tail_key) + tail_at,
                          static_cast<const __nv_bfloat16*>(p.cache.tail_value) + tail_at, p.new_k + new_at,
                          p.new_v + new_at, tail, tail + it.r0 + it.rows};
      const int end = min(min(ue, it.row_units) * kRowUnit, src.count);
      const int diagonal = tail + it.r0 + 1;                 // keys from here on are not seen by every row
#pragma unroll 1
      for (int t = ub * kRowUnit; t < end; t += 16)
        row_step(st, qa, src, t, diagonal + n, diagonal, p.scale_log2);
    }
    if (pb < pe) {
      // Q to halves: rows n and n + 8, each times 2^(14 - e)
      float f[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t top = 0;
#pragma unroll
        for (int i = x; i < 32; i += 2) top = max(top, max(qa[i] & 0x7fffu, (qa[i] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max(static_cast<int>(top >> 7) - 127, -100), 120);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
        f[x] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
        for (int i = x; i < 32; i += 2)
          qa[i] = pack_f16x2(__uint_as_float(qa[i] << 16) * up, __uint_as_float(qa[i] & 0xffff0000u) * up);
      }
#pragma unroll 1
      for (int page = pb; page < pe && alive; ++page) {
        if (page - chunk == 32) {
          load_ids(page);
          fp = page;                                         // (a chunk's stages are all used: none is ahead)
          while (ahead < kStagesA && fp < min(pe, chunk + 32)) fill_one();
        }
        if (__shfl_sync(0xffffffffu, id, page - chunk) < 0) continue;
        const float pks = __shfl_sync(0xffffffffu, ks, page - chunk), pvs = __shfl_sync(0xffffffffu, vs, page - chunk);
        const int stop = min(pe, chunk + 32);
        auto wait = [&]() {
          alive = __all_sync(0xffffffffu, mbar_wait(use.bar(), use.parity)) != 0;
          return alive;
        };
        auto release = [&]() {                               // every lane has read the stage
          use.next();
          --ahead;
          __syncwarp();
          if (fp < stop) fill_one();
        };
        float s[8][4];
#pragma unroll
        for (int u = 0; u < 8; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
        // S: column n of tile u = 2 t + x is key 16 (n / 2) + 4 t + 2 x + n % 2
        const uint32_t k_at = (16 * (n >> 1) + (n & 1)) * 64 + 16 * c;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!wait()) break;
          const uint32_t at = use.addr() + k_at;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const uint4 w = lds128(at + 2 * u * 64);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t b0, b1;
              decode4<kCode>(ww[x], b0, b1);
              mma_f16(s[u], *reinterpret_cast<const uint32_t(*)[4]>(&qa[16 * j + 4 * x]), b0, b1);
            }
          }
          release();
        }
        if (!alive) break;
        const float f0 = f[0] * pks, f1 = f[1] * pks;
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          s[u][0] *= f0;
          s[u][1] *= f0;
          s[u][2] *= f1;
          s[u][3] *= f1;
          m0 = fmaxf(m0, fmaxf(s[u][0], s[u][1]));
          m1 = fmaxf(m1, fmaxf(s[u][2], s[u][3]));
        }
        st.raise(quad_max(m0), quad_max(m1));
        uint32_t pa[4][4];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][e] = ex2(s[u][e] - st.m[e >> 1]);
            st.l[e >> 1] += s[u][e];
          }
          pa[u >> 1][2 * (u & 1)] = pack_f16x2(s[u][0], s[u][1]);
          pa[u >> 1][2 * (u & 1) + 1] = pack_f16x2(s[u][2], s[u][3]);
        }
        // O: column n of tile (j, r) is dim 64 j + 16 (n / 2) + 2 r + n % 2
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!wait()) break;
          const uint32_t at = use.addr() + k_at;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const uint4 w = lds128(at + 2 * r * 64);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
            float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t b0, b1;
              decode4<kCode>(ww[x], b0, b1);
              mma_f16(t, pa[x], b0, b1);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[j][r][e] = fmaf(t[e], pvs, st.o[j][r][e]);
          }
          release();
        }
      }
      if (!alive) break;
    }
    float l0 = st.l[0], l1 = st.l[1];
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (ub > 0 || ue < units) {
      float* part = p.part + part_index(blockIdx.x, idx == range.x ? 0 : 1, h);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            __stcg(reinterpret_cast<float4*>(part + (n + 8 * x) * kHeadDim + 64 * j + 16 * c + 4 * r),
                   make_float4(st.o[j][2 * r][2 * x], st.o[j][2 * r][2 * x + 1], st.o[j][2 * r + 1][2 * x],
                               st.o[j][2 * r + 1][2 * x + 1]));
        if (c == 0)
          __stcg(reinterpret_cast<float2*>(part + 16 * kHeadDim) + n + 8 * x, make_float2(st.m[x], x ? l1 : l0));
      }
    } else if (n < it.rows) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float inv = 1.f / (x ? l1 : l0);
        __nv_bfloat16* out = p.out + (static_cast<size_t>(it.q0 + n) * kQHeads + 2 * h + x) * kHeadDim + 16 * c;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              w[r] = pack_bf16x2(st.o[j][4 * y + r][2 * x] * inv, st.o[j][4 * y + r][2 * x + 1] * inv);
            *reinterpret_cast<uint4*>(out + 64 * j + 8 * y) = make_uint4(w[0], w[1], w[2], w[3]);
          }
      }
    }
  }
  if (!alive) {                                              // copies in flight land before the CTA exits
    for (int s = 0; s < kStagesA; ++s)
      if (use.stage != fill.stage || use.parity != fill.parity) {
        mbar_wait(use.bar(), use.parity);
        use.next();
      }
  }
}

// Grid (CTAs, 8): CTA (c, h) merges head h of the cut item whose first contributor is c.
// Thread (row, part) = (tid / 8, tid % 8) holds dims 16 part .. + 15 of a row.
__global__ void __launch_bounds__(128) quant_merge_kernel(const AttnParamsQ p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c0 = blockIdx.x, h = blockIdx.y, row = threadIdx.x >> 3, d0 = 16 * (threadIdx.x & 7);
  if (p.plan[kQMagic] != kPlanMagicQ || p.plan[kQGrid] != p.grid) return;
  const int4 merge = __ldg(reinterpret_cast<const int4*>(p.plan + plan_merge_at(p.grid)) + c0);
  if (merge.x < 0 || merge.x >= p.plan[kQItems] || merge.y <= c0 || merge.y >= p.grid) return;
  const ItemQ it = load_item_q(p, merge.x);
  const int x = row >> 3, r = row & 7;
  if (r >= it.rows || it.q0 < 0 || it.q0 + it.rows > p.batch.rows) return;
  auto at = [&](int k) { return p.part + part_index(k, k == c0 ? (merge.z & 1) : 0, h); };
  auto stat = [&](int k) { return __ldcg(reinterpret_cast<const float2*>(at(k) + 16 * kHeadDim) + row); };
  float m = kNoMaxQ;
  for (int k = c0; k <= merge.y; ++k) m = fmaxf(m, stat(k).x);
  float l = 0.f, o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
#pragma unroll 2
  for (int k = c0; k <= merge.y; ++k) {
    const float2 ml = stat(k);
    const float w = ex2(ml.x - m);
    l = fmaf(ml.y, w, l);
    const float4* src = reinterpret_cast<const float4*>(at(k) + row * kHeadDim + d0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldcg(src + i);
      o[4 * i] = fmaf(v.x, w, o[4 * i]);
      o[4 * i + 1] = fmaf(v.y, w, o[4 * i + 1]);
      o[4 * i + 2] = fmaf(v.z, w, o[4 * i + 2]);
      o[4 * i + 3] = fmaf(v.w, w, o[4 * i + 3]);
    }
  }
  const float inv = 1.f / l;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
  uint4* out = reinterpret_cast<uint4*>(p.out + (static_cast<size_t>(it.q0 + r) * kQHeads + 2 * h + x) * kHeadDim + d0);
  out[0] = make_uint4(w[0], w[1], w[2], w[3]);
  out[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

}  // namespace quant
}  // namespace dspark
