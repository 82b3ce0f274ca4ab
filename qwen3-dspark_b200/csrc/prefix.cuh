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
#include "train.cuh"

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

// ---------------------------------------------------------------------------
// bf16 tensor-core kernel (tcgen05), one persistent CTA per SM over the plan's items.
//
// An item is up to 128 query rows x the two query heads of a KV head = two MMA tiles A
// and B of 128 rows (row m of a tile = 2 * query row + head) that share every K/V block
// of 128 keys, so a block crosses from L2 once per 256 rows. Roles (384 threads):
//   warps 0-3, 4-7  softmax of tile A / B: one thread per row, whole rows of S in
//                   registers (no exchange between threads); P (bf16) overwrites its S
//                   columns in TMEM; the running maximum is raised, and O rescaled, only
//                   when it grows by more than 2^8 (exact: O / l does not depend on it);
//   warps 8, 9      MMA issuers of tile A / B (one thread each): S = Q K^T, O += P V. The
//                   MMAs of one thread execute in order, so S(i + 1) may follow PV(i)
//                   over the P it reads without a wait, and the tiles alternate on the
//                   tensor pipe: one tile's products run under the other's softmax;
//   warp 10         TMA producer: Q per item, K and V blocks through one ring of 32 KB
//                   stages in the order K0 V0 K1 V1 ..;
//   warp 11         zeroes the V rows between a short block's keys and the next multiple of
//                   16 (they may hold anything, and 0 * NaN is NaN).
// Short blocks load only boxes of 32 rows that hold keys, and multiply only N =
// keys rounded up to 16. Every wait is bounded; a timed-out wait raises the CTA abort
// flag, copies and MMAs in flight are drained and TMEM is released.
constexpr int kStagesN = 5;
constexpr int kAttThreads = 12 * 32;
constexpr uint32_t kSmemQ = 0;                             // 2 tiles x 32 KB
constexpr uint32_t kSmemRing = 2 * 32768;
constexpr uint32_t kSmemBar = kSmemRing + kStagesN * 32768;
enum Bar {
  kBQFull = 0, kBQEmpty, kBFull, kBEmpty = kBFull + kStagesN, kBFixed = kBEmpty + kStagesN,
  kBSFull = kBFixed + kStagesN, kBPFull = kBSFull + 2, kBODone = kBPFull + 2, kBOFree = kBODone + 2,
  kBDrain = kBOFree + 2, kNumBars
};
constexpr uint32_t kSmemSlot = kSmemBar + kNumBars * 8;
constexpr uint32_t kSmemAbort = kSmemSlot + 4;
constexpr uint32_t kSmemBytes = 1024 + kSmemAbort + 4;
constexpr uint32_t kTmemS = 0, kTmemO = 256;              // tile x: S at 128 x, O at 256 + 128 x
constexpr int kBoxRows = 32;

struct Maps {
  CUtensorMap q, kv[6];                                   // kv[2 s], kv[2 s + 1]: K and V of source s
};

struct ItemView {
  int q0, nq, head, slot, visible, nsegs, blocks;
  int src[kMaxSegs], row[kMaxSegs], len[kMaxSegs], pos[kMaxSegs];
};

__device__ __forceinline__ bool load_item(const Params& p, int idx, ItemView& x) {
  const int4* w = reinterpret_cast<const int4*>(p.plan + p.plan[kHItemsAt] + static_cast<size_t>(idx) * kItemWords);
  const int4 a = __ldg(w), b = __ldg(w + 1);
  x.q0 = a.x;
  x.nq = a.y;
  x.head = a.z;
  x.slot = a.w;
  x.visible = b.x;
  x.nsegs = b.y;
  x.blocks = 0;
  bool ok = x.nq >= 1 && x.nq <= kTileRows && x.q0 >= 0 && x.q0 <= p.total_q - x.nq && x.head >= 0 &&
            x.head < kHeads && x.nsegs >= 0 && x.nsegs <= kMaxSegs && x.slot < p.slots - (x.nq > kHalfTile ? 1 : 0);
#pragma unroll
  for (int s = 0; s < kMaxSegs; ++s) {
    const int4 g = __ldg(w + 2 + s);
    const bool used = s < x.nsegs;
    x.src[s] = g.x;
    x.row[s] = g.y;
    x.len[s] = used ? g.z : 0;
    x.pos[s] = g.w;
    if (used) {
      const Source& q = p.src[g.x == 0 ? 0 : (g.x == 1 ? 1 : 2)];
      ok = ok && g.x >= 0 && g.x < 3 && g.z >= 1 && g.z <= (1 << 30) && g.y >= 0 && q.off + g.y + g.z <= q.rows;
      x.blocks += (g.z + kBlock - 1) / kBlock;
    }
  }
  return ok;
}

// Walks an item's key blocks.
struct BlockWalk {
  int seg = 0, at = 0;
  __device__ __forceinline__ int keys(const ItemView& x) const {
    const int len = seg == 0 ? x.len[0] : (seg == 1 ? x.len[1] : x.len[2]);
    return min(kBlock, len - at);
  }
  __device__ __forceinline__ int pos(const ItemView& x) const {
    return (seg == 0 ? x.pos[0] : (seg == 1 ? x.pos[1] : x.pos[2])) + at;
  }
  __device__ __forceinline__ int row(const ItemView& x) const {
    return (seg == 0 ? x.row[0] : (seg == 1 ? x.row[1] : x.row[2])) + at;
  }
  __device__ __forceinline__ int src(const ItemView& x) const {
    return seg == 0 ? x.src[0] : (seg == 1 ? x.src[1] : x.src[2]);
  }
  __device__ __forceinline__ void next(const ItemView& x) {
    at += kBlock;
    if (at >= (seg == 0 ? x.len[0] : (seg == 1 ? x.len[1] : x.len[2]))) {
      at = 0;
      ++seg;
    }
  }
};

__host__ __device__ constexpr uint32_t instr_desc_n(uint32_t b_mn, uint32_t n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// Position in the ring of 32 KB stages.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStagesN) {
      stage = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ void producer_role(const Params& p, const Maps& maps, int first, int last, uint32_t sbase,
                                              uint32_t bars, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  Ring ring;
  int it = 0, armed_q = 0;
  uint32_t last_full[kStagesN] = {};      // phase + 1 of the last load into each stage
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x) || x.blocks == 0) continue;
    if (!(ok = train::wait_or_abort(bar(kBQEmpty), (it & 1) ^ 1, abort_flag))) break;
    const int tiles = x.nq > kHalfTile ? 2 : 1;
    mbar_arrive_expect_tx(bar(kBQFull), 32768u * tiles);
    for (int t = 0; t < tiles; ++t) {
      tma_load_3d(sbase + kSmemQ + t * 32768, &maps.q, 0, 2 * x.head, x.q0 + t * kHalfTile, bar(kBQFull));
      tma_load_3d(sbase + kSmemQ + t * 32768 + 16384, &maps.q, 64, 2 * x.head, x.q0 + t * kHalfTile, bar(kBQFull));
    }
    ++armed_q;
    BlockWalk w;
    for (int b = 0; b < x.blocks && ok; ++b, w.next(x)) {
      const int boxes = (w.keys(x) + kBoxRows - 1) / kBoxRows, src = w.src(x);
      const int row = static_cast<int>(p.src[src].off) + w.row(x);
      for (int v = 0; v < 2; ++v) {
        if (!(ok = train::wait_or_abort(bar(kBEmpty + ring.stage), ring.phase ^ 1, abort_flag))) break;
        const uint32_t full = bar(kBFull + ring.stage), dst = sbase + kSmemRing + ring.stage * 32768;
        mbar_arrive_expect_tx(full, static_cast<uint32_t>(boxes) * kBoxRows * 256u);
        const CUtensorMap* m = &maps.kv[2 * src + v];
        for (int i = 0; i < boxes; ++i) {
          tma_load_3d(dst + i * kBoxRows * 128, m, 0, x.head, row + i * kBoxRows, full);
          tma_load_3d(dst + 16384 + i * kBoxRows * 128, m, 64, x.head, row + i * kBoxRows, full);
        }
#pragma unroll
        for (int s = 0; s < kStagesN; ++s)
          if (s == ring.stage) last_full[s] = ring.phase + 1;
        ring.next();
      }
    }
    ++it;
  }
  if (!ok) *abort_flag = 1;
  // Copies in flight land before the CTA can exit (a no-op when all were consumed).
  volatile int never = 0;
  if (armed_q) train::wait_or_abort(bar(kBQFull), (armed_q - 1) & 1, &never);
#pragma unroll
  for (int s = 0; s < kStagesN; ++s)
    if (last_full[s]) train::wait_or_abort(bar(kBFull + s), last_full[s] - 1, &never);
}

__device__ __forceinline__ void issue_role(const Params& p, int tile, int first, int last, uint32_t sbase,
                                           uint32_t bars, uint32_t tmem, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  Ring ring;
  int it = 0, mine = 0;                   // items with blocks; of them, items with this tile
  uint32_t p_phase = 0, fixed_phase = 0;  // fixed_phase: one parity bit per stage
  const uint32_t s_col = tmem + kTmemS + tile * 128, o_col = tmem + kTmemO + tile * 128;
  const uint32_t qbase = sbase + kSmemQ + tile * 32768;
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x) || x.blocks == 0) continue;
    if (tile == 1 && x.nq <= kHalfTile) {
      // no rows in this tile: release the stages as they fill (every phase is waited for, so
      // no barrier runs two phases ahead of this thread)
      ok = train::wait_or_abort(bar(kBQFull), it & 1, abort_flag);
      BlockWalk w;
      for (int b = 0; b < x.blocks && ok; ++b, w.next(x)) {
        for (int v = 0; v < 2 && ok; ++v) {
          ok = train::wait_or_abort(bar(kBFull + ring.stage), ring.phase, abort_flag);
          if (!ok) break;
          if (v == 1 && (w.keys(x) & 15)) fixed_phase ^= 1u << ring.stage;
          mbar_arrive(bar(kBEmpty + ring.stage));
          ring.next();
        }
      }
      if (ok) mbar_arrive(bar(kBQEmpty));
      ++it;
      continue;
    }
    if (!(ok = train::wait_or_abort(bar(kBQFull), it & 1, abort_flag))) break;
    BlockWalk w;
    auto qk = [&](int keys, bool final) {
      if (!(ok = train::wait_or_abort(bar(kBFull + ring.stage), ring.phase, abort_flag))) return;
      train::tc_fence_after();
      const uint32_t kbase = sbase + kSmemRing + ring.stage * 32768;
      const uint32_t idesc = instr_desc_n(0, static_cast<uint32_t>((keys + 15) & ~15));
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
        train::umma_bf16(s_col, train::smem_desc(qbase + off, 16, 1024), train::smem_desc(kbase + off, 16, 1024),
                         idesc, kk > 0);
      }
      train::umma_commit(bar(kBSFull + tile));
      train::umma_commit(bar(kBEmpty + ring.stage));
      if (final) train::umma_commit(bar(kBQEmpty));
      ring.next();
    };
    qk(w.keys(x), x.blocks == 1);
    for (int b = 0; b < x.blocks && ok; ++b) {
      const int keys = w.keys(x);
      if (!(ok = train::wait_or_abort(bar(kBPFull + tile), p_phase, abort_flag))) break;
      p_phase ^= 1;
      if (b == 0 && !(ok = train::wait_or_abort(bar(kBOFree + tile), (mine & 1) ^ 1, abort_flag))) break;
      if (!(ok = train::wait_or_abort(bar(kBFull + ring.stage), ring.phase, abort_flag))) break;
      if (keys & 15) {
        if (!(ok = train::wait_or_abort(bar(kBFixed + ring.stage), (fixed_phase >> ring.stage) & 1, abort_flag))) break;
        fixed_phase ^= 1u << ring.stage;
      }
      train::tc_fence_after();
      const uint32_t vbase = sbase + kSmemRing + ring.stage * 32768;
      const int steps = (keys + 15) >> 4;
      if (steps == 8) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          train::umma_bf16_ts(o_col, s_col + kk * 8, train::smem_desc(vbase + kk * 2048, 16384, 1024),
                              instr_desc_n(1, 128), (b > 0 || kk > 0) ? 1u : 0u);
      } else {
        for (int kk = 0; kk < steps; ++kk)
          train::umma_bf16_ts(o_col, s_col + kk * 8, train::smem_desc(vbase + kk * 2048, 16384, 1024),
                              instr_desc_n(1, 128), (b > 0 || kk > 0) ? 1u : 0u);
      }
      train::umma_commit(bar(kBEmpty + ring.stage));
      ring.next();
      if (b + 1 == x.blocks) {
        train::umma_commit(bar(kBODone + tile));
      } else {
        w.next(x);
        qk(w.keys(x), b + 2 == x.blocks);
      }
    }
    ++it;
    ++mine;
  }
  if (!ok) *abort_flag = 1;
  // Every MMA issued above completes before TMEM is released.
  train::umma_commit(bar(kBDrain));
  volatile int never = 0;
  train::wait_or_abort(bar(kBDrain), 0, &never);
}

// Zeroes the V rows behind a short block's keys up to the next multiple of 16 (whole warp).
__device__ __forceinline__ void fix_role(const Params& p, int first, int last, uint8_t* smem, uint32_t bars,
                                         volatile int* abort_flag) {
  const int lane = threadIdx.x & 31;
  Ring ring;
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x) || x.blocks == 0) continue;
    BlockWalk w;
    for (int b = 0; b < x.blocks && ok; ++b, w.next(x)) {
      const int keys = w.keys(x);
      for (int v = 0; v < 2 && ok; ++v, ring.next()) {
        ok = train::wait_or_abort(bars + 8u * (kBFull + ring.stage), ring.phase, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (v == 1 && (keys & 15)) {
          uint8_t* stage = smem + kSmemRing + ring.stage * 32768;
          const int rows = ((keys + 15) & ~15) - keys;
          for (int u = lane; u < rows * 16; u += 32)
            *reinterpret_cast<uint4*>(stage + ((u >> 3) & 1) * 16384 + (keys + (u >> 4)) * 128 + (u & 7) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + 8u * (kBFixed + ring.stage));
        }
        // one of the three releases of a stage: this warp stays within a phase of the ring
        if (lane == 0) mbar_arrive(bars + 8u * (kBEmpty + ring.stage));
      }
    }
  }
  if (!ok) *abort_flag = 1;
}

template <int N>
__device__ __forceinline__ float max_n(const float (&s)[N]) {
  float a[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int i = 4; i + 8 <= N; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = train::max3f(a[k], s[i + 2 * k], s[i + 2 * k + 1]);
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = fmaxf(a[k], s[N - 4 + k]);
  return fmaxf(train::max3f(a[0], a[1], a[2]), a[3]);
}

struct RowState {
  float m, l;                             // running maximum (log2 units), sum of 2^(s - m)
};

// One block of a row: kCols scores from TMEM, probabilities back as packed bf16. `see`
// scores are visible.
template <int kCols>
__device__ __forceinline__ void softmax_block(uint32_t s_addr, uint32_t o_addr, int see, float scale_log2, bool first,
                                              RowState& st) {
  float s[kCols];
  if constexpr (kCols == 128) {
    train::tmem_ld128(s_addr, s);
  } else {
#pragma unroll
    for (int c = 0; c < kCols / 32; ++c) train::tmem_ld32(s_addr + 32 * c, *reinterpret_cast<float(*)[32]>(&s[32 * c]));
  }
  if (!__all_sync(0xffffffffu, see >= kCols)) {
#pragma unroll
    for (int i = 0; i < kCols; ++i) s[i] = i < see ? s[i] : -INFINITY;
  }
  const float m_new = fmaxf(st.m, max_n(s) * scale_log2);
  const bool raise = m_new > st.m + 8.f;
  float alpha = 1.f;
  if (raise) {
    alpha = ex2(st.m - m_new);
    st.m = m_new;
  }
  if (!first && __any_sync(0xffffffffu, raise)) {
    // the block's S was committed behind the previous PV: O is complete
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float o[32];
      train::tmem_ld32(o_addr + 32 * c, o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] *= alpha;
      train::tmem_st32(o_addr + 32 * c, o);
    }
  }
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < kCols / 64 + (kCols < 64); ++c) {
    constexpr int kW = kCols < 64 ? kCols / 2 : 32;
    uint32_t pk[32];
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      const float a = ex2(fmaf(s[64 * c + 2 * i], scale_log2, -st.m));
      const float b = ex2(fmaf(s[64 * c + 2 * i + 1], scale_log2, -st.m));
      sum[i & 3] += a + b;
      pk[i] = pack_bf16x2(a, b);
    }
    if constexpr (kW == 32) {
      train::tmem_st32(s_addr + 32 * c, *reinterpret_cast<const float(*)[32]>(pk));
    } else {
#pragma unroll
      for (int i = kW; i < 32; ++i) pk[i] = 0u;
      train::tmem_st32(s_addr + 32 * c, *reinterpret_cast<const float(*)[32]>(pk));
    }
  }
  st.l = st.l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
}

__device__ __forceinline__ void softmax_role(const Params& p, float* part, int first, int last, uint32_t bars,
                                             uint32_t tmem, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = warp >> 2, quarter = warp & 3;
  const int m = quarter * 32 + lane;                        // row of the tile == TMEM lane
  const int lt = tile * kHalfTile + (m >> 1);               // query row of the item
  const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
  const uint32_t s_addr = tmem + lanes + kTmemS + tile * 128, o_addr = tmem + lanes + kTmemO + tile * 128;
  uint32_t s_phase = 0, o_phase = 0;
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x)) {
      if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
      continue;
    }
    if (tile == 1 && x.nq <= kHalfTile) continue;
    const bool row_ok = lt < x.nq;
    const bool warp_ok = tile * kHalfTile + quarter * 16 < x.nq;
    RowState st{-1e30f, 0.f};
    if (x.blocks > 0) {
      BlockWalk w;
      for (int b = 0; b < x.blocks; ++b, w.next(x)) {
        ok = train::wait_or_abort(bar(kBSFull + tile), s_phase, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        s_phase ^= 1;
        if (warp_ok) {
          train::tc_fence_after();
          const int keys = w.keys(x);
          const int see = row_ok ? min(keys, x.visible + lt - w.pos(x)) : 0;
          if (keys > 64)
            softmax_block<128>(s_addr, o_addr, see, p.scale_log2, b == 0, st);
          else if (keys > 32)
            softmax_block<64>(s_addr, o_addr, see, p.scale_log2, b == 0, st);
          else
            softmax_block<32>(s_addr, o_addr, see, p.scale_log2, b == 0, st);
          train::tc_fence_before();
        }
        mbar_arrive(bar(kBPFull + tile));
      }
      if (!ok) break;
      ok = train::wait_or_abort(bar(kBODone + tile), o_phase, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      o_phase ^= 1;
      train::tc_fence_after();
    }
    if (warp_ok) {
      const float inv = st.l > 0.f ? 1.f / st.l : 0.f;
      __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.out) +
                            (static_cast<size_t>(x.q0 + (row_ok ? lt : 0)) * kQHeads + 2 * x.head + (m & 1)) * kHeadDim;
      const size_t slot = static_cast<size_t>(max(x.slot, 0) + tile);
      float* prow = part + slot * (kSlotFloats + 128) + static_cast<size_t>(m) * kHeadDim;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float o[32];
        if (x.blocks > 0) {
          train::tmem_ld32(o_addr + 32 * c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = st.l > 0.f ? o[i] * inv : 0.f;
        if (row_ok && x.slot < 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 v;
            v.x = pack_bf16x2(o[8 * j], o[8 * j + 1]);
            v.y = pack_bf16x2(o[8 * j + 2], o[8 * j + 3]);
            v.z = pack_bf16x2(o[8 * j + 4], o[8 * j + 5]);
            v.w = pack_bf16x2(o[8 * j + 6], o[8 * j + 7]);
            *reinterpret_cast<uint4*>(orow + 32 * c + 8 * j) = v;
          }
        } else if (row_ok) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(reinterpret_cast<float4*>(prow + 32 * c + 4 * j),
                   make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]));
        }
      }
      if (row_ok && x.slot >= 0)
        __stcg(part + slot * (kSlotFloats + 128) + kSlotFloats + m, st.l > 0.f ? st.m + log2f(st.l) : -INFINITY);
    }
    if (x.blocks > 0) {
      train::tc_fence_before();
      mbar_arrive(bar(kBOFree + tile));
    }
  }
  if (!ok) *abort_flag = 1;
}

__global__ void __launch_bounds__(kAttThreads, 1)
    prefix_attn_kernel(const __grid_constant__ Maps maps, const Params p, float* part) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem), bars = sbase + kSmemBar;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemAbort);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  int first = 0, last = 0;
  if (plan_ok(p) && p.plan[kHGrid] == static_cast<int>(gridDim.x)) {
    const int* offs = p.plan + p.plan[kHCtaAt] + blockIdx.x;
    first = offs[0];
    last = offs[1];
    if (first < 0 || last < first || last > p.plan[kHItems]) first = last = 0;
  } else if (threadIdx.x == 0) {
    atomicOr(&g_device_status, kStatusBadArgument);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) {
      uint32_t count = 1;
      if (i == kBQEmpty || i == kBDrain) count = 2;                     // both issuers
      if (i >= kBEmpty && i < kBEmpty + kStagesN) count = 3;            // both issuers and warp 11
      if ((i >= kBPFull && i < kBPFull + 2) || (i >= kBOFree && i < kBOFree + 2)) count = 128;
      mbar_init(bars + 8u * i, count);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) train::tmem_alloc(sbase + kSmemSlot, 512);
  train::tc_fence_before();
  __syncthreads();
  train::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kSmemSlot);
  if (warp < 8) {
    softmax_role(p, part, first, last, bars, tmem, abort_flag);
  } else if (warp < 10) {
    if (lane == 0) issue_role(p, warp - 8, first, last, sbase, bars, tmem, abort_flag);
    __syncwarp();
  } else if (warp == 10) {
    if (lane == 0) producer_role(p, maps, first, last, sbase, bars, abort_flag);
    __syncwarp();
  } else {
    fix_role(p, first, last, smem, bars, abort_flag);
  }
  train::tc_fence_before();
  __syncthreads();
  train::tc_fence_after();
  if (warp == 8) train::tmem_dealloc(tmem, 512);
}

// Combines the partial rows: one warp per (query row, head), lane l owns d = 4 l ..
//   out = sum_c 2^(L_c - M) o_c / sum_c 2^(L_c - M),  M = max_c L_c
__global__ void __launch_bounds__(256) prefix_merge_kernel(const Params p, const float* part) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!plan_ok(p)) return;
  const int lane = threadIdx.x & 31;
  const long long u = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (u >= static_cast<long long>(p.total_q) * kQHeads) return;
  const int t = static_cast<int>(u / kQHeads), h = static_cast<int>(u % kQHeads);
  const int run = p.plan[p.plan[kHTokenRunAt] + t];
  if (run < 0 || run >= p.plan[kHRuns]) return;
  const int* w = p.plan + p.plan[kHRunsAt] + static_cast<size_t>(run) * kRunWords;
  const int tiles = w[kRunTiles];
  const int n0 = w[kRunTile0 + 1], total = n0 + (tiles > 1 ? w[kRunTile0 + kRunTileWords + 1] : 0);
  // slot and row of contribution c
  auto where = [&](int c) -> size_t {
    const int* k = w + kRunTile0 + (c < n0 ? 0 : kRunTileWords);
    const int piece = c < n0 ? c : c - n0, lt = t - k[3];
    const int slot = min(max(k[0] + (piece * kHeads + (h >> 1)) * k[2] + (lt >> 6), 0), p.slots - 1);
    return static_cast<size_t>(slot) * (kSlotFloats + 128);
  };
  const int* k0 = w + kRunTile0;
  const int* k1 = w + kRunTile0 + kRunTileWords;
  auto row_of = [&](int c) { return 2 * ((t - (c < n0 ? k0[3] : k1[3])) & 63) + (h & 1); };
  float top = -INFINITY;
  for (int c = lane; c < total; c += 32) top = fmaxf(top, __ldcg(part + where(c) + kSlotFloats + row_of(c)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
  if (top > -INFINITY) {
    for (int c0 = 0; c0 < total; c0 += 32) {
      const int c = c0 + lane;
      const float mine = c < total ? ex2(__ldcg(part + where(c) + kSlotFloats + row_of(c)) - top) : 0.f;
      const int n = min(32, total - c0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float f = __shfl_sync(0xffffffffu, mine, i);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(
            part + where(c0 + i) + static_cast<size_t>(row_of(c0 + i)) * kHeadDim + 4 * lane));
        den += f;
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
    }
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  uint2 res;
  res.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  res.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) +
                            (static_cast<size_t>(t) * kQHeads + h) * kHeadDim + 4 * lane) = res;
}

}  // namespace prefix
}  // namespace dspark
