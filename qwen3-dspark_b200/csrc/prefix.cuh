// Attention of a batch whose requests share long prefixes (16 query heads, 8 KV heads,
// head dim 128; query head h reads KV head h / 2).
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / 2]) v[j, h / 2]
//
// over the visible keys j of row t's request: its group's prefix rows, then its own
// cached rows, then its new rows, read in place from three sources. With `causal`, row
// x of a request with q rows and n keys sees keys j <= n - q + x. A row without a
// visible key gives zeros. Keys behind a row's limit may hold anything; values there are
// multiplied by zero weights, so an infinity or NaN in a later row of the request shows.
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
  int check, total_q, grid, slots, part_rows, items_at, runs, runs_at, parts_at, token_run_at;
  Source src[3];     // prefix, own, new
  float scale, scale_log2;
};

// Partial rows of one MMA tile, a slot of R = part_pitch workspace rows: R x 128 fp32
// (normalised) as [d / 4][row][4], so that the 32 rows of a warp store 512 contiguous bytes
// (row by row, each store instruction touched 32 lines: 7,000 cycles a tile), then each row's
// maximum and sum. The two stay apart: where scores are large, m + log2(l) would round away
// how many keys a part holds.
constexpr int kPartRowFloats = kHeadDim + 2;
inline size_t workspace_bytes(int part_rows) { return static_cast<size_t>(part_rows) * kPartRowFloats * sizeof(float); }
__device__ __forceinline__ size_t part_at(int row) { return static_cast<size_t>(row) * kPartRowFloats; }

__device__ __forceinline__ bool plan_ok(const Params& p) {
  return p.plan[kHMagic] == kPlanMagic && p.plan[kHCheck] == p.check && p.plan[kHTotalQ] == p.total_q;
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
//   warps 8, 9      MMA issuers of tile A / B (an elected lane each): S = Q K^T, O += P V.
//                   The MMAs of one thread execute in order, so S(i + 1) may follow PV(i)
//                   over the P it reads without a wait, and the tiles alternate on the
//                   tensor pipe: one tile's products run under the other's softmax;
//   warp 10         TMA producer: Q per item, K and V blocks through one ring of 32 KB
//                   stages in the order K0 V0 K1 V1 ..;
//   warp 11         zeroes the V rows between a short block's keys and the next multiple of
//                   16 (they may hold anything, and 0 * NaN is NaN).
// Short blocks load only boxes of 32 rows that hold keys, and multiply only N =
// keys rounded up to 16. Every wait is bounded; a timed-out wait raises the CTA abort
// flag, copies and MMAs in flight are drained and TMEM is released.
//
// The probabilities are rounded to bf16 for the second product (the MMA takes both operands
// in one type; their sum l is of the unrounded ones): at most 2^-8 of each weight, which takes
// the relative error of an output from 0.0017 (its own rounding) to 0.0023.
//
// Bound by the softmax chain where there are many rows (1024 rows x 32768 keys: 269 us,
// 1,021 TFLOP/s of 1,666; a block of both tiles takes 3,700 cycles of which the MMAs are
// 2,048) and by DRAM and the latency of short items where there are few (8 rows x 32768 keys:
// 40 us with the merge; the keys alone take 21). 28 bytes of a softmax thread spill.
constexpr int kStagesN = 5;
constexpr int kAttThreads = 12 * 32;
constexpr uint32_t kSmemQ = 0;                             // 2 tiles x 32 KB
constexpr uint32_t kSmemRing = 2 * 32768;
constexpr uint32_t kSmemBar = kSmemRing + kStagesN * 32768;
enum Bar {
  kBQFull = 0, kBQEmpty, kBFull, kBEmpty = kBFull + kStagesN, kBFixed = kBEmpty + kStagesN,
  kBSFull = kBFixed + kStagesN, kBPFull = kBSFull + 2, kBODone = kBPFull + 2, kBOFree = kBODone + 2,
  kBTurn = kBOFree + 2, kBDrain = kBTurn + 2, kNumBars
};
// Registers per thread of the softmax warpgroups and of the third one after setmaxnreg; the
// launch's own (kAttThreads x the kernel's count, checked when the device is set up) cover them.
constexpr int kSoftmaxRegs = 200, kOtherRegs = 96;
constexpr uint32_t kSmemSlot = kSmemBar + kNumBars * 8;
constexpr uint32_t kSmemAbort = kSmemSlot + 4;
constexpr uint32_t kSmemBytes = 1024 + kSmemAbort + 4;
constexpr uint32_t kTmemS = 0, kTmemO = 256;              // tile x: S at 128 x, O at 256 + 128 x
constexpr int kBoxRows = 32;

struct Maps {
  CUtensorMap q;                                          // boxes of 32 query rows x 2 heads x 64 d
  CUtensorMap block[6], box[6];                           // [2 s], [2 s + 1]: K and V of source s
};

struct ItemView {
  int q0, nq, head, slot, part, visible, nsegs, blocks;
  bool dual;
  int src[kMaxSegs], row[kMaxSegs], len[kMaxSegs], pos[kMaxSegs];
};

__device__ __forceinline__ bool load_item(const Params& p, int idx, ItemView& x) {
  const int4* w = reinterpret_cast<const int4*>(p.plan + p.items_at + static_cast<size_t>(idx) * kItemWords);
  const int4 a = __ldg(w), b = __ldg(w + 1);
  x.q0 = a.x;
  x.nq = a.y;
  x.head = a.z;
  x.slot = a.w;
  x.visible = b.x;
  x.nsegs = b.y;
  x.dual = b.z != 0;
  x.part = b.w;
  x.blocks = 0;
  bool ok = item_fits(x.q0, x.nq, x.head, x.slot, x.part, x.nsegs, x.dual, p.total_q, p.slots, p.part_rows);
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
  return ok && (!x.dual || x.blocks >= 2);
}

// Walks an item's key blocks.
struct BlockWalk {
  int seg = 0, at = 0;
  __device__ __forceinline__ int keys(const ItemView& x) const {
    const int len = seg == 0 ? x.len[0] : (seg == 1 ? x.len[1] : x.len[2]);
    return min(kBlock, len - at);
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

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elected() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}

// First row of tile B in a dual item: up to 64 rows move to the other two warps' lanes, so
// that the tiles' softmax warps with rows lie on different SM quarters.
__device__ __forceinline__ int dual_shift(int nq) { return nq <= 32 ? 64 : 0; }

// A whole block of 128 keys is one copy: the map's dimensions (64 d, row, half, head) put
// the 16 KB halves of 128-byte rows one behind the other. A short block takes boxes of 32
// rows per half. (Boxes throughout, issued by one lane of a divergent warp, cost 1,050
// cycles a stage and bounded every memory-bound case.)
__device__ __forceinline__ void producer_role(const Params& p, const Maps& maps, int first, int last, uint32_t sbase,
                                              uint32_t bars, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  auto wait = [&](int i, uint32_t parity) {
    return __all_sync(0xffffffffu, train::wait_or_abort(bar(i), parity, abort_flag)) != 0;
  };
  const uint32_t leader = elected();
  Ring ring;
  int it = 0, uses = 0;
  if (leader) prefetch_tmap(&maps.q);
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x) || x.blocks == 0) continue;
    if (!(ok = wait(kBQEmpty, (it & 1) ^ 1))) break;
    if (leader) {
      // 32 query rows (64 MMA rows, 8 KB per half) a box
      const int boxes = (x.nq + 31) >> 5;
      mbar_arrive_expect_tx(bar(kBQFull), 16384u * boxes * (x.dual ? 2 : 1));
      for (int t = 0; t < boxes; ++t) {
        const uint32_t dst = sbase + kSmemQ + (t >> 1) * 32768 + (t & 1) * 8192;
        tma_load_3d(dst, &maps.q, 0, 2 * x.head, x.q0 + 32 * t, bar(kBQFull));
        tma_load_3d(dst + 16384, &maps.q, 64, 2 * x.head, x.q0 + 32 * t, bar(kBQFull));
        if (x.dual) {
          // tile B holds the same rows, from row dual_shift on
          const uint32_t d2 = sbase + kSmemQ + 32768 + ((t ^ (dual_shift(x.nq) >> 6)) & 1) * 8192;
          tma_load_3d(d2, &maps.q, 0, 2 * x.head, x.q0 + 32 * t, bar(kBQFull));
          tma_load_3d(d2 + 16384, &maps.q, 64, 2 * x.head, x.q0 + 32 * t, bar(kBQFull));
        }
      }
    }
    __syncwarp();
    BlockWalk w;
    for (int b = 0; b < x.blocks && ok; ++b, w.next(x)) {
      const int keys = w.keys(x), src = w.src(x);
      const int row = static_cast<int>(p.src[src].off) + w.row(x);
      for (int v = 0; v < 2; ++v) {
        if (!(ok = wait(kBEmpty + ring.stage, ring.phase ^ 1))) break;
        const uint32_t full = bar(kBFull + ring.stage), dst = sbase + kSmemRing + ring.stage * 32768;
        if (leader) {
          if (keys == kBlock) {
            mbar_arrive_expect_tx(full, 32768u);
            tma_load_4d(dst, &maps.block[2 * src + v], 0, row, 0, x.head, full);
          } else {
            const int boxes = (keys + kBoxRows - 1) / kBoxRows;
            mbar_arrive_expect_tx(full, static_cast<uint32_t>(boxes) * kBoxRows * 256u);
            for (int i = 0; i < boxes; ++i) {
              tma_load_3d(dst + i * kBoxRows * 128, &maps.box[2 * src + v], 0, x.head, row + i * kBoxRows, full);
              tma_load_3d(dst + 16384 + i * kBoxRows * 128, &maps.box[2 * src + v], 64, x.head, row + i * kBoxRows,
                          full);
            }
          }
        }
        __syncwarp();
        ++uses;
        ring.next();
      }
    }
    ++it;
  }
  if (!ok) *abort_flag = 1;
  // Copies in flight land before the CTA can exit (a no-op when all were consumed): the
  // last load of each stage that was used.
  volatile int never = 0;
  if (it) train::wait_or_abort(bar(kBQFull), (it - 1) & 1, &never);
  for (int s = 0; s < kStagesN && s < uses; ++s) {
    const int last_use = uses - 1 - (uses - 1 - s) % kStagesN;
    train::wait_or_abort(bar(kBFull + s), (last_use / kStagesN) & 1, &never);
  }
}

// The whole warp runs the issue loop, so that descriptors stay in uniform registers; one
// elected lane issues each MMA and commit. (A role run by one lane of a divergent warp
// took 105-115 cycles per MMA of 64.)
__device__ __forceinline__ void issue_role(const Params& p, int tile, int first, int last, uint32_t sbase,
                                           uint32_t bars, uint32_t tmem, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  auto wait = [&](int i, uint32_t parity) {
    return __all_sync(0xffffffffu, train::wait_or_abort(bar(i), parity, abort_flag)) != 0;
  };
  const uint32_t leader = elected();
  Ring ring;
  int it = 0, mine = 0;                   // items with blocks; of them, items with this tile
  uint32_t p_phase = 0, fixed_phase = 0;  // fixed_phase: one parity bit per stage
  uint32_t turns = 0;                     // turns taken
  const uint32_t s_col = tmem + kTmemS + tile * 128, o_col = tmem + kTmemO + tile * 128;
  const uint64_t k_desc = train::smem_desc(sbase + kSmemRing, 16, 1024);
  const uint64_t v_desc = train::smem_desc(sbase + kSmemRing, 16384, 1024);
  bool ok = true;
  for (int idx = first; idx < last && ok; ++idx) {
    ItemView x;
    if (!load_item(p, idx, x) || x.blocks == 0) continue;
    if (!(ok = wait(kBQFull, it & 1))) break;
    BlockWalk w;
    // releases the stages of a block that this tile does not use, as they fill (every phase
    // is waited for, so no barrier runs two phases ahead of this warp)
    auto skip_block = [&]() {
      for (int v = 0; v < 2 && ok; ++v) {
        if (!(ok = wait(kBFull + ring.stage, ring.phase))) return;
        if (v == 1 && (w.keys(x) & 15)) fixed_phase ^= 1u << ring.stage;
        if (leader) mbar_arrive(bar(kBEmpty + ring.stage));
        ring.next();
      }
      w.next(x);
    };
    if (tile == 1 && x.nq <= kHalfTile && !x.dual) {
      for (int b = 0; b < x.blocks && ok; ++b) skip_block();
      if (ok && leader) mbar_arrive(bar(kBQEmpty));
      ++it;
      continue;
    }
    const int step = x.dual ? 2 : 1, b0 = x.dual ? tile : 0;
    const uint64_t q_desc = train::smem_desc(sbase + kSmemQ + tile * 32768, 16, 1024);
    if (b0 > 0) skip_block();
    if (!ok) break;
    // The issuers of a two-tile item take turns, A before B: a turn is PV(b) and QK(b + 1)
    // of one tile, so the tiles stay half a block apart and each one's softmax runs under
    // the other's products. Issuing freely, both tiles' MMAs interleave on the pipe, both
    // softmaxes start together and the pipe idles under them (5,800 cycles a block).
    const bool paired = x.nq > kHalfTile;
    auto take_turn = [&]() {
      if (!paired) return true;
      const bool got = wait(kBTurn + tile, (turns & 1) ^ (tile == 0 ? 1u : 0u));
      ++turns;
      return got;
    };
    auto pass_turn = [&]() {
      if (paired && leader) mbar_arrive(bar(kBTurn + (tile ^ 1)));
    };
    auto issue_qk = [&](int stage, int keys) {
      const uint64_t kd = k_desc + static_cast<uint32_t>(stage * (32768 >> 4));
      const uint32_t idesc = instr_desc_n(0, static_cast<uint32_t>((keys + 15) & ~15));
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
        train::umma_bf16(s_col, q_desc + off, kd + off, idesc, kk > 0);
      }
    };
    // S of the first block
    if (!(ok = wait(kBFull + ring.stage, ring.phase)) || !(ok = take_turn())) break;
    train::tc_fence_after();
    if (leader) {
      issue_qk(ring.stage, w.keys(x));
      train::umma_commit(bar(kBSFull + tile));
      train::umma_commit(bar(kBEmpty + ring.stage));
      if (b0 + step >= x.blocks) train::umma_commit(bar(kBQEmpty));
    }
    __syncwarp();
    pass_turn();
    ring.next();
    for (int b = b0; b < x.blocks && ok; b += step) {
      const int keys = w.keys(x), vs = ring.stage;
      const bool more = b + step < x.blocks;
      if (b == b0 && !(ok = wait(kBOFree + tile, (mine & 1) ^ 1))) break;
      if (!(ok = wait(kBFull + vs, ring.phase))) break;
      if (keys & 15) {
        if (!(ok = wait(kBFixed + vs, (fixed_phase >> vs) & 1))) break;
        fixed_phase ^= 1u << vs;
      }
      ring.next();
      w.next(x);
      auto issue_pv = [&]() {
        const uint64_t vd = v_desc + static_cast<uint32_t>(vs * (32768 >> 4));
        const int steps = (keys + 15) >> 4;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (kk < steps)
            train::umma_bf16_ts(o_col, s_col + kk * 8, vd + kk * (2048 >> 4), instr_desc_n(1, 128),
                                (b > b0 || kk > 0) ? 1u : 0u);
      };
      if (x.dual) {
        // Two chains over one ring: PV(b) releases its stage as soon as P is there; waiting
        // for K(b + 2) first would leave every load in the ring behind the next one.
        if (!(ok = wait(kBPFull + tile, p_phase))) break;
        p_phase ^= 1;
        train::tc_fence_after();
        if (leader) {
          issue_pv();
          train::umma_commit(bar(kBEmpty + vs));
          if (!more) train::umma_commit(bar(kBODone + tile));
        }
        __syncwarp();
        if (b + 1 < x.blocks) skip_block();
        if (!ok) break;
        if (more) {
          if (!(ok = wait(kBFull + ring.stage, ring.phase))) break;
          if (leader) {
            issue_qk(ring.stage, w.keys(x));
            train::umma_commit(bar(kBSFull + tile));
            train::umma_commit(bar(kBEmpty + ring.stage));
            if (b + 2 * step >= x.blocks) train::umma_commit(bar(kBQEmpty));
          }
          __syncwarp();
          ring.next();
        }
        continue;
      }
      // every wait comes before the first MMA, every commit behind the last: PV(b) and
      // QK(b + 1) run back to back on the pipe
      if (more && !(ok = wait(kBFull + ring.stage, ring.phase))) break;
      if (!(ok = take_turn())) break;
      if (!(ok = wait(kBPFull + tile, p_phase))) break;
      p_phase ^= 1;
      train::tc_fence_after();
      if (leader) {
        issue_pv();
        if (more) {
          issue_qk(ring.stage, w.keys(x));
          train::umma_commit(bar(kBSFull + tile));
          train::umma_commit(bar(kBEmpty + ring.stage));
          if (b + 2 == x.blocks) train::umma_commit(bar(kBQEmpty));
        } else {
          train::umma_commit(bar(kBODone + tile));
        }
        train::umma_commit(bar(kBEmpty + vs));
      }
      __syncwarp();
      if (more) ring.next();
      pass_turn();
    }
    ++it;
    ++mine;
  }
  if (!ok) *abort_flag = 1;
  // Every MMA issued above completes before TMEM is released.
  if (leader) train::umma_commit(bar(kBDrain));
  __syncwarp();
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

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct RowState {
  float m, l;                             // running maximum (log2 units), sum of 2^(s - m)
};
constexpr float kNoMax = -3.402823466e38f;   // m before a visible key: below every score

// O *= alpha for the warp's rows, 16 columns at a time (the rows' scores are live in registers).
__device__ __forceinline__ void rescale_o(uint32_t o_addr, float alpha) {
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    uint32_t o[16];
    tmem_ld16(o_addr + 16 * c, o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st16(o_addr + 16 * c, o);
  }
  tmem_st_wait();
}

// 2^(s scale - m) is one fma and one ex2, exact in its argument; m is the rounded product, so
// the largest score's argument is that rounding error, up to |m| 2^-24. From |m| = 2^24 on it
// would count (at 2^31 it overflows ex2): there far_block computes the probabilities, product
// and difference rounded one by one, as m was, so that the largest argument is 0. Few rows
// ever come there: 16 scores at a time, read from TMEM again (P takes the columns of scores
// already read), so that the usual path carries no code or registers for it.
__device__ __forceinline__ bool is_far(float m) {            // 2^24 <= |m| < 2^127: not kNoMax, not infinite
  constexpr uint32_t kLow = 0x4b800000u, kHigh = 0x7f000000u;
  return (__float_as_uint(m) & 0x7fffffffu) - kLow < kHigh - kLow;
}
__device__ __noinline__ float far_block(uint32_t s_addr, uint32_t o_addr, int cols, int see, float scale_log2,
                                        bool rescale, float alpha, float m) {
  if (rescale) rescale_o(o_addr, alpha);
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < cols; c += 16) {
    uint32_t v[16], pk[8];
    tmem_ld16(s_addr + c, v);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float a = c + i < see ? ex2(__fsub_rn(__fmul_rn(__uint_as_float(v[i]), scale_log2), m)) : 0.f;
      const float b = c + i + 1 < see ? ex2(__fsub_rn(__fmul_rn(__uint_as_float(v[i + 1]), scale_log2), m)) : 0.f;
      sum += a + b;
      pk[i >> 1] = pack_bf16x2(a, b);
    }
    tmem_st8(s_addr + (c >> 1), pk);
  }
  tmem_st_wait();
  return sum;
}

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
  const float m_new = fmaxf(st.m, __fmul_rn(max_n(s), scale_log2));
  const bool raise = m_new > st.m + 8.f;
  float alpha = 1.f;
  if (raise) {
    alpha = ex2(st.m - m_new);
    st.m = m_new;
  }
  if (__any_sync(0xffffffffu, is_far(st.m))) {
    st.l = st.l * alpha + far_block(s_addr, o_addr, kCols, see, scale_log2, !first, alpha, st.m);
    return;
  }
  // the block's S was committed behind the previous PV: O is complete
  if (!first && __any_sync(0xffffffffu, raise)) rescale_o(o_addr, alpha);
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < kCols / 32; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float a = ex2(fmaf(s[32 * c + 2 * i], scale_log2, -st.m));
      const float b = ex2(fmaf(s[32 * c + 2 * i + 1], scale_log2, -st.m));
      sum[i & 1] += a + b;
      pk[i] = pack_bf16x2(a, b);
    }
    tmem_st16(s_addr + 16 * c, pk);
  }
  tmem_st_wait();
  st.l = st.l * alpha + (sum[0] + sum[1]);
}

__device__ __forceinline__ void softmax_role(const Params& p, float* part, int first, int last, uint32_t bars,
                                             uint32_t tmem, volatile int* abort_flag) {
  auto bar = [&](int i) { return bars + 8u * i; };
  const int tile = threadIdx.x >> 7;
  const int m = threadIdx.x & 127;                          // row of the tile == TMEM lane
  const uint32_t lanes = static_cast<uint32_t>(m & ~31) << 16;
  const uint32_t s_addr = tmem + lanes + kTmemS + tile * 128, o_addr = tmem + lanes + kTmemO + tile * 128;
  uint32_t s_phase = 0, o_phase = 0;
  bool ok = true;
  ItemView nx;                                              // the next item, loaded a step ahead
  bool nx_ok = first < last && load_item(p, first, nx);
#pragma unroll 1
  for (int idx = first; idx < last; ++idx) {
    // what the block loop keeps of the item; its keys are consecutive chain positions
    const bool valid = nx_ok, dual = nx.dual;
    const int nq = nx.nq, blocks = nx.blocks;
    const int rm = dual && tile == 1 ? (m + dual_shift(nq)) & 127 : m;     // row of the MMA tile's rows
    const int lt = (dual ? 0 : tile * kHalfTile) + (rm >> 1);  // query row of the item
    const bool active = valid && (tile == 0 || dual || nq > kHalfTile);
    const bool row_ok = lt < nq, warp_ok = lt - ((rm & 31) >> 1) < nq;
    int len0 = nx.len[0], len1 = nx.len[1], len2 = nx.len[2];
    int see0 = row_ok ? nx.visible + lt - nx.pos[0] : 0;
    if (!valid && threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    RowState st{kNoMax, 0.f};
    if (active) {
      const int b0 = dual ? tile : 0;
#pragma unroll 1
      for (int b = 0; b < blocks; ++b) {
        const int keys = min(kBlock, len0);
        if (!dual || (b & 1) == tile) {
          ok = train::wait_or_abort(bar(kBSFull + tile), s_phase, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          s_phase ^= 1;
          if (warp_ok) {
            train::tc_fence_after();
            if (keys > 32)
              softmax_block<128>(s_addr, o_addr, min(keys, see0), p.scale_log2, b == b0, st);
            else
              softmax_block<32>(s_addr, o_addr, min(keys, see0), p.scale_log2, b == b0, st);
            train::tc_fence_before();
          }
          __syncwarp();
          if ((threadIdx.x & 31) == 0) mbar_arrive(bar(kBPFull + tile));
        }
        see0 -= keys;
        len0 -= keys;
        if (len0 == 0) {
          len0 = len1;
          len1 = len2;
          len2 = 0;
        }
      }
      if (!ok) break;
    }
    const int4 where = __ldg(reinterpret_cast<const int4*>(p.plan + p.items_at + static_cast<size_t>(idx) * kItemWords));
    const int q0 = where.x, head = where.z, slot = where.w;    // (their registers were the scores')
    nx_ok = idx + 1 < last && load_item(p, idx + 1, nx);
    if (!active) continue;
    if (blocks > 0) {
      ok = train::wait_or_abort(bar(kBODone + tile), o_phase, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      o_phase ^= 1;
      train::tc_fence_after();
    }
    const float inv = st.l > 0.f ? 1.f / st.l : (st.l != st.l ? st.l : 0.f);   // (a NaN sum stays NaN)
    const int pitch = part_pitch(nq);
    float* prow = part;
    if (slot >= 0)
      prow += part_at(__ldg(p.plan + p.items_at + static_cast<size_t>(idx) * kItemWords + kIPart) + tile * pitch);
    __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.out) +
                          (static_cast<size_t>(q0 + (row_ok ? lt : 0)) * kQHeads + 2 * head + (rm & 1)) * kHeadDim;
    if (warp_ok) {
      // (small code: a launch meets it cold, and unrolled over the row the first epilogue took
      // 5,000 cycles of instruction fetches)
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float o[32];
        float* prow_c = prow + 4 * (8 * c * pitch + rm);
        train::tmem_ld32(o_addr + 32 * c, o);
        // (without a visible key O was never written, or holds products of zeros)
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = inv != 0.f ? o[i] * inv : 0.f;
        if (row_ok && slot < 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(orow + 32 * c + 8 * j) =
                make_uint4(pack_bf16x2(o[8 * j], o[8 * j + 1]), pack_bf16x2(o[8 * j + 2], o[8 * j + 3]),
                           pack_bf16x2(o[8 * j + 4], o[8 * j + 5]), pack_bf16x2(o[8 * j + 6], o[8 * j + 7]));
        } else if (row_ok) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(reinterpret_cast<float4*>(prow_c + 4 * j * pitch),
                   make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]));
        }
      }
      if (row_ok && slot >= 0)
        __stcg(reinterpret_cast<float2*>(prow + kHeadDim * pitch) + rm, make_float2(st.m, st.l));
    }
    if (blocks > 0) {
      train::tc_fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(bar(kBOFree + tile));
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
  const int warp = threadIdx.x >> 5;
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
      if ((i >= kBPFull && i < kBPFull + 2) || (i >= kBOFree && i < kBOFree + 2)) count = 4;   // softmax warps
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
  // 384 threads are launched with 168 registers each (64,512). A softmax thread holds a row
  // of 128 scores: its warpgroups grow to 200 each out of what the third one gives back
  // (2 x 128 x 200 + 128 x 96 = 63,488); without this the row spills to local memory (444
  // instead of 724 us at 1024 query rows x 32768 shared keys with 512 own keys a request).
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  }
  if (warp < 8) {
    softmax_role(p, part, first, last, bars, tmem, abort_flag);
  } else if (warp < 10) {
    issue_role(p, warp - 8, first, last, sbase, bars, tmem, abort_flag);
  } else if (warp == 10) {
    producer_role(p, maps, first, last, sbase, bars, abort_flag);
  } else {
    fix_role(p, first, last, smem, bars, abort_flag);
  }
  train::tc_fence_before();
  __syncthreads();
  train::tc_fence_after();
  if (warp == 8) train::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// fp32 kernel (CUDA cores) over the same plan: products, softmax and sums in fp32.
//
// CTA (item, 32 query rows of it): 64 rows of S, 32 keys at a time in shared memory. A
// thread owns kRpt rows and one sixteenth of the keys, then of d; the 16 lanes that share
// its rows reduce the maximum and the sum by shuffles and pass P through shared memory
// inside their warp. The FMA rate bounds it; items of at most 8 query rows take kRpt = 1 (16
// rows) instead of multiplying 48 empty ones. A dual item's keys all go to its first slot.
constexpr int kF32Threads2 = 256, kF32Keys2 = 32, kF32Sub = 32;
constexpr int kF32Pitch = kHeadDim + 4;
constexpr size_t kF32SmemBytes = (64 * kF32Pitch + kF32Keys2 * kF32Pitch + kF32Keys2 * kHeadDim + 64 * 33) * sizeof(float);

template <int kRpt>
__device__ __forceinline__ void f32_item(const Params& p, const ItemView& x, int sub, float* smem, float* part) {
  float* sq = smem;
  float* sk = sq + 64 * kF32Pitch;
  float* sv = sk + kF32Keys2 * kF32Pitch;
  float* sp = sv + kF32Keys2 * kHeadDim;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int rows = 2 * min(kF32Sub, x.nq - sub);           // rows of S: 2 * query row + head
  const float* qg = static_cast<const float*>(p.q);
  for (int u = tid; u < 16 * kRpt * (kHeadDim / 4); u += kF32Threads2) {
    const int m = u >> 5, d = (u & 31) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m < rows)
      v = *reinterpret_cast<const float4*>(
          qg + (static_cast<size_t>(x.q0 + sub + (m >> 1)) * kQHeads + 2 * x.head + (m & 1)) * kHeadDim + d);
    *reinterpret_cast<float4*>(sq + m * kF32Pitch + d) = v;
  }
  float mrow[kRpt], lrow[kRpt], acc[kRpt][8];
#pragma unroll
  for (int i = 0; i < kRpt; ++i) {
    mrow[i] = -INFINITY;
    lrow[i] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[i][d] = 0.f;
  }
#pragma unroll 1
  for (int s = 0; s < x.nsegs; ++s) {
    const Source& src = p.src[x.src[s]];
    const float* kg = static_cast<const float*>(src.k);
    const float* vg = static_cast<const float*>(src.v);
    const long long row0 = src.off + x.row[s];
#pragma unroll 1
    for (int k0 = 0; k0 < x.len[s]; k0 += kF32Keys2) {
      const int keys = min(kF32Keys2, x.len[s] - k0);
      __syncthreads();
      for (int u = tid; u < kF32Keys2 * (kHeadDim / 4); u += kF32Threads2) {
        const int n = u >> 5, d = (u & 31) * 4;
        float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
        if (n < keys) {
          const size_t off = (static_cast<size_t>(row0 + k0 + n) * kKVHeads + x.head) * kHeadDim + d;
          kv = __ldg(reinterpret_cast<const float4*>(kg + off));
          vv = __ldg(reinterpret_cast<const float4*>(vg + off));
        }
        *reinterpret_cast<float4*>(sk + n * kF32Pitch + d) = kv;
        *reinterpret_cast<float4*>(sv + n * kHeadDim + d) = vv;
      }
      __syncthreads();
      float dot[kRpt][2] = {};
#pragma unroll 4
      for (int d = 0; d < kHeadDim; d += 4) {
        const float4 ka = *reinterpret_cast<const float4*>(sk + tx * kF32Pitch + d);
        const float4 kb = *reinterpret_cast<const float4*>(sk + (tx + 16) * kF32Pitch + d);
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
          const float4 q = *reinterpret_cast<const float4*>(sq + (ty * kRpt + i) * kF32Pitch + d);
          dot[i][0] = fmaf(q.x, ka.x, fmaf(q.y, ka.y, fmaf(q.z, ka.z, fmaf(q.w, ka.w, dot[i][0]))));
          dot[i][1] = fmaf(q.x, kb.x, fmaf(q.y, kb.y, fmaf(q.z, kb.z, fmaf(q.w, kb.w, dot[i][1]))));
        }
      }
#pragma unroll
      for (int i = 0; i < kRpt; ++i) {
        const int m = ty * kRpt + i;
        const int see = min(keys, x.visible + sub + (m >> 1) - (x.pos[s] + k0));
        const float a = tx < see ? dot[i][0] * p.scale : -INFINITY, b = tx + 16 < see ? dot[i][1] * p.scale : -INFINITY;
        float mx = fmaxf(a, b);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(mrow[i], mx), mu = mn == -INFINITY ? 0.f : mn;
        const float alpha = expf(mrow[i] - mu), ea = expf(a - mu), eb = expf(b - mu);
        float ps = ea + eb;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
        lrow[i] = lrow[i] * alpha + ps;
        mrow[i] = mn;
        sp[m * 33 + tx] = ea;
        sp[m * 33 + tx + 16] = eb;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[i][d] *= alpha;
      }
      __syncwarp();
#pragma unroll 4
      for (int n = 0; n < kF32Keys2; ++n) {
        const float4 va = *reinterpret_cast<const float4*>(sv + n * kHeadDim + 4 * tx);
        const float4 vb = *reinterpret_cast<const float4*>(sv + n * kHeadDim + 64 + 4 * tx);
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
          const float e = sp[(ty * kRpt + i) * 33 + n];
          acc[i][0] = fmaf(e, va.x, acc[i][0]);
          acc[i][1] = fmaf(e, va.y, acc[i][1]);
          acc[i][2] = fmaf(e, va.z, acc[i][2]);
          acc[i][3] = fmaf(e, va.w, acc[i][3]);
          acc[i][4] = fmaf(e, vb.x, acc[i][4]);
          acc[i][5] = fmaf(e, vb.y, acc[i][5]);
          acc[i][6] = fmaf(e, vb.z, acc[i][6]);
          acc[i][7] = fmaf(e, vb.w, acc[i][7]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kRpt; ++i) {
    const int m = ty * kRpt + i;
    if (m >= rows) continue;
    const int lt = sub + (m >> 1);
    const bool any = lrow[i] > 0.f || lrow[i] != lrow[i];   // (a NaN sum stays NaN)
    const float inv = any ? 1.f / lrow[i] : 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[i][d] = any ? acc[i][d] * inv : 0.f;
    const float4 a = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    const float4 b = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
    if (x.slot < 0) {
      float* dst = static_cast<float*>(p.out) +
                   (static_cast<size_t>(x.q0 + lt) * kQHeads + 2 * x.head + (m & 1)) * kHeadDim;
      *reinterpret_cast<float4*>(dst + 4 * tx) = a;
      *reinterpret_cast<float4*>(dst + 64 + 4 * tx) = b;
    } else {
      const int rm = 2 * (lt & 63) + (m & 1), pitch = part_pitch(x.nq);
      float* prow = part + part_at(x.part + (x.dual ? 0 : lt >> 6) * pitch);
      *reinterpret_cast<float4*>(prow + 4 * (tx * pitch + rm)) = a;
      *reinterpret_cast<float4*>(prow + 4 * ((16 + tx) * pitch + rm)) = b;
      if (tx == 0) reinterpret_cast<float2*>(prow + kHeadDim * pitch)[rm] = make_float2(mrow[i], lrow[i]);
      if (x.dual) {                              // the second slot holds nothing
        float* empty = prow + part_at(pitch);
        *reinterpret_cast<float4*>(empty + 4 * (tx * pitch + rm)) = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(empty + 4 * ((16 + tx) * pitch + rm)) = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tx == 0) reinterpret_cast<float2*>(empty + kHeadDim * pitch)[rm] = make_float2(-INFINITY, 0.f);
      }
    }
  }
}

__global__ void __launch_bounds__(kF32Threads2) prefix_f32_kernel(const Params p, float* part) {
  extern __shared__ float f32_smem[];
  if (!plan_ok(p)) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  ItemView x;
  const bool ok = static_cast<int>(blockIdx.x) < p.plan[kHItems] && load_item(p, blockIdx.x, x);
  const int sub = blockIdx.y * kF32Sub;
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  if (sub >= x.nq) return;
  if (x.nq - sub <= 8)
    f32_item<1>(p, x, sub, f32_smem, part);
  else
    f32_item<4>(p, x, sub, f32_smem, part);
}

// Combines the partial rows of a query row's head pair (adjacent rows of a slot, so a lane
// reads whole 32-byte sectors); lane l owns d = 4 l ..
//   out = sum_c w_c o_c / sum_c w_c,  w_c = l_c 2^(m_c - M),  M = max_c m_c
// (m of the float32 kernel in natural units)
// kWarps = 1: a warp per (query row, KV head), 8 to a CTA. kWarps = 8: a CTA per pair, its
// warps taking every eighth contribution, for few rows, whose warps alone would not fill the
// GPU (CTA against warp a pair, whole call: 4 rows of 32 parts 27 / 35 us, of 7 parts 16.5 /
// 18.6; 32 rows of 38 parts 41 / 49, of 4 parts 24.1 / 24.7; 64 rows equal; 96 rows of 3
// parts 51.4 / 49.8, 256 rows 121 / 115).
constexpr int kMergeWidePairs = 64 * kHeads;

template <typename T, int kWarps>
__global__ void __launch_bounds__(256, 4) prefix_merge_kernel(const Params p, const float* part) {
  __shared__ float s_acc[kWarps > 1 ? 8 : 1][8][33];
  __shared__ float2 s_den[8];
  if (!plan_ok(p)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long u = kWarps > 1 ? static_cast<long long>(blockIdx.x) : static_cast<long long>(blockIdx.x) * 8 + warp;
  if (u >= static_cast<long long>(p.total_q) * kHeads) return;
  const int t = static_cast<int>(u / kHeads), h = static_cast<int>(u % kHeads);
  const int run = p.plan[p.token_run_at + t];
  if (run < 0 || run >= p.runs) return;
  const int* w = p.plan + p.runs_at + static_cast<size_t>(run) * kRunWords;
  const int4 k0 = *reinterpret_cast<const int4*>(w + kRunTile0);
  const int4 k1 = *reinterpret_cast<const int4*>(w + kRunTile0 + kRunTileWords);
  const int4 at = *reinterpret_cast<const int4*>(p.plan + p.parts_at + static_cast<size_t>(run) * kPartWords);
  // (a dual tile's pieces are two contributions each, in consecutive slots)
  const bool d0 = k0.z == kDualSlots, d1 = k1.z == kDualSlots;
  const int n0 = k0.y << d0, total = n0 + (w[kRunTiles] > 1 ? k1.y << d1 : 0);
  const int lt0 = t - k0.w, lt1 = t - k1.w;
  auto base = [&](int c) -> const float* {
    const bool first = c < n0;
    const bool dual = first ? d0 : d1;
    const int4 k = first ? k0 : k1;
    const int i = first ? c : c - n0, lt = first ? lt0 : lt1;
    const int slot = dual ? ((i >> 1) * kHeads + h) * 2 + (i & 1) : (i * kHeads + h) * k.z + (lt >> 6);
    const int pitch = first ? at.y : at.w, row = (first ? at.x : at.z) + slot * pitch;
    return part + part_at(min(max(row, 0), p.part_rows - pitch));
  };
  auto pitch_of = [&](int c) { return c < n0 ? at.y : at.w; };
  auto row_of = [&](int c) { return 2 * ((c < n0 ? lt0 : lt1) & 63); };
  // (m, l) of the two heads' rows
  auto stats = [&](int c) { return __ldcg(reinterpret_cast<const float4*>(base(c) + kHeadDim * pitch_of(c) + 2 * row_of(c))); };
  constexpr float kUnit = sizeof(T) == 4 ? 1.4426950408889634f : 1.f;
  float2 top = make_float2(-INFINITY, -INFINITY);
  for (int c = lane; c < total; c += 32) {
    const float4 v = stats(c);
    top.x = fmaxf(top.x, v.x);
    top.y = fmaxf(top.y, v.z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top.x = fmaxf(top.x, __shfl_xor_sync(0xffffffffu, top.x, o));
    top.y = fmaxf(top.y, __shfl_xor_sync(0xffffffffu, top.y, o));
  }
  // a row whose contributions all see nothing: weights 0
  const float mx = top.x > -INFINITY ? top.x : 0.f, my = top.y > -INFINITY ? top.y : 0.f;
  float a[8] = {}, den0 = 0.f, den1 = 0.f;
  const int c_first = kWarps > 1 ? warp : 0;
#pragma unroll 4
  for (int c = c_first; c < total; c += kWarps) {
    const float4 f = stats(c);
    const float4* src = reinterpret_cast<const float4*>(base(c) + 4 * (lane * pitch_of(c) + row_of(c)));
    const float4 v0 = __ldcg(src), v1 = __ldcg(src + 1);
    const float f0 = ex2((f.x - mx) * kUnit) * f.y, f1 = ex2((f.z - my) * kUnit) * f.w;
    den0 += f0;
    den1 += f1;
    a[0] = fmaf(f0, v0.x, a[0]);
    a[1] = fmaf(f0, v0.y, a[1]);
    a[2] = fmaf(f0, v0.z, a[2]);
    a[3] = fmaf(f0, v0.w, a[3]);
    a[4] = fmaf(f1, v1.x, a[4]);
    a[5] = fmaf(f1, v1.y, a[5]);
    a[6] = fmaf(f1, v1.z, a[6]);
    a[7] = fmaf(f1, v1.w, a[7]);
  }
  if (kWarps > 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_acc[warp][i][lane] = a[i];
    if (lane == 0) s_den[warp] = make_float2(den0, den1);
    __syncthreads();
    if (warp != 0) return;
    for (int o = 1; o < 8; ++o) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += s_acc[o][i][lane];
      den0 += s_den[o].x;
      den1 += s_den[o].y;
    }
  }
  auto inverse = [](float d) { return d > 0.f ? 1.f / d : (d != d ? d : 0.f); };
  const float i0 = inverse(den0), i1 = inverse(den1);
  T* dst = static_cast<T*>(p.out) + (static_cast<size_t>(t) * kQHeads + 2 * h) * kHeadDim + 4 * lane;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(a[0] * i0, a[1] * i0, a[2] * i0, a[3] * i0);
    *reinterpret_cast<float4*>(dst + kHeadDim) = make_float4(a[4] * i1, a[5] * i1, a[6] * i1, a[7] * i1);
  } else {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(a[0] * i0, a[1] * i0), pack_bf16x2(a[2] * i0, a[3] * i0));
    *reinterpret_cast<uint2*>(dst + kHeadDim) =
        make_uint2(pack_bf16x2(a[4] * i1, a[5] * i1), pack_bf16x2(a[6] * i1, a[7] * i1));
  }
}

}  // namespace prefix
}  // namespace dspark
