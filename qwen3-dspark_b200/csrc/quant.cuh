// Paged KV cache in 8 bits: the exact float32 attention over it, the quantising append and
// the page copies (16 query heads, 8 KV heads, head dim 128; pages of 64 tokens). The bf16
// tensor-core attention is in quant_attn.cuh.
//
// A page of one layer holds, per KV head, 64 x 128 codes of K and of V (int8 or e4m3) with one
// float32 scale each: value = scale * code. Codes lie in the order in which the tensor-core
// kernel reads them with 16-byte loads, 8 KB a (page, head):
//   K [half of the head dim][token][64]: the 16 bytes of a thread are one token's dims,
//     and the 4 KB of a half is one contiguous copy;
//   V [dim][token]: the 16 bytes are 16 consecutive keys of one dim, which is what the second
//     product contracts over, so no transposition is left for the attention.
// A request of n tokens owns the n / 64 pages of its page table row; its last n % 64 tokens
// wait unquantised in block (n / 64) & 1 of its slot's two tail blocks [2][64][8][128]. Blocks
// alternate, so an append that fills one writes the rows behind it into the other.
#pragma once
#include "attention.cuh"

namespace dspark {
namespace quant {

constexpr int kPage = 64;                                   // tokens of a page
constexpr int kHeadBytes = kPage * kHeadDim;                // codes of one (page, head): K or V
constexpr size_t kPageBytes = static_cast<size_t>(kKVHeads) * kHeadBytes;
constexpr int kRowElems = kKVHeads * kHeadDim;              // elements of a token's K (or V) row
enum Code : int { kInt8 = 0, kE4M3 = 1 };

template <int kCode>
__device__ __forceinline__ float code_max() { return kCode == kInt8 ? 127.f : 448.f; }

// One layer's cache, and the metadata of a batch.
struct Cache {
  uint8_t* key;              // [pages][8][2][64][64]
  uint8_t* value;            // [pages][8][128][64]
  float* key_scale;          // [pages][8]
  float* value_scale;
  void* tail_key;            // [slots][2][64][8][128], the rows' type
  void* tail_value;
  int pages, slots;
};
struct Batch {
  const int* cu_q;           // [R + 1] rows of the new tokens
  const int* ctx;            // [R] tokens in the cache
  const int* table;          // [R][width] page ids
  const int* slot;           // [R] tail slots
  int requests, rows, width;
};

// One request of a batch; ok is false (and nothing else is used) where its metadata does not
// fit the cache or the rows.
struct Request {
  int q0, q_len, ctx, slot;
  const int* table;
  bool ok;
};
__device__ __forceinline__ Request load_request(const Batch& b, const Cache& c, int i) {
  Request r;
  r.q0 = b.cu_q[i];
  r.q_len = b.cu_q[i + 1] - r.q0;
  r.ctx = b.ctx[i];
  r.slot = b.slot[i];
  r.table = b.table + static_cast<size_t>(i) * b.width;
  r.ok = r.q0 >= 0 && r.q_len >= 0 && r.q0 <= b.rows - r.q_len && r.ctx >= 0 && r.ctx / kPage <= b.width &&
         r.slot >= 0 && r.slot < c.slots;
  return r;
}
__device__ __forceinline__ size_t tail_row(int slot, int token) {
  return (static_cast<size_t>(slot) * 2 + ((token / kPage) & 1)) * kPage + (token & (kPage - 1));
}

// Four e4m3 codes of a word as two pairs of halves; every e4m3 value is a half.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 p, q;\n\tmov.b32 {p, q}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, p;\n\tcvt.rn.f16x2.e4m3x2 %1, q;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
template <int kCode>
__device__ __forceinline__ float2 decode2(uint32_t two) {
  if (kCode == kInt8)
    return make_float2(static_cast<float>(static_cast<int8_t>(two & 0xff)),
                       static_cast<float>(static_cast<int8_t>((two >> 8) & 0xff)));
  uint32_t h, unused;
  e4m3x4_to_f16x4(two, h, unused);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ---------------------------------------------------------------------------
// Float32 attention on the CUDA cores: one CTA per (request, 8 query rows, KV head), a warp
// per (row, query head). 64 keys at a time are decoded into shared memory; lane l scores keys
// l and l + 32 and then holds dims 4 l .. 4 l + 3 of the output.
constexpr int kF32AttnThreads = 16 * 32;
constexpr int kF32KPitch = kHeadDim + 4;                    // float4 reads of 8 rows hit distinct banks
constexpr size_t kF32AttnSmem = sizeof(float) * (kPage * kF32KPitch + kPage * kHeadDim + 16 * kHeadDim);

struct F32Params {
  const float* q;            // [rows, 16, 128]
  const float* new_k;        // [rows, 8, 128]
  const float* new_v;
  float* out;
  Cache cache;
  Batch batch;
  float scale;
};

template <int kCode>
__global__ void __launch_bounds__(kF32AttnThreads) f32_attn_kernel(const F32Params p) {
  extern __shared__ float4 smem4[];
  float* sk = reinterpret_cast<float*>(smem4);
  float* sv = sk + kPage * kF32KPitch;
  float* sq = sv + kPage * kHeadDim;
  const int h = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Request req = load_request(p.batch, p.cache, blockIdx.x);
  const int r0 = blockIdx.y * kQBlock;
  if (!req.ok) {
    if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  if (r0 >= req.q_len) return;
  const int row = r0 + (warp & 7), head = 2 * h + (warp >> 3);
  const bool live = row < req.q_len;
  const size_t q_at = (static_cast<size_t>(req.q0 + (live ? row : r0)) * kQHeads + head) * kHeadDim;
  *reinterpret_cast<float4*>(sq + warp * kHeadDim + 4 * lane) = *reinterpret_cast<const float4*>(p.q + q_at + 4 * lane);
  const int full = req.ctx / kPage, tail = req.ctx % kPage;
  const int visible = tail + min(r0 + kQBlock, req.q_len);   // unquantised keys that a row of this CTA sees
  const float* tk = static_cast<const float*>(p.cache.tail_key) + tail_row(req.slot, req.ctx - tail) * kRowElems + h * kHeadDim;
  const float* tv = static_cast<const float*>(p.cache.tail_value) + tail_row(req.slot, req.ctx - tail) * kRowElems + h * kHeadDim;
  const float* nk = p.new_k + static_cast<size_t>(req.q0) * kRowElems + h * kHeadDim;
  const float* nv = p.new_v + static_cast<size_t>(req.q0) * kRowElems + h * kHeadDim;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < full + (visible + kPage - 1) / kPage; ++step) {
    float ks = 1.f, vs = 1.f;
    int keys = kPage, limit = kPage;                          // keys loaded; keys that this warp's row sees
    __syncthreads();
    if (step < full) {
      const int id = req.table[step];
      if (id < 0 || id >= p.cache.pages) {                    // (uniform over the CTA)
        if (tid == 0) atomicOr(&g_device_status, kStatusBadArgument);
        continue;
      }
      const size_t at = static_cast<size_t>(id) * kKVHeads + h;
      ks = p.cache.key_scale[at];
      vs = p.cache.value_scale[at];
      const uint4 kc = reinterpret_cast<const uint4*>(p.cache.key + at * kHeadBytes)[tid];
      const uint4 vc = reinterpret_cast<const uint4*>(p.cache.value + at * kHeadBytes)[tid];
      const uint32_t kw[4] = {kc.x, kc.y, kc.z, kc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
      float* kd = sk + ((tid & 255) >> 2) * kF32KPitch + (tid >> 8) * 64 + (tid & 3) * 16;
      float* vd = sv + (tid & 3) * 16 * kHeadDim + (tid >> 2);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 a = decode2<kCode>(kw[w]), b = decode2<kCode>(kw[w] >> 16);
        *reinterpret_cast<float4*>(kd + 4 * w) = make_float4(a.x, a.y, b.x, b.y);
        const float2 c = decode2<kCode>(vw[w]), d = decode2<kCode>(vw[w] >> 16);
        vd[(4 * w + 0) * kHeadDim] = c.x;
        vd[(4 * w + 1) * kHeadDim] = c.y;
        vd[(4 * w + 2) * kHeadDim] = d.x;
        vd[(4 * w + 3) * kHeadDim] = d.y;
      }
    } else {
      const int t0 = (step - full) * kPage;
      keys = min(kPage, visible - t0);
      limit = min(keys, tail + row + 1 - t0);
      for (int u = tid; u < keys * 32; u += kF32AttnThreads) {
        const int t = t0 + (u >> 5), d = 4 * (u & 31);
        const size_t at = static_cast<size_t>(t < tail ? t : t - tail) * kRowElems + d;
        *reinterpret_cast<float4*>(sk + (u >> 5) * kF32KPitch + d) = *reinterpret_cast<const float4*>((t < tail ? tk : nk) + at);
        *reinterpret_cast<float4*>(sv + (u >> 5) * kHeadDim + d) = *reinterpret_cast<const float4*>((t < tail ? tv : nv) + at);
      }
    }
    __syncthreads();
    float s[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = lane + 32 * e;
      float dot = 0.f;
      if (j < limit) {
        const float4* kr = reinterpret_cast<const float4*>(sk + j * kF32KPitch);
        const float4* qr = reinterpret_cast<const float4*>(sq + warp * kHeadDim);
#pragma unroll 8
        for (int d = 0; d < 32; ++d) {
          const float4 a = qr[d], b = kr[d];
          dot = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, dot))));
        }
      }
      s[e] = j < limit ? dot * (ks * p.scale) : -INFINITY;
    }
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn, alpha = expf(m - mu);
    const float e0 = expf(s[0] - mu), e1 = expf(s[1] - mu);
    float sum = e0 + e1;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * alpha + sum;
    m = mn;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < limit; ++j) {                         // (keys that the row does not see are not touched)
      const float w = __shfl_sync(0xffffffffu, j < 32 ? e0 : e1, j & 31);
      const float4 v = *reinterpret_cast<const float4*>(sv + j * kHeadDim + 4 * lane);
      a[0] = fmaf(w, v.x, a[0]);
      a[1] = fmaf(w, v.y, a[1]);
      a[2] = fmaf(w, v.z, a[2]);
      a[3] = fmaf(w, v.w, a[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(a[i], vs, o[i] * alpha);
  }
  if (live)
    *reinterpret_cast<float4*>(p.out + q_at + 4 * lane) = make_float4(o[0] / l, o[1] / l, o[2] / l, o[3] / l);
}

// ---------------------------------------------------------------------------
// Append: the first n_i new rows of request i follow its ctx_i tokens, in all layers in one
// launch. A block of 64 rows that gets full is quantised per KV head with a = max |x|:
//   scale = a / qmax,   code = round(x qmax / a)  (to nearest, ties to even)
// and the rows of the block that stays open are copied to the tail. A zero block has scale
// and codes 0; a block with an infinity or NaN gets that scale, which makes all of its values NaN.
//
// The quotient: q = x * fl(qmax / a) is off by 2^-23 of itself at most, and for bf16 x and a the
// true quotient is either exactly between two codes or at least 2^-16 of itself away from there
// (127 X / A with 8-bit X against an odd multiple of 1/2: the difference is a multiple of
// 1 / (2 A), A <= 127 X / q; e4m3's midpoints have 5 bits and stay further away). Rounding q to
// 20 bits therefore gives the exact tie where there is one and moves nothing across one. Float32
// rows, of which that does not hold, divide in float64.
struct AppendParams {
  const void* new_k;         // [layers][new_rows][8][128]
  const void* new_v;
  long long new_rows;        // rows between the layers of new_k / new_v
  Cache cache;               // layer 0
  int layers, blocks;        // blocks: full blocks a request can get (grid x / requests)
  Batch batch;
  const int* counts;         // [R], or null: every new row
};

template <typename T>
struct Vec8;                 // 8 elements of a row
template <>
struct Vec8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = a; }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};

// Codes of one block and head. Small maxima are scaled up first, or qmax / a would overflow.
template <typename T, int kCode>
struct Quantizer {
  float a, pre, inv, scale;
  __device__ __forceinline__ explicit Quantizer(uint32_t max_bits) {
    a = __uint_as_float(max_bits);
    scale = __fdiv_rn(a, code_max<kCode>());
    pre = a < 0x1p-64f ? 0x1p64f : 1.f;
    a *= pre;
    inv = a > 0.f ? __fdiv_rn(code_max<kCode>(), a) : 0.f;
  }
  __device__ __forceinline__ float quotient(float x) const {
    if (sizeof(T) == 4) {
      const double q = static_cast<double>(x * pre) * static_cast<double>(code_max<kCode>()) / static_cast<double>(a);
      if (kCode == kInt8) return static_cast<float>(rint(q));
      // to odd, so that the second rounding (to e4m3) is the only one that counts
      float f = __double2float_rz(q);
      if (static_cast<double>(f) != q) f = __uint_as_float(__float_as_uint(f) | 1u);
      return f;
    }
    return __uint_as_float((__float_as_uint(x * pre * inv) + 8u) & ~15u);
  }
  // 4 codes in a word, x[0] lowest
  __device__ __forceinline__ uint32_t code4(float x0, float x1, float x2, float x3) const {
    if (!(a > 0.f)) return 0u;                                // a zero block; a NaN one, whose scale says so
    const float q[4] = {quotient(x0), quotient(x1), quotient(x2), quotient(x3)};
    if (kCode == kInt8) {
      uint32_t w = 0;                                         // rint by adding 1.5 * 2^23: the low byte is the code
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (__float_as_uint(__fadd_rn(q[i], 12582912.f)) & 0xffu) << (8 * i);
      return w;
    }
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 x;\n\tcvt.rn.satfinite.e4m3x2.f32 x, %2, %1;\n\tcvt.u32.u16 %0, x;\n\t}" : "=r"(lo) : "f"(q[0]), "f"(q[1]));
    asm("{\n\t.reg .b16 x;\n\tcvt.rn.satfinite.e4m3x2.f32 x, %2, %1;\n\tcvt.u32.u16 %0, x;\n\t}" : "=r"(hi) : "f"(q[2]), "f"(q[3]));
    return lo | (hi << 16);
  }
};

// Quantises K and V of one (block, head): rows base(t) for t = 0 .. 63. Thread (g, c) of the
// 256 takes rows 4 g .. 4 g + 3 (g = 2 warp + lane / 16) and dims 8 c .. 8 c + 7, so that a
// warp's loads are whole 256-byte rows and a thread holds four tokens of a dim, one word of V.
struct QuantSmem {
  uint32_t top[2][8];
  uint32_t v[kHeadDim * 16];                                  // [dim][token / 4], columns rotated by dim / 8
};
template <typename T, int kCode, typename RowOf>
__device__ __forceinline__ void quantize_block(const Cache& c, size_t page_head, const RowOf& row_of, QuantSmem& sm) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = 2 * warp + (lane >> 4), d0 = 8 * (lane & 15);
  Vec8<T> x[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T *k, *v;
    row_of(4 * g + i, k, v);
    x[0][i].load(k + d0);
    x[1][i].load(v + d0);
  }
  uint32_t top[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    top[s] = 0u;                                              // of the bits without the sign: a NaN is the largest
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[8];
      x[s][i].get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) top[s] = max(top[s], __float_as_uint(f[e]) & 0x7fffffffu);
    }
    top[s] = __reduce_max_sync(0xffffffffu, top[s]);
    if (lane == 0) sm.top[s][warp] = top[s];
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int w = 0; w < 8; ++w) top[s] = max(top[s], sm.top[s][w]);
  }
  const Quantizer<T, kCode> qk(top[0]), qv(top[1]);
  uint8_t* kd = c.key + page_head * kHeadBytes + (d0 >> 6) * (kPage * 64) + (d0 & 63);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[8];
    x[0][i].get(f);
    *reinterpret_cast<uint2*>(kd + (4 * g + i) * 64) =
        make_uint2(qk.code4(f[0], f[1], f[2], f[3]), qk.code4(f[4], f[5], f[6], f[7]));
  }
  float f[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[1][i].get(f[i]);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    sm.v[(d0 + e) * 16 + (g ^ (lane & 15))] = qv.code4(f[0][e], f[1][e], f[2][e], f[3][e]);
  __syncthreads();
  uint4* vd = reinterpret_cast<uint4*>(c.value + page_head * kHeadBytes);
#pragma unroll
  for (int u = tid; u < kHeadDim * 4; u += 256) {
    const int d = u >> 2, w = 4 * (u & 3);
    const uint32_t* s = sm.v + d * 16;
    const int rot = (d >> 3) & 15;
    vd[u] = make_uint4(s[w ^ rot], s[(w + 1) ^ rot], s[(w + 2) ^ rot], s[(w + 3) ^ rot]);
  }
  if (tid == 0) {
    c.key_scale[page_head] = qk.scale;
    c.value_scale[page_head] = qv.scale;
  }
  __syncthreads();                                            // sm is written again
}

// Grid (requests x blocks, layers, 8 / kHeads): CTA b of a request quantises its b-th block
// that gets full; the first one also copies the rows that stay open, behind the block that it
// reads (with 128 or more new rows both may lie in the same tail block).
template <typename T, int kCode, int kHeads>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  __shared__ QuantSmem sm;
  const int i = blockIdx.x / p.blocks, b = blockIdx.x % p.blocks, layer = blockIdx.y, h0 = blockIdx.z * kHeads;
  const Request r = load_request(p.batch, p.cache, i);
  const int n = p.counts != nullptr ? p.counts[i] : r.q_len;
  const int first = r.ctx / kPage, end = r.ok && n >= 0 ? (r.ctx + n) / kPage : 0;
  if (!r.ok || n < 0 || n > r.q_len || end > p.batch.width || end - first > p.blocks) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  if (n == 0 || (b > 0 && first + b >= end)) return;
  Cache c = p.cache;
  c.key += static_cast<size_t>(layer) * c.pages * kPageBytes;
  c.value += static_cast<size_t>(layer) * c.pages * kPageBytes;
  c.key_scale += static_cast<size_t>(layer) * c.pages * kKVHeads;
  c.value_scale += static_cast<size_t>(layer) * c.pages * kKVHeads;
  const size_t tail_layer = static_cast<size_t>(layer) * c.slots * 2 * kPage;
  T* tk = static_cast<T*>(c.tail_key) + tail_layer * kRowElems;
  T* tv = static_cast<T*>(c.tail_value) + tail_layer * kRowElems;
  const size_t new0 = (static_cast<size_t>(layer) * p.new_rows + r.q0) * kRowElems;
  const T* nk = static_cast<const T*>(p.new_k) + new0;
  const T* nv = static_cast<const T*>(p.new_v) + new0;
  if (first + b < end) {
    const int id = r.table[first + b];
    if (id < 0 || id >= c.pages) {
      if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
      return;
    }
#pragma unroll 1
    for (int h = h0; h < h0 + kHeads; ++h) {
      quantize_block<T, kCode>(c, static_cast<size_t>(id) * kKVHeads + h, [&](int t, const T*& k, const T*& v) {
        const int token = (first + b) * kPage + t;
        const bool old = token < r.ctx;
        const size_t at = (old ? tail_row(r.slot, token) : static_cast<size_t>(token - r.ctx)) * kRowElems + h * kHeadDim;
        k = (old ? tk : nk) + at;
        v = (old ? tv : nv) + at;
      }, sm);
    }
  }
  if (b > 0) return;
  const int low = max(r.ctx, end * kPage), rows = r.ctx + n - low;
  constexpr int kVecs = kHeads * kHeadDim / 8;
  for (int u = threadIdx.x; u < rows * kVecs; u += 256) {
    const int token = low + u / kVecs, e = h0 * kHeadDim + (u % kVecs) * 8;
    const size_t from = static_cast<size_t>(token - r.ctx) * kRowElems + e, to = tail_row(r.slot, token) * kRowElems + e;
    Vec8<T> a, v;
    a.load(nk + from);
    v.load(nv + from);
    a.store(tk + to);
    v.store(tv + to);
  }
}

// ---------------------------------------------------------------------------
// Copies: pages src -> dst (codes and scales) and the open tail rows of slots src -> dst, in all
// layers in one launch. Targets are distinct and no source is a target.
struct CopyParams {
  Cache cache;               // layer 0
  int layers, num, tails, row_bytes;
  const int* src;
  const int* dst;
  const int* tail_src;
  const int* tail_dst;
  const int* tail_len;       // tokens of the source request
};
constexpr int kCopyParts = 8;                               // CTAs of a page: one per head's K and V

__device__ __forceinline__ void copy_vecs(uint4* dst, const uint4* src, int n) {
  int u = threadIdx.x;
  for (; u + 3 * 256 < n; u += 4 * 256) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __ldg(src + u + 256 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[u + 256 * i] = x[i];
  }
  for (; u < n; u += 256) dst[u] = __ldg(src + u);
}

// Grid (num * 8 + tails * 2, layers)
__global__ void __launch_bounds__(256) copy_kernel(const CopyParams p) {
  const Cache& c = p.cache;
  const int layer = blockIdx.y, x = blockIdx.x;
  if (x < p.num * kCopyParts) {
    const int i = x / kCopyParts, h = x % kCopyParts, s = p.src[i], d = p.dst[i];
    if (s < 0 || s >= c.pages || d < 0 || d >= c.pages) {
      if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
      return;
    }
    const size_t from = (static_cast<size_t>(layer) * c.pages + s) * kKVHeads + h;
    const size_t to = (static_cast<size_t>(layer) * c.pages + d) * kKVHeads + h;
    const uint4* sk = reinterpret_cast<const uint4*>(c.key + from * kHeadBytes) + threadIdx.x;
    const uint4* sv = reinterpret_cast<const uint4*>(c.value + from * kHeadBytes) + threadIdx.x;
    const uint4 k0 = __ldg(sk), k1 = __ldg(sk + 256), v0 = __ldg(sv), v1 = __ldg(sv + 256);
    uint4* dk = reinterpret_cast<uint4*>(c.key + to * kHeadBytes) + threadIdx.x;
    uint4* dv = reinterpret_cast<uint4*>(c.value + to * kHeadBytes) + threadIdx.x;
    dk[0] = k0;
    dk[256] = k1;
    dv[0] = v0;
    dv[256] = v1;
    if (threadIdx.x == 0) c.key_scale[to] = c.key_scale[from];
    if (threadIdx.x == 32) c.value_scale[to] = c.value_scale[from];
    return;
  }
  const int i = (x - p.num * kCopyParts) >> 1, value = x & 1;
  const int s = p.tail_src[i], d = p.tail_dst[i], n = p.tail_len[i];
  if (s < 0 || s >= c.slots || d < 0 || d >= c.slots || n < 0) {
    if (threadIdx.x == 0) atomicOr(&g_device_status, kStatusBadArgument);
    return;
  }
  const int open = n % kPage;
  const size_t row0 = static_cast<size_t>(layer) * c.slots * 2 * kPage;
  uint8_t* base = static_cast<uint8_t*>(value ? c.tail_value : c.tail_key);
  copy_vecs(reinterpret_cast<uint4*>(base + (row0 + tail_row(d, n - open)) * p.row_bytes),
            reinterpret_cast<const uint4*>(base + (row0 + tail_row(s, n - open)) * p.row_bytes),
            open * (p.row_bytes / 16));
}

}  // namespace quant
}  // namespace dspark
