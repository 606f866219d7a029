// kv4.cu — the 4-bit key/value cache: quantizing append, read-back, causal
// attention over the cache and eviction by accumulated attention weight.
//
// The format and the row layouts are stated at mri_kv4_cache in mri_gpu.h.
// Offsets into the cache are size_t throughout: 32 heads of a long cache pass
// 2^31 bytes.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "internal.h"
#include "kv4_walk.h"
#include "mri_gpu.h"

namespace {

constexpr int kThreads = 256;

#define KV4_CUDA_TRY(expr)                                                                        \
  do {                                                                                            \
    cudaError_t _e = (expr);                                                                      \
    if (_e != cudaSuccess) return mri::set_error(MRI_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
  } while (0)

// Launch with programmatic dependent launch (unless the context has it off).
// `cluster`: blocks of a cluster.
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(mri_ctx* ctx, int cluster, void (*k)(KArgs...), unsigned grid, int threads, size_t smem,
                            Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (ctx->dev.opt.pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  ctx->ls.launches++;
  return cudaLaunchKernelEx(&cfg, k, static_cast<KArgs>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch(mri_ctx* ctx, void (*k)(KArgs...), unsigned grid, int threads, size_t smem, Args... args) {
  return launch_clusters(ctx, 1, k, grid, threads, smem, args...);
}

// Lets the next kernel be scheduled, and waits until the one before has ended.
__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A cache as the kernels see it.
struct Cache {
  uint8_t* k;
  uint8_t* v;
  uint16_t* ks;
  uint16_t* vs;
  float* weight;
  int batch, heads, hd, nb;
  size_t cap;
  __device__ __forceinline__ size_t row(int b, int h, size_t pos) const {
    return (static_cast<size_t>(b) * heads + h) * cap + pos;
  }
};

// ── append and read ──────────────────────────────────────────────────────────

// create_q4_0_block's scale (gguf/dequant.rs:706-749, f16 by
// gguf/quantization.rs:464-498): the f32 value cut to f16, mantissa truncated,
// infinite from 65536 on (round-toward-zero alone would give 65504).  That
// codec flushes what falls below 2^-14; a cache keeps it as a subnormal, so
// that rows of small values do not vanish.
__device__ __forceinline__ uint16_t scale_bits(float s) {
  if (s >= 65536.0f) return 0x7C00u;
  return __half_as_ushort(__float2half_rz(s));
}

// The scale is max|x| times the float32 nearest to 1/7: within one unit of the
// file codec's quotient, which the cut to f16 hides but for a block in some
// thousands, and without a division in the block's critical path.
constexpr float kSeventh = 1.0f / 7.0f;

// clamp(round(v * inv)) + 8, halves away from 0; NaN gives 8, which stands for 0.
__device__ __forceinline__ uint32_t code_of(float v, float inv) {
  const float r = roundf(__fmul_rn(v, inv));
  if (r != r) return 8u;
  return static_cast<uint32_t>(fminf(fmaxf(r, -8.0f), 7.0f) + 8.0f);
}
// The same where v * inv is finite and at most 7 and a rounding: adding the float
// below 1/2 with v's sign and cutting rounds halves away from 0.
__device__ __forceinline__ uint32_t code_in_range(float v, float inv) {
  const float r = __fmul_rn(v, inv);
  return static_cast<uint32_t>(__float2int_rz(__fadd_rn(r, copysignf(0.49999997f, r))) + 8);
}
// max(|a|, |b|) that passes a NaN on.
__device__ __forceinline__ float absmax_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(b)));
  return m;
}

// Rows are numbered (entry, token, head); 4 NB threads take one, a thread 8
// neighbouring values: word t of block b.
template <int NB>
struct RowThread {
  static constexpr int kPer = 4 * NB, kRows = kThreads / kPer;  // threads of a row, rows of a block
  int b, t, h, bi, ti;
  size_t tok;
  bool live;  // the threads of a row agree
  __device__ __forceinline__ RowThread(const Cache& c, unsigned rows, unsigned n_tokens, unsigned block) {
    const unsigned at = threadIdx.x / kPer, w = threadIdx.x % kPer, row = block * kRows + at;
    live = at < kRows && row < rows;
    b = static_cast<int>(w >> 2);
    t = static_cast<int>(w & 3);
    const unsigned token = (live ? row : 0u) / static_cast<unsigned>(c.heads);
    h = static_cast<int>((live ? row : 0u) % static_cast<unsigned>(c.heads));
    bi = static_cast<int>(token / n_tokens);
    ti = static_cast<int>(token % n_tokens);
    tok = token;
  }
};

// Bound by HBM (8 d bytes read, d + 4 NB + 4 written a row): all of a thread's
// loads are issued before the first is used.  2047 tokens of 32 heads of 128: 18 us,
// 4.3 TB/s.  vec: 16-byte aligned rows.
template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Cache c, const float* __restrict__ k,
                                                              const float* __restrict__ v, size_t ld,
                                                              unsigned n_tokens,
                                                              const int32_t* __restrict__ start,
                                                              unsigned rows, bool vec) {
  pdl_enter();
  const RowThread<NB> r(c, rows, n_tokens, blockIdx.x);
  const int64_t pos = static_cast<int64_t>(mri::ld_act(start + r.bi)) + r.ti;
  const bool store = r.live && pos >= 0 && pos < static_cast<int64_t>(c.cap);
  const size_t src = r.tok * ld + static_cast<size_t>(r.h) * (32 * NB) + 32 * r.b + 8 * r.t;
  const size_t dst = store ? c.row(r.bi, r.h, static_cast<size_t>(pos)) : 0;
  float x[2][8];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* p = (which ? v : k) + src;
    if (r.live && vec) {
      const float4 a = mri::ld_act(reinterpret_cast<const float4*>(p)), b = mri::ld_act(reinterpret_cast<const float4*>(p) + 1);
      x[which][0] = a.x, x[which][1] = a.y, x[which][2] = a.z, x[which][3] = a.w;
      x[which][4] = b.x, x[which][5] = b.y, x[which][6] = b.z, x[which][7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[which][i] = r.live ? mri::ld_act(p + i) : 0.0f;
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = absmax_nan(m, x[which][i]);
    m = absmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));  // the 4 threads of a block of 32
    m = absmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float s = __fmul_rn(m, kSeventh);
    float inv = __fdiv_rn(1.0f, s);
    uint32_t word = 0;
    const bool plain = s > 0.0f && s < INFINITY && inv < INFINITY;
    if (plain) {
#pragma unroll
      for (int i = 0; i < 8; ++i) word |= code_in_range(x[which][i], inv) << (4 * i);
    }
    if (__any_sync(0xffffffffu, !plain)) {
      // Blocks of zeros, with an inf or NaN, or so small that 1 / s overflows.
      float c = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) c = mri::absmax_acc(c, x[which][i]);
      c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 1));
      c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 2));
      if (!plain) {
        s = __fmul_rn(c, kSeventh);
        inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= (s > 0.0f ? code_of(x[which][i], inv) : 8u) << (4 * i);
      }
    }
    // Value codes: the half-words of pieces 2 t and 2 t + 1.  The threads of
    // blocks b and b ^ 1 (4 lanes apart) each put one whole word together.
    uint32_t pair = 0;
    if (which == 1 && NB % 2 == 0) {
      const bool odd = r.b & 1;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? word << 16 : word >> 16, 4);
      pair = odd ? (got & 0xFFFFu) | (word & 0xFFFF0000u) : (word & 0xFFFFu) | (got & 0xFFFF0000u);
    }
    if (!store) continue;
    if (which == 0) {
      reinterpret_cast<uint32_t*>(c.k + dst * (16 * NB))[r.t * NB + r.b] = word;
      if (r.t == 0) c.ks[dst * NB + r.b] = scale_bits(s);
      if (r.t == 0 && r.b == 0) c.weight[dst] = 0.0f;
    } else {
      uint16_t* o = reinterpret_cast<uint16_t*>(c.v + dst * (16 * NB));
      if (NB % 2 == 0) {
        *reinterpret_cast<uint32_t*>(o + (2 * r.t + (r.b & 1)) * NB + (r.b & ~1)) = pair;
      } else {
        o[(2 * r.t) * NB + r.b] = static_cast<uint16_t>(word);
        o[(2 * r.t + 1) * NB + r.b] = static_cast<uint16_t>(word >> 16);
      }
      if (r.t == 0) c.vs[dst * NB + r.b] = scale_bits(s);
    }
  }
}

// Bound by the writes (d + 4 NB bytes read, 8 d written a row): 128000 rows of 128 in 36 us,
// 4.1 TB/s.  Each of a thread's two 16-byte writes is half a sector, and a warp's cover 1 KB
// by halves.  Two rows a thread were slower.
template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Cache c, const int32_t* __restrict__ start,
                                                            unsigned n_tokens, float* __restrict__ k,
                                                            float* __restrict__ v, unsigned rows, bool vec) {
  pdl_enter();
  const RowThread<NB> r(c, rows, n_tokens, blockIdx.x);
  if (!r.live) return;
  const int64_t pos = static_cast<int64_t>(start ? mri::ld_act(start + r.bi) : 0) + r.ti;
  const bool there = pos >= 0 && pos < static_cast<int64_t>(c.cap);
  const size_t src = there ? c.row(r.bi, r.h, static_cast<size_t>(pos)) : 0;
  const size_t dst = (r.tok * c.heads + r.h) * (32 * NB) + 32 * r.b + 8 * r.t;
  uint32_t word[2] = {0x88888888u, 0x88888888u};
  uint32_t scale[2] = {0, 0};
  if (there) {
    word[0] = mri::ld_act(reinterpret_cast<const uint32_t*>(c.k + src * (16 * NB)) + r.t * NB + r.b);
    const uint16_t* p = reinterpret_cast<const uint16_t*>(c.v + src * (16 * NB)) + 2 * r.t * NB + r.b;
    word[1] = mri::ld_act(p) | static_cast<uint32_t>(mri::ld_act(p + NB)) << 16;
    scale[0] = mri::ld_act(c.ks + src * NB + r.b);
    scale[1] = mri::ld_act(c.vs + src * NB + r.b);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float s = mri::f16_bits_to_f32(scale[which]);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)  // 2^23 + code, less 2^23 + 8
      y[i] = __fmul_rn(__fsub_rn(__uint_as_float(((word[which] >> (4 * i)) & 15u) | 0x4B000000u), 8388616.0f), s);
    float* o = (which ? v : k) + dst;
    if (vec) {
      __stcs(reinterpret_cast<float4*>(o), make_float4(y[0], y[1], y[2], y[3]));
      __stcs(reinterpret_cast<float4*>(o) + 1, make_float4(y[4], y[5], y[6], y[7]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = y[i];
    }
  }
}

// ── attention ────────────────────────────────────────────────────────────────
//
// One key/value head's cache is read by G = n_heads / n_kv_heads query heads for
// each of n_tokens tokens: G * n_tokens rows (row r: token r / G, head r % G).
// A warp walks keys 16 at a time on mma.sync m16n8k16 (f16 in, f32 out); the matrix
// work of a decode step has 8 rows at most, too few for the 128-row tiles of
// tcgen05 (tried at 8 to 509 rows: 1.2 to 2.3 times slower, since the unpacked codes
// then go through shared memory).  Up to 8 rows, the A tile's 16 rows are the rows' high
// and low f16 parts (22 bits), so one MMA returns both halves of the product and a
// lane adds D[g] + D[g + 8].  More rows: 16 a warp, high and low parts as two
// MMAs, which unpacks a code for twice the rows.  Codes are exact in f16.
//
//   A code becomes f16 by one AND-OR that puts its 4 bits under the exponent
//   of 1024 (1024 + c; the nibble above gives 1024 + 16 c) and one subtraction
//   for two codes: c - 8 or 16 (c - 8), normal numbers.  (As f16 subnormals c *
//   2^-24 the codes would need the AND alone, but the tensor core aligns its
//   sums by exponents, and a subnormal's leading zeros then cost 8 of the
//   result's bits: 9e-6 off instead of 5e-7.)
//   S = Q K^T: B is 8 keys' codes.  The scale differs by block and key, so each
//   32-wide block is its own sum, scaled afterwards.
//   O += P V: the scales belong to keys, the summed index, so they go into
//   P: per block, A = f16 high and low parts of P * scale, B = the codes.
//
// An f16 pair holds P * scale to 22 bits from 2^-2 up, and to 2^-25 below.  P is taken
// relative to a reference below the row's running maximum, moved (and the sums rescaled)
// only when a score passes the old maximum by 2^kRise; value scales by a factor of their
// block (the same 32 columns) that brings the largest one the warp has seen below
// 2^kTop, moved when one passes that.  So a block of small values is as exact as one of
// large ones.  Within a block a key has its 22 bits down to 2^-11 of the row's
// largest P times the block's largest scale, whoever's that is, and a bit less with every
// factor of 2 from there: keys beside one of 2^11 times their values, in a row in
// which that one counts for nothing, are where f32 products would hold more.
// exp2 of log2-scaled scores; sums and scores in f32.

constexpr int kStep = 32;        // keys that are scored together; a ring's stage is one or two steps
constexpr int kMaxWarps = 4;     // of a block: rings of their own (up to 8 rows) or 16-row tiles that share one
constexpr size_t kBlockBytes = 74 * 1024 + 256;  // shared memory of a block of four warps: three fit an SM
constexpr int kMinKeys = 128;    // a block's keys before the next block is used
constexpr int kMaxStages = 4;
constexpr int kFlushKeys = 512;  // keys whose products a warp leaves to the tensor core's own sums
// P is 2^kHead at most when a row's reference is set and 2^(kHead + kRise) before it is
// moved; with scales below 2^kTop, P * scale is below 2^15.  With this kTop the factors of
// scales from 2^-23 to 2^16 are f16 numbers.  24 x 8 heads of up to 32K keys, and 16 x 8 of up
// to 4K with 40 rows: 153 and 100 us with kRise 5; 153 and 99 with 8, which leaves three bits
// less below the largest; 154 and 102 with 3.  A factor for the block's scales costs 1 to 2 us
// of these, and 1.4 of 57 in a tracked decode step.
constexpr int kTop = -8;
constexpr float kHead = 18.0f, kRise = 5.0f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The warp's largest |x|.
__device__ __forceinline__ float warp_absmax(float x) {
  float y;
  asm("redux.sync.max.abs.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// Two floats as f16 pairs hi = f16(x), lo = f16(x - hi).
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_half2(x0, x1);
  const float2 h = unpack_half2(hi);
  lo = pack_half2(__fsub_rn(x0, h.x), __fsub_rn(x1, h.y));
}

// Two floats in one 64-bit register: one instruction does both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair2(float x, float y) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float2 unpair2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// A pair as f16 hi = f16(x) and lo = f16(hi - x): the rest with its sign changed,
// which the f16 - f32 subtraction gives in one instruction a value.
__device__ __forceinline__ void split2_neg(f32x2 x, uint32_t& hi, uint32_t& lo) {
  const float2 v = unpair2(x);
  hi = pack_half2(v.x, v.y);
  float r0, r1;
  asm("{\n\t.reg .b16 h0, h1;\n\tmov.b32 {h0, h1}, %2;\n\t"
      "sub.f32.f16 %0, h0, %3;\n\tsub.f32.f16 %1, h1, %4;\n\t}"
      : "=f"(r0), "=f"(r1)
      : "r"(hi), "f"(v.x), "f"(v.y));
  lo = pack_half2(r0, r1);
}
__device__ __forceinline__ void split2_pos(f32x2 x, uint32_t& hi, uint32_t& lo) {
  split2_neg(x, hi, lo);
  lo ^= 0x80008000u;
}
// c - 8 of the codes in bits 0..3 of both halves of w, and 16 (c - 8) of those
// in bits 4..7.  One LOP3 ((w & mask) | 1024's exponent) and one subtraction;
// written out, since the compiler makes two of an AND and an OR with constants.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b32 x;\n\tlop3.b32 x, %1, 0x000F000F, %2, 0xEA;\n\tsub.rn.f16x2 %0, x, %3;\n\t}"
      : "=r"(d)
      : "r"(w), "r"(0x64006400u), "r"(0x64086408u));  // 1024, 1032
  return d;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b32 x;\n\tlop3.b32 x, %1, 0x00F000F0, %2, 0xEA;\n\tsub.rn.f16x2 %0, x, %3;\n\t}"
      : "=r"(d)
      : "r"(w), "r"(0x64006400u), "r"(0x64806480u));  // 1024, 1152
  return d;
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero sums.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}

struct AttnArgs {
  Cache c;
  const float* q;
  size_t ld;
  int n_tokens, n_heads, group;  // group = n_heads / c.heads
  const int32_t* lens;
  float scale;
  float* out;
  float2* stats;    // tracked calls: reference and 1 / sum of every row
  int rows;         // group * n_tokens
  int row_tiles;    // tiles of a row group = warps that share a ring
  int n_rows;       // of a row group
  int pad;          // places a unit counts besides its stages
  int keys;         // of a ring stage
  int row_groups;
  int splits;       // rings (key splits) of a block
  int stages;
  float* part;      // [2 * grid][n_rows][hd + 4]
  unsigned* ready;  // [grid], zero between calls
  int2* spans;      // of each unit: the first and the last block that have a part in it
  unsigned grid;    // blocks of the first kernel
  int* status;
  __device__ __forceinline__ int len(int b) const { return min(max(mri::ld_act(lens + b), 0), static_cast<int>(c.cap)); }
};

using mri::kv4::Plan;
using mri::kv4::Unit;
using mri::kv4::next_segment;
using mri::kv4::next_unit;
using mri::kv4::owner_of;
using mri::kv4::seek_stage;
using mri::kv4::unit_tiles;

// This block's share of the call's stages and the unit it begins in.
// Every thread calls it; sums over (entry, row group) pairs in shared memory.
__device__ __forceinline__ void make_plan(const AttnArgs& a, Plan* plan, unsigned* sh) {
  const unsigned threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned groups = static_cast<unsigned>(a.row_groups), heads = static_cast<unsigned>(a.c.heads);
  const unsigned pairs = static_cast<unsigned>(a.c.batch) * groups;
  const unsigned run = (pairs + threads - 1) / threads;
  const unsigned p0 = min(pairs, run * threadIdx.x), p1 = min(pairs, p0 + run);
  unsigned mine = 0;
#pragma unroll 1
  for (unsigned p = p0; p < p1; ++p)
    mine += static_cast<unsigned>(unit_tiles(a, static_cast<int>(p / groups), static_cast<int>(p % groups))) * heads;
  unsigned incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= static_cast<unsigned>(o)) incl += v;
  }
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  unsigned before = incl - mine, total = 0;
  for (unsigned w = 0; w < threads / 32; ++w) {
    if (w < warp) before += sh[w];
    total += sh[w];
  }
  Plan p;
  mri::kv4::share_out(a, total, blockIdx.x, gridDim.x, kMinKeys / static_cast<unsigned>(a.keys), p);
  if (threadIdx.x == 0) *plan = p;
  __syncthreads();
  if (p.x0 >= before && p.x0 - before < mine) mri::kv4::find_first(a, p.x0, before, p0, p1, plan->first);
  __syncthreads();
}

// One row tile's queries as A fragments: high parts in rows 0..7, low in
// 8..15, scaled by a power of two that brings the row's largest |q| near
// 2^13.  mult: score factor (log2 units) that undoes it.
template <int NB>
struct QueryTile {
  uint32_t a[NB][2][4];
  float mult;
};

template <int NB>
__device__ __forceinline__ void fetch_queries(const AttnArgs& a, int b, int h, int row, float (&x)[NB][8]) {
  const int t = threadIdx.x & 3;
  const bool live = row < a.rows;
  const float* src = a.q + (static_cast<size_t>(b) * a.n_tokens + (live ? row / a.group : 0)) * a.ld +
                     (static_cast<size_t>(h) * a.group + (live ? row % a.group : 0)) * (32 * NB) + 8 * t;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.ld * 4)) & 15) == 0;
#pragma unroll
  for (int bl = 0; bl < NB; ++bl) {
    if (live && vec) {
      const float4 u = mri::ld_act(reinterpret_cast<const float4*>(src + 32 * bl));
      const float4 v = mri::ld_act(reinterpret_cast<const float4*>(src + 32 * bl + 4));
      x[bl][0] = u.x, x[bl][1] = u.y, x[bl][2] = u.z, x[bl][3] = u.w;
      x[bl][4] = v.x, x[bl][5] = v.y, x[bl][6] = v.z, x[bl][7] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[bl][i] = live ? mri::ld_act(src + 32 * bl + i) : 0.0f;
    }
  }
}
template <int NB>
__device__ __forceinline__ void split_queries(const AttnArgs& a, float (&x)[NB][8], QueryTile<NB>& q) {
  float big = 0.0f;
#pragma unroll
  for (int bl = 0; bl < NB; ++bl)
#pragma unroll
    for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[bl][i]));
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
  // 2^up brings `big` into [2^13, 2^14); 0 and what is not finite stay.  In
  // two factors: up itself may pass f32's exponents.
  int up = 0;
  if (big > 0.0f && big < INFINITY) up = 140 - static_cast<int>(__float_as_uint(big) >> 23);  // subnormals as 2^-127
  const int up0 = max(-126, min(126, up));
  const float f0 = __int_as_float((up0 + 127) << 23), f1 = __int_as_float((up - up0 + 127) << 23);
  q.mult = __fmul_rn(__fmul_rn(__fmul_rn(a.scale, kLog2e), __int_as_float((127 - up0) << 23)),
                     __int_as_float((127 - (up - up0)) << 23));
#pragma unroll
  for (int bl = 0; bl < NB; ++bl) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[bl][i] = __fmul_rn(__fmul_rn(x[bl][i], f0), f1);
    // Step 0 takes code nibbles (0, 4) and (2, 6), step 1 (1, 5) and (3, 7)
    // as 16 (c - 8), so its q is a sixteenth.
    split2(x[bl][0], x[bl][4], q.a[bl][0][0], q.a[bl][0][1]);
    split2(x[bl][2], x[bl][6], q.a[bl][0][2], q.a[bl][0][3]);
    split2(x[bl][1] * 0.0625f, x[bl][5] * 0.0625f, q.a[bl][1][0], q.a[bl][1][1]);
    split2(x[bl][3] * 0.0625f, x[bl][7] * 0.0625f, q.a[bl][1][2], q.a[bl][1][3]);
  }
}

template <int NB>
__device__ __forceinline__ void load_queries(const AttnArgs& a, int b, int h, int row, QueryTile<NB>& q) {
  float x[NB][8];
  fetch_queries<NB>(a, b, h, row, x);
  split_queries<NB>(a, x, q);
}

// Scores (before mult) of 8 keys for the lane's row: keys 2t and 2t + 1.
// kw: the lane's piece (t) of key g's codes; ks: per block, the scales of keys
// 2t, 2t + 1.
template <int NB>
__device__ __forceinline__ f32x2 score8(const QueryTile<NB>& q, const uint32_t (&kw)[NB], const f32x2 (&ks)[NB]) {
  f32x2 s = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float d[4];
    const uint32_t w = kw[b], w8 = w >> 8;
    mma16816_first(d, q.a[b][0], low_codes(w), low_codes(w8));
    mma16816(d, q.a[b][1], high_codes(w), high_codes(w8));
    const f32x2 both = add2(pair2(d[0], d[1]), pair2(d[2], d[3]));
    s = b == 0 ? mul2(ks[b], both) : fma2(ks[b], both, s);
  }
  return s;
}

// A warp's queries: 8 rows, or 16 with high and low parts as products of their own,
// so that the same unpacked codes serve twice the rows.
template <int NB, int R>
struct WarpQueries {
  // 16 rows of 96 or 128 wide heads would take 48 or 64 registers: those lie in
  // shared memory, each lane's own where only it reads them, and are loaded once for
  // 32 keys.
  static constexpr bool kShared = R == 2 && NB > 2;
  static constexpr int kSharedItems = kShared ? 4 * NB * 32 : 0;
  uint32_t a[kShared ? 1 : R][NB][2][4];  // 16 rows: high parts, low parts
  uint4* shared;                          // [block][step][high, low][lane]
  float mult[R];                          // of rows g, g + 8

  __device__ __forceinline__ void load(const AttnArgs& args, int b, int h, int row, uint4* area) {
    QueryTile<NB> q[R];
    float x[R][NB][8];  // all loads first
#pragma unroll
    for (int i = 0; i < R; ++i) fetch_queries<NB>(args, b, h, row + 8 * i, x[i]);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      split_queries<NB>(args, x[i], q[i]);
      mult[i] = q[i].mult;
    }
    shared = area + (threadIdx.x & 31);
#pragma unroll
    for (int bl = 0; bl < NB; ++bl)
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if constexpr (R == 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x) a[0][bl][step][x] = q[0].a[bl][step][x];
          } else {
            const uint32_t f[4] = {q[0].a[bl][step][i], q[1].a[bl][step][i], q[0].a[bl][step][2 + i], q[1].a[bl][step][2 + i]};
            if constexpr (kShared)
              shared[((bl * 2 + step) * 2 + i) * 32] = make_uint4(f[0], f[1], f[2], f[3]);
            else
#pragma unroll
              for (int x = 0; x < 4; ++x) a[i][bl][step][x] = f[x];
          }
        }
  }
  // The fragments of a block.
  __device__ __forceinline__ void block(int bl, uint32_t (&f)[R][2][4]) const {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        if constexpr (kShared) {
          const uint4 v = shared[((bl * 2 + step) * 2 + i) * 32];
          f[i][step][0] = v.x, f[i][step][1] = v.y, f[i][step][2] = v.z, f[i][step][3] = v.w;
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) f[i][step][x] = a[i][bl][step][x];
        }
      }
  }
};

// score8 for the lane's rows: block bl of 8 keys, added to s.
template <int R>
__device__ __forceinline__ void score_block(const uint32_t (&q)[R][2][4], uint32_t w, f32x2 ks, bool first, f32x2 (&s)[R]) {
  float d[4];
  const uint32_t w8 = w >> 8;
  const uint32_t l0 = low_codes(w), l1 = low_codes(w8), h0 = high_codes(w), h1 = high_codes(w8);
  mma16816_first(d, q[0][0], l0, l1);
  mma16816(d, q[0][1], h0, h1);
  if constexpr (R == 2) {
    mma16816(d, q[R - 1][0], l0, l1);
    mma16816(d, q[R - 1][1], h0, h1);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const f32x2 sum = R == 1 ? add2(pair2(d[0], d[1]), pair2(d[2], d[3])) : pair2(d[2 * i], d[2 * i + 1]);
    s[i] = first ? mul2(ks, sum) : fma2(ks, sum, s[i]);
  }
}

// Scales of two keys as float pairs from shared memory.
template <int NB>
__device__ __forceinline__ void load_scales(const float* p, f32x2 (&s)[NB]) {
  if constexpr (NB % 2 == 0) {
#pragma unroll
    for (int b = 0; b < NB; b += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p + 2 * b);
      s[b] = v.x;
      s[b + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = *reinterpret_cast<const f32x2*>(p + 2 * b);
  }
}

template <int NB, int KEYS>
constexpr int stage_bytes() { return KEYS * NB * 36; }

// The f16 scales of 32 keys, as a lane reads them from a stage: key pairs and one
// or two blocks, keys' before values'.
template <int NB>
struct RawScales {
  static constexpr int kPer = NB % 2 ? 1 : 2;  // blocks of an item
  static constexpr int kItems = kStep / 2 * NB / kPer, kRounds = (2 * kItems + 31) / 32;
  uint32_t w[kRounds][2];  // of the pair's two keys: kPer halves each
};

// The powers of two that a warp's value scales are multiplied by, one a block.
template <int NB>
struct ValueFactors {
  unsigned fields;  // byte b: the exponent field of block b's
  uint32_t lane;    // f16, of the value scales that this lane converts (1 for key scales): of a round's two blocks, or of two rounds
  static constexpr int kLargest = 127 + 15, kSmallest = 127 - 24;  // f16's powers of two

  __device__ __forceinline__ float of(int b) const { return __uint_as_float((fields >> (8 * b) & 0xFFu) << 23); }
  __device__ __forceinline__ float inverse(int b) const { return __uint_as_float((254u - (fields >> (8 * b) & 0xFFu)) << 23); }
  __device__ __forceinline__ void set_lane() {
    using S = RawScales<NB>;
    const int i0 = 32 * (S::kRounds - (NB == 3 ? 2 : 1)) + (threadIdx.x & 31), i1 = NB == 3 ? i0 + 32 : i0;
    auto factor = [&](int i, int more) { return i < S::kItems ? 1.0f : of((i - S::kItems) % (NB / S::kPer) * S::kPer + more); };
    lane = pack_half2(factor(i0, 0), factor(i1, S::kPer - 1));
  }
  __device__ __forceinline__ void init() {
    fields = 0x01010101u * kLargest;
    set_lane();
  }
};
// x's half `high` times f's, exactly, in f32.
__device__ __forceinline__ float mul_halves(uint32_t x, int high, uint32_t f, int high_f) {
  float y;
  asm("{\n\t.reg .b16 a, b;\n\tcvt.u16.u32 a, %1;\n\tcvt.u16.u32 b, %2;\n\tfma.rn.f32.f16 %0, a, b, %3;\n\t}"
      : "=f"(y)
      : "r"(high ? x >> 16 : x), "r"(high_f ? f >> 16 : f), "f"(0.0f));
  return y;
}

// What a warp carries over its keys for its rows (lane: rows g and g + 8, columns by t).
template <int NB, int R>
struct RowState {
  // 8 rows: [0..1] by high parts, [2..3] by low ones, whose sign was changed; 16: rows g, g + 8.
  float o[NB * 4][4];
  float m[R];    // running maximum that the reference was set from (row)
  float ref[R];  // reference: P = exp2(score - ref)
  f32x2 l[R];    // sums of P over the lane's even and odd keys
  ValueFactors<NB> scaled;  // of the value scales; the sums count by them too
};

// ks, vs: the key and value scales of the 32 keys.
template <int NB>
__device__ __forceinline__ RawScales<NB> load_raw_scales(const uint8_t* ks, const uint8_t* vs) {
  using R = RawScales<NB>;
  const int lane = threadIdx.x & 31;
  R raw;
#pragma unroll
  for (int n = 0; n < R::kRounds; ++n) {
    const int i = 32 * n + lane;
    const bool value = i >= R::kItems, live = 2 * R::kItems % 32 == 0 || i < 2 * R::kItems;
    const int it = value ? i - R::kItems : i;
    const int pair = it / (NB / R::kPer), b = it % (NB / R::kPer) * R::kPer;
    const uint8_t* src = (value ? vs : ks) + (live ? pair : 0) * (4 * NB) + 2 * b;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      raw.w[n][c] = R::kPer == 2 ? *reinterpret_cast<const uint32_t*>(src + c * 2 * NB) : *reinterpret_cast<const uint16_t*>(src + c * 2 * NB);
  }
  return raw;
}

// The same as float32 [key pair][block][2], keys' first and then values', in shared
// memory: each is needed by 8 lanes, and is converted once.  Value scales are multiplied by
// the factors f of their blocks.  Keys from len on (whatever they hold) become 0.
// Returns the lane's largest value scale after that.
template <int NB, bool MASKED>
__device__ __forceinline__ float convert_scales(const RawScales<NB>& raw, float* to, int k0, int len, uint32_t f) {
  using R = RawScales<NB>;
  const int lane = threadIdx.x & 31;
  float dmax = 0.0f;
#pragma unroll
  for (int n = 0; n < R::kRounds; ++n) {
    const int i = 32 * n + lane;
    if (2 * R::kItems % 32 && i >= 2 * R::kItems) break;
    const bool value = i >= R::kItems;
    const int it = value ? i - R::kItems : i;
    const int pair = it / (NB / R::kPer), b = it % (NB / R::kPer) * R::kPer;
    float2 x[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (32 * n + 31 < R::kItems)  // key scales alone
        x[c] = unpack_half2(raw.w[n][c]);
      else
        x[c] = make_float2(mul_halves(raw.w[n][c], 0, f, NB == 3 ? n - 1 : 0), R::kPer == 2 ? mul_halves(raw.w[n][c], 1, f, 1) : 0.0f);
      if (MASKED && k0 + 2 * pair + c >= len) x[c] = make_float2(0.0f, 0.0f);
      if (value) dmax = fmaxf(dmax, R::kPer == 2 ? fmaxf(fabsf(x[c].x), fabsf(x[c].y)) : fabsf(x[c].x));
    }
    float* dst = to + (value ? kStep * NB : 0) + pair * (2 * NB) + 2 * b;
    if constexpr (R::kPer == 2)
      *reinterpret_cast<float4*>(dst) = make_float4(x[0].x, x[1].x, x[0].y, x[1].y);
    else
      *reinterpret_cast<float2*>(dst) = make_float2(x[0].x, x[1].x);
  }
  return dmax;
}

// The tensor core cuts its sums off instead of rounding them, which is a drift over
// a long run of keys: results 1.3e-6 off after 2048 keys of one warp.  So a warp
// adds its sums to float32 ones, rounded, every kFlushKeys keys (8 rows; 16 rows, of
// twice the products a key, every half of that): 2e-7 and 8e-7 off.  These lie in
// local memory (`volatile`): the loop has no registers for them.  24 x 8 heads of up
// to 32K keys: 153 us, 1 less every 1024 keys (2.7e-7).  They are relative to the
// reference of their time.
template <int NB, int R>
struct FlushedSums {
  volatile float o[NB * 8 * R];
  float ref[R];  // -inf: no key was seen (the sums are 0 or NaN); +inf: nothing was flushed

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < R; ++i) ref[i] = INFINITY;
  }
  __device__ __forceinline__ bool any() const { return ref[0] != INFINITY; }
  // Column c (0, 1) of the lane's row i, from the warp's sums.
  static __device__ __forceinline__ float sum(const RowState<NB, R>& r, int n, int i, int c) {
    return R == 1 ? __fsub_rn(r.o[n][c], r.o[n][2 + c]) : r.o[n][2 * i + c];
  }
  __device__ __forceinline__ float total(const RowState<NB, R>& r, int n, int i, int c) const {
    return any() ? o[(n * R + i) * 2 + c] : sum(r, n, i, c);
  }
  // The sums of a block whose value scales are divided by 2^less (byte b: block b).
  __device__ __forceinline__ void scale(unsigned less) {
#pragma unroll 1
    for (int n = 0; n < NB * 8 * R; ++n) o[n] = __fmul_rn(o[n], __uint_as_float((127u - (less >> (n / R & ~7) & 0xFFu)) << 23));
  }
  __device__ __forceinline__ void flush(RowState<NB, R>& r) {
    const bool add = any();
    float f[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      f[i] = ref[i] == r.ref[i] ? 1.0f : exp2_fast(ref[i] - r.ref[i]);
      ref[i] = r.m[i] == -INFINITY ? -INFINITY : r.ref[i];
    }
    constexpr int kRun = R == 1 ? NB * 4 : 4;  // all loads of a run before its first store
#pragma unroll
    for (int n0 = 0; n0 < NB * 4; n0 += kRun) {
      float old[kRun][R][2];
#pragma unroll
      for (int n = 0; n < kRun; ++n)
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            old[n][i][c] = 0.0f;
            if (add) old[n][i][c] = o[((n0 + n) * R + i) * 2 + c];
          }
#pragma unroll
      for (int n = 0; n < kRun; ++n)
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float x = sum(r, n0 + n, i, c);
            o[((n0 + n) * R + i) * 2 + c] = add ? __fmaf_rn(old[n][i][c], f[i], x) : x;
          }
    }
#pragma unroll
    for (int n = 0; n < NB * 4; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) r.o[n][x] = 0.0f;
  }
};

// 32 keys from k0 on: kc and vc their key and value codes, scales where their
// converted scales go.  row_end: keys before it are seen by the lane's rows; MASKED:
// some key is not, for some row.
template <int NB, int R, bool MASKED>
__device__ __forceinline__ void keys32(const uint8_t* kc, const uint8_t* vc, const RawScales<NB>& raw, float* scales, int k0,
                                       int len, const int (&row_end)[R], const WarpQueries<NB, R>& q, RowState<NB, R>& r,
                                       FlushedSums<NB, R>& flushed) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const float dmax = convert_scales<NB, MASKED>(raw, scales, k0, len, r.scaled.lane);
  __syncwarp();
  f32x2 z[4][R];  // keys 8 j + 2t, + 1
  if constexpr (WarpQueries<NB, R>::kShared) {
    uint32_t kw[4][NB];
#pragma unroll
    for (int j = 0; j < 4; ++j) load_words<NB>(kc + (8 * j + g) * (16 * NB) + t * (4 * NB), kw[j]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t f[R][2][4];
      q.block(b, f);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        score_block<R>(f, kw[j][b], *reinterpret_cast<const f32x2*>(scales + (4 * j + t) * (2 * NB) + 2 * b), b == 0, z[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t kw[NB];
      f32x2 ks[NB];
      load_words<NB>(kc + (8 * j + g) * (16 * NB) + t * (4 * NB), kw);
      load_scales<NB>(scales + (4 * j + t) * (2 * NB), ks);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t f[R][2][4];
        q.block(b, f);
        score_block<R>(f, kw[b], ks[b], b == 0, z[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < R; ++i) z[j][i] = mul2(z[j][i], pair2(q.mult[i], q.mult[i]));
  if constexpr (MASKED) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 v = unpair2(z[j][i]);
        const int key = k0 + 8 * j + 2 * t;
        z[j][i] = pair2(key < row_end[i] ? v.x : -INFINITY, key + 1 < row_end[i] ? v.y : -INFINITY);
      }
  }
  float zmax[R];
  constexpr float kTopScale = 1.0f / (1 << -kTop);
  bool moves = dmax >= kTopScale;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    zmax[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = unpair2(z[j][i]);
      zmax[i] = fmaxf(zmax[i], fmaxf(v.x, v.y));
    }
    moves = moves || zmax[i] > r.m[i] + kRise;
  }
  if (__any_sync(0xffffffffu, moves)) {
    float by[NB];
    unsigned less = 0;  // byte b: by how many powers of two
    if (__any_sync(0xffffffffu, dmax >= kTopScale)) {
      // A block with such a scale takes a smaller factor, and so do its sums.  An infinite
      // scale does not count: it spoils the sums of rows that see it, and no others.
      float* s = scales + kStep * NB + (lane >> 1) * (2 * NB) + (lane & 1);
#pragma unroll 1
      for (int b = 0; b < NB; ++b) {
        const float x = s[2 * b];
        const float top = warp_absmax(fabsf(x) < INFINITY ? x : 0.0f);
        const int over = static_cast<int>(__float_as_uint(top) >> 23) - (127 + kTop - 1);
        const int n = max(0, min(over, static_cast<int>(r.scaled.fields >> (8 * b) & 0xFFu) - ValueFactors<NB>::kSmallest));
        less |= static_cast<unsigned>(n) << (8 * b);
        s[2 * b] = __fmul_rn(x, __uint_as_float(static_cast<unsigned>(127 - n) << 23));
      }
      r.scaled.fields -= less;
      if (flushed.any()) flushed.scale(less);
      r.scaled.set_lane();
      __syncwarp();
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) by[b] = __uint_as_float((127u - (less >> (8 * b) & 0xFFu)) << 23);
    float f[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float mn = fmaxf(zmax[i], __shfl_xor_sync(0xffffffffu, zmax[i], 1));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
      mn = mn > r.m[i] + kRise ? mn : r.m[i];  // a row moves on its own scores only
      const float ref = mn == -INFINITY ? 0.0f : mn - kHead;
      f[i] = r.m[i] == -INFINITY ? 0.0f : exp2_fast(r.ref[i] - ref);
      r.m[i] = mn;
      r.ref[i] = ref;
      r.l[i] = mul2(r.l[i], pair2(f[i], f[i]));
    }
#pragma unroll
    for (int n = 0; n < NB * 4; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) r.o[n][x] = __fmul_rn(r.o[n][x], __fmul_rn(f[R == 1 ? 0 : x / 2], by[n / 4]));
  }
  f32x2 nref[R];
#pragma unroll
  for (int i = 0; i < R; ++i) nref[i] = pair2(-r.ref[i], -r.ref[i]);
  // Value codes: piece g of keys 2t, 2t + 1 (tile j), both halves of a word
  // from the two keys.  Odd t loads the pair in the other order: rows of
  // both parities in one load, half the bank conflicts.
  constexpr int VW = NB % 2 ? NB : NB / 2;  // registers of a piece: words, or half-words where a piece is no whole word
  const int odd = t & 1;
  const uint32_t sel_lo = odd ? 0x1054u : 0x5410u, sel_hi = odd ? 0x3276u : 0x7632u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x2 p[2][R], dv[2][NB];
    uint32_t vx[2][VW], vy[2][VW];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = 16 * h + 8 * j + 2 * t;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 e = unpair2(add2(z[2 * h + j][i], nref[i]));
        p[j][i] = pair2(exp2_fast(e.x), exp2_fast(e.y));
        r.l[i] = add2(r.l[i], p[j][i]);
      }
      load_scales<NB>(scales + kStep * NB + key * NB, dv[j]);
      const uint8_t* px = vc + (key + odd) * (16 * NB) + g * (2 * NB);
      const uint8_t* py = vc + (key + 1 - odd) * (16 * NB) + g * (2 * NB);
      if constexpr (NB % 2 == 0) {
        load_words<VW>(px, vx[j]);
        load_words<VW>(py, vy[j]);
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          vx[j][b] = reinterpret_cast<const uint16_t*>(px)[b];
          vy[j][b] = reinterpret_cast<const uint16_t*>(py)[b];
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // P times the scale of key pair j, row i; where some key is hidden, 0 for it:
      // 0 times its scale, if that is infinite, is not.
      auto scaled = [&](int j, int i) {
        f32x2 x = mul2(p[j][i], dv[j][b]);
        if constexpr (MASKED) {
          const float2 v = unpair2(x);
          const int key = k0 + 16 * h + 8 * j + 2 * t;
          x = pair2(key < row_end[i] ? v.x : 0.0f, key + 1 < row_end[i] ? v.y : 0.0f);
        }
        return x;
      };
      uint32_t a[R][4];
      if constexpr (R == 1) {
        split2_neg(scaled(0, 0), a[0][0], a[0][1]);
        split2_neg(scaled(1, 0), a[0][2], a[0][3]);
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) split2_pos(scaled(x / 2, x & 1), a[0][x], a[1][x]);
      }
      uint32_t w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (NB % 2 == 0)
          w[j] = __byte_perm(vx[j][b / 2], vy[j][b / 2], b & 1 ? sel_hi : sel_lo);
        else
          w[j] = __byte_perm(vx[j][b], vy[j][b], sel_lo);
      }
      const uint32_t u0 = w[0] >> 8, u1 = w[1] >> 8;
      const uint32_t c[4][2] = {{low_codes(w[0]), low_codes(w[1])}, {high_codes(w[0]), high_codes(w[1])},
                                {low_codes(u0), low_codes(u1)}, {high_codes(u0), high_codes(u1)}};
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n) mma16816(r.o[4 * b + n], a[i], c[n][0], c[n][1]);
    }
  }
}

// One stage, 32 keys at a time.
template <int NB, int R, int KEYS, bool MASKED>
__device__ __forceinline__ void stage_keys(const uint8_t* st, float* scales, int k0, int len, const int (&row_end)[R],
                                           const WarpQueries<NB, R>& q, RowState<NB, R>& r, FlushedSums<NB, R>& flushed) {
#pragma unroll 1
  for (int h = 0; h < KEYS; h += kStep) {
    if (KEYS > kStep) __syncwarp();  // the scales of the step before are read
    const RawScales<NB> raw = load_raw_scales<NB>(st + KEYS * NB * 32 + h * (2 * NB), st + KEYS * NB * 34 + h * (2 * NB));
    keys32<NB, R, MASKED>(st + h * (16 * NB), st + (KEYS + h) * (16 * NB), raw, scales, k0 + h, len, row_end, q, r, flushed);
  }
}

// A row's four columns, and the row's reference and sum of P, of one partial result
// or of several merged ones.
struct Merged {
  float ref, sum;  // ref -inf: no key seen
  float4 o;
};
template <int N>
__device__ __forceinline__ void merge_into(Merged& m, const float2 (&st)[N], const float4 (&v)[N]) {
  float to_ref = m.ref;
#pragma unroll
  for (int y = 0; y < N; ++y) to_ref = fmaxf(to_ref, st[y].x);
  if (to_ref == -INFINITY) return;  // no key seen so far
  const float f0 = m.ref == -INFINITY ? 0.0f : exp2_fast(m.ref - to_ref);
  m.sum = __fmul_rn(m.sum, f0);
  m.o = make_float4(__fmul_rn(m.o.x, f0), __fmul_rn(m.o.y, f0), __fmul_rn(m.o.z, f0), __fmul_rn(m.o.w, f0));
  m.ref = to_ref;
#pragma unroll
  for (int y = 0; y < N; ++y) {
    if (st[y].x == -INFINITY) continue;
    const float f = exp2_fast(st[y].x - to_ref);
    m.sum = __fmaf_rn(st[y].y, f, m.sum);
    m.o.x = __fmaf_rn(v[y].x, f, m.o.x);
    m.o.y = __fmaf_rn(v[y].y, f, m.o.y);
    m.o.z = __fmaf_rn(v[y].z, f, m.o.z);
    m.o.w = __fmaf_rn(v[y].w, f, m.o.w);
  }
}

// A row's result: four columns of an output row, and its statistics.
template <int NB>
__device__ __forceinline__ void put_out(const AttnArgs& a, const Unit& u, int row, int col, float ref, float inv, float4 o) {
  const size_t out_row = (static_cast<size_t>(u.b) * a.n_tokens + row / a.group) * a.n_heads +
                         static_cast<size_t>(u.h) * a.group + row % a.group;
  float4* dst = reinterpret_cast<float4*>(a.out + out_row * (32 * NB) + col);
  const float4 x = make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
  if ((reinterpret_cast<uintptr_t>(a.out) & 15) == 0) {
    *dst = x;
  } else {
    float* d = reinterpret_cast<float*>(dst);
    d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w;
  }
  if (a.stats && col == 0) a.stats[out_row] = make_float2(ref, inv);
}

// Merges `parts` partial results of a unit's rows ([n_rows][hd sums, reference,
// sum of P, 2 unused] at src(p)) in order, into the outputs and statistics or
// (to given) one more partial result: places [i0, n) of rows and groups of four
// columns, by the block's threads.  SHARED: the parts are in shared memory; else each
// thread has kMergeItems places' loads of four parts in flight.
constexpr int kMergeItems = 2;
template <int NB, bool SHARED, typename Src>
__device__ __forceinline__ void merge_rows(const AttnArgs& a, const Unit& u, int parts, Src src, float* to, int i0, int n) {
  constexpr int HD = 32 * NB, PR = HD + 4, Y = SHARED ? 1 : kMergeItems;
#pragma unroll 1
  for (i0 += threadIdx.x; i0 < n; i0 += Y * blockDim.x) {
    Merged m[Y];
#pragma unroll
    for (int y = 0; y < Y; ++y) m[y] = Merged{-INFINITY, 0.0f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if constexpr (SHARED) {
      for (int p = 0; p < parts; ++p) {
        const float* s = src(p) + static_cast<size_t>(i0 / (HD / 4)) * PR;
        const float2 st[1] = {*reinterpret_cast<const float2*>(s + HD)};
        const float4 v[1] = {*reinterpret_cast<const float4*>(s + 4 * (i0 % (HD / 4)))};
        merge_into(m[0], st, v);
      }
    } else {
      for (int p0 = 0; p0 < parts; p0 += 4) {
        float2 st[Y][4];
        float4 v[Y][4];
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          const int i = i0 + y * blockDim.x;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            st[y][p] = make_float2(-INFINITY, 0.0f);
            v[y][p] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p0 + p < parts && i < n) {
              const float* s = src(p0 + p) + static_cast<size_t>(i / (HD / 4)) * PR;
              st[y][p] = __ldcg(reinterpret_cast<const float2*>(s + HD));
              v[y][p] = __ldcg(reinterpret_cast<const float4*>(s + 4 * (i % (HD / 4))));
            }
          }
        }
#pragma unroll
        for (int y = 0; y < Y; ++y) merge_into(m[y], st[y], v[y]);
      }
    }
#pragma unroll
    for (int y = 0; y < Y; ++y) {
      const int i = i0 + y * blockDim.x, rr = i / (HD / 4), d4 = i % (HD / 4);
      if (i >= n) break;
      if (to) {
        float* dst = to + static_cast<size_t>(rr) * PR;
        __stcg(reinterpret_cast<float4*>(dst + 4 * d4), m[y].o);
        if (d4 == 0) __stcg(reinterpret_cast<float2*>(dst + HD), make_float2(m[y].ref, m[y].sum));
        continue;
      }
      const int row = u.rg * a.n_rows + rr;
      if (row < a.rows)
        put_out<NB>(a, u, row, 4 * d4, m[y].ref, m[y].ref == -INFINITY ? 0.0f : __fdiv_rn(1.0f, m[y].sum), m[y].o);
    }
  }
}

// The part of a unit, whose first block is c0, that block cta holds.
template <int NB>
__device__ __forceinline__ float* part_at(const AttnArgs& a, int cta, int c0) {
  return a.part + static_cast<size_t>(cta == c0 ? 2 * cta + 1 : 2 * cta) * a.n_rows * (32 * NB + 4);
}

// R = 1: 8 rows, four warps with a ring each, whose results meet in shared memory;
// stages of 32 keys; the block that finishes a unit merges its parts.  R = 2: a warp
// for each 16 rows, one ring; stages of 64 keys; results go from registers to memory,
// and a kernel of its own merges what several blocks had a part in (the last block
// alone took 30K clocks for 40 rows of 128).
// Bound by instruction issue at three warps of 168 registers a scheduler.  24 x 8 heads
// of up to 32K keys, 8 rows of 128: 153 us, 3.0 TB/s, 53 % of issue slots.  16 x 8
// heads of up to 4K keys, 40 rows: 82 us (all 8 rows a warp: 107).  2 x 32 heads of 64,
// 509 rows: 111 us (8 rows a warp: 159).
template <int NB, int R>
__global__ void __launch_bounds__(kMaxWarps * 32, 3) kv4_attend_kernel(AttnArgs a) {
  constexpr int KEYS = R * kStep, kFlushStages = kFlushKeys / R / KEYS;  // 16 rows: twice the products a key
  constexpr int HD = 32 * NB, PR = HD + 4;  // floats of a partial row
  constexpr int SB = stage_bytes<NB, KEYS>();
  static_assert(R == 2 || 8 * PR * sizeof(float) <= SB, "a warp's rows fit a stage");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Plan plan;
  __shared__ Unit ahead[kMaxWarps];
  __shared__ unsigned sh[kMaxWarps];
  __shared__ uint64_t full[kMaxWarps * kMaxStages], empty[kMaxWarps * kMaxStages];
  __shared__ int free_slot[kMaxWarps];
  __shared__ int last_block;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp % a.row_tiles, wk = warp / a.row_tiles;
  const int n_rows = a.n_rows;
  uint8_t* ring = smem + wk * a.stages * SB;
  float* scales_sh = reinterpret_cast<float*>(smem + a.splits * a.stages * SB) + warp * (2 * kStep * NB);
  uint4* queries_sh = reinterpret_cast<uint4*>(smem + a.splits * a.stages * SB + (blockDim.x / 32) * (2 * kStep * NB * sizeof(float))) +
                      warp * WarpQueries<NB, R>::kSharedItems;
  if (threadIdx.x < a.splits * a.stages) {
    mri::mbar_init(&full[threadIdx.x], 1);
    mri::mbar_init(&empty[threadIdx.x], a.row_tiles);
    mri::fence_barrier_init();
  }
  pdl_enter();
  make_plan(a, &plan, sh);
  const int count = plan.count;
  if (count == 0) return;
  uint64_t* fullw = full + wk * a.stages;
  uint64_t* emptyw = empty + wk * a.stages;
  // Ring wk holds the block's stages wk, wk + splits, ...; the first four lanes of its
  // first warp issue them (key codes, value codes, key scales, value scales), stages - 1
  // ahead, across units.
  const bool producer = wr == 0;
  bool dead = false;  // a wait gave up: nothing more is issued or read
  int next = wk, issued = 0, slot = 0, stop = 0;  // stop: end of the stages that src reaches by stepping
  unsigned slot_parity = 0;
  const uint8_t* src = nullptr;  // this lane's part of the stage `next`
  const int width = lane < 2 ? 16 * NB : 2 * NB;  // bytes a row of this lane's part
  const int step = a.splits * KEYS * width;
  uint8_t* const dst = ring + (lane < 2 ? lane * (KEYS * NB * 16) : (28 + 2 * lane) * (KEYS * NB));
  auto issue = [&](bool reused) {
    if (next >= stop) {
      if (next >= count) return;
      __syncwarp();
      if (lane == 0) next = seek_stage(a, ahead[wk], next, count);
      __syncwarp();  // lane 0's unit is read by all lanes: a shuffle alone orders no memory
      next = __shfl_sync(0xffffffffu, next, 0);
      if (next >= count) return;
      const Unit& v = ahead[wk];
      stop = min(count, v.end);
      const uint8_t* base = lane == 0 ? a.c.k : lane == 1 ? a.c.v : reinterpret_cast<const uint8_t*>(lane == 2 ? a.c.ks : a.c.vs);
      src = base + a.c.row(v.b, v.h, static_cast<size_t>(next - (v.end - v.tiles + a.pad)) * KEYS) * width;
    }
    // A ring of one warp needs no "empty" barriers: the warp itself has read the slot.
    if (a.row_tiles > 1 && reused) {
      if (!dead && !mri::mbar_wait(&emptyw[slot], slot_parity, a.status)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
    }
    if (dead) return;
    if (lane == 0) mri::mbar_arrive_expect_tx(&fullw[slot], SB);
    __syncwarp();
    if (lane < 4) mri::bulk_copy_g2s(dst + slot * SB, src, KEYS * width, &fullw[slot]);
    src += step;
    next += a.splits;
    ++issued;
    if (++slot == a.stages) {
      slot = 0;
      if (reused) slot_parity ^= 1;
    }
  };
  if (producer) {
    if (lane == 0) ahead[wk] = plan.first;
    for (int i = 0; i < a.stages - 1; ++i) issue(false);
  }

  Unit u = plan.first;
  int x = 0, unit_begin, seg_end;  // the unit's stages of this block: [x, seg_end)
  int s = 0, used = 0;             // s: the ring's next slot
  unsigned parity = 0;
  while (next_segment(a, u, x, count, unit_begin, seg_end)) {
    const int row = u.rg * n_rows + wr * (8 * R) + g;
    const int len = a.len(u.b);
    WarpQueries<NB, R> q;
    q.load(a, u.b, u.h, row, queries_sh);
    RowState<NB, R> r;
#pragma unroll
    for (int n = 0; n < NB * 4; ++n) r.o[n][0] = r.o[n][1] = r.o[n][2] = r.o[n][3] = 0.0f;
    int row_end[R];
    // Stages that end by `clear` need no mask for any live row of the warp.
    int clear = INT32_MAX;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int x = row + 8 * i;
      row_end[i] = x < a.rows ? len - a.n_tokens + 1 + x / a.group : 0;
      if (x < a.rows) clear = min(clear, row_end[i]);
      r.m[i] = -INFINITY;
      r.ref[i] = 0.0f;
      r.l[i] = 0;
    }
    r.scaled.init();
    FlushedSums<NB, R> flushed;
    flushed.init();
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) clear = min(clear, __shfl_xor_sync(0xffffffffu, clear, o));
    // From the first of this ring's stages at or after x.
    for (int y = x + (a.splits + wk - x % a.splits) % a.splits; y < seg_end; y += a.splits) {
      if (producer) issue(used >= 1);
      if (used % kFlushStages == kFlushStages - 1) flushed.flush(r);
      ++used;
      if (!dead && !mri::mbar_wait(&fullw[s], parity, a.status)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (!dead) {
        const int k0 = (y - unit_begin) * KEYS;
        if (k0 + KEYS > clear)
          stage_keys<NB, R, KEYS, true>(ring + s * SB, scales_sh, k0, len, row_end, q, r, flushed);
        else
          stage_keys<NB, R, KEYS, false>(ring + s * SB, scales_sh, k0, len, row_end, q, r, flushed);
      }
      __syncwarp();
      if (a.row_tiles > 1 && lane == 0) mri::mbar_arrive(&emptyw[s]);
      if (++s == a.stages) {
        s = 0;
        parity ^= 1;
      }
    }
    if (flushed.any()) flushed.flush(r);
    const bool whole = x == unit_begin && seg_end == u.end;
    // Where this block's part of the unit goes if others have one too.
    const int c0 = owner_of(plan, plan.x0 + static_cast<unsigned>(unit_begin)),
              c1 = owner_of(plan, plan.x0 + static_cast<unsigned>(u.end - 1));
    auto part_of = [&](int cta) { return part_at<NB>(a, cta, c0); };
    // R = 1: the warp's rows go into the ring's slot that was consumed last, the one
    // that is issued next.
    auto rows_of = [&](int p) -> float* { return reinterpret_cast<float*>(smem + (p * a.stages + free_slot[p]) * SB); };
    if (R == 1) {
      if (lane == 0) free_slot[wk] = (s + a.stages - 1) % a.stages;
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float2 l2 = unpair2(r.l[i]);
      float l = __fadd_rn(l2.x, l2.y);
      l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 1));
      l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 2));
      const float ref = r.m[i] == -INFINITY && l == l ? -INFINITY : r.ref[i];  // -inf: no key seen
      const float inv = ref == -INFINITY ? 0.0f : __fdiv_rn(1.0f, l);
      float* mine = (R == 1 ? rows_of(wk) : part_of(static_cast<int>(blockIdx.x))) + (wr * (8 * R) + 8 * i + g) * PR;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // odd places of each four were 16-fold
          const float unit = r.scaled.inverse(b), part = __fmul_rn(unit, 0.0625f);
          float4 v;
          v.x = __fmul_rn(flushed.total(r, 4 * b, i, c), unit);
          v.y = __fmul_rn(flushed.total(r, 4 * b + 1, i, c), part);
          v.z = __fmul_rn(flushed.total(r, 4 * b + 2, i, c), unit);
          v.w = __fmul_rn(flushed.total(r, 4 * b + 3, i, c), part);
          const int col = 32 * b + 8 * t + 4 * c;
          if (R == 1)
            *reinterpret_cast<float4*>(mine + col) = v;
          else if (!whole)
            __stcg(reinterpret_cast<float4*>(mine + col), v);
          else if (row + 8 * i < a.rows)
            put_out<NB>(a, u, row + 8 * i, col, ref, inv, v);
        }
      if (t == 0 && (R == 1 || !whole)) {
        mine[HD] = ref;
        mine[HD + 1] = l;
      }
    }
    if (R == 2 && x == unit_begin && threadIdx.x == 0)
      a.spans[(static_cast<size_t>(u.b) * a.row_groups + u.rg) * a.c.heads + u.h] = make_int2(c0, c1);
    if constexpr (R == 1) {
      __syncthreads();
      const int places = n_rows * (HD / 4);
      merge_rows<NB, true>(a, u, a.splits, rows_of, whole ? nullptr : part_of(static_cast<int>(blockIdx.x)), 0, places);
      if (!whole) {
        // This block's part is in memory; the block that arrives last merges all.
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          last_block = atomicAdd(&a.ready[c0], 1u) == static_cast<unsigned>(c1 - c0);
          if (last_block) a.ready[c0] = 0;
        }
        __syncthreads();
        if (last_block) {
          __threadfence();
          merge_rows<NB, false>(a, u, c1 - c0 + 1, [&](int p) { return part_of(c0 + p); }, nullptr, 0, places);
        }
      }
      // The slots were written by threads; the next copies into them are asynchronous.
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
    }
    x = seg_end;
    next_unit(a, u);
  }
  // After a wait that gave up: the copies still in flight end before the block does.
  if (producer && dead)
    for (int n = max(0, issued - a.stages); n < issued; ++n)
      mri::mbar_wait(&fullw[n % a.stages], (n / a.stages) & 1, a.status);
}

// What several blocks have a part in, after the first kernel (R = 2): kMergeThreads x
// kMergeItems places a block, so that all SMs read parts.  Bound by latency: three
// rounds of loads.
constexpr int kMergeThreads = 128;
template <int NB>
__global__ void __launch_bounds__(kMergeThreads) kv4_merge_kernel(AttnArgs a, unsigned blocks_per_unit) {
  pdl_enter();
  const unsigned unit = blockIdx.x / blocks_per_unit, pair = unit / static_cast<unsigned>(a.c.heads);
  const int2 span = mri::ld_act(a.spans + unit);
  const int c0 = span.x, c1 = span.y;
  // One block's, or (lengths that changed) no block began the unit.
  if (static_cast<unsigned>(c0) >= static_cast<unsigned>(c1) || static_cast<unsigned>(c1) >= a.grid) return;
  const unsigned groups = static_cast<unsigned>(a.row_groups);
  const Unit u{static_cast<int>(pair / groups), static_cast<int>(pair % groups), static_cast<int>(unit % static_cast<unsigned>(a.c.heads)), 0, 0};
  const int i0 = static_cast<int>(blockIdx.x % blocks_per_unit) * (kMergeThreads * kMergeItems);
  merge_rows<NB, false>(a, u, c1 - c0 + 1, [&](int p) { return part_at<NB>(a, c0 + p, c0); }, nullptr, i0,
                        min(a.n_rows * (8 * NB), i0 + kMergeThreads * kMergeItems));
}

// Tracked calls, second pass: with every row's reference and sum known, a warp
// scores keys of one head against all rows that see them (the same products as
// above) and adds each key's weights, rows in order, to its total: no atomics, one
// owner a key.  Two forms, by which operand is worth keeping in registers:
//   up to 8 rows (a decode step): the queries, over kTrackRun keys a warp;
//   more: 32 unpacked keys, over all rows, whose A fragments a small kernel has
//   prepared once (splitting 8 rows' queries costs twice what scoring them does).
// 8 x 8 heads of 4001 to 8192 keys, 4 rows: 22 us (35 with the second form alone); 2 x
// 32 heads of 1021 to 2048 keys, 509 rows: 70 us (170 with the queries split by every
// warp; 16 keys a warp 104, fragments by way of shared memory 75).
constexpr int kTrackWarps = 4;
constexpr int kTrackRun = 128;

// The lane's weight sums of keys key0 + 8 j + 2t, + 1 over the rows g, added to the totals.
template <int TILES>
__device__ __forceinline__ void add_weights(float* weight, int key0, int len, float (&sum)[TILES][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < TILES; ++j) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) sum[j][i] = __fadd_rn(sum[j][i], __shfl_xor_sync(0xffffffffu, sum[j][i], o));
    const int key = key0 + 8 * j + 2 * t;
    if (g == j) {
      float* w = weight + 8 * j + 2 * t;
      if (key < len) w[0] = __fadd_rn(w[0], sum[j][0]);
      if (key + 1 < len) w[1] = __fadd_rn(w[1], sum[j][1]);
    }
  }
}

// The scales of keys 2t, 2t + 1 of 8 keys from cache row `row` on.
template <int NB>
__device__ __forceinline__ void load_key_scales(const Cache& c, size_t row, f32x2 (&ks)[NB]) {
  const int t = threadIdx.x & 3;
  uint32_t raw[NB];
  load_words<NB>(reinterpret_cast<const uint8_t*>(c.ks + (row + 2 * t) * NB), raw);
#pragma unroll
  for (int b = 0; b < NB; ++b)  // halves [key][block] of two keys
    ks[b] = pair2(mri::f16_bits_to_f32(b & 1 ? raw[b / 2] >> 16 : raw[b / 2]),
                  mri::f16_bits_to_f32((NB + b) & 1 ? raw[(NB + b) / 2] >> 16 : raw[(NB + b) / 2]));
}

// Row r of a head: the key it sees up to, and its statistics (or nothing).
__device__ __forceinline__ float2 row_stats(const AttnArgs& a, int b, int h, int row, int len, int* end) {
  *end = 0;
  if (row >= a.rows) return make_float2(0.0f, 0.0f);
  *end = len - a.n_tokens + 1 + row / a.group;
  return mri::ld_act(a.stats + (static_cast<size_t>(b) * a.n_tokens + row / a.group) * a.n_heads +
                     static_cast<size_t>(h) * a.group + row % a.group);
}

template <int NB>
__global__ void __launch_bounds__(kTrackWarps * 32) kv4_track_few_kernel(AttnArgs a, unsigned blocks_per_head) {
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const unsigned head = blockIdx.x / blocks_per_head;
  const int h = static_cast<int>(head % a.c.heads), b = static_cast<int>(head / a.c.heads);
  const int len = a.len(b);
  const int64_t first = (static_cast<int64_t>(blockIdx.x % blocks_per_head) * kTrackWarps + warp) * kTrackRun;
  if (first >= len) return;
  QueryTile<NB> q;
  load_queries<NB>(a, b, h, g, q);
  int end;
  const float2 st = row_stats(a, b, h, g, len, &end);
#pragma unroll 1
  for (int key0 = static_cast<int>(first); key0 < min(len, static_cast<int>(first) + kTrackRun); key0 += 32) {
    const size_t row0 = a.c.row(b, h, static_cast<size_t>(key0));
    uint32_t kw[4][NB];
    f32x2 ks[4][NB];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      load_words<NB>(a.c.k + (row0 + 8 * j + g) * (16 * NB) + t * (4 * NB), kw[j]);
      load_key_scales<NB>(a.c, row0 + 8 * j, ks[j]);
    }
    float sum[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 z = unpair2(score8<NB>(q, kw[j], ks[j]));
      const int key = key0 + 8 * j + 2 * t;
      sum[j][0] = key < end ? __fmul_rn(exp2_fast(__fsub_rn(__fmul_rn(z.x, q.mult), st.x)), st.y) : 0.0f;
      sum[j][1] = key + 1 < end ? __fmul_rn(exp2_fast(__fsub_rn(__fmul_rn(z.y, q.mult), st.x)), st.y) : 0.0f;
    }
    add_weights(a.c.weight + row0, key0, len, sum);
  }
}

// Every 8-row tile's A fragments [block][step][lane] (16 bytes), and of each row
// its score factor, reference, 1 / sum and the key it sees up to.
template <int NB>
__global__ void __launch_bounds__(kTrackWarps * 32) kv4_fragments_kernel(AttnArgs a, uint4* __restrict__ frags,
                                                                         float4* __restrict__ about, unsigned tiles) {
  pdl_enter();
  const unsigned tile = blockIdx.x * kTrackWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (tile >= tiles) return;
  const unsigned per = static_cast<unsigned>((a.rows + 7) / 8), head = tile / per;
  const int entry = static_cast<int>(head / a.c.heads), h = static_cast<int>(head % a.c.heads);
  const int row = static_cast<int>(tile % per) * 8 + (lane >> 2);
  QueryTile<NB> q;
  load_queries<NB>(a, entry, h, row, q);
  int end;
  const float2 st = row_stats(a, entry, h, row, a.len(entry), &end);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      frags[(static_cast<size_t>(tile) * (2 * NB) + 2 * b + i) * 32 + lane] = make_uint4(q.a[b][i][0], q.a[b][i][1], q.a[b][i][2], q.a[b][i][3]);
  if ((lane & 3) == 0) about[static_cast<size_t>(tile) * 8 + (lane >> 2)] = make_float4(q.mult, st.x, st.y, __int_as_float(end));
}

template <int NB>
__global__ void __launch_bounds__(kTrackWarps * 32) kv4_track_many_kernel(AttnArgs a, const uint4* __restrict__ frags,
                                                                          const float4* __restrict__ about,
                                                                          unsigned blocks_per_head) {
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const unsigned head = blockIdx.x / blocks_per_head;
  const int h = static_cast<int>(head % a.c.heads), b = static_cast<int>(head / a.c.heads);
  const int64_t first = (static_cast<int64_t>(blockIdx.x % blocks_per_head) * kTrackWarps + warp) * 32;
  const int len = a.len(b);
  if (first >= len) return;
  const int key0 = static_cast<int>(first);
  const size_t row0 = a.c.row(b, h, static_cast<size_t>(key0));
  uint32_t codes[4][NB][4];
  f32x2 ks[4][NB];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t kw[NB];
    load_words<NB>(a.c.k + (row0 + 8 * j + g) * (16 * NB) + t * (4 * NB), kw);
    load_key_scales<NB>(a.c, row0 + 8 * j, ks[j]);
#pragma unroll
    for (int bl = 0; bl < NB; ++bl) {
      codes[j][bl][0] = low_codes(kw[bl]);
      codes[j][bl][1] = low_codes(kw[bl] >> 8);
      codes[j][bl][2] = high_codes(kw[bl]);
      codes[j][bl][3] = high_codes(kw[bl] >> 8);
    }
  }
  float sum[4][2] = {};
  // Row r sees keys before len - n_tokens + 1 + r / group.
  const int64_t token0 = max(int64_t{0}, static_cast<int64_t>(key0) - (len - a.n_tokens));
  const int from = static_cast<int>(min(token0 * a.group, static_cast<int64_t>(a.rows)));
  const unsigned tiles = static_cast<unsigned>((a.rows + 7) / 8);
  // What is known of the next tile's rows is on its way while this one is scored.
  const size_t tile0 = static_cast<size_t>(head) * tiles;
  float4 ahead = from < a.rows ? mri::ld_act(about + (tile0 + from / 8) * 8 + g) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int r0 = from & ~7; r0 < a.rows; r0 += 8) {
    const size_t tile = tile0 + r0 / 8;
    const float4 now = ahead;
    if (r0 + 8 < a.rows) ahead = mri::ld_act(about + (tile + 1) * 8 + g);
    const float mult = now.x;
    const float2 st = make_float2(now.y, now.z);
    const int end = __float_as_int(now.w);
    f32x2 z[4];
#pragma unroll
    for (int bl = 0; bl < NB; ++bl) {
      const uint4 f0 = mri::ld_act(frags + (tile * (2 * NB) + 2 * bl) * 32 + lane);
      const uint4 f1 = mri::ld_act(frags + (tile * (2 * NB) + 2 * bl + 1) * 32 + lane);
      const uint32_t a0[4] = {f0.x, f0.y, f0.z, f0.w}, a1[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float d[4];
        mma16816_first(d, a0, codes[j][bl][0], codes[j][bl][1]);
        mma16816(d, a1, codes[j][bl][2], codes[j][bl][3]);
        const f32x2 both = add2(pair2(d[0], d[1]), pair2(d[2], d[3]));
        z[j] = bl == 0 ? mul2(ks[j][bl], both) : fma2(ks[j][bl], both, z[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = unpair2(z[j]);
      const int key = key0 + 8 * j + 2 * t;
      const float p0 = __fmul_rn(exp2_fast(__fsub_rn(__fmul_rn(v.x, mult), st.x)), st.y);
      const float p1 = __fmul_rn(exp2_fast(__fsub_rn(__fmul_rn(v.y, mult), st.x)), st.y);
      if (key < end) sum[j][0] = __fadd_rn(sum[j][0], p0);
      if (key + 1 < end) sum[j][1] = __fadd_rn(sum[j][1], p1);
    }
  }
  add_weights(a.c.weight + row0, key0, len, sum);
}

template <int NB>
int launch_attention(mri_ctx* ctx, AttnArgs a, bool track) {
  // Up to 8 rows (a decode step): one warp a ring, its A fragments the queries' high
  // and low parts.  More: 16 rows a warp, which unpacks the keys once for all of them.
  const bool few = a.rows <= 8;
  const int tile = few ? 8 : 16, tiles = (a.rows + tile - 1) / tile;
  const int most = NB > 2 ? 3 : kMaxWarps;
  a.row_groups = (tiles + most - 1) / most;
  a.row_tiles = (tiles + a.row_groups - 1) / a.row_groups;
  a.row_groups = (tiles + a.row_tiles - 1) / a.row_tiles;
  a.n_rows = a.row_tiles * tile;
  a.splits = few ? kMaxWarps : 1;
  const int warps = a.row_tiles * a.splits, threads = warps * 32;
  const size_t part_row = 32 * NB + 4;
  // Stages of 64 keys where warps share rings and what a stage costs besides its keys
  // (40 rows, 8 a warp: 126 us with 32, 110 with 64); of 32 where a block has four rings
  // (ragged batch: 180 and 189: with 64 two slots of each fit, and shares round to more keys).
  // At most three tiles of 96 or 128 wide heads: four warps' queries would leave room
  // for one stage.
  a.keys = few ? kStep : 2 * kStep;
  const auto kernel = few ? kv4_attend_kernel<NB, 1> : kv4_attend_kernel<NB, 2>;
  // A unit's queries, results and merge take as long as some of its stages, so shares
  // of equal stages are not of equal time.  24 x 8 heads of up to 32K keys: 192 us
  // counting stages alone, 152 with 12 more, 153 with 20; 40 rows (drafts, 16 x 8
  // heads of up to 4K keys): 115 us, 93 with 1, 87 with 2, 88 with 4.
  a.pad = few ? 12 : 2;
  const size_t stage = static_cast<size_t>(a.keys) * NB * 36;
  const size_t scales = warps * 2 * kStep * NB * sizeof(float);
  const size_t queries = few ? 0 : warps * WarpQueries<NB, 2>::kSharedItems * sizeof(uint4);
  // A block's share of the SM by its warps; a lone 16-row tile takes what two stages need.
  const size_t block_bytes = std::max(kBlockBytes / 4 * warps, scales + queries + 2 * a.splits * stage);
  a.stages = std::min<int>(kMaxStages, static_cast<int>((block_bytes - scales - queries) / (a.splits * stage)));
  const size_t smem = static_cast<size_t>(a.splits) * a.stages * stage + scales + queries;
  const size_t stages = ((a.c.cap + a.keys - 1) / a.keys + a.pad) * a.c.heads;
  if (stages > UINT32_MAX / (static_cast<size_t>(a.c.batch) * a.row_groups))
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_attention: cache and rows too large for one call");
  int& fit = ctx->kv4_fit[NB - 1][few ? 0 : a.row_tiles];  // blocks that fit an SM; asked for once
  if (fit == 0) {
    KV4_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kBlockBytes)));
    KV4_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, smem));
    fit = std::max(1, fit);
  }
  const unsigned grid = std::min<unsigned>(static_cast<unsigned>(fit) * ctx->dev.sm_count, mri_ctx::kSyncAttnBlocks);
  const size_t part_bytes = (2 * grid * a.n_rows * part_row * sizeof(float) + 255) / 256 * 256;
  const size_t all_rows = static_cast<size_t>(a.c.batch) * a.n_tokens * a.n_heads;
  const size_t stat_bytes = track ? (all_rows * sizeof(float2) + 255) / 256 * 256 : 0;
  const size_t q_tiles = static_cast<size_t>(a.c.batch) * a.c.heads * ((a.rows + 7) / 8);  // of 8 rows
  const size_t frag_bytes = track && !few ? q_tiles * (2 * NB * 32 * sizeof(uint4) + 8 * sizeof(float4)) : 0;
  const size_t units = static_cast<size_t>(a.c.batch) * a.row_groups * a.c.heads;
  const size_t span_bytes = few ? 0 : (units * sizeof(int2) + 255) / 256 * 256;
  if (int rc = mri::ctx_reserve_scratch(ctx, part_bytes + stat_bytes + span_bytes + frag_bytes)) return rc;
  a.part = reinterpret_cast<float*>(ctx->scratch);
  a.stats = track ? reinterpret_cast<float2*>(ctx->scratch + part_bytes) : nullptr;
  a.spans = reinterpret_cast<int2*>(ctx->scratch + part_bytes + stat_bytes);
  a.ready = ctx->d_sync + mri_ctx::kSyncAttn;
  a.grid = grid;
  a.status = ctx->d_status;
  KV4_CUDA_TRY(launch(ctx, kernel, grid, threads, smem, a));
  if (!few) {
    const unsigned per = static_cast<unsigned>((a.n_rows * 8 * NB + kMergeThreads * kMergeItems - 1) / (kMergeThreads * kMergeItems));
    const size_t blocks = units * per;
    if (blocks > (size_t{1} << 31) - 1)
      return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_attention: cache and rows too large for one call");
    KV4_CUDA_TRY(launch(ctx, kv4_merge_kernel<NB>, static_cast<unsigned>(blocks), kMergeThreads, 0, a, per));
  }
  if (track) {
    const size_t keys = kTrackWarps * (few ? kTrackRun : 32);
    const size_t per_head = (a.c.cap + keys - 1) / keys, blocks = per_head * a.c.heads * a.c.batch;
    if (blocks > (size_t{1} << 31) - 1)
      return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_attention: cache too large for one tracked call");
    const unsigned grid_t = static_cast<unsigned>(blocks), per = static_cast<unsigned>(per_head);
    if (few) {
      KV4_CUDA_TRY(launch(ctx, kv4_track_few_kernel<NB>, grid_t, kTrackWarps * 32, 0, a, per));
    } else {
      uint4* frags = reinterpret_cast<uint4*>(ctx->scratch + part_bytes + stat_bytes + span_bytes);
      float4* about = reinterpret_cast<float4*>(frags + q_tiles * (2 * NB) * 32);
      KV4_CUDA_TRY(launch(ctx, kv4_fragments_kernel<NB>, static_cast<unsigned>((q_tiles + kTrackWarps - 1) / kTrackWarps),
                          kTrackWarps * 32, 0, a, frags, about, static_cast<unsigned>(q_tiles)));
      KV4_CUDA_TRY(launch(ctx, kv4_track_many_kernel<NB>, grid_t, kTrackWarps * 32, 0, a,
                          static_cast<const uint4*>(frags), static_cast<const float4*>(about), per));
    }
  }
  return MRI_OK;
}

// ── eviction ─────────────────────────────────────────────────────────────────

// A weight as an unsigned number of the same order; what is not a positive
// number counts as 0.
__device__ __forceinline__ uint32_t weight_key(float w) { return w > 0.0f ? __float_as_uint(w) : 0u; }

// One cluster of blocks per (entry, head).  Selection: the budget - recent largest of
// the older keys' weights, by a radix search for the smallest kept weight (four
// histograms, of 8, 8, 8 and 7 bits).  The blocks split the keys, count into their
// own shared memory and add up all blocks' counts from there; then every thread
// counts and places the kept of a run of consecutive keys, so that they come out in
// order; of keys equal to that weight the first ones stay.  The weights are read
// once where they fit shared memory.  Then the blocks split the kept rows evenly
// and move them, 8 threads a row, in pieces of 16 bytes, kMoveRows rows in flight.
// The selection is bound by latency (five cluster barriers and four walks of its
// share a thread), the move by HBM.
constexpr int kMaxCluster = 8, kSelThreads = 512;
constexpr int kSelRounds = 4, kSelBins = 256;
constexpr int kSelKeys = 40960;  // weights a block holds in shared memory at most
constexpr int kMoveRows = 2;

struct SelectShared {
  uint32_t hist[kSelRounds][kSelBins];  // one a round: other blocks read it until the next barrier but one
  unsigned long long totals[kMaxCluster];
  unsigned long long sums[kSelThreads / 32];
  uint32_t digit, above;
};
// A held key's place: runs of a thread's keys do not meet in one bank.
__host__ __device__ constexpr int held_at(int i) { return i + (i >> 5); }

// The sum of the warps' totals before this warp's.
__device__ __forceinline__ unsigned long long sum_before(const unsigned long long* sums, int warp, int lane) {
  unsigned long long v = lane < warp ? sums[lane] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Positions kept of one head to out, by the whole cluster.  old: candidates, keys
// [0, old); want: how many of them stay (0 < want < old).
__device__ __forceinline__ void select_keys(SelectShared& sh, uint32_t* held, int hold, const float* w, int old,
                                            uint32_t want, int rank, int blocks, int32_t* out) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = ((old + blocks - 1) / blocks + 3) & ~3;
  const int k0 = min(old, rank * per), count = min(old - k0, per);
  const bool in_shared = per <= hold;
  w += k0;
  auto key_of = [&](int i) { return in_shared ? held[held_at(i)] : weight_key(mri::ld_act(w + i)); };
  // thr: the digits found of the smallest kept weight; left: how many of the keys
  // that begin with them stay.
  uint32_t thr = 0, left = want;
#pragma unroll 1
  for (int round = 0; round < kSelRounds; ++round) {
    // The sign is 0: the exponent's 8 bits, then 8, 8 and 7.
    const int shift = round == 3 ? 0 : 23 - 8 * round, bits = round == 3 ? 7 : 8;
    uint32_t* hist = sh.hist[round];
    auto add = [&](uint32_t key) {
      const uint32_t d = (key >> shift) & ((1u << bits) - 1u);
      // Where all lanes have the same digit (unused keys weigh 0), one atomic.
      const unsigned on = __activemask();
      int same;
      __match_all_sync(on, d, &same);
      if (!same)
        atomicAdd(&hist[d], 1u);
      else if (lane == __ffs(on) - 1)
        atomicAdd(&hist[d], static_cast<uint32_t>(__popc(on)));
    };
    if (round == 0) {
      // 16-byte loads, four in flight: a head's weights start 256-byte aligned, and
      // a share is a multiple of four keys.
#pragma unroll 4
      for (int i = 4 * tid; i < count; i += 4 * kSelThreads) {
        const float4 q = mri::ld_act(reinterpret_cast<const float4*>(w + i));
        const uint32_t key[4] = {weight_key(q.x), weight_key(q.y), weight_key(q.z), weight_key(q.w)};
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (i + y < count) {
            if (in_shared) held[held_at(i + y)] = key[y];
            add(key[y]);
          }
      }
    } else {
      const uint32_t prefix = thr >> (shift + bits);
      for (int i = tid; i < count; i += kSelThreads) {
        const uint32_t key = key_of(i);
        if (key >> (shift + bits) == prefix) add(key);
      }
    }
    mri::cluster_sync();
    // From the top: the bin where the count of larger keys first reaches `left`.
    // Thread t holds bin 255 - t.
    uint32_t mine = 0;
    if (tid < kSelBins) {
      uint32_t v[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        v[r] = 0;
        if (r < blocks)
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(mri::cluster_addr(hist + kSelBins - 1 - tid, r)));
      }
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) mine += v[r];
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh.sums[warp] = incl;
    __syncthreads();
    const uint32_t before = incl - mine + static_cast<uint32_t>(sum_before(sh.sums, warp, lane));
    if (before < left && before + mine >= left) {
      sh.digit = kSelBins - 1 - tid;
      sh.above = before;
    }
    __syncthreads();
    thr |= sh.digit << shift;
    left -= sh.above;
  }
  // Every thread's run of keys: how many lie above the threshold and at it.
  const int each = (count + kSelThreads - 1) / kSelThreads;
  const int i0 = min(count, tid * each), i1 = min(count, i0 + each);
  uint32_t above = 0, ties = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t key = key_of(i);
    above += key > thr;
    ties += key == thr;
  }
  const unsigned long long mine = (static_cast<unsigned long long>(above) << 32) | ties;
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.sums[warp] = incl;
  __syncthreads();
  unsigned long long before = incl - mine + sum_before(sh.sums, warp, lane);
  // The block's total to every block after it (the last thread's inclusive one).
  if (tid == kSelThreads - 1)
    for (int r = rank + 1; r < blocks; ++r)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mri::cluster_addr(&sh.totals[rank], r)), "l"(before + mine) : "memory");
  mri::cluster_sync();
  for (int r = 0; r < rank; ++r) before += sh.totals[r];
  uint32_t tie = static_cast<uint32_t>(before);
  uint32_t at = static_cast<uint32_t>(before >> 32) + min(tie, left);
  if (above + ties > 0)
    for (int i = i0; i < i1; ++i) {
      const uint32_t key = key_of(i);
      if (key > thr || (key == thr && tie < left)) out[at++] = k0 + i;
      tie += key == thr;
    }
}

// Rows r0, r0 + step, ... below end of a head to their new places: 8 threads a row, in
// pieces of 16 bytes, kMoveRows rows in flight.
template <int NB>
__device__ __forceinline__ void move_rows(const Cache& src, const Cache& dst, size_t head, const int32_t* out, int r0,
                                          int end, int step) {
  const int part = threadIdx.x & 7;
  for (; r0 < end; r0 += kMoveRows * step) {
    int32_t from[kMoveRows];
#pragma unroll
    for (int y = 0; y < kMoveRows; ++y) {
      const int r = r0 + y * step;
      from[y] = r < end ? mri::ld_act(out + r) : -1;
    }
    uint4 k[kMoveRows], v[kMoveRows];
    uint16_t sc[kMoveRows][NB];
    float w[kMoveRows];
#pragma unroll
    for (int y = 0; y < kMoveRows; ++y) {
      k[y] = v[y] = make_uint4(0u, 0u, 0u, 0u);
      w[y] = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b) sc[y][b] = 0;
      if (from[y] < 0) continue;
      const size_t s = head * src.cap + from[y];
      if (part < NB) {
        k[y] = mri::ld_act(reinterpret_cast<const uint4*>(src.k + s * (16 * NB)) + part);
        v[y] = mri::ld_act(reinterpret_cast<const uint4*>(src.v + s * (16 * NB)) + part);
      } else if (part == 4 || part == 5) {
#pragma unroll
        for (int b = 0; b < NB; ++b) sc[y][b] = mri::ld_act((part == 4 ? src.ks : src.vs) + s * NB + b);
      } else if (part == 6) {
        w[y] = mri::ld_act(src.weight + s);
      }
    }
#pragma unroll
    for (int y = 0; y < kMoveRows; ++y) {
      const int r = r0 + y * step;
      if (r >= end) continue;
      const size_t d = head * dst.cap + r;
      if (part < NB) {
        reinterpret_cast<uint4*>(dst.k + d * (16 * NB))[part] = k[y];
        reinterpret_cast<uint4*>(dst.v + d * (16 * NB))[part] = v[y];
      } else if (part == 4 || part == 5) {
#pragma unroll
        for (int b = 0; b < NB; ++b) (part == 4 ? dst.ks : dst.vs)[d * NB + b] = sc[y][b];
      } else if (part == 6) {
        dst.weight[d] = w[y];
      }
    }
  }
}

template <int NB>
__global__ void __launch_bounds__(kSelThreads, 2)
    kv4_evict_kernel(Cache src, Cache dst, const int32_t* __restrict__ lens, int budget, int recent, int hold, int blocks,
                     int32_t* __restrict__ new_lens, int32_t* kept, bool move) {
  extern __shared__ __align__(16) uint8_t sel_smem[];
  SelectShared& sh = *reinterpret_cast<SelectShared*>(sel_smem);
  uint32_t* held = reinterpret_cast<uint32_t*>(sel_smem + sizeof(SelectShared));
  const int tid = threadIdx.x;
  for (int i = tid; i < kSelRounds * kSelBins; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
  __syncthreads();
  pdl_enter();
  const int rank = static_cast<int>(blockIdx.x % static_cast<unsigned>(blocks));
  const size_t head = blockIdx.x / static_cast<unsigned>(blocks);
  const int bi = static_cast<int>(head / src.heads);
  const int n = min(max(mri::ld_act(lens + bi), 0), static_cast<int>(src.cap));
  int32_t* out = kept + head * budget;
  const int total = min(n, budget), first = rank * kSelThreads + tid;
  const int all = blocks * kSelThreads;
  if (head % src.heads == 0 && first == 0) new_lens[bi] = total;
  for (int i = total + first; i < budget; i += all) out[i] = -1;
  if (n <= budget) {
    for (int i = first; i < n; i += all) out[i] = i;
  } else {
    const int old = n - recent, want = budget - recent;
    for (int i = first; i < recent; i += all) out[want + i] = old + i;
    if (want > 0) select_keys(sh, held, hold, src.weight + head * src.cap, old, static_cast<uint32_t>(want), rank, blocks, out);
  }
  if (!move) return;
  mri::cluster_sync();
  move_rows<NB>(src, dst, head, out, rank * (kSelThreads / 8) + tid / 8, budget, all / 8);
}

// The move alone, by blocks of the whole GPU.
template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_move_kernel(Cache src, Cache dst, int budget,
                                                            const int32_t* __restrict__ kept, unsigned per_head) {
  pdl_enter();
  const size_t head = blockIdx.x / per_head;
  const int r0 = static_cast<int>(blockIdx.x % per_head) * (kMoveRows * kThreads / 8);
  move_rows<NB>(src, dst, head, kept + head * budget, r0 + threadIdx.x / 8,
                min(budget, r0 + kMoveRows * kThreads / 8), kThreads / 8);
}

// ── host side ────────────────────────────────────────────────────────────────

// Checks a cache's description and fills the kernels' view of it.
int view(const char* fn, const mri_kv4_cache* c, Cache* out) {
  if (!c) return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  if (c->head_dim < 32 || c->head_dim > 128 || c->head_dim % 32)
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "%s: head_dim=%zu is not 32, 64, 96 or 128", fn, c->head_dim);
  if (c->capacity == 0 || c->capacity % 64 || c->capacity > (size_t{1} << 30))
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "%s: capacity=%zu is not a positive multiple of 64 up to 2^30", fn,
                          c->capacity);
  if (c->n_kv_heads == 0 || c->n_kv_heads > 65536 || c->batch > (size_t{1} << 20) ||
      c->batch * c->n_kv_heads > (size_t{1} << 24))
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "%s: batch=%zu, n_kv_heads=%zu out of range", fn, c->batch,
                          c->n_kv_heads);
  const uintptr_t all = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
                        reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) |
                        reinterpret_cast<uintptr_t>(c->weight);
  if (c->batch && (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->weight || (all & 15)))
    return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "%s: null or not 16-byte aligned cache buffer", fn);
  *out = Cache{c->k, c->v, c->k_scale, c->v_scale, c->weight, static_cast<int>(c->batch),
               static_cast<int>(c->n_kv_heads), static_cast<int>(c->head_dim), static_cast<int>(c->head_dim / 32),
               c->capacity};
  return MRI_OK;
}

int check_tokens(const char* fn, size_t n_tokens, size_t rows_each, size_t batch) {
  if (n_tokens > (size_t{1} << 24) || n_tokens * rows_each * batch > (size_t{1} << 31) - 1)
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "%s: n_tokens=%zu with batch=%zu and %zu heads is too large", fn,
                          n_tokens, batch, rows_each);
  return MRI_OK;
}

// A buffer that a call reads or writes.
struct Span {
  const void* p;
  size_t bytes;
};
// The five buffers of a cache, to to[0..4].
void spans_of(const Cache& c, Span* to) {
  const size_t rows = static_cast<size_t>(c.batch) * c.heads * c.cap, nb = c.nb;
  const Span all[5] = {{c.k, rows * 16 * nb}, {c.v, rows * 16 * nb}, {c.ks, rows * 2 * nb}, {c.vs, rows * 2 * nb}, {c.weight, rows * 4}};
  std::copy(all, all + 5, to);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int NB>
cudaError_t launch_append(mri_ctx* ctx, const Cache& c, const float* k, const float* v, size_t ld, size_t n_tokens,
                          const int32_t* start) {
  const unsigned rows = static_cast<unsigned>(c.batch * n_tokens * c.heads), per = RowThread<NB>::kRows;
  return launch(ctx, kv4_append_kernel<NB>, (rows + per - 1) / per, kThreads, 0, c, k, v, ld, static_cast<unsigned>(n_tokens),
                start, rows, aligned16(k) && aligned16(v) && ld % 4 == 0);
}

template <int NB>
cudaError_t launch_read(mri_ctx* ctx, const Cache& c, const int32_t* start, size_t n_tokens, float* k, float* v) {
  const unsigned rows = static_cast<unsigned>(c.batch * n_tokens * c.heads), per = RowThread<NB>::kRows;
  return launch(ctx, kv4_read_kernel<NB>, (rows + per - 1) / per, kThreads, 0, c, start, static_cast<unsigned>(n_tokens), k, v,
                rows, aligned16(k) && aligned16(v));
}

template <int NB>
cudaError_t launch_evict(mri_ctx* ctx, const Cache& s, const Cache& d, const int32_t* lens, size_t budget, size_t recent,
                         int32_t* new_lens, int32_t* kept) {
  // Blocks of a cluster: as many as the GPU still takes at once, two an SM, but no
  // more than leave each 1024 keys (below, barriers cost more than they save: 32 heads
  // of 2048 keys, 512 kept: 11.9 us with 2, 13.6 with 8; with 1 13.4, or 10.8 with the
  // move as a second kernel, whose launch costs the host 2.4), and enough that two
  // blocks' shares fit an SM's shared memory.  64 heads of up to 32768 keys, 2000 kept:
  // 46 us with 2, 32 with 4, 39 with 8; one of 262144: 46 us with 8, 456 with one block
  // of 1024 threads.
  const size_t heads = static_cast<size_t>(s.batch) * s.heads, sms = static_cast<size_t>(ctx->dev.sm_count);
  int blocks = kMaxCluster;
  while (blocks > 1 && (heads * blocks > 2 * sms || s.cap < static_cast<size_t>(1024 * blocks)) &&
         s.cap <= static_cast<size_t>(kSelKeys / 4 * blocks))
    blocks /= 2;
  // Few blocks and many rows: the move is a kernel of its own, which fills the GPU.
  // 8 heads, 30000 rows each: 98 us in one kernel of 32 blocks, 29 in two.
  const bool move = heads * blocks >= sms || budget <= static_cast<size_t>(blocks * (2 * kMoveRows * kSelThreads / 8));
  // Shared memory for a block's share of the weights where it fits.
  auto bytes = [](int keys) { return sizeof(SelectShared) + (held_at(keys) + 1) * sizeof(uint32_t); };
  const int hold = static_cast<int>(std::min<size_t>(s.cap / blocks + 4, kSelKeys));
  if (!(ctx->kv4_evict_ready >> NB & 1)) {
    if (cudaError_t e = cudaFuncSetAttribute(kv4_evict_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(bytes(kSelKeys))))
      return e;
    ctx->kv4_evict_ready |= 1u << NB;
  }
  if (cudaError_t e = launch_clusters(ctx, blocks, kv4_evict_kernel<NB>, static_cast<unsigned>(heads * blocks), kSelThreads,
                                      bytes(hold), s, d, lens, static_cast<int>(budget), static_cast<int>(recent), hold,
                                      blocks, new_lens, kept, move))
    return e;
  if (move) return cudaSuccess;
  const unsigned per_head = static_cast<unsigned>((budget + kMoveRows * kThreads / 8 - 1) / (kMoveRows * kThreads / 8));
  return launch(ctx, kv4_move_kernel<NB>, static_cast<unsigned>(heads) * per_head, kThreads, 0, s, d, static_cast<int>(budget),
                static_cast<const int32_t*>(kept), per_head);
}

// f<NB>(...) for the cache's blocks a row.
#define KV4_BY_BLOCKS(nb, f, ...)                                                        \
  ((nb) == 1 ? f<1>(__VA_ARGS__) : (nb) == 2 ? f<2>(__VA_ARGS__) : (nb) == 3 ? f<3>(__VA_ARGS__) : f<4>(__VA_ARGS__))

}  // namespace

extern "C" {

int mri_kv4_append(mri_ctx* ctx, const mri_kv4_cache* cache, const float* k_dev, const float* v_dev, size_t ld,
                   size_t n_tokens, const int32_t* start_dev) {
  if (int rc = mri::enter_ctx(ctx)) return rc;
  Cache c;
  if (int rc = view("mri_kv4_append", cache, &c)) return rc;
  if (int rc = check_tokens("mri_kv4_append", n_tokens, c.heads, c.batch)) return rc;
  if (ld < static_cast<size_t>(c.heads) * c.hd)
    return mri::set_error(MRI_ERR_SHAPE_MISMATCH, "mri_kv4_append: expected rows of %d values, got ld=%zu",
                          c.heads * c.hd, ld);
  if (c.batch == 0 || n_tokens == 0) return MRI_OK;
  if (!k_dev || !v_dev || !start_dev) return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_append: null pointer");
  KV4_CUDA_TRY(KV4_BY_BLOCKS(c.nb, launch_append, ctx, c, k_dev, v_dev, ld, n_tokens, start_dev));
  return MRI_OK;
}

int mri_kv4_read(mri_ctx* ctx, const mri_kv4_cache* cache, const int32_t* start_dev, size_t n_tokens, float* k_dev,
                 float* v_dev) {
  if (int rc = mri::enter_ctx(ctx)) return rc;
  Cache c;
  if (int rc = view("mri_kv4_read", cache, &c)) return rc;
  if (int rc = check_tokens("mri_kv4_read", n_tokens, c.heads, c.batch)) return rc;
  if (c.batch == 0 || n_tokens == 0) return MRI_OK;
  if (!k_dev || !v_dev) return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_read: null pointer");
  KV4_CUDA_TRY(KV4_BY_BLOCKS(c.nb, launch_read, ctx, c, start_dev, n_tokens, k_dev, v_dev));
  return MRI_OK;
}

int mri_kv4_attention(mri_ctx* ctx, const mri_kv4_cache* cache, const float* q_dev, size_t ld, size_t n_tokens,
                      size_t n_heads, const int32_t* lens_dev, float scale, int track, float* out_dev) {
  if (int rc = mri::enter_ctx(ctx)) return rc;
  Cache c;
  if (int rc = view("mri_kv4_attention", cache, &c)) return rc;
  if (n_heads == 0 || n_heads % c.heads || n_heads > 65536)
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_attention: n_heads=%zu is not a multiple of n_kv_heads=%d",
                          n_heads, c.heads);
  if (int rc = check_tokens("mri_kv4_attention", n_tokens, n_heads, c.batch)) return rc;
  if (ld < n_heads * c.hd)
    return mri::set_error(MRI_ERR_SHAPE_MISMATCH, "mri_kv4_attention: expected rows of %zu values, got ld=%zu",
                          n_heads * c.hd, ld);
  const size_t rows = static_cast<size_t>(c.batch) * n_tokens * n_heads;
  if (rows == 0) return MRI_OK;
  if (!q_dev || !lens_dev || !out_dev)
    return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_attention: null pointer");
  // A unit's outputs are the places of its own queries, and are written when all of its
  // blocks have those in registers, so out may be q itself.  Not in tracked calls, whose
  // second pass reads the queries again.
  const size_t tokens = static_cast<size_t>(c.batch) * n_tokens, row_bytes = n_heads * c.hd * sizeof(float);
  const bool in_place = out_dev == q_dev && ld == n_heads * c.hd && !track;
  const Span tracked{track ? c.weight : nullptr, static_cast<size_t>(c.batch) * c.heads * c.cap * sizeof(float)};
  Span reads[6];
  spans_of(c, reads);
  reads[5] = {lens_dev, static_cast<size_t>(c.batch) * sizeof(int32_t)};
  bool shared = !in_place && mri::overlaps(out_dev, tokens * row_bytes, q_dev, row_bytes, tokens, ld * sizeof(float));
  shared |= mri::overlaps(tracked.p, tracked.bytes, q_dev, row_bytes, tokens, ld * sizeof(float));
  shared |= mri::overlaps(tracked.p, tracked.bytes, lens_dev, reads[5].bytes);
  for (const Span& r : reads) shared |= mri::overlaps(out_dev, tokens * row_bytes, r.p, r.bytes);
  if (shared)
    return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_attention: an output buffer overlaps an input%s",
                          track ? " (a tracked call reads the queries again after its outputs)" : "");
  AttnArgs a{};
  a.c = c;
  a.q = q_dev;
  a.ld = ld;
  a.n_tokens = static_cast<int>(n_tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.group = static_cast<int>(n_heads) / c.heads;
  a.lens = lens_dev;
  a.scale = scale;
  a.out = out_dev;
  a.rows = a.group * a.n_tokens;
  switch (c.nb) {
    case 1: return launch_attention<1>(ctx, a, track != 0);
    case 2: return launch_attention<2>(ctx, a, track != 0);
    case 3: return launch_attention<3>(ctx, a, track != 0);
    default: return launch_attention<4>(ctx, a, track != 0);
  }
}

int mri_kv4_evict(mri_ctx* ctx, const mri_kv4_cache* src, const int32_t* lens_dev, const mri_kv4_cache* dst,
                  size_t budget, size_t recent, int32_t* new_lens_dev, int32_t* kept_dev) {
  if (int rc = mri::enter_ctx(ctx)) return rc;
  Cache s, d;
  if (int rc = view("mri_kv4_evict: source", src, &s)) return rc;
  if (int rc = view("mri_kv4_evict: destination", dst, &d)) return rc;
  if (s.batch != d.batch || s.heads != d.heads || s.hd != d.hd)
    return mri::set_error(MRI_ERR_SHAPE_MISMATCH, "mri_kv4_evict: expected [%d, %d, ., %d], got [%d, %d, ., %d]", s.batch,
                          s.heads, s.hd, d.batch, d.heads, d.hd);
  if (budget == 0 || budget > d.cap || recent > budget)
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_evict: budget=%zu, recent=%zu for a destination of %zu rows",
                          budget, recent, d.cap);
  if (s.batch == 0) return MRI_OK;
  if (!lens_dev || !new_lens_dev) return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_evict: null pointer");
  const size_t rows = static_cast<size_t>(s.batch) * s.heads * budget;
  if (rows > (size_t{1} << 31) - 1)
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_kv4_evict: %zu rows are too many for one call", rows);
  // Blocks write while others still read: no output may lie in an input or in another output.
  const size_t lens_bytes = static_cast<size_t>(s.batch) * sizeof(int32_t);
  Span reads[6], writes[7];
  spans_of(s, reads);
  reads[5] = {lens_dev, lens_bytes};
  spans_of(d, writes);
  writes[5] = {new_lens_dev, lens_bytes};
  writes[6] = {kept_dev, rows * sizeof(int32_t)};
  for (int i = 0; i < 7; ++i) {
    bool shared = false;
    for (const Span& r : reads) shared |= mri::overlaps(writes[i].p, writes[i].bytes, r.p, r.bytes);
    for (int j = 0; j < i; ++j) shared |= mri::overlaps(writes[i].p, writes[i].bytes, writes[j].p, writes[j].bytes);
    if (shared)
      return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_kv4_evict: an output buffer overlaps an input or another output");
  }
  if (!kept_dev) {
    if (int rc = mri::ctx_reserve_scratch(ctx, rows * sizeof(int32_t))) return rc;
    kept_dev = reinterpret_cast<int32_t*>(ctx->scratch);
  }
  KV4_CUDA_TRY(KV4_BY_BLOCKS(s.nb, launch_evict, ctx, s, d, lens_dev, budget, recent, new_lens_dev, kept_dev));
  return MRI_OK;
}

}  // extern "C"
