// verify.cu — verification of drafted tokens against the target model's
// probabilities (speculative sampling) from given random numbers; the rule is
// stated at mri_verify_draft in mri_gpu.h.
#include <cuda_runtime.h>

#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "internal.h"
#include "mri_gpu.h"

namespace {

// A thread's values in one pass: 16 in blocks of 256 threads where those fill the GPU,
// which spends the least on each; else 8, in blocks of as many threads as a
// part has use for, since then the passes' round trips count.
constexpr int kPerMany = 16, kManyThreads = 256, kPerFew = 8, kFewThreads = 512, kMaxWarps = kFewThreads / 32;
constexpr int kMaxCluster = 8;   // blocks of a sequence
constexpr size_t kMaxDrafts = 64;

#define VERIFY_CUDA_TRY(expr)                                                                     \
  do {                                                                                            \
    cudaError_t _e = (expr);                                                                      \
    if (_e != cudaSuccess) return mri::set_error(MRI_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
  } while (0)

// What a part of a row says: its maximum and where it is first, and the sum of
// exp((x - maximum) / temperature).
struct __align__(16) Stat {
  float top, sum;
  int at, pad;
};
// The best of a part for the token after the accepted ones: of w / race and, for
// a row whose w is 0 everywhere, of p / race.
struct __align__(16) Pick {
  float left, all, most;
  int left_at, all_at;
  float left_x, all_x;  // their logits
  int pad;
};

struct Args {
  const float* logits;
  const int32_t* drafts;
  const float* uniforms;
  const float* races;
  const float* q;
  const float* temperature;
  int n_drafts;
  int vocab, blocks;  // blocks of a sequence's cluster
  int32_t* tokens;
  int32_t* accepted;
  float* logprobs;
};

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// NaN -> -inf, +inf -> the largest finite value (fmaxf drops a NaN).
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

// 1 / temperature; greedy entries (temperature 0) are scored at 1.  At most 2^127, so that
// it and its product with log2 e are finite: subnormal temperatures below 2^-127 count as
// that, at which logits 2^-119 apart are past exp's range already.
__device__ __forceinline__ float inverse_temperature(const Args& a, int b, bool* greedy) {
  const float t = a.temperature ? mri::ld_act(a.temperature + b) : 1.0f;
  *greedy = t == 0.0f;
  return t > 0.0f && !isinf(t) ? fminf(__fdiv_rn(1.0f, t), 1.7014118346046923e38f) : 1.0f;
}

// A value with its index; the larger value wins, of equal ones the lower index.
__device__ __forceinline__ void take(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) {
    v = ov;
    i = oi;
  }
}
// The same with what belongs to the winner.
__device__ __forceinline__ void take(float& v, int& i, float& x, float ov, int oi, float ox) {
  if (ov > v || (ov == v && oi < i)) {
    v = ov;
    i = oi;
    x = ox;
  }
}
__device__ __forceinline__ void warp_take(float& v, int& i, float& x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, o), ox = __shfl_xor_sync(0xffffffffu, x, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    take(v, i, x, ov, oi, ox);
  }
}
__device__ __forceinline__ void warp_take(float& v, int& i) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    take(v, i, ov, oi);
  }
}

// Of values that are no NaN.
__device__ __forceinline__ float warp_max_fast(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// Index of value c of this thread in the pass that begins at base: in fours where
// rows are aligned.
template <int PER, bool VEC>
__device__ __forceinline__ int index_of(int base, int c) {
  const int threads = static_cast<int>(blockDim.x);
  return base + (VEC ? (c / 4 * threads + static_cast<int>(threadIdx.x)) * 4 + c % 4
                     : c * threads + static_cast<int>(threadIdx.x));
}
// The thread's values of a row in a pass, `fill` from `end` on; all loads first.
template <int PER, bool VEC>
__device__ __forceinline__ void load_pass(const float* x, int base, int end, float fill, float (&v)[PER]) {
  if constexpr (VEC) {
#pragma unroll
    for (int c = 0; c < PER; c += 4) {
      const int i = index_of<PER, VEC>(base, c);
      const float4 q = i < end ? mri::ld_act(reinterpret_cast<const float4*>(x + i)) : make_float4(fill, fill, fill, fill);
      v[c] = q.x, v[c + 1] = q.y, v[c + 2] = q.z, v[c + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int i = index_of<PER, VEC>(base, c);
      v[c] = i < end ? mri::ld_act(x + i) : fill;
    }
  }
}
// Two 16-byte halves of p to the same place in the cluster's block `rank`.
__device__ __forceinline__ void put_remote(const void* p, int rank, int4 v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mri::cluster_addr(p, rank)), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

// One cluster of blocks a sequence, which split the vocabulary.  Every block reads its
// part of each row of logits once, the next pass's values on their way while one is
// summed; a warp's maxima and sums stay with it until all rows are read.  The blocks
// tell each other their rows' statistics, each merges them and decides how many
// drafts stand, and scores its part of the next token's row, which is in L2 by
// then; the first block takes the best of all.  Exponentials of the rows are ex2.approx of
// an argument rounded to f32: 2 units in the last place near p = 1, some 20 at p =
// e^-20 (the acceptance test and the merges use expf).  Bound by instruction issue and HBM
// for a batch (256 sequences of 5 rows of 32000: 48 us, 3.5 TB/s), by latency for one
// sequence (5 rows of 32000: 8.5 us): a round trip a row, two cluster barriers, the second
// row's loads.  Two kernels with a block for each 1024 or 4096 values of a row took 74 us
// for the 256 sequences, but 7.7 for the one, and 12.5 for 16 of 4 rows of 50001 where this
// takes 17; against that stand 2.5 us a call of the host, which is what a lone call waits
// for (and which a CUDA graph does not pay).
template <int PER, bool VEC>
__global__ void __launch_bounds__(PER == kPerMany ? kManyThreads : kFewThreads, PER == kPerMany ? 4 : 2) verify_kernel(Args a) {
  __shared__ Stat sh_warp[kMaxDrafts + 1][kMaxWarps];       // of this block's warps
  __shared__ Stat sh_block[kMaxDrafts + 1][kMaxCluster];  // of the cluster's blocks
  __shared__ float sh_top[kMaxDrafts + 1], sh_sum[kMaxDrafts + 1], sh_log[kMaxDrafts + 1];
  __shared__ int sh_at[kMaxDrafts + 1];
  __shared__ int sh_n;
  __shared__ Pick sh_pick[kMaxWarps], sh_best[kMaxCluster];
  mri::cluster_arrive();
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x, warps = threads / 32;
  const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.blocks));
  const int rank = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.blocks));
  const int part = ((a.vocab + a.blocks - 1) / a.blocks + 3) & ~3;
  const int begin = min(a.vocab, rank * part), end = min(a.vocab, begin + part);
  bool greedy;
  const float inv_t = inverse_temperature(a, b, &greedy), scale = __fmul_rn(inv_t, kLog2e);
  const float* logits = a.logits + static_cast<size_t>(b) * (a.n_drafts + 1) * a.vocab;
  const float* races = a.races + static_cast<size_t>(b) * a.vocab;
  if (tid == 0) sh_n = a.n_drafts;
  // Each draft's own values, on their way while the rows are read.
  int32_t d_mine = -1;
  float x_mine = 0.0f, q_mine = 1.0f, u_mine = 0.0f;
  if (tid < a.n_drafts) {
    const size_t at = static_cast<size_t>(b) * a.n_drafts + tid;
    d_mine = mri::ld_act(a.drafts + at);
    u_mine = mri::ld_act(a.uniforms + at);
    if (d_mine >= 0 && d_mine < a.vocab) {
      x_mine = mri::ld_act(logits + static_cast<size_t>(tid) * a.vocab + d_mine);
      if (a.q) q_mine = mri::ld_act(a.q + at * a.vocab + d_mine);
    }
  }
  float next[PER];
  load_pass<PER, VEC>(logits, begin, end, -INFINITY, next);
  for (int j = 0; j <= a.n_drafts; ++j) {
    const float* x = logits + static_cast<size_t>(j) * a.vocab;
    float top = -INFINITY, sum = 0.0f;
    int at = INT_MAX;
    int base = begin;
    do {
      float v[PER];
#pragma unroll
      for (int c = 0; c < PER; ++c) v[c] = clean(next[c]);
      const int after = base + threads * PER;
      if (after < end)
        load_pass<PER, VEC>(x, after, end, -INFINITY, next);
      else if (j < a.n_drafts)
        load_pass<PER, VEC>(x + a.vocab, begin, end, -INFINITY, next);
      float most = top;
#pragma unroll
      for (int c = 0; c < PER; ++c) most = fmaxf(most, v[c]);
      if (greedy && most > top)  // where it is first matters for greedy entries only
#pragma unroll
        for (int c = PER - 1; c >= 0; --c)
          if (v[c] == most) at = index_of<PER, VEC>(base, c);
      if (most > -INFINITY) {
        sum = __fmul_rn(sum, exp2_fast(__fmul_rn(__fsub_rn(top, most), scale)));
        top = most;
        float part_sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < PER; ++c)
          part_sum[c & 1] = __fadd_rn(part_sum[c & 1], exp2_fast(__fmul_rn(__fsub_rn(v[c], top), scale)));
        sum = __fadd_rn(sum, __fadd_rn(part_sum[0], part_sum[1]));
      }
      base = after;
    } while (base < end);
    const float all = warp_max_fast(top);
    if (greedy) at = __reduce_min_sync(0xffffffffu, top == all ? at : INT_MAX);
    if (top > -INFINITY) sum = __fmul_rn(sum, exp2_fast(__fmul_rn(__fsub_rn(top, all), scale)));
    sum = mri::warp_sum_f(sum);
    if (lane == 0) sh_warp[j][warp] = Stat{all, sum, at, 0};
  }
  __syncthreads();
  mri::cluster_wait();  // every block has begun: its shared memory may be written
  // A warp a row: the block's statistics, to every block.
  for (int j = warp; j <= a.n_drafts; j += warps) {
    const Stat st = lane < warps ? sh_warp[j][lane] : Stat{-INFINITY, 0.0f, INT_MAX, 0};
    float top = st.top;
    int at = st.at;
    warp_take(top, at);
    float sum = st.top > -INFINITY ? __fmul_rn(st.sum, expf(__fmul_rn(__fsub_rn(st.top, top), inv_t))) : 0.0f;
    sum = mri::warp_sum_f(sum);
    if (lane < a.blocks) put_remote(&sh_block[j][rank], lane, make_int4(__float_as_int(top), __float_as_int(sum), at, 0));
  }
  mri::cluster_sync();
  if (tid <= a.n_drafts) {
    float top = -INFINITY, sum = 0.0f;
    int at = INT_MAX;
    for (int c = 0; c < a.blocks; ++c) take(top, at, sh_block[tid][c].top, sh_block[tid][c].at);
    for (int c = 0; c < a.blocks; ++c) {
      const Stat st = sh_block[tid][c];
      if (st.top > -INFINITY) sum = __fmaf_rn(st.sum, expf(__fmul_rn(__fsub_rn(st.top, top), inv_t)), sum);
    }
    sh_top[tid] = top;
    sh_sum[tid] = sum;
    sh_at[tid] = at == INT_MAX ? 0 : at;
    if (tid < a.n_drafts) {
      bool ok = false;
      if (d_mine >= 0 && d_mine < a.vocab) {
        const float z = __fmul_rn(__fsub_rn(clean(x_mine), top), inv_t);
        ok = greedy ? d_mine == sh_at[tid] : __fmul_rn(u_mine, q_mine) < __fdiv_rn(expf(z), sum);
        sh_log[tid] = __fsub_rn(z, logf(sum));
      }
      if (!ok) atomicMin(&sh_n, tid);
    }
  }
  __syncthreads();
  const int n = sh_n;
  const bool last = n == a.n_drafts;
  const float* x = logits + static_cast<size_t>(n) * a.vocab;
  const float top = sh_top[n], sum = sh_sum[n];
  int pick_at = sh_at[n];
  float pick_x = top;
  if (!greedy) {
    const float* q = !last && a.q ? a.q + (static_cast<size_t>(b) * a.n_drafts + n) * a.vocab : nullptr;
    const int32_t d = last || a.q ? -1 : mri::ld_act(a.drafts + static_cast<size_t>(b) * a.n_drafts + n);
    const float share = __fdiv_rn(1.0f, sum);
    Pick p{-INFINITY, -INFINITY, 0.0f, INT_MAX, INT_MAX, 0.0f, 0.0f, 0};
    for (int base = begin; base < end; base += threads * PER) {
      float vx[PER], vr[PER], vq[PER];
      load_pass<PER, VEC>(x, base, end, -INFINITY, vx);
      if (q) load_pass<PER, VEC>(q, base, end, 0.0f, vq);
      load_pass<PER, VEC>(races, base, end, 1.0f, vr);
#pragma unroll
      for (int c = 0; c < PER; ++c) {
        const int i = index_of<PER, VEC>(base, c);
        if (i >= end) continue;
        const float xc = clean(vx[c]);
        const float pr = __fmul_rn(exp2_fast(__fmul_rn(__fsub_rn(xc, top), scale)), share);
        const float w = q ? fmaxf(__fsub_rn(pr, vq[c]), 0.0f) : i == d ? 0.0f : pr;
        p.most = fmaxf(p.most, w);
        take(p.left, p.left_at, p.left_x, __fdividef(w, vr[c]), i, xc);
        if (!last) take(p.all, p.all_at, p.all_x, __fdividef(pr, vr[c]), i, xc);
      }
    }
    warp_take(p.left, p.left_at, p.left_x);
    warp_take(p.all, p.all_at, p.all_x);
    p.most = mri::warp_max(p.most);
    if (lane == 0) sh_pick[warp] = p;
    __syncthreads();
    if (warp == 0) {
      Pick m = lane < warps ? sh_pick[lane] : Pick{-INFINITY, -INFINITY, 0.0f, INT_MAX, INT_MAX, 0.0f, 0.0f, 0};
      warp_take(m.left, m.left_at, m.left_x);
      warp_take(m.all, m.all_at, m.all_x);
      m.most = mri::warp_max(m.most);
      if (lane == 0) {
        put_remote(&sh_best[rank], 0, make_int4(__float_as_int(m.left), __float_as_int(m.all), __float_as_int(m.most), m.left_at));
        put_remote(reinterpret_cast<const int4*>(&sh_best[rank]) + 1, 0,
                   make_int4(m.all_at, __float_as_int(m.left_x), __float_as_int(m.all_x), 0));
      }
    }
    mri::cluster_sync();
    if (rank != 0) return;
    Pick m = sh_best[0];
    for (int c = 1; c < a.blocks; ++c) {
      const Pick o = sh_best[c];
      take(m.left, m.left_at, m.left_x, o.left, o.left_at, o.left_x);
      take(m.all, m.all_at, m.all_x, o.all, o.all_at, o.all_x);
      m.most = fmaxf(m.most, o.most);
    }
    const bool left = last || m.most > 0.0f;
    pick_at = left ? m.left_at : m.all_at;
    pick_x = left ? m.left_x : m.all_x;
    if (pick_at == INT_MAX) {  // a row of nothing but -inf
      pick_at = 0;
      pick_x = -INFINITY;
    }
  } else if (rank != 0) {
    return;
  }
  for (int j = tid; j <= a.n_drafts; j += threads) {
    const size_t o = static_cast<size_t>(b) * (a.n_drafts + 1) + j;
    int32_t token = -1;
    float lp = 0.0f;
    if (j < n) {
      token = mri::ld_act(a.drafts + static_cast<size_t>(b) * a.n_drafts + j);
      lp = sh_log[j];
    } else if (j == n) {
      token = pick_at;
      lp = __fsub_rn(__fmul_rn(__fsub_rn(pick_x, top), inv_t), logf(sum));
    }
    a.tokens[o] = token;
    if (a.logprobs) a.logprobs[o] = lp;
  }
  if (tid == 0) a.accepted[b] = n;
}

cudaError_t launch(mri_ctx* ctx, void (*k)(Args), unsigned grid, int threads, const Args& args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (ctx->dev.opt.pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (args.blocks > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(args.blocks);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  ctx->ls.launches++;
  return cudaLaunchKernelEx(&cfg, k, args);
}

}  // namespace

extern "C" int mri_verify_draft(mri_ctx* ctx, const float* target_logits_dev, const int32_t* draft_tokens_dev,
                                const float* uniforms_dev, const float* races_dev, const float* draft_probs_dev,
                                const float* temperature_dev, size_t batch, size_t n_drafts, size_t vocab,
                                int32_t* tokens_dev, int32_t* accepted_dev, float* logprobs_dev) {
  if (int rc = mri::enter_ctx(ctx)) return rc;
  if (vocab == 0 || vocab > (size_t{1} << 30) || n_drafts > kMaxDrafts || batch > (size_t{1} << 24))
    return mri::set_error(MRI_ERR_INVALID_SHAPE, "mri_verify_draft: batch=%zu, n_drafts=%zu (up to %zu), vocab=%zu", batch,
                          n_drafts, kMaxDrafts, vocab);
  if (batch == 0) return MRI_OK;
  if (!target_logits_dev || !races_dev || !tokens_dev || !accepted_dev ||
      (n_drafts && (!draft_tokens_dev || !uniforms_dev)))
    return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_verify_draft: null pointer");
  // A sequence's outputs are written while others still read their inputs; only a lone
  // sequence's tokens may take the place of its drafts (its blocks have read them).
  struct Span {
    const void* p;
    size_t bytes;
  };
  const size_t drafts = batch * n_drafts * 4, given = batch * (n_drafts + 1) * 4, row = batch * vocab * 4;
  const Span reads[] = {{target_logits_dev, row * (n_drafts + 1)}, {draft_probs_dev, row * n_drafts}, {races_dev, row},
                        {uniforms_dev, drafts}, {temperature_dev, batch * 4}, {draft_tokens_dev, drafts}};
  const Span writes[] = {{tokens_dev, given}, {accepted_dev, batch * 4}, {logprobs_dev, given}};
  for (const Span& w : writes) {
    bool shared = false;
    for (const Span& r : reads)
      if (!(batch == 1 && r.p == draft_tokens_dev && w.p == tokens_dev && r.p == w.p))
        shared |= mri::overlaps(w.p, w.bytes, r.p, r.bytes);
    for (const Span* o = writes; o != &w; ++o) shared |= mri::overlaps(w.p, w.bytes, o->p, o->bytes);
    if (shared)
      return mri::set_error(MRI_ERR_INVALID_ARGUMENT, "mri_verify_draft: an output overlaps an input or another output");
  }
  // Blocks of a sequence: as many as the GPU still takes at once, each with at least
  // 2048 values of a row.  48 sequences of 8 rows of 32000: 21 us with 16 values a
  // thread, 31 with 8; one of 5 rows: 9.0 and 8.2 to 8.5; 16 of 4 rows of 50001: 17 us in
  // blocks of up to 512 threads, 23 of up to 1024 (not all clusters run at once).
  const size_t sms = static_cast<size_t>(ctx->dev.sm_count);
  size_t blocks = kMaxCluster;
  while (blocks > 1 && (batch * blocks > 4 * sms || vocab < 2048 * blocks)) blocks /= 2;
  const bool many = batch * blocks > 2 * sms;
  int threads = kManyThreads;
  while (!many && threads < kFewThreads && static_cast<size_t>(threads * kPerFew) * blocks < vocab) threads *= 2;
  Args a{target_logits_dev, draft_tokens_dev, uniforms_dev, races_dev, draft_probs_dev, temperature_dev,
         static_cast<int>(n_drafts), static_cast<int>(vocab), static_cast<int>(blocks), tokens_dev, accepted_dev, logprobs_dev};
  const uintptr_t all = reinterpret_cast<uintptr_t>(target_logits_dev) | reinterpret_cast<uintptr_t>(races_dev) |
                        reinterpret_cast<uintptr_t>(draft_probs_dev);
  const bool vec = vocab % 4 == 0 && (all & 15) == 0;
  const auto kernel = many ? (vec ? verify_kernel<kPerMany, true> : verify_kernel<kPerMany, false>)
                           : (vec ? verify_kernel<kPerFew, true> : verify_kernel<kPerFew, false>);
  VERIFY_CUDA_TRY(launch(ctx, kernel, static_cast<unsigned>(batch * blocks), threads, a));
  return MRI_OK;
}
