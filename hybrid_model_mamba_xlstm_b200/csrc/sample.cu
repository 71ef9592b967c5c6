// sample.cu — one token per row of logits: temperature, top-k, top-p, min-p, and the draw from a
// given uniform number, in one launch (sm_100a).
//
// Replaces the sampling of HybridLanguageModel.generate (hybrid_xmamba/models/hybrid_lm.py:238-262:
// topk, sort, softmax, cumsum, multinomial) without a sort: the logits are read from HBM once and
// stay in shared memory as order-preserving 32-bit keys, one thread-block cluster per row; the top-k
// and top-p borders are found by radix selection (8 bits of the key a pass) over counts and weights.
//
// Weights w = exp((logit - max) / temperature) are formed in 64 bits and held as integers of 2^-44:
// their sums are exact, so no order of additions (atomics, cluster size) changes a result, and a
// vocabulary of up to 2^18 tokens stays below 2^62.  In 32 bits the sum over a vocabulary is off by
// more than its smallest weights, and a border would fall between other tokens.
#include <cooperative_groups.h>

#include "capi_internal.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace hxm {
namespace sample {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr double kOne = 17592186044416.0;  // 2^44
constexpr int kMaxVocab = 1 << 18;
typedef unsigned long long u64;

struct Params {
  int vocab, slice;  // slice: tokens per CTA of the cluster
  const void* logits;
  int64_t row_stride;
  const float* uniforms;
  float temperature;
  const float* temperature_rows;
  int top_k;
  const int32_t* top_k_rows;
  float top_p;
  const float* top_p_rows;
  float min_p;
  const float* min_p_rows;
  int64_t* tokens;
  float* logprob;
};

// Keys rise with the logit; 0 marks a masked one (-inf, NaN), so that real keys start above it.
HXM_DEV uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 and 0 are one logit
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
HXM_DEV float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Shared {
  u64 hist[2][256];    // this CTA's sums per bin, double-buffered between passes
  u64 total[256];      // the cluster's
  u64 scan[2][kWarps]; // block scans
  u64 mine[2][2];      // this CTA's totals, double-buffered, for the cluster to read
  uint32_t wmax[kWarps];
  uint32_t cmax;
  int pick;
  u64 above;
};

struct Ctx {
  cg::cluster_group cl;
  Shared* s;
  const uint32_t* keys;
  int n;        // this CTA's tokens
  int e;        // tokens per thread (odd: a thread's run of keys starts in a bank of its own)
  double max, t;
  uint32_t kmax;
  int flip;
};

HXM_DEV double weight_d(const Ctx& c, uint32_t key) {
  if (key == c.kmax) return 1.0;
  return exp(((double)logit_of(key) - c.max) / c.t);
}
HXM_DEV u64 weight(const Ctx& c, uint32_t key) { return (u64)__double2ll_rn(weight_d(c, key) * kOne); }

// Sum of v over the cluster, to every thread; `before`: over the CTAs of lower rank.
HXM_DEV u64 cluster_sum(Ctx& c, u64 v, u64* before) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) c.s->scan[0][threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 a = 0;
    for (int i = 0; i < kWarps; ++i) a += c.s->scan[0][i];
    c.s->mine[c.flip][0] = a;
  }
  c.cl.sync();
  u64 all = 0, pre = 0;
  for (unsigned r = 0; r < c.cl.num_blocks(); ++r) {
    const u64 x = c.cl.map_shared_rank(&c.s->mine[c.flip][0], r)[0];
    if (r < c.cl.block_rank()) pre += x;
    all += x;
  }
  c.flip ^= 1;  // the next call writes the other copy, so no peer still reads this one
  if (before) *before = pre;
  return all;
}

// Exclusive sum of v over the block's threads before this one.
HXM_DEV u64 block_before(Ctx& c, u64 v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 a = v;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, a, o);
    if (lane >= o) a += x;
  }
  __syncthreads();
  if (lane == 31) c.s->scan[1][warp] = a;
  __syncthreads();
  u64 pre = a - v;
  for (int i = 0; i < warp; ++i) pre += c.s->scan[1][i];
  return pre;
}

// The key at which the sum of f over larger keys first reaches past `target`: largest key K with
// sum(f, key > K) <= target < sum(f, key >= K); `above` = sum(f, key > K).  The total exceeds target.
template <typename F>
HXM_DEV uint32_t select(Ctx& c, u64 target, u64* above, F f) {
  uint32_t prefix = 0;
  u64 over = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    u64* hist = c.s->hist[(shift >> 3) & 1];
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < c.n; i += kThreads) {
      const uint32_t k = c.keys[i];
      if (k && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))) {
        const u64 v = f(k, i);
        if (v) atomicAdd(&hist[(k >> shift) & 255], v);
      }
    }
    c.cl.sync();
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      u64 a = 0;
      for (unsigned r = 0; r < c.cl.num_blocks(); ++r) a += c.cl.map_shared_rank(hist, r)[i];
      c.s->total[i] = a;
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // from the top: 8 bins a lane
      const int lane = threadIdx.x;
      u64 mine = 0;
      for (int j = 0; j < 8; ++j) mine += c.s->total[255 - (lane * 8 + j)];
      u64 a = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, a, o);
        if (lane >= o) a += x;
      }
      u64 run = over + a - mine;
      if (run <= target && target < over + a) {
        for (int j = 0; j < 8; ++j) {
          const int bin = 255 - (lane * 8 + j);
          const u64 v = c.s->total[bin];
          if (target < run + v) {
            c.s->pick = bin;
            c.s->above = run;
            break;
          }
          run += v;
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)c.s->pick << shift;
    over = c.s->above;
  }
  *above = over;
  return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ Shared sh;
  Ctx c{cg::this_cluster(), &sh, keys, 0, 0, 0, 1, 0, 0};
  const int row = blockIdx.x / c.cl.num_blocks(), rank = c.cl.block_rank();
  const int i0 = rank * p.slice;
  c.n = max(0, min(p.slice, p.vocab - i0));
  c.e = ((c.n + kThreads - 1) / kThreads) | 1;
  const T* lg = static_cast<const T*>(p.logits) + row * p.row_stride + i0;
  // logits -> keys, and the largest
  uint32_t m = 0;
  constexpr int V = 16 / sizeof(T);
  if (reinterpret_cast<uintptr_t>(lg) % 16 == 0) {
    const int nv = c.n / V;
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += kThreads) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(lg) + i);
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const uint32_t k = key_of(to_f32<T>(x[j]));
        keys[i * V + j] = k;
        m = max(m, k);
      }
    }
    for (int i = nv * V + threadIdx.x; i < c.n; i += kThreads) {
      const uint32_t k = key_of(to_f32<T>(lg[i]));
      keys[i] = k;
      m = max(m, k);
    }
  } else {
    for (int i = threadIdx.x; i < c.n; i += kThreads) {
      const uint32_t k = key_of(to_f32<T>(lg[i]));
      keys[i] = k;
      m = max(m, k);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) sh.wmax[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWarps; ++i) m = max(m, sh.wmax[i]);
    sh.cmax = m;
  }
  c.cl.sync();
  for (unsigned r = 0; r < c.cl.num_blocks(); ++r) c.kmax = max(c.kmax, *c.cl.map_shared_rank(&sh.cmax, r));
  if (c.kmax == 0) {  // nothing left (every CTA of the cluster agrees)
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
    }
    c.cl.sync();
    return;
  }
  const float temp = p.temperature_rows ? p.temperature_rows[row] : p.temperature;
  const bool greedy = !(temp > 0.f);
  int k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  if (greedy) k = 1;
  const float top_p = greedy ? 1.f : p.top_p_rows ? p.top_p_rows[row] : p.top_p;
  const float min_p = greedy ? 0.f : p.min_p_rows ? p.min_p_rows[row] : p.min_p;
  c.max = (double)logit_of(c.kmax);
  c.t = greedy ? 1.0 : (double)temp;

  // kept: key > thr, and the first `ties` tokens whose key is thr
  uint32_t thr = 0;
  u64 ties = 0;
  if (k == 1) {
    thr = c.kmax;
    ties = 1;
  } else if (k > 0 && k < p.vocab) {
    u64 valid = 0;
    for (int i = threadIdx.x; i < c.n; i += kThreads) valid += keys[i] != 0;
    if (cluster_sum(c, valid, nullptr) > (u64)k) {
      u64 above;
      thr = select(c, (u64)(k - 1), &above, [](uint32_t, int) { return (u64)1; });
      ties = (u64)k - above;
    }
  }
  auto kept_weight = [&](uint32_t key) { return key > thr ? weight(c, key) : (u64)0; };
  if (top_p < 1.f && k != 1) {
    u64 mine = 0;
    for (int i = threadIdx.x; i < c.n; i += kThreads) mine += keys[i] ? kept_weight(keys[i]) : (u64)0;
    const u64 wt = thr ? weight(c, thr) : 0;
    const u64 total = cluster_sum(c, mine, nullptr) + ties * wt;
    const double border = fmax((double)top_p, 0.0) * (double)total;  // a token stays with at most this before it
    const u64 target = (u64)floor(border);
    if (target < total) {
      u64 above;
      // the tied tokens at the top-k border count `ties` times, once for the cluster
      u64 in_larger = total - ties * wt;
      if (in_larger > target) {
        const uint32_t t2 = select(c, target, &above, [&](uint32_t key, int) { return kept_weight(key); });
        ties = (target - above) / weight(c, t2) + 1;
        thr = t2;
      } else {
        const u64 stay = wt ? (target - in_larger) / wt + 1 : ties;
        ties = min(ties, stay);
      }
    }
  }
  // drop by min-p, then the draw: runs of c.e tokens per thread, in the order of the tokens
  const int lo = min(c.n, (int)threadIdx.x * c.e), hi = min(c.n, lo + c.e);
  u64 tied = 0;
  for (int i = lo; i < hi; ++i) tied += thr && keys[i] == thr;
  u64 tie_pre = 0;
  cluster_sum(c, tied, &tie_pre);
  tie_pre += block_before(c, tied);
  auto draw_weight = [&](uint32_t key, u64& rank_of_tie) -> u64 {
    if (key == 0 || key < thr) return 0;
    if (key == thr && rank_of_tie++ >= ties) return 0;
    const double w = weight_d(c, key);
    return w >= (double)min_p || key == c.kmax ? (u64)__double2ll_rn(w * kOne) : 0;
  };
  u64 mine = 0, rk = tie_pre;
  for (int i = lo; i < hi; ++i) mine += draw_weight(keys[i], rk);
  u64 before = 0;
  const u64 total = cluster_sum(c, mine, &before);
  before += block_before(c, mine);
  const double u = fmin(fmax((double)p.uniforms[row], 0.0), 1.0);
  u64 target = (u64)floor(u * (double)total);
  if (target >= total) target = total - 1;
  if (before <= target && target < before + mine) {
    rk = tie_pre;
    u64 run = before;
    for (int i = lo; i < hi; ++i) {
      const u64 w = draw_weight(keys[i], rk);
      run += w;
      if (target < run) {
        p.tokens[row] = i0 + i;
        if (p.logprob) p.logprob[row] = keys[i] == c.kmax && w == total
                                            ? 0.f
                                            : (float)(((double)logit_of(keys[i]) == c.max ? 0.0 : ((double)logit_of(keys[i]) - c.max) / c.t) -
                                                      log((double)total * (1.0 / kOne)));
        break;
      }
    }
  }
  c.cl.sync();  // a peer may still read this CTA's shared memory
}

template <typename T>
static hxm_status launch(Params p, int rows, cudaStream_t st) {
  // CTAs per row: as many as keep the slices within shared memory, more while the SMs are not full
  int cl = 1;
  while ((p.vocab + cl - 1) / cl > 50 * 1024) cl *= 2;
  while (cl < 8 && (int64_t)rows * cl < 148 && p.vocab / cl > 4 * kThreads) cl *= 2;
  p.slice = ((p.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t smem = (size_t)p.slice * sizeof(uint32_t);
  HXM_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cl));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  HXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_kernel<T>, p));
  return check_launch("hxm_sample_tokens");
}

}  // namespace sample
}  // namespace hxm

extern "C" hxm_status hxm_sample_tokens(const hxm_sample_args* a, void* stream) {
  using namespace hxm;
  clear_error();
  HXM_REQUIRE(a != nullptr, "hxm_sample_tokens: args is NULL");
  HXM_REQUIRE(a->struct_size == sizeof(hxm_sample_args), "hxm_sample_tokens: struct_size %zu != %zu", a->struct_size,
              sizeof(hxm_sample_args));
  HXM_REQUIRE(a->rows >= 0 && a->vocab >= 1, "hxm_sample_tokens: bad dims rows=%d vocab=%d", a->rows, a->vocab);
  HXM_REQUIRE(a->io_dtype == HXM_F32 || a->io_dtype == HXM_BF16 || a->io_dtype == HXM_F16, "hxm_sample_tokens: bad io_dtype %d",
              (int)a->io_dtype);
  HXM_REQUIRE_SUPPORTED(a->vocab <= sample::kMaxVocab, "hxm_sample_tokens: vocab %d (at most %d)", a->vocab, sample::kMaxVocab);
  HXM_REQUIRE_SUPPORTED(a->rows <= (1 << 27), "hxm_sample_tokens: %d rows", a->rows);
  if (a->rows == 0) return HXM_OK;
  HXM_REQUIRE(a->logits && a->uniforms && a->tokens, "hxm_sample_tokens: NULL tensor pointer");
  sample::Params p{};
  p.vocab = a->vocab;
  p.logits = a->logits; p.row_stride = a->logits_row_stride; p.uniforms = a->uniforms;
  p.temperature = a->temperature; p.temperature_rows = a->temperature_rows;
  p.top_k = a->top_k; p.top_k_rows = a->top_k_rows;
  p.top_p = a->top_p; p.top_p_rows = a->top_p_rows;
  p.min_p = a->min_p; p.min_p_rows = a->min_p_rows;
  p.tokens = a->tokens; p.logprob = a->logprob;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->io_dtype == HXM_F32) return sample::launch<float>(p, a->rows, st);
  return a->io_dtype == HXM_BF16 ? sample::launch<__nv_bfloat16>(p, a->rows, st) : sample::launch<__half>(p, a->rows, st);
}
