// sample.cu — one token per row of logits: temperature, top-k, top-p, min-p, and the draw from a
// given uniform number, in one launch (sm_100a).
//
// Replaces the sampling of HybridLanguageModel.generate (hybrid_xmamba/models/hybrid_lm.py:238-262:
// topk, sort, softmax, cumsum, multinomial) without a sort of the vocabulary.  One thread-block
// cluster takes a row: the logits are read from HBM once and stay in shared memory as order-preserving
// keys (16 bits for 16-bit logits).  What is left is a chain of passes over shared memory, and the
// number of passes and of 64-bit exponentials in them is the cost:
//   - counts of the logits in 2048 bins, 1/64 of exp's unit wide, below the largest one;
//   - top_k up to 400: the tokens of the bins that hold the k largest (a few more than k) go to a list,
//     which alone is ranked, cut and drawn from;
//   - a larger top_k: the border's bin is known from the counts, and its keys are listed;
//   - top_p: counts and mean places in the bins bound the weight above every bin to 1 part in 10^4, so the
//     border lies in a bin or a few; the pass that sums all weights also sums those before them and lists their keys;
//   - a list of keys is searched for the border by radix, 8 bits of the key a pass; so are all keys where
//     the list would not fit (a border among thousands of tokens: logits of few values).
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

constexpr int kThreads = 512;  // two CTAs of 64 registers a thread fit an SM: one's barriers hide behind the other
constexpr int kWarps = kThreads / 32;
constexpr int kMaxVocab = 1 << 18;
constexpr int kBins = 4 * kThreads;
constexpr float kBinsPerUnit = 64.f;   // 32 units in all: weights behind them are below 2^-46
constexpr int kList = kThreads;  // tokens ranked one by one
constexpr int kTopKList = 400;   // top_k up to which the kept tokens are listed
constexpr int kSubs = 4 * kWarps;  // runs of tokens whose weights are summed apart
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
// -0 and 0 are one logit.
template <typename T> struct Key;
template <> struct Key<float> {
  typedef uint32_t type;
  static constexpr int kBits = 32;
  static HXM_DEV uint32_t make(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static HXM_DEV float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
};
template <typename T> struct Key16 {
  typedef uint16_t type;
  static constexpr int kBits = 16;
  static HXM_DEV uint32_t make(T x) {
    const float f = to_f32<T>(x);
    if (!(f > -INFINITY)) return 0u;
    uint32_t b = *reinterpret_cast<const uint16_t*>(&x);
    if (f == 0.f) b = 0;
    return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
  }
  static HXM_DEV float value(uint32_t k) {
    const uint16_t b = (uint16_t)(k & 0x8000u ? k & 0x7fffu : ~k);
    return to_f32<T>(*reinterpret_cast<const T*>(&b));
  }
};
template <> struct Key<__nv_bfloat16> : Key16<__nv_bfloat16> {};
template <> struct Key<__half> : Key16<__half> {};

struct Shared {
  double pow2[64];  // 2^(j / 64)
  u64 scan[32];     // by warp; the rest stay 0
  u64 mine[2][2];   // this CTA's totals, double-buffered, for the cluster to read
  u64 sub[kSubs];
  u64 hist[256];    // select_listed
  uint32_t wred[32];
  float wredf[2][kWarps];
  uint32_t cmax;
  uint32_t cmin[1];
  int pick, pick2;
  u64 above;
  int run_at;
  u64 run_sum;
  uint32_t n_list;
  // rank 0's verdict on a top-p border
  uint32_t thr;
  u64 ties;
};
// One region after the keys: the bins, then a list and its ranking, or the radix selection's sums.
struct Bins { uint32_t n[kBins], pos[kBins]; };  // tokens, and their summed positions in the bin in 1/1024
struct Lists { u64 item[kList]; u64 weight[kList]; };
struct Radix { u64 hist[2][256]; u64 total[256]; };
// Keys listed at a border.
template <typename K> struct Keys { static constexpr int kMax = (int)(sizeof(Bins) / sizeof(K)); K key[kMax]; };
constexpr size_t kRegion = sizeof(Bins);
static_assert(kThreads * 4 <= kRegion / 2 && kThreads * 8 <= kRegion / 2, "select_few");
static_assert(sizeof(Lists) <= kRegion && sizeof(Radix) <= kRegion, "region");

template <typename T>
struct Ctx {
  typedef typename Key<T>::type K;
  cg::cluster_group cl;
  Shared* s;
  unsigned char* region;
  const K* keys;
  int n;        // this CTA's tokens
  double max, c;  // weight of x: 2^((x - max) c)
  float fmax, per_bin;
  uint32_t kmax;
  int flip;
};

// 2^44 2^t for t = (x - max) log2(e) / temperature <= 0, not yet rounded to an integer: t = n / 64 + r,
// a table for n mod 64 and the series of 2^r, whose next term is below 4e-17.  0 below 2^-46.
template <typename T>
HXM_DEV double weight_d(const Ctx<T>& c, uint32_t key) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: its sum with |y| < 2^31 ends in round(y)
  constexpr double kLn2_ = 0.69314718055994530942;
  if (key == c.kmax) return 17592186044416.0;
  const double t = ((double)Key<T>::value(key) - c.max) * c.c;
  if (!(t > -46.0)) return 0.0;
  const double z = fma(t, 64.0, kShift);
  const int n = (int)__double2loint(z);
  const double r = fma(z - kShift, -1.0 / 64.0, t) * kLn2_;
  const double p = fma(r, fma(r, fma(r, fma(r, fma(r, 1.0 / 120.0, 1.0 / 24.0), 1.0 / 6.0), 0.5), 1.0), 1.0);
  const double m = c.s->pow2[n & 63] * p;
  return __hiloint2double(__double2hiint(m) + (((n >> 6) + 44) << 20), __double2loint(m));
}
HXM_DEV u64 to_fixed(double w) {
  return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;  // w < 2^45: the sum's last bits
}
template <typename T>
HXM_DEV u64 weight(const Ctx<T>& c, uint32_t key) { return to_fixed(weight_d(c, key)); }

// Bins of falling logits: 0 next to the largest, the last one open.
template <typename T>
HXM_DEV float place_of(const Ctx<T>& c, uint32_t key) {
  return key == c.kmax ? 0.f : fminf((c.fmax - Key<T>::value(key)) * c.per_bin, (float)(kBins - 1));
}
template <typename T>
HXM_DEV int bin_of(const Ctx<T>& c, uint32_t key) { return (int)place_of(c, key); }

HXM_DEV u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
HXM_DEV u64 warp_prefix(u64 v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Inclusive sum over the block's threads up to this one.
HXM_DEV u64 block_prefix(Shared* s, u64 v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 a = warp_prefix(v);
  __syncthreads();
  if (lane == 31) s->scan[warp] = a;
  __syncthreads();
  const u64 w = lane < warp ? s->scan[lane] : 0;
  return a + warp_sum(w);
}

// Sums over the cluster of this CTA's values v0, v1 (same in all its threads); `before`: v0 over lower ranks.
template <typename T>
HXM_DEV void cluster_sum(Ctx<T>& c, u64 v0, u64 v1, u64& all0, u64& all1, u64& before) {
  if (threadIdx.x == 0) {
    c.s->mine[c.flip][0] = v0;
    c.s->mine[c.flip][1] = v1;
  }
  c.cl.sync();
  all0 = all1 = before = 0;
  for (unsigned r = 0; r < c.cl.num_blocks(); ++r) {
    const u64* m = c.cl.map_shared_rank(&c.s->mine[c.flip][0], r);
    const u64 x = m[0];
    if (r < c.cl.block_rank()) before += x;
    all0 += x;
    all1 += m[1];
  }
  c.flip ^= 1;  // the next call writes the other copy, so no peer still reads this one
}
// The block's sum of v, to all of its threads.
HXM_DEV u64 block_sum(Shared* s, u64 v) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s->scan[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(s->scan[threadIdx.x & 31]);
}

// The bin of 256 sums, from the top, at which `over` + the sum passes target (s->pick), and the sum before (s->above).
HXM_DEV void pick_bin(Shared* s, const u64* sums, u64 over, u64 target) {
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;  // 8 bins a lane
  u64 mine = 0;
  for (int j = 0; j < 8; ++j) mine += sums[255 - (lane * 8 + j)];
  const u64 a = warp_prefix(mine);
  u64 run = over + a - mine;
  if (run <= target && target < over + a)
    for (int j = 0; j < 8; ++j) {
      const int bin = 255 - (lane * 8 + j);
      const u64 v = sums[bin];
      if (target < run + v) {
        s->pick = bin;
        s->above = run;
        break;
      }
      run += v;
    }
}

// The key at which the sum of f over larger keys first reaches past `target`: largest key K with
// sum(f, key > K) <= target < sum(f, key >= K); `above` = sum(f, key > K).  The total exceeds target.
template <typename T, typename F>
HXM_DEV uint32_t select(Ctx<T>& c, u64 target, u64* above, F f) {
  Radix* rx = reinterpret_cast<Radix*>(c.region);
  uint32_t prefix = 0;
  u64 over = 0;
  c.cl.sync();  // the region's last readers are done
  for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
    u64* hist = rx->hist[(shift >> 3) & 1];
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i0 = threadIdx.x & ~31; i0 < c.n; i0 += kThreads) {
      const int i = i0 + (threadIdx.x & 31);
      const uint32_t k = i < c.n ? c.keys[i] : 0;
      const bool in = k && (shift == Key<T>::kBits - 8 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
      const uint32_t who = __ballot_sync(0xffffffffu, in);
      if (who == 0) continue;
      const u64 v = in ? f(k) : 0;
      const uint32_t bin = (k >> shift) & 255;
      // the warps of a row of few values share a bin: one addition for all of their tokens
      const uint32_t b0 = __shfl_sync(0xffffffffu, bin, __ffs(who) - 1);
      if (__all_sync(0xffffffffu, !in || bin == b0)) {
        const u64 sum = warp_sum(v);
        if ((threadIdx.x & 31) == 0) atomicAdd(&hist[b0], sum);
      } else if (v) {
        atomicAdd(&hist[bin], v);
      }
    }
    c.cl.sync();
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      u64 a = 0;
      for (unsigned r = 0; r < c.cl.num_blocks(); ++r) a += c.cl.map_shared_rank(hist, r)[i];
      rx->total[i] = a;
    }
    __syncthreads();
    pick_bin(c.s, rx->total, over, target);
    __syncthreads();
    prefix |= (uint32_t)c.s->pick << shift;
    over = c.s->above;
  }
  c.cl.sync();
  *above = over;
  return prefix;
}

// Appends the key of every lane with `want` to rank 0's list (the whole warp calls; the order is arbitrary).
template <typename T>
HXM_DEV void append(Keys<typename Key<T>::type>* list, uint32_t* count, bool want, uint32_t key) {
  const uint32_t who = __ballot_sync(0xffffffffu, want);
  if (who == 0) return;
  const int lane = threadIdx.x & 31, first = __ffs(who) - 1;
  uint32_t at = 0;
  if (lane == first) at = atomicAdd(count, (uint32_t)__popc(who));
  at = __shfl_sync(0xffffffffu, at, first) + __popc(who & ((1u << lane) - 1));
  if (want && at < Keys<typename Key<T>::type>::kMax) list->key[at] = (typename Key<T>::type)key;
}

// select() over a list of n keys, by rank 0's CTA alone; `over`: the sum before the list.
template <typename T, typename F>
HXM_DEV uint32_t select_listed(Ctx<T>& c, int n, u64 over, u64 target, u64* above, F f) {
  const Keys<typename Key<T>::type>* list = reinterpret_cast<const Keys<typename Key<T>::type>*>(c.region);
  uint32_t prefix = 0;
  for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) c.s->hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t k = list->key[i];
      if (shift == Key<T>::kBits - 8 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&c.s->hist[(k >> shift) & 255], f(k));
    }
    __syncthreads();
    pick_bin(c.s, c.s->hist, over, target);
    __syncthreads();
    prefix |= (uint32_t)c.s->pick << shift;
    over = c.s->above;
  }
  *above = over;
  return prefix;
}

// The same for n <= kThreads keys: every thread sums f over the keys above its own.
template <typename T, typename F>
HXM_DEV uint32_t select_few(Ctx<T>& c, int n, u64 over, u64 target, u64* above, F f) {
  const Keys<typename Key<T>::type>* list = reinterpret_cast<const Keys<typename Key<T>::type>*>(c.region);
  u64* w = reinterpret_cast<u64*>(c.region + kRegion / 2);
  const int tid = threadIdx.x;
  const uint32_t mine = tid < n ? list->key[tid] : 0;
  const u64 v = tid < n ? f(mine) : 0;
  w[tid] = v;
  __syncthreads();
  if ((tid & ~31) < n) {
    u64 larger = over, same = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const uint32_t k = list->key[j];
      larger += k > mine ? w[j] : 0;
      same += k == mine ? w[j] : 0;
    }
    if (tid < n && larger <= target && target < larger + same) {  // all threads of this key agree
      c.s->pick = (int)mine;
      c.s->above = larger;
    }
  }
  __syncthreads();
  *above = c.s->above;
  return (uint32_t)c.s->pick;
}

// Puts the tokens whose key passes `want` into rank 0's list, as (key, ~token): larger is better.
// The list's order is arbitrary; it is ranked next.
template <typename T, typename F>
HXM_DEV void gather(Ctx<T>& c, int i0, F want) {
  Lists* ls = reinterpret_cast<Lists*>(c.cl.map_shared_rank(c.region, 0));
  uint32_t* count = c.cl.map_shared_rank(&c.s->n_list, 0);
  for (int i = threadIdx.x; i < c.n; i += kThreads) {
    const uint32_t k = c.keys[i];
    if (k && want(k)) {
      const uint32_t at = atomicAdd(count, 1u);
      if (at < kList) ls->item[at] = ((u64)k << 32) | (0xffffffffu - (uint32_t)(i0 + i));
    }
  }
}
// This thread's item of n <= kList listed ones, in rank order (0 past the end); rank 0's CTA only.
template <typename T>
HXM_DEV u64 ranked(Ctx<T>& c, int n) {
  Lists* ls = reinterpret_cast<Lists*>(c.region);
  u64 mine = 0;
  int rank = 0;
  if ((int)threadIdx.x < n) {
    mine = ls->item[threadIdx.x];
    for (int j = 0; j < n; ++j) rank += ls->item[j] > mine;
  }
  __syncthreads();
  if ((int)threadIdx.x < n) ls->item[rank] = mine;
  __syncthreads();
  return (int)threadIdx.x < n ? ls->item[threadIdx.x] : 0;
}

// From the counts and mean places in the bins (this thread: 4 tid ..): tokens of bins below b0 lie before
// the border, a share of the whole weight, for certain, and those of bins behind b1 after it.  The
// weights of n tokens of one bin, 1/64 wide, sum to n e^-(mean place) times at most 1 + (1/64)^2 / 8
// (Jensen's inequality from below, the largest variance from above); with the places' rounding that is
// 1 part in 10^4.  `split`: a bin of which only some tokens count: bounded by its ends.
HXM_DEV void border_bins(Shared* s, const uint32_t (&cnt)[4], const uint32_t (&pos)[4], int split, float share, int& b0, int& b1) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float hi[4], lo[4], hs = 0.f, ls = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = 4 * tid + j;
    const float n = (float)cnt[j], mean = cnt[j] ? (float)pos[j] * (1.f / 1024.f) / n : 0.f;
    const bool open = b == kBins - 1, part = b == split;
    hi[j] = n * expf(-((float)b + (part || open ? 0.f : mean)) / kBinsPerUnit) * 1.0001f;
    lo[j] = open ? 0.f : n * expf(-((float)b + (part ? 1.f : mean + 1.f / 1024.f)) / kBinsPerUnit) * 0.9999f;
    hs += hi[j];
    ls += lo[j];
  }
  float hp = hs, lp = ls;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float a = __shfl_up_sync(0xffffffffu, hp, o), b = __shfl_up_sync(0xffffffffu, lp, o);
    if (lane >= o) {
      hp += a;
      lp += b;
    }
  }
  __syncthreads();
  if (lane == 31) {
    s->wredf[0][warp] = hp;
    s->wredf[1][warp] = lp;
  }
  if (tid == 0) s->pick = s->pick2 = kBins - 1;
  __syncthreads();
  float ha = 0.f, la = 0.f, hr = hp - hs, lr = lp - ls;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      hr += s->wredf[0][w];
      lr += s->wredf[1][w];
    }
    ha += s->wredf[0][w];
    la += s->wredf[1][w];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    hr += hi[j];
    lr += lo[j];
    if (hr >= share * la && cnt[j]) atomicMin(&s->pick, 4 * tid + j);
    if (lr > share * ha) atomicMin(&s->pick2, 4 * tid + j);
  }
  __syncthreads();
  b0 = s->pick;
  b1 = max(b0, s->pick2);
  __syncthreads();
}

template <typename T>
HXM_DEV float log_prob(const Ctx<T>& c, uint32_t key, u64 w, u64 total) {
  if (w == total) return 0.f;
  const double t = key == c.kmax ? 0.0 : ((double)Key<T>::value(key) - c.max) * c.c * 0.69314718055994530942;
  return (float)(t - log((double)total * (1.0 / 17592186044416.0)));
}

// floor(u * total), held below total
HXM_DEV u64 draw_target(float u, u64 total) {
  const u64 t = (u64)floor(fmin(fmax((double)u, 0.0), 1.0) * (double)total);
  return t < total ? t : total - 1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
  typedef typename Key<T>::type K;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  __shared__ Shared sh;
  unsigned char* region = raw_smem;
  K* keys = reinterpret_cast<K*>(raw_smem + kRegion);
  Ctx<T> c{cg::this_cluster(), &sh, region, keys, 0, 0, 0, 0.f, 0.f, 0, 0};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / c.cl.num_blocks(), rank = c.cl.block_rank();
  const int i0 = rank * p.slice;
  c.n = max(0, min(p.slice, p.vocab - i0));
  if (tid < 64) sh.pow2[tid] = exp2(tid / 64.0);
  if (tid == 0) sh.n_list = 0;
  if (tid < 32) sh.scan[tid] = sh.wred[tid] = 0;
  for (int i = tid; i < 2 * kBins; i += kThreads) reinterpret_cast<Bins*>(region)->n[i] = 0;

  // ---- logits -> keys, and the largest ----
  const T* lg = static_cast<const T*>(p.logits) + row * p.row_stride + i0;
  uint32_t m = 0;
  constexpr int V = 16 / sizeof(T);
  int done = 0;
  if (reinterpret_cast<uintptr_t>(lg) % 16 == 0) {
    const int nv = c.n / V;
#pragma unroll 4
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(lg) + i);
      const T* x = reinterpret_cast<const T*>(&raw);
      uint4 packed;
      K* k = reinterpret_cast<K*>(&packed);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const uint32_t key = Key<T>::make(x[j]);
        k[j] = (K)key;
        m = max(m, key);
      }
      reinterpret_cast<uint4*>(keys)[i] = packed;
    }
    done = nv * V;
  }
  for (int i = done + tid; i < c.n; i += kThreads) {
    const uint32_t key = Key<T>::make(lg[i]);
    keys[i] = (K)key;
    m = max(m, key);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  __syncthreads();
  if (lane == 0) sh.wred[warp] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, sh.wred[lane]);
  if (tid == 0) sh.cmax = m;
  c.cl.sync();
  for (unsigned r = 0; r < c.cl.num_blocks(); ++r) c.kmax = max(c.kmax, *c.cl.map_shared_rank(&sh.cmax, r));

  const float temp = p.temperature_rows ? p.temperature_rows[row] : p.temperature;
  int k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  const float top_p = p.top_p_rows ? p.top_p_rows[row] : p.top_p;
  const float min_p = p.min_p_rows ? p.min_p_rows[row] : p.min_p;
  if (c.kmax == 0) {  // nothing left (every CTA of the cluster agrees)
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
    }
    c.cl.sync();
    return;
  }
  if (!(temp > 0.f) || k == 1) {  // the lowest token with the largest logit
    uint32_t at = 0xffffffffu;
    for (int i = tid; i < c.n; i += kThreads)
      if (keys[i] == c.kmax) {
        at = i0 + i;
        break;
      }
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (lane == 0) sh.wred[warp] = at;
    __syncthreads();
    if (warp == 0) {
      at = __reduce_min_sync(0xffffffffu, lane < kWarps ? sh.wred[lane] : 0xffffffffu);
      if (lane == 0) sh.cmin[0] = at;
    }
    c.cl.sync();
    if (rank == 0 && tid == 0) {
      for (unsigned r = 1; r < c.cl.num_blocks(); ++r) at = min(at, *c.cl.map_shared_rank(&sh.cmin[0], r));
      p.tokens[row] = at;
      if (p.logprob) p.logprob[row] = 0.f;
    }
    c.cl.sync();
    return;
  }
  c.fmax = Key<T>::value(c.kmax);
  c.max = (double)c.fmax;
  c.c = 1.4426950408889634074 / (double)temp;
  c.per_bin = kBinsPerUnit / temp;
  const double min_w = (double)min_p * 17592186044416.0;
  const float u = p.uniforms[row];

  // kept: key > thr, and the first `ties` tokens whose key is thr
  uint32_t thr = 0;
  u64 ties = 0;
  bool all_ties = true;  // no token of key thr is dropped
  if ((k > 0 && k < p.vocab) || top_p < 1.f) {
    // ---- counts per bin, over the cluster; this thread: bins 4 tid .. ----
    Bins* bins = reinterpret_cast<Bins*>(region);
    const bool cut = top_p < 1.f;
#pragma unroll 4
    for (int i = tid; i < c.n; i += kThreads) {
      const uint32_t key = keys[i];
      if (key) {
        const float at = place_of(c, key);
        const int bin = (int)at;
        atomicAdd(&bins->n[bin], 1u);
        if (cut) atomicAdd(&bins->pos[bin], (uint32_t)((at - (float)bin) * 1024.f));
      }
    }
    c.cl.sync();
    uint32_t cnt[4] = {0, 0, 0, 0}, pos[4] = {0, 0, 0, 0};
    for (unsigned r = 0; r < c.cl.num_blocks(); ++r) {
      const Bins* peer = c.cl.map_shared_rank(bins, r);
      const uint4 x = reinterpret_cast<const uint4*>(peer->n)[tid], y = reinterpret_cast<const uint4*>(peer->pos)[tid];
      cnt[0] += x.x;
      cnt[1] += x.y;
      cnt[2] += x.z;
      cnt[3] += x.w;
      pos[0] += y.x;
      pos[1] += y.y;
      pos[2] += y.z;
      pos[3] += y.w;
    }
    const uint32_t four = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    const uint32_t upto = (uint32_t)block_prefix(&sh, four), from = upto - four;
    __syncthreads();
    if (tid == kThreads - 1) sh.pick = (int)upto;
    __syncthreads();
    const int valid = sh.pick;
    if (k >= valid) k = 0;
    c.cl.sync();  // every CTA has read the bins: the region is free
    Keys<K>* keys0 = reinterpret_cast<Keys<K>*>(c.cl.map_shared_rank(region, 0));
    uint32_t* count0 = c.cl.map_shared_rank(&sh.n_list, 0);
    int split = -1;
    if (k > 0) {
      uint32_t run = from;
      for (int j = 0; j < 4; ++j) {
        if (run < (uint32_t)k && (uint32_t)k <= run + cnt[j]) {
          sh.pick = 4 * tid + j;
          sh.pick2 = (int)(run + cnt[j]);
        }
        run += cnt[j];
      }
      __syncthreads();
      const int last = sh.pick, listed = sh.pick2;
      if (k <= kTopKList && listed <= kList) {
        // ---- the k largest as a list in rank 0: rank, cut, draw ----
        gather(c, i0, [&](uint32_t key) { return bin_of(c, key) <= last; });
        c.cl.sync();
        if (rank != 0) return;
        Lists* ls = reinterpret_cast<Lists*>(region);
        const u64 item = ranked(c, listed);
        const uint32_t key = (uint32_t)(item >> 32);
        const double wd = tid < k ? weight_d(c, key) : 0.0;
        const u64 w = to_fixed(wd);
        const u64 incl = block_prefix(&sh, w);
        ls->weight[tid] = incl;
        __syncthreads();
        const u64 all = ls->weight[kThreads - 1];
        const u64 border = top_p < 1.f ? (u64)floor(fmax((double)top_p, 0.0) * (double)all) : all;
        // a first run of the ranking: both cuts fall with the weight
        const bool keep = tid < k && (tid == 0 || incl - w <= border) && (wd >= min_w || key == c.kmax);
        const int kept = __syncthreads_count(keep);
        const u64 total = ls->weight[kept - 1];
        const u64 target = draw_target(u, total);
        __syncthreads();
        ls->weight[tid] = keep ? w : 0;
        __syncthreads();
        if (tid < kept) {  // the weights of the kept tokens up to this one, in the order of the tokens
          u64 sum = 0;
          const uint32_t me = (uint32_t)item;  // ~token: larger for lower tokens
          for (int j = 0; j < kept; ++j) sum += (uint32_t)ls->item[j] >= me ? ls->weight[j] : 0;
          if (target < sum && sum - w <= target) {
            p.tokens[row] = (int64_t)(0xffffffffu - me);
            if (p.logprob) p.logprob[row] = log_prob(c, key, w, total);
          }
        }
        return;
      }
      // ---- the border's bin: its keys listed, the k-th largest found among them ----
      __syncthreads();
      if (tid == last / 4) {
        uint32_t r = from;
        for (int j = 0; j < last % 4; ++j) r += cnt[j];
        sh.pick = (int)r;  // tokens before the bin
      }
      __syncthreads();
      const int ahead = sh.pick;
      if (listed - ahead <= Keys<K>::kMax) {
        for (int i = warp * 32; i < c.n; i += kThreads) {
          const uint32_t key = i + lane < c.n ? keys[i + lane] : 0;
          append<T>(keys0, count0, key && bin_of(c, key) == last, key);
        }
        c.cl.sync();
        if (rank == 0) {
          u64 above;
          const int n = listed - ahead;
          auto one = [](uint32_t) { return (u64)1; };
          const uint32_t t = n <= kThreads ? select_few(c, n, (u64)ahead, (u64)(k - 1), &above, one)
                                           : select_listed(c, n, (u64)ahead, (u64)(k - 1), &above, one);
          if (tid == 0) {
            sh.thr = t;
            sh.ties = (u64)k - above;
            sh.n_list = 0;
          }
        }
        c.cl.sync();
        thr = *c.cl.map_shared_rank(&sh.thr, 0);
        ties = *c.cl.map_shared_rank(&sh.ties, 0);
        c.cl.sync();
      } else {
        u64 above;
        thr = select(c, (u64)(k - 1), &above, [](uint32_t) { return (u64)1; });
        ties = (u64)k - above;
      }
      all_ties = false;
      split = last;
      // from here on the counts are those of the kept tokens
      uint32_t r = from;
      for (int j = 0; j < 4; ++j) {
        const uint32_t now = cnt[j];
        cnt[j] = r >= (uint32_t)k ? 0 : min(now, (uint32_t)k - r);
        r += now;
      }
    }
    if (top_p < 1.f) {
      // ---- the bins that may hold the border; all weights, those before the bins, and the bins' keys ----
      int b0, b1;
      const float share = fmaxf(top_p, 0.f);
      border_bins(&sh, cnt, pos, split, share, b0, b1);
      u64 sum = 0, before = 0;
#pragma unroll 2
      for (int i = warp * 32; i < c.n; i += kThreads) {
        const uint32_t key = i + lane < c.n ? keys[i + lane] : 0;
        const bool in = key > thr;
        const int bin = in ? bin_of(c, key) : kBins;
        const u64 w = in ? weight(c, key) : 0;
        sum += w;
        if (bin < b0) before += w;
        append<T>(keys0, count0, in && bin >= b0 && bin <= b1, key);
      }
      sum = block_sum(&sh, sum);
      before = block_sum(&sh, before);
      u64 larger, pre, unused;
      cluster_sum(c, sum, before, larger, pre, unused);
      // the tokens tied at the top-k border count `ties` times
      const u64 wt = thr ? weight(c, thr) : 0;
      const u64 total = larger + ties * wt;
      const u64 target = (u64)floor(fmax((double)top_p, 0.0) * (double)total);  // a token stays with at most this before it
      const int n = (int)*c.cl.map_shared_rank(count0, 0);
      if (target < total) {
        if (target >= larger) {
          const u64 stay = wt ? (target - larger) / wt + 1 : ties;
          ties = min(ties, stay);
          all_ties = false;
        } else if (n <= Keys<K>::kMax) {
          if (rank == 0) {
            u64 above;
            auto weighed = [&](uint32_t key) { return weight(c, key); };
            const uint32_t t = n <= kThreads ? select_few(c, n, pre, target, &above, weighed) : select_listed(c, n, pre, target, &above, weighed);
            uint32_t same = 0;
            const Keys<K>* list = reinterpret_cast<const Keys<K>*>(region);
            for (int i = tid; i < n; i += kThreads) same += list->key[i] == t;
            const u64 all = block_sum(&sh, same), stay = (target - above) / weight(c, t) + 1;
            if (tid == 0) {
              sh.thr = t;
              sh.ties = min(all, stay);
              sh.pick = all <= stay;
            }
          }
          c.cl.sync();
          thr = *c.cl.map_shared_rank(&sh.thr, 0);
          ties = *c.cl.map_shared_rank(&sh.ties, 0);
          all_ties = *c.cl.map_shared_rank(&sh.pick, 0) != 0;
          c.cl.sync();
        } else {
          const uint32_t floor_key = thr;
          u64 above;
          thr = select(c, target, &above, [&](uint32_t key) { return key > floor_key ? weight(c, key) : (u64)0; });
          ties = (target - above) / weight(c, thr) + 1;
          all_ties = false;
        }
      }
    }
  }

  // ---- the draw, in the order of the tokens: sums of kSubs runs, four per warp ----
  const int run = ((c.n + kSubs - 1) / kSubs + 31) / 32 * 32;
  u64 tie_pre[4] = {0, 0, 0, 0};  // tied tokens before each of this warp's runs
  if (!all_ties) {
    u64 mine = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t t = 0;
      const int lo = (4 * warp + q) * run, hi = min(c.n, lo + run);
      for (int i = lo + lane; i < hi; i += 32) t += keys[i] == thr;
      tie_pre[q] = mine;
      mine += __reduce_add_sync(0xffffffffu, t);
    }
    const u64 incl = block_prefix(&sh, lane == 0 ? mine : 0);  // up to this warp's end
    if (tid == kThreads - 1) sh.above = incl;
    __syncthreads();
    u64 all, unused, before;
    cluster_sum(c, sh.above, 0, all, unused, before);
#pragma unroll
    for (int q = 0; q < 4; ++q) tie_pre[q] += before + incl - mine;
  }
  // weight of token i (within the warp's step of 32 tokens) given the tied tokens before the step
  auto drawn = [&](int i, int hi, u64& tied) -> u64 {
    const uint32_t key = i < hi ? keys[i] : 0;
    bool keep = key > thr;
    if (thr) {
      const bool tie = key == thr;
      const uint32_t same = __ballot_sync(0xffffffffu, tie);
      if (tie) keep = all_ties || tied + __popc(same & ((1u << lane) - 1)) < ties;
      tied += __popc(same);
    }
    if (!keep) return 0;
    const double w = weight_d(c, key);
    return w >= min_w || key == c.kmax ? to_fixed(w) : 0;
  };
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int lo = (4 * warp + q) * run, hi = min(c.n, lo + run);
    u64 sum = 0, tied = tie_pre[q];
#pragma unroll 2
    for (int i = lo; i < hi; i += 32) sum += drawn(i + lane, hi, tied);
    sum = warp_sum(sum);
    if (lane == 0) sh.sub[4 * warp + q] = sum;
  }
  if (tid == 0) sh.run_at = -1;
  __syncthreads();
  constexpr int kPer = kSubs / 32;
  u64 part[kPer] = {}, mine = 0, upto = 0;
  if (warp == 0) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      part[q] = sh.sub[kPer * lane + q];
      mine += part[q];
    }
    upto = warp_prefix(mine);
    if (lane == 31) sh.above = upto;
  }
  __syncthreads();
  u64 total, unused, before;
  cluster_sum(c, sh.above, 0, total, unused, before);
  const u64 target = draw_target(u, total);
  if (warp == 0) {  // the run that holds the target
    u64 at = before + upto - mine;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      if (at <= target && target < at + part[q]) {
        sh.run_at = kPer * lane + q;
        sh.run_sum = at;
      }
      at += part[q];
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (sh.run_at != 4 * warp + q) continue;
    const int lo = (4 * warp + q) * run, hi = min(c.n, lo + run);
    u64 sum = sh.run_sum, tied = tie_pre[q];
    for (int i = lo; i < hi; i += 32) {
      const u64 w = drawn(i + lane, hi, tied);
      const u64 incl = sum + warp_prefix(w);
      if (target < incl && incl - w <= target) {
        p.tokens[row] = i0 + i + lane;
        if (p.logprob) p.logprob[row] = log_prob(c, (uint32_t)keys[i + lane], w, total);
      }
      sum = __shfl_sync(0xffffffffu, incl, 31);
      if (target < sum) break;
    }
  }
  c.cl.sync();  // a peer may still read this CTA's shared memory
}

template <typename T>
static hxm_status launch(Params p, int rows, cudaStream_t st) {
  typedef typename Key<T>::type K;
  // CTAs per row: as many as leave room for two on an SM (92 KB of keys each; 8 CTAs reach 2^18 tokens
  // of 32 bits with one on an SM), more while that leaves SMs idle: a thread then has fewer tokens
  int cl = 1;
  while (cl < 8 && (size_t)((p.vocab + cl - 1) / cl) * sizeof(K) > 92 * 1024) cl *= 2;
  while (cl < 8 && (int64_t)rows * cl * 2 <= 2 * 148 && p.vocab / cl > 4 * kThreads) cl *= 2;
  p.slice = ((p.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t smem = kRegion + (size_t)p.slice * sizeof(K);
  HXM_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  HXM_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
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
