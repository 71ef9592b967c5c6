// sample.cu — one token per row of logits: temperature, top-k, top-p, min-p, and the draw from a
// given uniform number, in one launch (sm_100a).
//
// Replaces the sampling of HybridLanguageModel.generate (hybrid_xmamba/models/hybrid_lm.py:238-262:
// topk, sort, softmax, cumsum, multinomial) without a sort of the vocabulary.  One thread-block
// cluster takes a row: the logits are read from HBM once and stay in shared memory as order-preserving
// keys (16 bits for 16-bit logits).  What is left is a chain of passes over shared memory, bound by the
// instructions issued (some 30 a token where a 64-bit weight is formed) and, for few rows, by the meetings
// of the cluster between them:
//   - small top_k: the threads' own largest logits give a lower bound of the border, so one pass lists a few more
//     than k tokens, which alone are ranked, cut and drawn from;
//   - larger top_k: counts of the logits in 2048 bins, 1/64 of exp's unit wide, give the border's bin, and its
//     keys are listed;
//   - top_p: the weights' sums in the bins are right to 1 part in 10^4, so the border lies in a bin or a few; a
//     pass sums all weights and those before these bins and lists the bins' keys; the border is found among them;
//   - lists are ranked against themselves up to 512 keys, longer ones searched by radix, 8 bits of the key a
//     pass; so are all keys where the list would not fit (logits of few values);
//   - the draw: sums of runs of 128 tokens (of which the pass before has most already), the run that holds the
//     target, the token in it.
// 256 x 50304 bf16, a call among others: greedy 18.6 us, top_k 50 26.8, all tokens 41, top_p 0.9 85 (with cold
// caches and the profiler's clocks 20, 29, 47 and 92); 1 x 50304 fp32, GPU time: 7, 12, 10 and 22; 32 x 131072 fp32,
// top_p 0.9: 43.
//
// Weights w = exp((logit - max) / temperature) are formed in 64 bits and held as integers of 2^-44:
// their sums are exact, so no order of additions (atomics, cluster size) changes a result, and a
// vocabulary of up to 2^18 tokens stays below 2^62.  In 32 bits the sum over a vocabulary is off by
// more than its smallest weights, and a border would fall between other tokens.
#include <cooperative_groups.h>
#include <type_traits>

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
constexpr int kBatch = 4;           // tokens in a row that a lane takes at once
constexpr int kRun = 32 * kBatch;   // tokens whose weights are summed apart
constexpr int kMaxRuns = 384;       // of a CTA: 82 KB of 16-bit keys
static_assert(kMaxRuns <= kThreads && kWarps == 16, "one run a thread; two sums in scan");
constexpr int kTabBits = 8, kTab = 1 << kTabBits;
typedef unsigned long long u64;

// 2^(i / 16), 2^(i / 256): each entry of the table is a product of two.
__constant__ double kSixteenths[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0,
};
__constant__ double kRest[16] = {
    0x1.0000000000000p+0, 0x1.00b1afa5abcbfp+0, 0x1.0163da9fb3335p+0, 0x1.02168143b0281p+0,
    0x1.02c9a3e778061p+0, 0x1.037d42e11bbccp+0, 0x1.04315e86e7f85p+0, 0x1.04e5f72f654b1p+0,
    0x1.059b0d3158574p+0, 0x1.0650a0e3c1f89p+0, 0x1.0706b29ddf6dep+0, 0x1.07bd42b72a836p+0,
    0x1.0874518759bc8p+0, 0x1.092bdf66607e0p+0, 0x1.09e3ecac6f383p+0, 0x1.0a9c79b1f3919p+0,
};
static_assert(kTab == 256, "the two tables");

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
  // the key of the smallest logit of at least x (0 for -inf and NaN)
  static HXM_DEV uint32_t floor_of(float x) { return make(x); }
  // 16 bytes of logits; m: the largest key so far
  static HXM_DEV uint4 vector(const uint4& raw, uint32_t& m) {
    const uint4 k = make_uint4(make(__uint_as_float(raw.x)), make(__uint_as_float(raw.y)), make(__uint_as_float(raw.z)),
                               make(__uint_as_float(raw.w)));
    m = max(m, max(max(k.x, k.y), max(k.z, k.w)));
    return k;
  }
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
  static HXM_DEV uint32_t floor_of(float x) {
    const uint32_t k = Key<float>::make(x);
    // bf16 keys are the upper halves; below zero the lower half of a bf16's 32-bit key is full
    if (std::is_same<T, __nv_bfloat16>::value) return (k & 0x80000000u ? k + 0xffffu : k) >> 16;
    const __half h = __float2half_ru(x);
    return make(*reinterpret_cast<const T*>(&h));
  }
  // two logits a word; zeros, infinities and NaN go one by one
  static HXM_DEV uint4 vector(const uint4& raw, uint32_t& m) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t k[4], least = 0xffffffffu, most = 0, top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = w[j] & 0x7fff7fffu, s = (w[j] >> 15) & 0x00010001u;
      least = __vminu2(least, a);
      most = __vmaxu2(most, a);
      k[j] = w[j] ^ (s * 0x7fffu) ^ 0x80008000u;
      top = __vmaxu2(top, k[j]);
    }
    constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    if ((most & 0xffffu) >= inf || (most >> 16) >= inf || (least & 0xffffu) == 0 || (least >> 16) == 0) {
      const T* x = reinterpret_cast<const T*>(&raw);
      top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[j] = make(x[2 * j]) | make(x[2 * j + 1]) << 16;
        top = __vmaxu2(top, k[j]);
      }
    }
    m = max(m, max(top & 0xffffu, top >> 16));
    return make_uint4(k[0], k[1], k[2], k[3]);
  }
};
template <> struct Key<__nv_bfloat16> : Key16<__nv_bfloat16> {};
template <> struct Key<__half> : Key16<__half> {};

struct Shared {
  double pow2[kTab];  // 2^44 2^(j / kTab)
  u64 scan[32];     // by warp; the rest stay 0
  u64 mine[2][2];   // this CTA's totals, double-buffered, for the cluster to read
  u64 sub[kMaxRuns];
  uint32_t tied[kMaxRuns];  // tokens tied at the border before each run
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
struct Bins { uint32_t n[kBins]; };  // tokens, or their weights relative to the bin's start in 2^-16
struct Lists { u64 item[kList]; u64 weight[kList]; };
struct Few { u64 weight[kThreads]; uint32_t key[kThreads], sorted[kThreads], count[kThreads]; };
struct Radix { u64 hist[2][256]; u64 total[256]; };
constexpr size_t kRegion = 20480;
// Keys listed at a border.
template <typename K> struct Keys { static constexpr int kMax = (int)(kRegion / sizeof(K)); K key[kMax]; };
static_assert(kThreads * 4 <= kRegion / 2, "select_few");
static_assert(2 * sizeof(Bins) <= kRegion && sizeof(Lists) <= kRegion && sizeof(Radix) <= kRegion, "region");

template <typename T>
struct Ctx {
  typedef typename Key<T>::type K;
  cg::cluster_group cl;
  Shared* s;
  unsigned char* region;
  const K* keys;
  int n;        // this CTA's tokens
  double max, c;  // weight of x: 2^((x - max) c / kTab); max is finite
  float fmax, half;  // the largest logit, and half of it
  float per_bin;     // places in a difference of 2; a bin has 1024
  uint32_t kmax, live;  // of the largest logit; below it no weight
  int flip;
};

// 2^44 2^(t / kTab) for t = kTab (x - max) log2(e) / temperature <= 0, not yet rounded to an integer:
// t = n + r, a table for n mod kTab and the series of 2^(r / kTab), |r| <= 1/2, whose next term is below
// 4e-17.  For t > -46 kTab only (smaller weights round to 0).  Without branches, so that several of these
// chains of dependent operations run at once.
template <typename T>
HXM_DEV double scaled(const Ctx<T>& c, uint32_t key) { return ((double)Key<T>::value(key) - c.max) * c.c; }
template <typename T>
HXM_DEV double weight_d(const Ctx<T>& c, uint32_t key) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: its sum with |y| < 2^31 ends in round(y)
  constexpr double k1 = 0.69314718055994530942 / kTab, k2 = k1 * k1 / 2, k3 = k2 * k1 / 3, k4 = k3 * k1 / 4;
  const double t = scaled(c, key), z = t + kShift;
  const int n = __double2loint(z);
  const double r = t - (z - kShift);
  const double p = fma(r, fma(r, fma(r, fma(r, k4, k3), k2), k1), 1.0);
  const double m = c.s->pow2[n & (kTab - 1)] * p;  // the table holds 2^44 2^(j / kTab)
  return __hiloint2double(__double2hiint(m) + ((n & -kTab) << (20 - kTabBits)), __double2loint(m));
}
// Rounded to an integer; w < 2^45, so the sum's last bits are it.
HXM_DEV u64 to_fixed(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull; }
// Keys below `live` have no weight.
template <typename T>
HXM_DEV u64 weight(const Ctx<T>& c, uint32_t key) { return key >= c.live ? to_fixed(weight_d(c, key)) : 0; }

// Places below the largest logit, in 1/1024 of a bin; the last bin is open.  diff / 2 * per_bin + 2^23 ends
// in the integer; anything larger than the last place (NaN too) has larger bits.  (Half of a difference: a whole one
// may be beyond fp32, and an infinite one lies in the last bin at any temperature.)
template <typename T>
HXM_DEV uint32_t place_of(const Ctx<T>& c, uint32_t key) {
  constexpr uint32_t k23 = 0x4b000000u;  // 2^23
  return min(__float_as_uint(fmaf(fmaf(Key<T>::value(key), -0.5f, c.half), c.per_bin, 8388608.f)), k23 + ((kBins - 1) << 10)) - k23;
}
// The smallest key in [1, kmax] for which pass(key) holds; it rises with the key and holds for kmax (a whole
// warp calls: the 32 keys around a guess, then 33 parts a step).
template <typename T, typename F>
HXM_DEV uint32_t first_key(const Ctx<T>& c, float guess, F pass) {
  uint32_t lo = 0, hi = c.kmax;  // hi passes, lo does not
  uint32_t step = 1, base = min(max(Key<T>::floor_of(guess), 17u), hi) - 17u;
  while (hi - lo > 1) {
    const uint32_t at = base + step * ((threadIdx.x & 31) + 1);
    const uint32_t who = __ballot_sync(0xffffffffu, at >= hi || (at > lo && pass(at)));
    const int f = who ? __ffs(who) - 1 : 32;
    if (f < 32) hi = min(hi, base + step * (f + 1));
    if (f > 0) lo = max(lo, base + step * f);
    step = (hi - lo + 32) / 33;
    base = lo;
  }
  return hi;
}
// The smallest key whose bin is at most b, above every key for b < 0.
template <typename T>
HXM_DEV uint32_t bin_floor(const Ctx<T>& c, int b) {
  if (b < 0) return c.kmax + 1;
  return first_key(c, c.fmax - (float)((b + 1) << 11) / c.per_bin, [&](uint32_t key) { return (int)(place_of(c, key) >> 10) <= b; });
}

// The keys of kBatch tokens in a row from i on, 0 behind the last one.
template <typename T>
HXM_DEV void read_keys(const Ctx<T>& c, int i, uint32_t (&key)[kBatch]) {
  if (Key<T>::kBits == 32) {
    const uint4 r = i < c.n ? *reinterpret_cast<const uint4*>(c.keys + i) : make_uint4(0, 0, 0, 0);
    key[0] = r.x;
    key[1] = r.y;
    key[2] = r.z;
    key[3] = r.w;
  } else {
    const uint2 r = i < c.n ? *reinterpret_cast<const uint2*>(c.keys + i) : make_uint2(0, 0);
    key[0] = r.x & 0xffffu;
    key[1] = r.x >> 16;
    key[2] = r.y & 0xffffu;
    key[3] = r.y >> 16;
  }
}
// f(keys of kBatch tokens in a row, the first one's place) for all of this CTA's tokens, every lane of a
// warp the same number of times; keys behind the last token are 0.
template <typename T, typename F>
HXM_DEV void each_key(const Ctx<T>& c, F f) {
  const int nr = (c.n + kRun - 1) / kRun;
  for (int r = threadIdx.x >> 5; r < nr; r += kWarps) {
    const int i = r * kRun + (threadIdx.x & 31) * kBatch;
    uint32_t key[kBatch];
    read_keys(c, i, key);
    f(key, i);
  }
}

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
  const unsigned r = threadIdx.x & 31;  // a lane per CTA: one round trip
  u64 x = 0, y = 0;
  if (r < c.cl.num_blocks()) {
    const u64* m = c.cl.map_shared_rank(&c.s->mine[c.flip][0], r);
    x = m[0];
    y = m[1];
  }
  before = warp_sum(r < c.cl.block_rank() ? x : 0);
  all0 = warp_sum(x);
  all1 = warp_sum(y);
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

// Appends the keys in [lo, up), lo > 0, to this CTA's list (the whole warp calls; the order is arbitrary).
template <typename T>
HXM_DEV void append(Ctx<T>& c, const uint32_t (&key)[kBatch], uint32_t lo, uint32_t up) {
  typedef Keys<typename Key<T>::type> List;
  int mine = 0;
#pragma unroll
  for (int j = 0; j < kBatch; ++j) mine += key[j] >= lo && key[j] < up;
  if (mine == 0) return;
  uint32_t at = atomicAdd(&c.s->n_list, (uint32_t)mine);
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (key[j] >= lo && key[j] < up) {
      if (at < List::kMax) reinterpret_cast<List*>(c.region)->key[at] = (typename Key<T>::type)key[j];
      ++at;
    }
}

// The length of all CTAs' lists of E together; if that is at most `most`, rank 0 brings them behind its own.
// Between two meetings of the cluster.
template <typename E, typename T>
HXM_DEV int collect(Ctx<T>& c, int most) {
  const int lane = threadIdx.x & 31, nb = (int)c.cl.num_blocks();
  const uint32_t mine = lane < nb ? *c.cl.map_shared_rank(&c.s->n_list, lane) : 0;
  const int n = (int)__reduce_add_sync(0xffffffffu, min(mine, (uint32_t)kMaxVocab));
  if (n > most || c.cl.block_rank() != 0) return n;
  E* list = reinterpret_cast<E*>(c.region);
  int at = __shfl_sync(0xffffffffu, (int)mine, 0);
  for (int r = 1; r < nb; ++r) {
    const int more = __shfl_sync(0xffffffffu, (int)mine, r);
    const E* from = reinterpret_cast<const E*>(c.cl.map_shared_rank(c.region, r));
    for (int i = threadIdx.x; i < more; i += kThreads) list[at + i] = from[i];
    at += more;
  }
  __syncthreads();
  return n;
}

// select() over a list of n <= kThreads keys, by rank 0's CTA alone; `over`: the sum before the list.  Every
// thread counts the keys above its own, and the sums run over the places found.  `same`: keys of the result.
template <typename T, typename F>
HXM_DEV uint32_t select_few(Ctx<T>& c, int n, u64 over, u64 target, u64* above, uint32_t* same, F f) {
  const Keys<typename Key<T>::type>* list = reinterpret_cast<const Keys<typename Key<T>::type>*>(c.region);
  Few* few = reinterpret_cast<Few*>(c.region + kRegion / 2);
  const int tid = threadIdx.x;
  const uint32_t mine = tid < n ? list->key[tid] : 0;
  few->key[tid] = mine;
  few->count[tid] = 0;
  __syncthreads();
  if (tid < n) {
    uint32_t larger = 0;
    for (int j = 0; j < n; j += 4) {  // 0 behind the list
      const uint4 k = *reinterpret_cast<const uint4*>(&few->key[j]);
      larger += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
    }
    // the place of a key's first copy stands for all of them
    few->weight[larger] = f(mine);
    few->sorted[larger] = mine;
    atomicAdd(&few->count[larger], 1u);
  }
  __syncthreads();
  const uint32_t equal = few->count[tid];
  const u64 v = equal ? few->weight[tid] * equal : 0, upto = over + block_prefix(c.s, v);
  if (equal && upto - v <= target && target < upto) {
    c.s->pick = (int)few->sorted[tid];
    c.s->pick2 = (int)equal;
    c.s->above = upto - v;
  }
  __syncthreads();
  *above = c.s->above;
  *same = (uint32_t)c.s->pick2;
  return (uint32_t)c.s->pick;
}

// The same for a list of any length.
template <typename T, typename F>
HXM_DEV uint32_t select_listed(Ctx<T>& c, int n, u64 over, u64 target, u64* above, uint32_t* same, F f) {
  if (n <= kThreads) return select_few(c, n, over, target, above, same, f);
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
  uint32_t equal = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) equal += list->key[i] == prefix;
  *same = (uint32_t)block_sum(c.s, equal);
  return prefix;
}

// Puts the tokens with keys of at least `from` > 0 into this CTA's list, as (key, ~token): larger is better.
// The list's order is arbitrary; it is ranked next.
template <typename T>
HXM_DEV void gather(Ctx<T>& c, int i0, uint32_t from) {
  Lists* ls = reinterpret_cast<Lists*>(c.region);
  each_key(c, [&](const uint32_t (&key)[kBatch], int i) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) any |= key[j] >= from;
    if (!any) return;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (key[j] >= from) {
        const uint32_t at = atomicAdd(&c.s->n_list, 1u);
        if (at < kList) ls->item[at] = ((u64)key[j] << 32) | (0xffffffffu - (uint32_t)(i0 + i + j));
      }
  });
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

// This thread's four of the cluster's bins, 4 tid .., summed.  The region is free when it returns.  Every CTA
// sums its share of the bins and all of them read the sums: 2 * 8 KB over the cluster's network for each,
// where every CTA reading all bins of the others would take 8 KB times the CTAs (8: 7.3 K cycles).
template <typename T, typename N>
HXM_DEV void read_bins(Ctx<T>& c, N (&sum)[4]) {
  const int tid = threadIdx.x, nb = (int)c.cl.num_blocks(), share = kThreads / nb;  // threads a CTA's share
  uint4* mine = reinterpret_cast<uint4*>(c.region + sizeof(Bins));  // 16-byte pieces of this share, by CTA
  c.cl.sync();
  mine[tid] = reinterpret_cast<const uint4*>(c.cl.map_shared_rank(c.region, tid / share))[c.cl.block_rank() * share + tid % share];
  __syncthreads();
  struct alignas(16) Four { N n[4]; };
  Four all = {};
  if (tid < share)
    for (int r = 0; r < nb; ++r) {
      const uint4 x = mine[r * share + tid];
      all.n[0] += (N)x.x;
      all.n[1] += (N)x.y;
      all.n[2] += (N)x.z;
      all.n[3] += (N)x.w;
    }
  __syncthreads();
  if (tid < share) reinterpret_cast<Four*>(mine)[tid] = all;
  c.cl.sync();
  all = reinterpret_cast<const Four*>(c.cl.map_shared_rank(reinterpret_cast<unsigned char*>(mine), tid / share))[tid % share];
  c.cl.sync();
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = all.n[j];
}

// From the weights in the bins (this thread: 4 tid ..): tokens of bins below b0 lie before the border, a
// share of the whole weight, for certain, and those of bins behind b1 after it.  A bin's sum of rounded
// relative weights, its places' rounding and the sums here are off by less than 1 part in 10^4.  `after`:
// weight behind all bins.
HXM_DEV void border_bins(Shared* s, const float (&sum)[4], float after, float share, int& b0, int& b1) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float hi[4], lo[4], hs = 0.f, ls = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = 4 * tid + j;
    const float w = sum[j] * (1.f / 65536.f) * expf(-(float)b / kBinsPerUnit);
    hi[j] = w * 1.0001f;
    lo[j] = b == kBins - 1 ? 0.f : w * 0.9999f;  // the last one is open
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
  float ha = after * 1.0001f, la = after * 0.9999f, hr = hp - hs, lr = lp - ls;
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
    if (hr >= share * la && sum[j] != 0.f) atomicMin(&s->pick, 4 * tid + j);
    if (lr > share * ha) atomicMin(&s->pick2, 4 * tid + j);
  }
  __syncthreads();
  b0 = s->pick;
  b1 = max(b0, s->pick2);
  __syncthreads();
}

// Sum over the warp of values below 2^46.
HXM_DEV u64 warp_sum46(u64 v) {
  const u64 low = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0xffffffu);
  return ((u64)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24)) << 24) + low;
}

template <typename T>
HXM_DEV float log_prob(const Ctx<T>& c, uint32_t key, u64 w, u64 total) {
  if (w == total) return 0.f;
  const double t = scaled(c, key) * (0.69314718055994530942 / kTab);
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
  Ctx<T> c{cg::this_cluster(), &sh, region, keys, 0, 0, 0, 0.f, 0.f, 0.f, 0, 0, 0};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / c.cl.num_blocks(), rank = c.cl.block_rank();
  int i0 = rank * p.slice;
  c.n = max(0, min(p.slice, p.vocab - i0));
  if (tid == 0) sh.n_list = 0;
  if (tid < 32) sh.scan[tid] = sh.wred[tid] = 0;
  Bins* bins = reinterpret_cast<Bins*>(region);
  reinterpret_cast<uint4*>(bins)[tid] = make_uint4(0, 0, 0, 0);

  // ---- logits -> keys, and the largest ----
  const T* lg = static_cast<const T*>(p.logits) + row * p.row_stride + i0;
  uint32_t m = 0;
  constexpr int V = 16 / sizeof(T);
  // as many empty places first as bring the vectors of logits and of keys into line
  const int pad = (int)(reinterpret_cast<uintptr_t>(lg) % 16 / sizeof(T));
  lg -= pad;
  i0 -= pad;
  c.n += c.n ? pad : 0;
  const int v0 = pad ? 1 : 0, v1 = c.n / V;
#pragma unroll 4
  for (int i = v0 + tid; i < v1; i += kThreads)
    reinterpret_cast<uint4*>(keys)[i] = Key<T>::vector(__ldg(reinterpret_cast<const uint4*>(lg) + i), m);
  // the first and the last vector, if they are not whole
  if (tid < 2 * V) {
    const int i = tid < V ? tid : v1 * V + tid - V;
    if (tid < V ? v0 == 1 : i < (c.n + 7) / 8 * 8 && v1 >= v0) {
      const uint32_t key = i >= pad && i < c.n ? Key<T>::make(lg[i]) : 0;
      keys[i] = (K)key;
      m = max(m, key);
    }
  }
  if (tid < kTab) sh.pow2[tid] = 17592186044416.0 * kSixteenths[tid >> 4] * kRest[tid & 15];
  uint32_t own = m;  // this thread's largest
  m = __reduce_max_sync(0xffffffffu, m);
  __syncthreads();
  if (lane == 0) sh.wred[warp] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, sh.wred[lane]);
  if (tid == 0) sh.cmax = m;
  c.cl.sync();
  c.kmax = __reduce_max_sync(0xffffffffu, lane < (int)c.cl.num_blocks() ? *c.cl.map_shared_rank(&sh.cmax, lane) : 0u);

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
  if (c.fmax == INFINITY) {  // such logits share all of the weight: as zeros, with the others masked
    constexpr uint32_t zero = 1u << (Key<T>::kBits - 1);
    __syncthreads();
    for (int i = tid; i < c.n; i += kThreads) keys[i] = (K)(keys[i] == c.kmax ? zero : 0);
    __syncthreads();
    own = own == c.kmax ? zero : 0;
    c.kmax = zero;
    c.fmax = 0.f;
  }
  c.max = (double)c.fmax;
  c.c = kTab * 1.4426950408889634074 / (double)temp;
  c.half = 0.5f * c.fmax;
  c.per_bin = fminf(2048.f * kBinsPerUnit / temp, 3e38f);
  // -45.5 in the exponent of two: weights below it round to 0, and any bound up to -46 would do
  c.live = max(Key<T>::floor_of(__double2float_ru(c.max - 45.5 * 0.69314718055994530942 * (double)temp)), 1u);
  const float u = p.uniforms[row];
  // the smallest key that min_p keeps
  const double min_w = fmin((double)min_p, 1.0) * 17592186044416.0;
  const uint32_t least = min_w > 0 ? first_key(c, c.fmax + temp * logf(min_p), [&](uint32_t key) { return key >= c.live && weight_d(c, key) >= min_w; }) : 1;

  // kept: key > thr, and the first `ties` tokens whose key is thr
  uint32_t thr = 0;
  u64 ties = 0;
  bool all_ties = true;  // no token of key thr is dropped
  uint32_t sure = 0xffffffffu;  // keys from here on are kept and already summed in the runs
  bool clean = true;  // the bins are zero
  // Empties the bins, and the list's count; ends before any CTA uses them again.
  auto clear = [&]() {
    c.cl.sync();
    reinterpret_cast<uint4*>(bins)[tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) sh.n_list = 0;
    c.cl.sync();
  };
  if (k > 0 && k < p.vocab) {
    // Where every CTA has k / CTAs threads whose own largest logit lies in its bin `last` or above, k tokens do: a lower
    // bound of the border from 512 logits a CTA, for one look at all of them.  Up to a quarter of the threads, few more
    // than k tokens pass; a longer list, or a larger k, takes counts of all tokens.
    const int nb = (int)c.cl.num_blocks();
    for (int pass = k <= kThreads / 4 * nb && k <= kTopKList ? 0 : 1; pass < 2; ++pass) {
      if (!clean) clear();
      clean = false;
      int last, ahead = 0, listed = 0;
      if (pass == 0) {
        if (own) atomicAdd(&bins->n[place_of(c, own) >> 10], 1u);
        if (tid == 0) sh.pick = kBins - 1;
        __syncthreads();
        const uint4 x = reinterpret_cast<const uint4*>(bins->n)[tid];
        const uint32_t cnt[4] = {x.x, x.y, x.z, x.w}, share = (uint32_t)(k + nb - 1) / nb;
        const uint32_t four = x.x + x.y + x.z + x.w;
        uint32_t run = (uint32_t)block_prefix(&sh, four) - four;
        for (int j = 0; j < 4; ++j) {
          if (run < share && share <= run + cnt[j]) sh.pick = 4 * tid + j;
          run += cnt[j];
        }
        c.cl.sync();
        last = (int)__reduce_max_sync(0xffffffffu, lane < nb ? (uint32_t)*c.cl.map_shared_rank(&sh.pick, lane) : 0u);
        if (last == kBins - 1) continue;  // a CTA with fewer logits, or too far below the largest
      } else {
        each_key(c, [&](const uint32_t (&key)[kBatch], int) {
          uint32_t at[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) at[j] = place_of(c, key[j]) >> 10;
#pragma unroll
          for (int j = 0; j < kBatch; ++j)
            if (key[j]) atomicAdd(&bins->n[at[j]], 1u);
        });
        uint32_t cnt[4];
        read_bins(c, cnt);
        const uint32_t four = cnt[0] + cnt[1] + cnt[2] + cnt[3];
        const uint32_t upto = (uint32_t)block_prefix(&sh, four), from = upto - four;
        __syncthreads();
        if (tid == kThreads - 1) sh.pick = (int)upto;
        __syncthreads();
        if (k >= sh.pick) {  // all of them stay
          k = 0;
          continue;
        }
        __syncthreads();
        uint32_t run = from;
        for (int j = 0; j < 4; ++j) {
          if (run < (uint32_t)k && (uint32_t)k <= run + cnt[j]) {
            sh.pick = 4 * tid + j;
            sh.pick2 = (int)(run + cnt[j]);
            sh.run_at = (int)run;  // tokens before the bin
          }
          run += cnt[j];
        }
        __syncthreads();
        last = sh.pick;
        listed = sh.pick2;
        ahead = sh.run_at;
      }
      if (pass == 0 || (k <= kTopKList && listed <= kList)) {
        gather(c, i0, bin_floor(c, last));
        c.cl.sync();
        listed = collect<u64>(c, kList);
        c.cl.sync();
        if (listed > kList) continue;  // pass 0 only
        if (rank != 0) return;
        Lists* ls = reinterpret_cast<Lists*>(region);
        const u64 item = ranked(c, listed);
        const uint32_t key = (uint32_t)(item >> 32);
        const u64 w = tid < k ? weight(c, key) : 0;
        const u64 incl = block_prefix(&sh, w);
        ls->weight[tid] = incl;
        __syncthreads();
        const u64 all = ls->weight[kThreads - 1];
        const u64 border = top_p < 1.f ? (u64)floor(fmax((double)top_p, 0.0) * (double)all) : all;
        // a first run of the ranking: both cuts fall with the weight
        const bool keep = tid < k && (tid == 0 || incl - w <= border) && key >= least;
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
      if (listed - ahead <= Keys<K>::kMax) {
        const uint32_t lo = bin_floor(c, last), up = bin_floor(c, last - 1);
        each_key(c, [&](const uint32_t (&key)[kBatch], int) { append(c, key, lo, up); });
        c.cl.sync();
        const int n = collect<K>(c, Keys<K>::kMax);
        if (rank == 0) {
          u64 above;
          auto one = [](uint32_t) { return (u64)1; };
          uint32_t same;
          const uint32_t t = select_listed(c, n, (u64)ahead, (u64)(k - 1), &above, &same, one);
          if (tid == 0) {
            sh.thr = t;
            sh.ties = (u64)k - above;
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
    }
  }
  if (top_p < 1.f) {
    // ---- weights in the bins; the bins that may hold the border; all weights, those before the bins (by
    // runs, for the draw), and the bins' keys ----
    if (!clean) clear();
    each_key(c, [&](const uint32_t (&key)[kBatch], int) {
      uint32_t at[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) at[j] = place_of(c, key[j]);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t x = at[j] & 1023;  // 2^16 e^(-x / 2^16)
        if (key[j] > thr) atomicAdd(&bins->n[at[j] >> 10], 65536u - x + (x * x >> 17));
      }
    });
    float sums[4];
    read_bins(c, sums);
    int b0, b1;
    const float after = thr ? (float)ties * expf((float)place_of(c, thr) * (-1.f / 1024.f / kBinsPerUnit)) : 0.f;
    border_bins(&sh, sums, after, fmaxf(top_p, 0.f), b0, b1);
    u64 sum = 0, before = 0;
    const uint32_t from_key = max(thr + 1, c.live), lo = max(bin_floor(c, b1), from_key), up = bin_floor(c, b0 - 1), up_live = max(up, from_key);
    each_key(c, [&](const uint32_t (&key)[kBatch], int i) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) any |= key[j] >= from_key;
      u64 rs = 0;
      if (__any_sync(0xffffffffu, any)) {
        double w[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) w[j] = weight_d(c, key[j]);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const u64 f = to_fixed(w[j]);
          if (key[j] >= from_key) sum += f;
          if (key[j] >= up_live) rs += f;
        }
      }
      before += rs;
      rs = warp_sum46(rs);
      if (lane == 0) sh.sub[i / kRun] = rs;
      append(c, key, lo, up);
    });
    if (least <= up_live) sure = up_live;
    sum = warp_sum(sum);
    before = warp_sum(before);
    if (lane == 0) {
      sh.scan[warp] = sum;
      sh.scan[16 + warp] = before;
    }
    __syncthreads();
    sum = warp_sum(lane < 16 ? sh.scan[lane] : 0);
    before = warp_sum(lane >= 16 ? sh.scan[lane] : 0);
    __syncthreads();
    if (tid >= 16 && tid < 32) sh.scan[tid] = 0;
    u64 larger, pre, unused;
    cluster_sum(c, sum, before, larger, pre, unused);
    // the tokens tied at the top-k border count `ties` times
    const u64 wt = thr ? weight(c, thr) : 0;
    const u64 total = larger + ties * wt;
    const u64 target = (u64)floor(fmax((double)top_p, 0.0) * (double)total);  // a token stays with at most this before it
    const int n = collect<K>(c, Keys<K>::kMax);
    if (target < total) {
      if (target >= larger) {
        const u64 stay = wt ? (target - larger) / wt + 1 : ties;
        ties = min(ties, stay);
        all_ties = false;
      } else if (n <= Keys<K>::kMax) {
        if (rank == 0) {
          u64 above;
          auto weighed = [&](uint32_t key) { return weight(c, key); };
          uint32_t same;
          const uint32_t t = select_listed(c, n, pre, target, &above, &same, weighed);
          __syncthreads();
          if (tid == 0) {
            const u64 all = same, stay = (target - above) / weight(c, t) + 1;
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
  // ---- the draw, in the order of the tokens: the sums of runs of kRun tokens, one a warp ----
  const int runs = (c.n + kRun - 1) / kRun;
  // the kept keys: at least `from`, and of those equal to thr the first `ties`
  const uint32_t from = max(max(thr + (all_ties ? 0 : 1), 1u), max(least, c.live));
  const bool some = !all_ties && thr >= max(least, c.live);
  each_key(c, [&](const uint32_t (&key)[kBatch], int i) {
    const int r = i / kRun;
    const uint32_t up = min(sure, c.kmax + 1);
    u64 sum = 0;
    bool any = false;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) any |= key[j] >= from && key[j] < up;
    if (__any_sync(0xffffffffu, any)) {
      double w[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) w[j] = weight_d(c, key[j]);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const u64 f = to_fixed(w[j]);
        if (key[j] >= from && key[j] < up) sum += f;
      }
      sum = warp_sum46(sum);
    }
    if (lane == 0) sh.sub[r] = sure == 0xffffffffu ? sum : sh.sub[r] + sum;
    if (some) {
      uint32_t t = 0;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) t += key[j] == thr;
      t = __reduce_add_sync(0xffffffffu, t);
      if (lane == 0) sh.tied[r] = t;
    }
  });
  if (tid == 0) sh.run_at = -1;
  __syncthreads();
  u64 part = tid < runs ? sh.sub[tid] : 0;
  const u64 tie_w = some ? weight(c, thr) : 0;
  if (some) {  // of the tied tokens the first `ties`
    const u64 mine = tid < runs ? sh.tied[tid] : 0, incl = block_prefix(&sh, mine);
    if (tid == kThreads - 1) sh.above = incl;
    __syncthreads();
    u64 all, unused, before;
    cluster_sum(c, sh.above, 0, all, unused, before);
    const u64 first = before + incl - mine;
    if (tid < runs) sh.tied[tid] = (uint32_t)first;
    part += tie_w * (first < ties ? min(mine, ties - first) : 0);
  }
  const u64 upto = block_prefix(&sh, part);
  if (tid == kThreads - 1) sh.above = upto;
  __syncthreads();
  u64 total, unused, before;
  cluster_sum(c, sh.above, 0, total, unused, before);
  const u64 target = draw_target(u, total);
  const u64 end = before + upto;
  if (target < end && end - part <= target) {  // the run that holds the target
    sh.run_at = tid;
    sh.run_sum = end - part;
  }
  __syncthreads();
  const int at = sh.run_at;
  if (at >= 0 && warp == 0) {
    uint32_t key[kBatch];
    read_keys(c, at * kRun + lane * kBatch, key);
    u64 w[kBatch], mine = 0, tied = 0;
    if (some) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) tied += key[j] == thr;
      tied = sh.tied[at] + warp_prefix(tied) - tied;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      w[j] = key[j] >= from ? to_fixed(weight_d(c, key[j])) : 0;
      if (some && key[j] == thr) w[j] = tied++ < ties ? tie_w : 0;
      mine += w[j];
    }
    u64 sum = sh.run_sum + warp_prefix(mine) - mine;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (sum <= target && target < sum + w[j]) {
        p.tokens[row] = i0 + at * kRun + lane * kBatch + j;
        if (p.logprob) p.logprob[row] = log_prob(c, key[j], w[j], total);
      }
      sum += w[j];
    }
  }
  c.cl.sync();  // a peer may still read this CTA's shared memory
}

template <typename T>
static hxm_status launch(Params p, int rows, cudaStream_t st) {
  typedef typename Key<T>::type K;
  // CTAs per row: as many as leave room for two on an SM (82 KB of keys each; 8 CTAs reach 2^18 tokens
  // of 32 bits with one on an SM), more while that leaves SMs idle: a thread then has fewer tokens
  int cl = 1;
  while (cl < 8 && (size_t)((p.vocab + cl - 1) / cl) * sizeof(K) > 82 * 1024) cl *= 2;
  while (cl < 8 && (int64_t)rows * cl * 2 <= 2 * 148 && p.vocab / cl > 4 * kThreads) cl *= 2;
  p.slice = ((p.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t smem = kRegion + (size_t)(p.slice + 8) * sizeof(K);  // 8: kernel's pad
  const hxm_status s = allow_shared_memory<sample_kernel<T>, true>();
  if (s != HXM_OK) return s;
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
