// qk_norm_rope.cu — RMS norm of every head of q and k with the position rotation in the same pass,
// and its gradients (sm_100a).
//
// Replaces the two per-head norms of mLSTMBlock.forward (hybrid_xmamba/layers/mlstm_block.py:113-114,
// RMSNorm.forward of layers/normalization.py:32-34) for layers that also rotate q and k.  HBM-bound:
// x is read once and y written once (gradients: x and dy read, dx written).
// 8 x 2048 tokens of 16 + 4 heads of 128, bf16: 33.5 us, 5.0 TB/s; gradients 62 us, 4.0 TB/s (latency: two blocks
// of 256 threads fit an SM), 68 with the join of the weights' sums.  fp32: 60 us, 5.6 TB/s, and 93 us.  Rows off
// their alignment (row_kernel): bf16 169 us and 390.
//
// A row is one head of one token.  With n = x / sqrt(mean x^2 + eps) and y = R (w * n), R turning the
// pairs, the gradients are g = R^T dy, dw = sum over rows of g * n, and
//   dx = (w g - n mean(w g n)) / sqrt(mean x^2 + eps).
// The angle positions * base^(-2p/rotary) is formed in 64 bits, in turns, and only its fraction goes
// to 32 bits: at position 10^6 a 32-bit angle would be off by 0.06.
#include "capi_internal.h"
#include "common.cuh"

namespace hxm {
namespace qknr {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;

struct Side {
  const void* x;
  int64_t sx[3];
  const float* w;
  void* out;  // y, or dx
  int64_t so[3];
  const void* g;  // gradients: dy
  int64_t sg[3];
  int heads;
};

struct Params {
  Side s[2];  // q, k
  int batch, seqlen, dim, rotary, interleaved;
  const int64_t* pos;
  int64_t spos[2];
  double log2_base;
  float eps;
  float* partial;  // gradients: (blocks, 2, dim) weight sums
  int tokens_per_block, blocks;
};

// cos, sin of every pair of `nt` tokens from token `tok0` on, into cs[token * rotary/2 + pair].
HXM_DEV void angles(const Params& p, int64_t tok0, int nt, float2* cs) {
  const int half = p.rotary / 2;
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int64_t tok = tok0 + i / half;
    const int pr = i % half;
    const int64_t at = p.pos[(tok / p.seqlen) * p.spos[0] + (tok % p.seqlen) * p.spos[1]];
    // turns = position * frequency / (2 pi)
    const double turns = (double)at * (exp2(-2.0 * pr / p.rotary * p.log2_base) * 0.15915494309189535);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(c, s);
  }
}

// How a lane holds its V elements of a row, and which of them are pairs.
enum Mode : int {
  kHalves = 0,  // V/2 elements from each half of the rotated part: pairs (j, j + V/2); behind it V in a row
  kRun = 1,     // V elements in a row: pairs (2j, 2j + 1), those behind `rotary` turn by 0
};

// 16 bytes of a row as float2s, and back (the one rounding of a 16-bit result).
template <typename T>
HXM_DEV void widen(const uint4& raw, float2 (&v)[8 / sizeof(T)]) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int j = 0; j < (int)(8 / sizeof(T)); ++j) v[j] = make_float2(to_f32<T>(e[2 * j]), to_f32<T>(e[2 * j + 1]));
}
template <typename T>
HXM_DEV uint4 narrow(const float2 (&v)[8 / sizeof(T)]) {
  uint4 raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int j = 0; j < (int)(8 / sizeof(T)); ++j) {
    e[2 * j] = from_f32<T>(v[j].x);
    e[2 * j + 1] = from_f32<T>(v[j].y);
  }
  return raw;
}
HXM_DEV float2 both(float a) { return make_float2(a, a); }

// Rows that fit the registers of G <= 32 lanes, NV * 16 bytes a lane.  A group of G lanes takes one token
// and every (256 / G / tokens_per_block)-th of its heads, so a lane's cosines and sines serve all of its
// rows; R rows are loaded before the first is worked on, for the latency of HBM.  The instructions weigh as
// much as the bytes (some 100 a row and lane), so the arithmetic goes two elements at a time.
template <typename T, int G, int NV, int MODE, bool BWD>
__global__ void __launch_bounds__(kThreads) vec_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T), H = V / 2, F = V / 2, A = V / 4, R = NV > 1 ? 2 : 4;
  extern __shared__ __align__(16) unsigned char shraw[];
  double* freq = reinterpret_cast<double*>(shraw);  // turns per position of each pair
  const int half = p.rotary / 2;
  const int gl = threadIdx.x & (G - 1), group = threadIdx.x / G;
  constexpr int kGroups = kThreads / G;
  const int it = group & (p.tokens_per_block - 1), h0 = group / p.tokens_per_block, hs = kGroups / p.tokens_per_block;
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  for (int i = threadIdx.x; i < half; i += kThreads)
    freq[i] = exp2(-2.0 * i / p.rotary * p.log2_base) * 0.15915494309189535;
  __syncthreads();
  // column of element j of this lane's vector i
  auto col = [&](int i, int j) {
    const int v = i * G + gl;
    return MODE == kHalves && v * V < p.rotary ? v * H + (j < H ? j : j - H + half) : v * V + j;
  };
  const bool has[2] = {gl * V < p.dim, NV > 1 && (G + gl) * V < p.dim};  // dim is a multiple of V
  float2 dw[2][NV][F];
  if (BWD) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) dw[s][i][j] = both(0.f);
  }
  auto load = [&](const T* row, int i) {
    if (MODE == kRun) return *reinterpret_cast<const uint4*>(row + (i * G + gl) * V);
    const uint2 a = *reinterpret_cast<const uint2*>(row + col(i, 0));
    const uint2 b = *reinterpret_cast<const uint2*>(row + col(i, H));
    return make_uint4(a.x, a.y, b.x, b.y);
  };
  auto store = [&](T* row, int i, const uint4& raw) {
    if (MODE == kRun) {
      *reinterpret_cast<uint4*>(row + (i * G + gl) * V) = raw;
    } else {
      *reinterpret_cast<uint2*>(row + col(i, 0)) = make_uint2(raw.x, raw.y);
      *reinterpret_cast<uint2*>(row + col(i, H)) = make_uint2(raw.z, raw.w);
    }
  };
  const float per_dim = 1.f / (float)p.dim;
  for (int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block; tok0 < tokens; tok0 += (int64_t)gridDim.x * p.tokens_per_block) {
    const int64_t tok = tok0 + it;
    const bool here = tok < tokens;
    const int64_t b = here ? tok / p.seqlen : 0, t = here ? tok - b * p.seqlen : 0;
    float2 cs[NV][A], sn[NV][A];  // of pairs 2j, 2j + 1 of this lane; the gradients turn back
    if (half) {
      const int64_t at = here ? p.pos[b * p.spos[0] + t * p.spos[1]] : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const int pr = (i * G + gl) * H + j;
          const double turns = (double)at * freq[pr < half ? pr : 0];
          float s, c;
          sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
          if (pr >= half) c = 1.f, s = 0.f;
          if (BWD) s = -s;
          (j & 1 ? cs[i][j / 2].y : cs[i][j / 2].x) = c;
          (j & 1 ? sn[i][j / 2].y : sn[i][j / 2].x) = s;
        }
    }
    auto turn = [&](float2 (&y)[F], int i) {
      if (!half) return;
      if (MODE == kHalves) {
#pragma unroll
        for (int j = 0; j < A; ++j) {
          const float2 u = y[j], v = y[A + j], c = cs[i][j], s = sn[i][j];
          y[j] = __ffma2_rn(u, c, __fmul2_rn(make_float2(-v.x, -v.y), s));
          y[A + j] = __ffma2_rn(v, c, __fmul2_rn(u, s));
        }
      } else {
#pragma unroll
        for (int j = 0; j < F; ++j) {
          const float c = j & 1 ? cs[i][j / 2].y : cs[i][j / 2].x, s = j & 1 ? sn[i][j / 2].y : sn[i][j / 2].x;
          const float2 u = y[j];
          y[j] = make_float2(u.x * c - u.y * s, u.y * c + u.x * s);
        }
      }
    };
#pragma unroll
    for (int sd = 0; sd < 2; ++sd) {
      const Side& s = p.s[sd];
      float2 w[NV][F];
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) w[i][j] = s.w && has[i] ? *reinterpret_cast<const float2*>(s.w + col(i, 2 * j)) : both(1.f);
      const T* xt = static_cast<const T*>(s.x) + b * s.sx[0] + t * s.sx[1] + h0 * s.sx[2];
      const T* gt = BWD ? static_cast<const T*>(s.g) + b * s.sg[0] + t * s.sg[1] + h0 * s.sg[2] : nullptr;
      T* ot = static_cast<T*>(s.out) + b * s.so[0] + t * s.so[1] + h0 * s.so[2];
      const int64_t xs = hs * s.sx[2], gs = BWD ? hs * s.sg[2] : 0, os = hs * s.so[2];
      const int rows = here ? s.heads - h0 : 0;  // of this lane: those r with r * hs < rows
      // every lane of the warp goes through the loop (the shuffles need them all)
      for (int hb = 0; hb < s.heads; hb += R * hs) {
        uint4 xr[R][NV], gr[R][NV];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const bool live = hb + r * hs < rows && has[i];
            xr[r][i] = live ? load(xt, i) : make_uint4(0, 0, 0, 0);
            if (BWD) gr[r][i] = live ? load(gt, i) : make_uint4(0, 0, 0, 0);
          }
          xt += xs;
          if (BWD) gt += gs;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (hb + r * hs >= s.heads) break;  // block-uniform
          float2 x[NV][F], sq = both(0.f);
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            widen<T>(xr[r][i], x[i]);
#pragma unroll
            for (int j = 0; j < F; ++j) sq = __ffma2_rn(x[i][j], x[i][j], sq);
          }
          float ssq = sq.x + sq.y;
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
          // a lane without a row adds nothing to the weight sums: there rsqrt would be infinite for eps = 0
          const float2 inv = both(!BWD || hb + r * hs < rows ? rsqrtf(fmaf(ssq, per_dim, p.eps)) : 0.f);
          if (!BWD) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
              for (int j = 0; j < F; ++j) x[i][j] = __fmul2_rn(__fmul2_rn(x[i][j], inv), w[i][j]);
              turn(x[i], i);
            }
          } else {
            float2 g[NV][F], mm = both(0.f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
              widen<T>(gr[r][i], g[i]);
              turn(g[i], i);
#pragma unroll
              for (int j = 0; j < F; ++j) {
                x[i][j] = __fmul2_rn(x[i][j], inv);
                const float2 gn = __fmul2_rn(g[i][j], x[i][j]);
                dw[sd][i][j] = __fadd2_rn(dw[sd][i][j], gn);  // 0 where this lane has no row
                mm = __ffma2_rn(gn, w[i][j], mm);
              }
            }
            float m = mm.x + mm.y;
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
            const float2 mean = both(-m * per_dim);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
              for (int j = 0; j < F; ++j) x[i][j] = __fmul2_rn(inv, __ffma2_rn(x[i][j], mean, __fmul2_rn(w[i][j], g[i][j])));
          }
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (hb + r * hs < rows && has[i]) store(ot, i, narrow<T>(x[i]));
          ot += os;
        }
      }
    }
  }
  if (BWD) {  // the block's weight sums: groups in order
    float* red = reinterpret_cast<float*>(shraw);  // [kGroups][dim]
#pragma unroll
    for (int sd = 0; sd < 2; ++sd) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i])
#pragma unroll
          for (int j = 0; j < F; ++j) *reinterpret_cast<float2*>(red + group * p.dim + col(i, 2 * j)) = dw[sd][i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.dim; c += kThreads) {
        float a = 0.f;
        for (int r = 0; r < kGroups; ++r) a += red[r * p.dim + c];
        p.partial[((int64_t)blockIdx.x * 2 + sd) * p.dim + c] = a;
      }
    }
  }
}

// Any other dim, stride or alignment: one warp a row, the row in shared memory.
template <typename T, bool BWD>
__global__ void __launch_bounds__(kThreads) row_kernel(const Params p) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ __align__(16) unsigned char shraw[];
  const int half = p.rotary / 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2* cs = reinterpret_cast<float2*>(shraw);
  float* buf = reinterpret_cast<float*>(cs + half) + warp * 2 * p.dim;  // this warp's row, and its gradient
  float* acc = reinterpret_cast<float*>(cs + half) + kWarps * 2 * p.dim;  // [2][kWarps][dim] weight sums
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  if (BWD)
    for (int i = threadIdx.x; i < 2 * kWarps * p.dim; i += kThreads) acc[i] = 0.f;
  for (int64_t tok = blockIdx.x; tok < tokens; tok += gridDim.x) {
    __syncthreads();
    if (half) angles(p, tok, 1, cs);
    __syncthreads();
    const int64_t b = tok / p.seqlen, t = tok % p.seqlen;
    for (int r = warp; r < p.s[0].heads + p.s[1].heads; r += kWarps) {
      const int sd = r >= p.s[0].heads;
      const Side& s = p.s[sd];
      const int h = sd ? r - p.s[0].heads : r;
      const T* x = static_cast<const T*>(s.x) + b * s.sx[0] + t * s.sx[1] + h * s.sx[2];
      T* out = static_cast<T*>(s.out) + b * s.so[0] + t * s.so[1] + h * s.so[2];
      float* xs = buf;
      float* gs = buf + p.dim;
      __syncwarp();
      float ssq = 0.f;
      for (int c = lane; c < p.dim; c += 32) {
        const float v = to_f32<T>(x[c]);
        xs[c] = v;
        ssq = fmaf(v, v, ssq);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
      const float inv = rsqrtf(ssq / (float)p.dim + p.eps);
      if (BWD) {
        const T* g = static_cast<const T*>(s.g) + b * s.sg[0] + t * s.sg[1] + h * s.sg[2];
        for (int c = lane; c < p.dim; c += 32) gs[c] = to_f32<T>(g[c]);
      }
      __syncwarp();
      float* src = BWD ? gs : xs;
      const float sign = BWD ? -1.f : 1.f;
      // element c of the rotated row: src (times the weight going forward) turned with its partner
      auto turned = [&](int c) {
        auto val = [&](int i) { return BWD ? src[i] : src[i] * inv * (s.w ? s.w[i] : 1.f); };
        if (c >= p.rotary) return val(c);
        const int pr = p.interleaved ? c >> 1 : (c < half ? c : c - half);
        const bool first = p.interleaved ? (c & 1) == 0 : c < half;
        const int mate = p.interleaved ? c ^ 1 : (first ? c + half : c - half);
        const float2 a = cs[pr];
        return first ? val(c) * a.x - val(mate) * (sign * a.y) : val(c) * a.x + val(mate) * (sign * a.y);
      };
      if (!BWD) {
        for (int c = lane; c < p.dim; c += 32) out[c] = from_f32<T>(turned(c));
      } else {
        float m = 0.f;
        for (int c = lane; c < p.dim; c += 32) {
          const float n = xs[c] * inv, g = turned(c);
          acc[(sd * kWarps + warp) * p.dim + c] += g * n;
          m = fmaf(g * n, s.w ? s.w[c] : 1.f, m);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        m /= (float)p.dim;
        for (int c = lane; c < p.dim; c += 32)
          out[c] = from_f32<T>(inv * ((s.w ? s.w[c] : 1.f) * turned(c) - xs[c] * inv * m));
      }
    }
  }
  if (BWD) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.dim; i += kThreads) {
      float a = 0.f;
      for (int w = 0; w < kWarps; ++w) a += acc[((i / p.dim) * kWarps + w) * p.dim + i % p.dim];
      p.partial[(int64_t)blockIdx.x * 2 * p.dim + i] = a;
    }
  }
}

// Joins the blocks' weight sums in a fixed order: one block per 32 columns, 8 rows at a time.
__global__ void __launch_bounds__(kThreads) join_kernel(const float* partial, int blocks, int dim, float* dwq, float* dwk) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, wr = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;  // column of the 2 * dim
  float a = 0.f;
  if (c < 2 * dim)
    for (int r = wr; r < blocks; r += 8) a += partial[(int64_t)r * 2 * dim + c];
  red[wr][lane] = a;
  __syncthreads();
  if (wr == 0 && c < 2 * dim) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) s += red[r][lane];
    float* out = c < dim ? dwq : dwk;
    if (out) out[c < dim ? c : c - dim] = s;
  }
}

constexpr int kSMs = 148;
// Blocks whose weight sums the gradients keep: the two per SM that are resident (with four, in two waves,
// 8 x 2048 x 20 x 128 took 75 us instead of 62), of the shared-memory kernel four (604 us with two, 357).
constexpr int kBwdBlocks = 2 * kSMs, kBwdBlocksRow = 4 * kSMs;

template <typename T, int G, int NV, int MODE, bool BWD>
static hxm_status launch_mode(Params& p, cudaStream_t st) {
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  // tokens a block takes at once: one while blocks are few, for their number; up to 16, so that a lane's
  // angles serve more rows (8 x 2048 x 20 x 128 bf16 33.5 us, with up to 8 36.5); gradients 8, whose blocks
  // then have even shares
  int tpb = 1;
  while (tpb < (BWD ? 8 : 16) && tpb * 2 <= kThreads / G && tokens / (tpb * 2) >= 4 * kSMs) tpb *= 2;
  p.tokens_per_block = tpb;
  int64_t grid = (tokens + tpb - 1) / tpb;
  if (grid > 16 * kSMs) grid = 16 * kSMs;  // the pairs' frequencies are made once a block
  size_t smem = (size_t)(p.rotary / 2) * sizeof(double);
  if (BWD) {
    const size_t red = (size_t)(kThreads / G) * p.dim * sizeof(float);
    if (red > smem) smem = red;
    // blocks that take no token write zeros: the join reads all sums
    grid = p.blocks = kBwdBlocks;
  }
  vec_kernel<T, G, NV, MODE, BWD><<<(unsigned)grid, kThreads, smem, st>>>(p);
  return check_launch("hxm_qk_norm_rope");
}

template <typename T, int G, int NV, bool BWD>
static hxm_status launch_vec(Params& p, cudaStream_t st) {
  return p.rotary == 0 || p.interleaved ? launch_mode<T, G, NV, kRun, BWD>(p, st) : launch_mode<T, G, NV, kHalves, BWD>(p, st);
}

template <typename T, bool BWD>
static hxm_status launch(Params& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // the register kernel: whole vectors, in the rotated part too where its pairs lie half of it apart
  bool vec = p.dim % V == 0 && p.dim <= 64 * V && (p.interleaved || p.rotary % V == 0);
  for (int i = 0; i < 2; ++i) {
    const Side& s = p.s[i];
    auto ok = [&](const void* ptr, const int64_t* st3) {
      return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && st3[0] % V == 0 && st3[1] % V == 0 && st3[2] % V == 0;
    };
    vec = vec && reinterpret_cast<uintptr_t>(s.w) % 8 == 0 && (s.heads == 0 || (ok(s.x, s.sx) && ok(s.out, s.so) && (!BWD || ok(s.g, s.sg))));
  }
  if (vec) {
    const int nvec = p.dim / V;
    if (nvec <= 4) return launch_vec<T, 4, 1, BWD>(p, st);
    if (nvec <= 8) return launch_vec<T, 8, 1, BWD>(p, st);
    if (nvec <= 16) return launch_vec<T, 16, 1, BWD>(p, st);
    if (nvec <= 32) return launch_vec<T, 32, 1, BWD>(p, st);
    return launch_vec<T, 32, 2, BWD>(p, st);
  }
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  const unsigned grid = BWD ? (unsigned)(p.blocks = kBwdBlocksRow) : (unsigned)(tokens < 16 * kSMs ? tokens : 16 * kSMs);
  const size_t smem = (size_t)(p.rotary / 2) * sizeof(float2) + sizeof(float) * p.dim * (kThreads / 32) * (BWD ? 4 : 2);
  const hxm_status s = allow_shared_memory<row_kernel<T, BWD>>();
  if (s != HXM_OK) return s;
  row_kernel<T, BWD><<<grid, kThreads, smem, st>>>(p);
  return check_launch("hxm_qk_norm_rope");
}

static hxm_status check_args(const hxm_qk_norm_rope_args* a, const char* who) {
  HXM_REQUIRE(a != nullptr, "%s: args is NULL", who);
  HXM_REQUIRE(a->struct_size == sizeof(hxm_qk_norm_rope_args), "%s: struct_size %zu != %zu", who, a->struct_size,
              sizeof(hxm_qk_norm_rope_args));
  HXM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->heads_q >= 0 && a->heads_k >= 0 && a->dim >= 1,
              "%s: bad dims B=%d L=%d Hq=%d Hk=%d dim=%d", who, a->batch, a->seqlen, a->heads_q, a->heads_k, a->dim);
  HXM_REQUIRE(a->io_dtype == HXM_F32 || a->io_dtype == HXM_BF16 || a->io_dtype == HXM_F16, "%s: bad io_dtype %d", who, (int)a->io_dtype);
  HXM_REQUIRE_SUPPORTED(a->dim <= kMaxDim, "%s: dim %d (at most %d)", who, a->dim, kMaxDim);
  HXM_REQUIRE(a->rotary >= 0 && a->rotary <= a->dim && a->rotary % 2 == 0, "%s: rotary %d must be even and at most dim %d", who,
              a->rotary, a->dim);
  HXM_REQUIRE(a->rotary == 0 || (a->rope_base > 0 && a->rope_base - a->rope_base == 0), "%s: rope_base must be positive and finite", who);
  HXM_REQUIRE(a->eps >= 0 && a->eps - a->eps == 0, "%s: eps must be finite and at least 0", who);
  HXM_REQUIRE_SUPPORTED((int64_t)a->heads_q + a->heads_k <= (1 << 20), "%s: %lld heads", who, (long long)a->heads_q + a->heads_k);
  return HXM_OK;
}

static Params make_params(const hxm_qk_norm_rope_args* a) {
  Params p{};
  auto side = [](Side& s, const void* x, const int64_t* sx, const float* w, void* o, const int64_t* so, int heads) {
    s.x = x; s.w = w; s.out = o; s.heads = heads;
    for (int i = 0; i < 3; ++i) { s.sx[i] = sx[i]; s.so[i] = so[i]; }
  };
  side(p.s[0], a->q, a->q_stride, a->q_weight, a->q_out, a->q_out_stride, a->heads_q);
  side(p.s[1], a->k, a->k_stride, a->k_weight, a->k_out, a->k_out_stride, a->heads_k);
  p.batch = a->batch; p.seqlen = a->seqlen; p.dim = a->dim; p.rotary = a->rotary; p.interleaved = a->interleaved;
  p.pos = a->positions; p.spos[0] = a->positions_stride[0]; p.spos[1] = a->positions_stride[1];
  p.log2_base = a->rotary ? log2(a->rope_base) : 0;
  p.eps = a->eps;
  return p;
}

}  // namespace qknr
}  // namespace hxm

using namespace hxm;
using namespace hxm::qknr;

extern "C" hxm_status hxm_qk_norm_rope_fwd(const hxm_qk_norm_rope_args* a, void* stream) {
  clear_error();
  const hxm_status s = check_args(a, "hxm_qk_norm_rope_fwd");
  if (s != HXM_OK) return s;
  if ((int64_t)a->batch * a->seqlen == 0 || a->heads_q + a->heads_k == 0) return HXM_OK;
  HXM_REQUIRE((a->heads_q == 0 || (a->q && a->q_out)) && (a->heads_k == 0 || (a->k && a->k_out)) && (a->rotary == 0 || a->positions),
              "hxm_qk_norm_rope_fwd: NULL tensor pointer");
  Params p = make_params(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->io_dtype == HXM_F32) return launch<float, false>(p, st);
  return a->io_dtype == HXM_BF16 ? launch<__nv_bfloat16, false>(p, st) : launch<__half, false>(p, st);
}

static hxm_status check_bwd(const hxm_qk_norm_rope_bwd_args* a, const char* who) {
  HXM_REQUIRE(a != nullptr, "%s: args is NULL", who);
  HXM_REQUIRE(a->struct_size == sizeof(hxm_qk_norm_rope_bwd_args), "%s: struct_size %zu != %zu", who, a->struct_size,
              sizeof(hxm_qk_norm_rope_bwd_args));
  return check_args(&a->fwd, who);
}

extern "C" size_t hxm_qk_norm_rope_bwd_workspace_size(const hxm_qk_norm_rope_bwd_args* a) {
  if (check_bwd(a, "hxm_qk_norm_rope_bwd_workspace_size") != HXM_OK) return 0;
  return sizeof(float) * 2 * (size_t)a->fwd.dim * kBwdBlocksRow;
}

extern "C" hxm_status hxm_qk_norm_rope_bwd(const hxm_qk_norm_rope_bwd_args* a, void* stream) {
  clear_error();
  const hxm_status s = check_bwd(a, "hxm_qk_norm_rope_bwd");
  if (s != HXM_OK) return s;
  const hxm_qk_norm_rope_args& f = a->fwd;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((int64_t)f.batch * f.seqlen == 0 || f.heads_q + f.heads_k == 0) {
    if (a->dq_weight) HXM_CUDA_TRY(cudaMemsetAsync(a->dq_weight, 0, sizeof(float) * f.dim, st));
    if (a->dk_weight) HXM_CUDA_TRY(cudaMemsetAsync(a->dk_weight, 0, sizeof(float) * f.dim, st));
    return HXM_OK;
  }
  HXM_REQUIRE((f.heads_q == 0 || (f.q && f.q_out && a->dq_out)) && (f.heads_k == 0 || (f.k && f.k_out && a->dk_out)) &&
                  (f.rotary == 0 || f.positions), "hxm_qk_norm_rope_bwd: NULL tensor pointer");
  const size_t need = sizeof(float) * 2 * (size_t)f.dim * kBwdBlocksRow;
  HXM_REQUIRE(a->workspace && a->workspace_bytes >= need, "hxm_qk_norm_rope_bwd: workspace %zu bytes < %zu", a->workspace_bytes, need);
  Params p = make_params(&f);
  p.s[0].g = a->dq_out; p.s[1].g = a->dk_out;
  for (int i = 0; i < 3; ++i) { p.s[0].sg[i] = a->dq_out_stride[i]; p.s[1].sg[i] = a->dk_out_stride[i]; }
  p.partial = static_cast<float*>(a->workspace);
  const hxm_status r = f.io_dtype == HXM_F32 ? launch<float, true>(p, st)
                       : f.io_dtype == HXM_BF16 ? launch<__nv_bfloat16, true>(p, st) : launch<__half, true>(p, st);
  if (r != HXM_OK || (!a->dq_weight && !a->dk_weight)) return r;
  join_kernel<<<(2 * f.dim + 31) / 32, kThreads, 0, st>>>(p.partial, p.blocks, f.dim, a->dq_weight, a->dk_weight);
  return check_launch("hxm_qk_norm_rope_bwd");
}
