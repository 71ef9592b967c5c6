// qk_norm_rope.cu — RMS norm of every head of q and k with the position rotation in the same pass,
// and its gradients (sm_100a).
//
// Replaces the two per-head norms of mLSTMBlock.forward (hybrid_xmamba/layers/mlstm_block.py:113-114,
// RMSNorm.forward of layers/normalization.py:32-34) for layers that also rotate q and k.  HBM-bound:
// x is read once and y written once (gradients: x and dy read, dx written).
//
// A row is one head of one token.  With n = x / sqrt(mean x^2 + eps) and y = R (w * n), R turning the
// pairs, the gradients are g = R^T dy, dw = sum over rows of g * n, and
//   dx = (w g - n mean(w g n)) / sqrt(mean x^2 + eps).
// The angle positions * base^(-2p/rotary) is formed in 64 bits, in turns, and only its fraction goes
// to 32 bits: at position 10^6 a 32-bit angle would be off by 0.06.  The cosines and sines of a token
// are made once for all of its heads, in shared memory.
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
  int tokens_per_block;
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

template <typename T, int V>
HXM_DEV void load_vec(const T* p, float (&v)[V]) {
  static_assert(V * sizeof(T) == 16, "16-byte vectors");
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = to_f32<T>(e[j]);
}
template <typename T, int V>
HXM_DEV void store_vec(T* p, const float (&v)[V]) {
  uint4 raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int j = 0; j < V; ++j) e[j] = from_f32<T>(v[j]);
  *reinterpret_cast<uint4*>(p) = raw;
}

// Turns this lane's vectors by sign * angle.  Lane `gl` of a row's G lanes holds vectors gl, gl + G, ..
// (NV of them); pairs of the half-split form sit in vectors half/V apart, fetched by shuffle.
template <int V, int NV>
HXM_DEV void rotate(float (&y)[NV][V], const Params& p, const float2* cs, int gl, int G, float sign) {
  if (p.rotary == 0) return;
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + gl) * V;
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        if (c + j < p.rotary) {
          const float2 t = cs[(c + j) >> 1];
          const float s = sign * t.y, a = y[i][j], b = y[i][j + 1];
          y[i][j] = a * t.x - b * s;
          y[i][j + 1] = b * t.x + a * s;
        }
      }
    }
    return;
  }
  const int half = p.rotary / 2, hv = half / V;  // half is a multiple of V on this path
  float other[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vi = i * G + gl;
    const int pv = vi < hv ? vi + hv : (vi < 2 * hv ? vi - hv : vi);
    const int src = ((threadIdx.x & 31) & ~(G - 1)) + (pv & (G - 1));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float r = __shfl_sync(0xffffffffu, y[0][j], src);
#pragma unroll
      for (int m = 1; m < NV; ++m) {
        const float t = __shfl_sync(0xffffffffu, y[m][j], src);
        if (pv / G == m) r = t;
      }
      other[i][j] = r;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vi = i * G + gl;
    if (vi < 2 * hv) {
      const bool first = vi < hv;
      const float2* t = cs + (first ? vi : vi - hv) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float s = sign * t[j].y;
        y[i][j] = first ? y[i][j] * t[j].x - other[i][j] * s : y[i][j] * t[j].x + other[i][j] * s;
      }
    }
  }
}

// Rows whose vectors fit the registers of G <= 32 lanes: dim a multiple of the 16-byte vector, NV
// vectors a lane.  A block takes tokens_per_block tokens with all of their heads; 256 / G rows at once.
template <typename T, int G, int NV, bool BWD>
__global__ void __launch_bounds__(kThreads) vec_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char shraw[];
  float2* cs = reinterpret_cast<float2*>(shraw);
  const int gl = threadIdx.x & (G - 1), group = threadIdx.x / G;
  constexpr int kGroups = kThreads / G;
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  const int half = p.rotary / 2;
  float dw[2][NV][V];
  if (BWD) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[s][i][j] = 0.f;
  }
  for (int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block; tok0 < tokens; tok0 += (int64_t)gridDim.x * p.tokens_per_block) {
    const int nt = (int)min((int64_t)p.tokens_per_block, tokens - tok0);
    if (half) {
      __syncthreads();
      angles(p, tok0, nt, cs);
      __syncthreads();
    }
#pragma unroll
    for (int sd = 0; sd < 2; ++sd) {
      const Side& s = p.s[sd];
      const int rows = nt * s.heads;
      float w[NV][V];
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (i * G + gl) * V + j;
          w[i][j] = c < p.dim ? (s.w ? s.w[c] : 1.f) : 0.f;
        }
      // every lane of the warp goes through the loop (the shuffles need them all)
      for (int r0 = 0; r0 < rows; r0 += kGroups) {
        const int r = r0 + group;
        const bool live = r < rows;
        const int it = live ? r / s.heads : 0, h = live ? r % s.heads : 0;
        const int64_t tok = tok0 + it, b = tok / p.seqlen, t = tok % p.seqlen;
        float x[NV][V];
        float ssq = 0.f;
        const T* xr = static_cast<const T*>(s.x) + b * s.sx[0] + t * s.sx[1] + h * s.sx[2];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * G + gl) * V;
#pragma unroll
          for (int j = 0; j < V; ++j) x[i][j] = 0.f;
          if (live && c < p.dim) load_vec<T, V>(xr + c, x[i]);
#pragma unroll
          for (int j = 0; j < V; ++j) ssq = fmaf(x[i][j], x[i][j], ssq);
        }
        float g[NV][V];
        if (BWD) {
          const T* gr = static_cast<const T*>(s.g) + b * s.sg[0] + t * s.sg[1] + h * s.sg[2];
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * G + gl) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) g[i][j] = 0.f;
            if (live && c < p.dim) load_vec<T, V>(gr + c, g[i]);
          }
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
        const float inv = rsqrtf(ssq / (float)p.dim + p.eps);
        T* orow = static_cast<T*>(s.out) + b * s.so[0] + t * s.so[1] + h * s.so[2];
        if (!BWD) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = x[i][j] * inv * w[i][j];
          rotate<V, NV>(x, p, cs + it * half, gl, G, 1.f);
        } else {
          rotate<V, NV>(g, p, cs + it * half, gl, G, -1.f);
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              x[i][j] *= inv;
              const float gn = g[i][j] * x[i][j];
              if (live) dw[sd][i][j] += gn;
              m = fmaf(gn, w[i][j], m);
            }
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
          m /= (float)p.dim;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = inv * (w[i][j] * g[i][j] - x[i][j] * m);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * G + gl) * V;
          if (live && c < p.dim) store_vec<T, V>(orow + c, x[i]);
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
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (i * G + gl) * V + j;
          if (c < p.dim) red[group * p.dim + c] = dw[sd][i][j];
        }
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
// Blocks whose weight sums the gradients keep: four per SM.
constexpr int kBwdBlocks = 4 * kSMs;

template <typename T, int G, int NV, bool BWD>
static hxm_status launch_vec(Params& p, cudaStream_t st) {
  const int64_t tokens = (int64_t)p.batch * p.seqlen;
  // tokens a block takes at once: more share the angles' latency, fewer fill the SMs
  int64_t tpb = tokens / (kSMs * 8);
  p.tokens_per_block = (int)(tpb < 1 ? 1 : (tpb > 8 ? 8 : tpb));
  int64_t grid = (tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  if (BWD && grid > kBwdBlocks) grid = kBwdBlocks;
  if (grid > 0x7fffffff) grid = 0x7fffffff;
  size_t smem = (size_t)p.tokens_per_block * (p.rotary / 2) * sizeof(float2);
  if (BWD) {
    const size_t red = (size_t)(kThreads / G) * p.dim * sizeof(float);
    if (red > smem) smem = red;
    // blocks that take no token write zeros: the join always reads kBwdBlocks sums
    grid = kBwdBlocks;
  }
  vec_kernel<T, G, NV, BWD><<<(unsigned)grid, kThreads, smem, st>>>(p);
  return check_launch("hxm_qk_norm_rope");
}

template <typename T, bool BWD>
static hxm_status launch(Params& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool vec = p.dim % V == 0 && p.dim <= 64 * V && (p.interleaved || (p.rotary / 2) % V == 0);
  for (int i = 0; i < 2; ++i) {
    const Side& s = p.s[i];
    auto ok = [&](const void* ptr, const int64_t* st3) {
      return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && st3[0] % V == 0 && st3[1] % V == 0 && st3[2] % V == 0;
    };
    vec = vec && (s.heads == 0 || (ok(s.x, s.sx) && ok(s.out, s.so) && (!BWD || ok(s.g, s.sg))));
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
  const unsigned grid = BWD ? kBwdBlocks : (unsigned)(tokens < 16 * kSMs ? tokens : 16 * kSMs);
  const size_t smem = (size_t)(p.rotary / 2) * sizeof(float2) + sizeof(float) * p.dim * (kThreads / 32) * (BWD ? 4 : 2);
  HXM_CUDA_TRY(cudaFuncSetAttribute(row_kernel<T, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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
  return sizeof(float) * 2 * (size_t)a->fwd.dim * kBwdBlocks;
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
  const size_t need = sizeof(float) * 2 * (size_t)f.dim * kBwdBlocks;
  HXM_REQUIRE(a->workspace && a->workspace_bytes >= need, "hxm_qk_norm_rope_bwd: workspace %zu bytes < %zu", a->workspace_bytes, need);
  Params p = make_params(&f);
  p.s[0].g = a->dq_out; p.s[1].g = a->dk_out;
  for (int i = 0; i < 3; ++i) { p.s[0].sg[i] = a->dq_out_stride[i]; p.s[1].sg[i] = a->dk_out_stride[i]; }
  p.partial = static_cast<float*>(a->workspace);
  const hxm_status r = f.io_dtype == HXM_F32 ? launch<float, true>(p, st)
                       : f.io_dtype == HXM_BF16 ? launch<__nv_bfloat16, true>(p, st) : launch<__half, true>(p, st);
  if (r != HXM_OK || (!a->dq_weight && !a->dk_weight)) return r;
  join_kernel<<<(2 * f.dim + 31) / 32, kThreads, 0, st>>>(p.partial, kBwdBlocks, f.dim, a->dq_weight, a->dk_weight);
  return check_launch("hxm_qk_norm_rope_bwd");
}
