// linear_attn.cu — linear attention with a constant decay per head: argument checks, dispatch, the
// CUDA-core kernel (fp32, and bf16 shapes that the tensor-core kernel does not take) and the
// single-token step (sm_100a).
//
// The reference has no such kernel; the recurrence is its mLSTM loop
// (hybrid_xmamba/kernels/tfla/tfla_interface.py:113-137) with a constant forget gate and without
// input gate and normalizer.
#include "linear_attn.h"

#include "capi_internal.h"
#include "common.cuh"

namespace hxm {
namespace lattn {

constexpr int kSMs = 148;

struct GenericParams {
  Common c;
  Problem p[3];
};

// g^n for n >= 0 from log2(g) in 64 bits: exponents reach the sequence length, where a 32-bit
// product n * log2(g) would lose the factor's low bits.
HXM_DEV float decay_pow(double lg2, int n) { return n == 0 ? 1.f : (float)exp2(lg2 * n); }

// Rows 0 .. C - 1 of a chunk to shared memory as fp32: row r is time t0 + r * dt (r < nc), `cols` columns, zeros
// elsewhere up to `pitch` (a multiple of 4).  Aligned fp32 rows by 16-byte copies that all are on their way at
// once (the caller waits), others eight elements a thread at a time.
template <typename T, int C>
HXM_DEV void load_rows(float* dst, int ld, int pitch, const T* src, int64_t stride, int64_t t0, int dt, int nc, int cols) {
  if (sizeof(T) == 4 && cols % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    const int pv = pitch / 4;
    for (int i = threadIdx.x; i < C * pv; i += 256) {
      const int r = i / pv, d = 4 * (i - r * pv);
      const bool in = r < nc && d < cols;
      const T* from = in ? src + (t0 + (int64_t)r * dt) * stride + d : src;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + r * ld + d)),
                   "l"(from), "r"(in ? 16 : 0)
                   : "memory");
    }
    return;
  }
  constexpr int B = 8;
  for (int i0 = threadIdx.x; i0 < C * pitch; i0 += 256 * B) {
    T x[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + 256 * k, r = i / pitch, d = i - r * pitch;
      x[k] = __ldg(src + (r < nc && d < cols ? (t0 + (int64_t)r * dt) * stride + d : t0 * stride));
    }
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + 256 * k, r = i / pitch, d = i - r * pitch;
      if (r < C) dst[r * ld + d] = r < nc && d < cols ? to_f32<T>(x[k]) : 0.f;
    }
  }
}
template <int N> struct Pairs { float2 v[N / 2]; };
template <int N> HXM_DEV Pairs<N> pairs(const float* at) { return *reinterpret_cast<const Pairs<N>*>(at); }
template <int N>
HXM_DEV void fma_row(Pairs<N>& acc, float a, const Pairs<N>& x) {
#pragma unroll
  for (int m = 0; m < N / 2; ++m) acc.v[m] = __ffma2_rn(make_float2(a, a), x.v[m], acc.v[m]);
}

// One CTA: (batch, head), TV value columns, one time segment, in chunks of C steps held in shared
// memory as fp32.  All sums are fp32 FMAs, so fp32 inputs keep their precision; per step and head
// that is 2 C dk (for each TV columns) + 2 C dv + 4 dk dv operations on the FP32 pipe, which bounds it: each of
// the 256 threads holds a tile of C / 16 rows by TV / 16 columns of the product at hand, so that a float4 of
// shared memory serves C / 16 or TV / 16 FMAs for each of its elements.  8 x 2048 x 16 heads of 128, fp32: 1.10 ms,
// of which the products take four fifths, at half of the pipe's rate: a warp's 16-byte read takes four cycles of
// shared memory, and eight of them serve 64 FMAs a thread.  2 x 513 x 4 heads of 64: 34 us, half of it joining the
// segments.
template <typename T, int C, int TV>
__global__ void __launch_bounds__(256, 1) generic_kernel(const __grid_constant__ GenericParams gp, int dkp, int state_only) {
  constexpr int M = C / 16, N = TV / 16;
  const Common& cm = gp.c;
  const int b = blockIdx.z % cm.batch;
  const Problem& p = gp.p[blockIdx.z / cm.batch];
  const int segs = cm.nseg - state_only;  // the last one's sum is nobody's entering state
  const int h = blockIdx.y, seg = blockIdx.x % segs, e0 = (blockIdx.x / segs) * TV;
  if (e0 >= p.dv) return;
  const int ld = dkp + 4;  // row pitch of Q, K
  extern __shared__ __align__(16) float sh[];
  float* Q = sh;             // [C][ld]
  float* K = Q + C * ld;     // [C][ld]
  float* V = K + C * ld;     // [C][TV]; times each row's weight in the state once the output has it
  float* X = V + C * TV;     // [dkp][TV]
  float* P = X + dkp * TV;   // [C][C]
  float* pw = P + C * C;     // [C + 1]: g^0 .. g^C
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, c0 = tx * N;
  const double lg2 = (double)cm.log_decay[h] * 1.4426950408889634;
  const int n = cm.lengths ? min(max(cm.lengths[b], 0), cm.seqlen) : cm.seqlen;
  const int u_lo = seg * cm.seg_len, u_hi = min(n, u_lo + cm.seg_len);
  const int is = p.reverse ? 0 : 1, fs = p.reverse ? 1 : 0;
  for (int i = tid; i <= C; i += 256) pw[i] = decay_pow(lg2, i);
  // the state entering the segment
  const int nprev = state_only || n == 0 ? 0 : min(seg, (n + cm.seg_len - 1) / cm.seg_len);
  const float f0 = state_only || !p.s0 ? 0.f : decay_pow(lg2, n == 0 ? 0 : u_lo + is) * p.s0_scale;
  __shared__ float join[kSMs];  // the earlier segments' factors; there are fewer segments than SMs
  for (int r = tid; r < nprev; r += 256) join[r] = decay_pow(lg2, u_lo - (r + 1) * cm.seg_len);
  __syncthreads();
  constexpr int B = 8;  // elements a thread has on their way (dkp * TV is a multiple of 128)
  for (int i0 = tid; i0 < dkp * TV; i0 += 256 * B) {
    float x[B], y[B];
    auto live = [&](int k) { return (i0 + 256 * k) / TV < p.dk && e0 + (i0 + 256 * k) % TV < p.dv; };
    // (absent elements read the first one: loads without branches, all on their way at once)
#pragma unroll
    for (int k = 0; k < B; ++k) x[k] = 0.f;
    if (f0 != 0.f) {
      const float* s0 = p.s0 + b * p.s0s[0] + h * p.s0s[1] + e0 * p.s0s[3];
#pragma unroll
      for (int k = 0; k < B; ++k) y[k] = __ldg(s0 + (live(k) ? (i0 + 256 * k) / TV * p.s0s[2] + (i0 + 256 * k) % TV * p.s0s[3] : 0));
#pragma unroll
      for (int k = 0; k < B; ++k) x[k] = live(k) ? f0 * y[k] : 0.f;
    }
    for (int r = 0; r < nprev; ++r) {
      const float* ws = p.ws + (((int64_t)b * cm.heads + h) * (cm.nseg - 1) + r) * p.dk * p.dv + e0;
#pragma unroll
      for (int k = 0; k < B; ++k) y[k] = __ldg(ws + (live(k) ? (int64_t)((i0 + 256 * k) / TV) * p.dv + (i0 + 256 * k) % TV : 0));
#pragma unroll
      for (int k = 0; k < B; ++k) x[k] = live(k) ? fmaf(join[r], y[k], x[k]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < B; ++k)
      if (i0 + 256 * k < dkp * TV) X[i0 + 256 * k] = x[k];
  }
  T* o = static_cast<T*>(p.o) + b * p.so[0] + h * p.so[2] + e0;
  const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + h * p.sq[2];
  const T* k = static_cast<const T*>(p.k) + b * p.sk[0] + h * p.sk[2];
  const T* v = static_cast<const T*>(p.v) + b * p.sv[0] + h * p.sv[2] + e0;
  if (!state_only) {  // rows past the sequence
    const int lo = max(n, u_lo), hi = min(cm.seqlen, u_lo + cm.seg_len);
    for (int64_t i = tid; i < (int64_t)(hi - lo) * TV; i += 256)
      if (e0 + i % TV < p.dv) o[(lo + i / TV) * p.so[1] + i % TV] = from_f32<T>(0.f);
  }
  const bool last_seg = n == 0 ? seg == 0 : (u_lo < n && u_hi == n);
  for (int u0 = u_lo; u0 < u_hi; u0 += C) {
    const int nc = min(C, u_hi - u0);
    const bool fin = !state_only && u0 + nc == n;  // exponents of the last state in the last chunk
    const int endexp = fin ? nc - 1 + fs : nc;
    const int64_t t0 = p.reverse ? n - 1 - u0 : u0;
    const int dt = p.reverse ? -1 : 1;
    __syncthreads();
    load_rows<T, C>(K, ld, dkp, k, p.sk[1], t0, dt, nc, p.dk);
    if (!state_only) load_rows<T, C>(Q, ld, dkp, q, p.sq[1], t0, dt, nc, p.dk);
    load_rows<T, C>(V, TV, TV, v, p.sv[1], t0, dt, nc, min(TV, p.dv - e0));
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (!state_only) {
      {  // P = (q_i . k_j) g^(i-j), j <= i
        float2 acc[M][M] = {};
#pragma unroll 2
        for (int d = 0; d < dkp; d += 4) {
          float4 a[M], c[M];
#pragma unroll
          for (int m = 0; m < M; ++m) {
            a[m] = *reinterpret_cast<const float4*>(Q + (ty + 16 * m) * ld + d);
            c[m] = *reinterpret_cast<const float4*>(K + (tx + 16 * m) * ld + d);
          }
#pragma unroll
          for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {  // columns of a later block of 16 lie behind all of the rows
              acc[i][j] = __ffma2_rn(make_float2(a[i].x, a[i].y), make_float2(c[j].x, c[j].y), acc[i][j]);
              acc[i][j] = __ffma2_rn(make_float2(a[i].z, a[i].w), make_float2(c[j].z, c[j].w), acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
          for (int j = 0; j < M; ++j) {
            const int r = ty + 16 * i, s = tx + 16 * j;
            P[r * C + s] = s <= r ? (acc[i][j].x + acc[i][j].y) * pw[r - s] : 0.f;
          }
      }
      __syncthreads();
      {  // out = scale (g^i Q X + P V)
        Pairs<N> acc[M] = {};
#pragma unroll 2
        for (int d = 0; d < dkp; d += 4) {
          float4 a[M];
#pragma unroll
          for (int i = 0; i < M; ++i) a[i] = *reinterpret_cast<const float4*>(Q + (ty + 16 * i) * ld + d);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const Pairs<N> x = pairs<N>(X + (d + m) * TV + c0);
#pragma unroll
            for (int i = 0; i < M; ++i) fma_row(acc[i], m == 0 ? a[i].x : m == 1 ? a[i].y : m == 2 ? a[i].z : a[i].w, x);
          }
        }
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
          for (int m = 0; m < N / 2; ++m) acc[i].v[m] = __fmul2_rn(make_float2(pw[ty + 16 * i], pw[ty + 16 * i]), acc[i].v[m]);
#pragma unroll 2
        for (int j = 0; j < nc; j += 4) {  // rows behind the last are zeros
          float4 a[M];
#pragma unroll
          for (int i = 0; i < M; ++i) a[i] = *reinterpret_cast<const float4*>(P + (ty + 16 * i) * C + j);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const Pairs<N> x = pairs<N>(V + (j + m) * TV + c0);
#pragma unroll
            for (int i = 0; i < M; ++i) fma_row(acc[i], m == 0 ? a[i].x : m == 1 ? a[i].y : m == 2 ? a[i].z : a[i].w, x);
          }
        }
        float2 odd = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
          for (int m = 0; m < N / 2; ++m) odd = __ffma2_rn(acc[i].v[m], make_float2(0.f, 0.f), odd);
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const int r = ty + 16 * i;
          if (r >= nc) continue;
          T* row = o + (t0 + (int64_t)r * dt) * p.so[1] + c0;
#pragma unroll
          for (int m = 0; m < N / 2; ++m) {
            if (e0 + c0 + 2 * m < p.dv) row[2 * m] = from_f32<T>(p.scale * acc[i].v[m].x);
            if (e0 + c0 + 2 * m + 1 < p.dv) row[2 * m + 1] = from_f32<T>(p.scale * acc[i].v[m].y);
          }
        }
        // An infinity or NaN in V reached the rows before it too (their weights are 0, and 0 * inf is NaN): a thread
        // with a sum that is not finite forms all of its sums again, each from the steps up to its row alone.
        if (odd.x + odd.y != 0.f) {
#pragma unroll 1
          for (int i = 0; i < M * N; ++i) {
            const int r = ty + 16 * (i / N), c = c0 + i % N;
            if (r >= nc || e0 + c >= p.dv) continue;
            float sum = 0.f;
#pragma unroll 1
            for (int d = 0; d < dkp; ++d) sum = fmaf(Q[r * ld + d], X[d * TV + c], sum);
            sum *= pw[r];
#pragma unroll 1
            for (int j = 0; j <= r; ++j) sum = fmaf(P[r * C + j], V[j * TV + c], sum);
            o[(t0 + (int64_t)r * dt) * p.so[1] + c] = from_f32<T>(p.scale * sum);
          }
        }
      }
      __syncthreads();
    }
    for (int i = tid; i < nc * TV; i += 256) V[i] *= pw[endexp - i / TV];
    __syncthreads();
    // X = g^endexp X + K^T V
    const float f = pw[endexp];
    for (int d = 4 * ty; d < dkp; d += 64) {
      Pairs<N> acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i] = pairs<N>(X + (d + i) * TV + c0);
#pragma unroll
        for (int m = 0; m < N / 2; ++m) acc[i].v[m] = __fmul2_rn(make_float2(f, f), acc[i].v[m]);
      }
#pragma unroll 4
      for (int j = 0; j < nc; ++j) {
        const float4 a = *reinterpret_cast<const float4*>(K + j * ld + d);
        const Pairs<N> x = pairs<N>(V + j * TV + c0);
        fma_row(acc[0], a.x, x);
        fma_row(acc[1], a.y, x);
        fma_row(acc[2], a.z, x);
        fma_row(acc[3], a.w, x);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<Pairs<N>*>(X + (d + i) * TV + c0) = acc[i];
    }
  }
  __syncthreads();
  if (state_only) {
    if (u_lo < n)
      for (int i = tid; i < dkp * TV; i += 256) {
        const int d = i / TV, e = e0 + i % TV;
        if (d < p.dk && e < p.dv) p.ws[((((int64_t)b * cm.heads + h) * (cm.nseg - 1) + seg) * p.dk + d) * p.dv + e] = X[i];
      }
  } else if (p.sT && last_seg) {
    for (int i = tid; i < dkp * TV; i += 256) {
      const int d = i / TV, e = e0 + i % TV;
      if (d < p.dk && e < p.dv) p.sT[b * p.sTs[0] + h * p.sTs[1] + d * p.sTs[2] + e * p.sTs[3]] = p.sT_scale * X[i];
    }
  }
}

// Rounded up so that rows stay float4-aligned.
static int padded_dk(int dk) { return (dk + 3) / 4 * 4; }

static size_t generic_smem(int C, int tv, int dkp) {
  return sizeof(float) * ((size_t)2 * C * (dkp + 4) + C * tv + (size_t)dkp * tv + C * C + C + 4);
}
// 64-step chunks and 64 columns while Q, K, X of the padded dk fit the shared memory of an SM (dk up to 256), else
// 32 and 32.
static int generic_tile(int dk) { return generic_smem(64, 64, padded_dk(dk)) + sizeof(float) * kSMs <= 227 * 1024 ? 64 : 32; }

template <typename T, int C>
static hxm_status launch_generic_c(const GenericParams& gp, int np, int dkp, int dv, bool state_only, cudaStream_t st) {
  const size_t smem = generic_smem(C, C, dkp);
  const hxm_status s = allow_shared_memory<generic_kernel<T, C, C>>();
  if (s != HXM_OK) return s;
  const dim3 grid((unsigned)((dv + C - 1) / C * (gp.c.nseg - (state_only ? 1 : 0))), (unsigned)gp.c.heads, (unsigned)(gp.c.batch * np));
  generic_kernel<T, C, C><<<grid, 256, smem, st>>>(gp, dkp, state_only ? 1 : 0);
  return check_launch("hxm_linear_attn");
}

static hxm_status launch_generic(const Common& c, const Problem* p, int np, hxm_dtype io, bool state_only, cudaStream_t st) {
  GenericParams gp{};
  gp.c = c;
  int dk = 0, dv = 0;
  for (int i = 0; i < np; ++i) {
    gp.p[i] = p[i];
    dk = p[i].dk > dk ? p[i].dk : dk;
    dv = p[i].dv > dv ? p[i].dv : dv;
  }
  const int dkp = padded_dk(dk);
  if (generic_tile(dk) == 64)
    return io == HXM_F32 ? launch_generic_c<float, 64>(gp, np, dkp, dv, state_only, st)
                         : launch_generic_c<__nv_bfloat16, 64>(gp, np, dkp, dv, state_only, st);
  return io == HXM_F32 ? launch_generic_c<float, 32>(gp, np, dkp, dv, state_only, st)
                       : launch_generic_c<__nv_bfloat16, 32>(gp, np, dkp, dv, state_only, st);
}

// ---- checks, time segments, dispatch -------------------------------------------------------------

static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Segments: the recurrence is sequential in time, so a call with fewer CTAs than SMs is cut along
// time; every segment but the last first sums its own k v^T (pass one), the others' sums are joined
// when a segment starts.  Pass one and the joining cost about half a chunk's and a few chunks' time on
// the tensor cores, so a segment has `least` chunks there (4); on the FP32 pipe a chunk takes so much
// longer that one will do (2 x 513 x 4 heads of 64, fp32: 34 us; two chunks 54, uncut 98).
static void set_segments(Common& c, int64_t ctas, int chunk, int least) {
  const int chunks = ceil_div(c.seqlen, chunk);
  int64_t want = ctas > 0 ? kSMs / ctas : 1;
  if (want > chunks / least) want = chunks / least;
  if (want < 2) want = 1;
  c.seg_len = (int)(ceil_div(chunks, want) * (int64_t)chunk);
  c.nseg = c.seqlen > 0 ? ceil_div(c.seqlen, c.seg_len) : 1;
}

static size_t ws_floats(const Common& c, const Problem& p) {
  return (size_t)c.batch * c.heads * (c.nseg - 1) * p.dk * p.dv;
}

static hxm_status check_args(const hxm_linear_attn_args* a, const char* who) {
  HXM_REQUIRE(a != nullptr, "%s: args is NULL", who);
  HXM_REQUIRE(a->struct_size == sizeof(hxm_linear_attn_args), "%s: struct_size %zu != %zu", who, a->struct_size,
              sizeof(hxm_linear_attn_args));
  HXM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->heads >= 0 && a->dk >= 1 && a->dv >= 1,
              "%s: bad dims B=%d L=%d H=%d dk=%d dv=%d", who, a->batch, a->seqlen, a->heads, a->dk, a->dv);
  HXM_REQUIRE(a->io_dtype == HXM_F32 || a->io_dtype == HXM_BF16, "%s: io_dtype must be f32 or bf16", who);
  HXM_REQUIRE_SUPPORTED(a->dk <= 512, "%s: dk %d (at most 512)", who, a->dk);
  HXM_REQUIRE_SUPPORTED((int64_t)a->batch * 3 <= 65535 && a->heads <= 65535, "%s: batch %d (at most 21845) or heads %d (at most 65535)", who,
                        a->batch, a->heads);
  HXM_REQUIRE_SUPPORTED(a->seqlen <= (1 << 30), "%s: seqlen %d (at most 2^30)", who, a->seqlen);
  // the gradients divide by it
  HXM_REQUIRE(fabsf(a->scale) >= 0x1p-126f && fabsf(a->scale) <= 0x1p126f, "%s: scale must be nonzero, of 2^-126 to 2^126", who);
  return HXM_OK;
}

static Common make_common(const hxm_linear_attn_args* a) {
  Common c{};
  c.batch = a->batch; c.heads = a->heads; c.seqlen = a->seqlen;
  c.log_decay = a->log_decay; c.lengths = a->lengths;
  c.error_flag = a->error_flag;
  c.wait_limit = a->wait_limit_cycles != 0 ? a->wait_limit_cycles : 4000000000ll;
  return c;
}

static Problem fwd_problem(const hxm_linear_attn_args* a) {
  Problem p{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->out;
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = a->q_stride[i]; p.sk[i] = a->k_stride[i]; p.sv[i] = a->v_stride[i]; p.so[i] = a->out_stride[i];
  }
  p.dk = a->dk; p.dv = a->dv;
  p.s0 = a->s0; p.sT = a->sT;
  for (int i = 0; i < 4; ++i) { p.s0s[i] = a->s0_stride[i]; p.sTs[i] = a->sT_stride[i]; }
  p.scale = a->scale; p.s0_scale = 1.f; p.sT_scale = 1.f;
  return p;
}

// The gradients' three runs (see linear_attn.h): dq, dv, dk.
static void bwd_problems(const hxm_linear_attn_bwd_args* a, Problem out[3]) {
  const hxm_linear_attn_args& f = a->fwd;
  const int64_t L = f.seqlen, H = f.heads;
  auto dense = [&](int64_t s[3], int d) { s[0] = L * H * d; s[1] = H * d; s[2] = d; };
  auto copy = [](int64_t* d, const int64_t* s, int n) { for (int i = 0; i < n; ++i) d[i] = s[i]; };
  auto turned = [](int64_t* d, const int64_t* s) { d[0] = s[0]; d[1] = s[1]; d[2] = s[3]; d[3] = s[2]; };
  for (int i = 0; i < 3; ++i) {
    out[i] = Problem{};
    out[i].scale = f.scale;
    out[i].s0_scale = 1.f;
    out[i].sT_scale = 1.f;
  }
  Problem& dq = out[0];
  dq.q = a->dout; dq.k = f.v; dq.v = f.k; dq.o = a->dq;
  copy(dq.sq, a->dout_stride, 3); copy(dq.sk, f.v_stride, 3); copy(dq.sv, f.k_stride, 3); dense(dq.so, f.dk);
  dq.dk = f.dv; dq.dv = f.dk;
  dq.s0 = f.s0; turned(dq.s0s, f.s0_stride);
  Problem& dv = out[1];
  dv.q = f.k; dv.k = f.q; dv.v = a->dout; dv.o = a->dv;
  copy(dv.sq, f.k_stride, 3); copy(dv.sk, f.q_stride, 3); copy(dv.sv, a->dout_stride, 3); dense(dv.so, f.dv);
  dv.dk = f.dk; dv.dv = f.dv; dv.reverse = 1;
  dv.s0 = a->dsT; copy(dv.s0s, a->dsT_stride, 4); dv.s0_scale = 1.f / f.scale;
  dv.sT = a->ds0; dv.sT_scale = f.scale;
  dv.sTs[0] = H * f.dk * f.dv; dv.sTs[1] = (int64_t)f.dk * f.dv; dv.sTs[2] = f.dv; dv.sTs[3] = 1;
  Problem& dk = out[2];
  dk.q = f.v; dk.k = a->dout; dk.v = f.q; dk.o = a->dk;
  copy(dk.sq, f.v_stride, 3); copy(dk.sk, a->dout_stride, 3); copy(dk.sv, f.q_stride, 3); dense(dk.so, f.dk);
  dk.dk = f.dv; dk.dv = f.dk; dk.reverse = 1;
  dk.s0 = a->dsT; turned(dk.s0s, a->dsT_stride); dk.s0_scale = 1.f / f.scale;
}

// Which kernel runs these problems, and the time segments.
static bool plan(Common& c, const Problem* p, int np, hxm_dtype io) {
  bool tc = true;
  int64_t ctas = 0;
  int dk = 0;
  for (int i = 0; i < np; ++i) {
    tc = tc && tc_ok(p[i], c.seqlen, io);
    dk = p[i].dk > dk ? p[i].dk : dk;
  }
  for (int i = 0; i < np; ++i) ctas += (int64_t)c.batch * c.heads * ceil_div(p[i].dv, tc ? 64 : generic_tile(dk));
  if (tc) set_segments(c, ctas, 128, 4);
  else set_segments(c, ctas, 64, 1);
  return tc;
}

static hxm_status run(Common c, Problem* p, int np, hxm_dtype io, float* ws, size_t ws_bytes, cudaStream_t st, const char* who) {
  const bool tc = plan(c, p, np, io);
  size_t need = 0;
  for (int i = 0; i < np; ++i) {
    p[i].ws = ws + need;
    need += ws_floats(c, p[i]);
  }
  HXM_REQUIRE(need == 0 || (ws && ws_bytes >= need * sizeof(float)), "%s: workspace %zu bytes < %zu", who, ws_bytes,
              need * sizeof(float));
  HXM_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(ws) % 16 == 0, "%s: workspace must be 16-byte aligned", who);
  for (int pass = c.nseg > 1 ? 0 : 1; pass < 2; ++pass) {
    if (!tc) {
      const hxm_status s = launch_generic(c, p, np, io, pass == 0, st);
      if (s != HXM_OK) return s;
      continue;
    }
    // runs of the same padded dk share a launch
    Problem group[3];
    for (int wide = 0; wide < 2; ++wide) {
      int n = 0;
      for (int i = 0; i < np; ++i)
        if ((p[i].dk > 128) == (wide == 1)) group[n++] = p[i];
      if (n) {
        const hxm_status s = launch_tc(c, group, n, pass == 0, st);
        if (s != HXM_OK) return s;
      }
    }
  }
  return HXM_OK;
}

// ---- single-token step -----------------------------------------------------------------------------

struct StepParams {
  int heads, dk, dv;
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t sq[2], sk[2], sv[2], so[2];
  const float* log_decay;
  float* s;
  int64_t ss[3];
  float scale;
};

// S = g S + k v^T and out = scale S^T q for one token: the state is read and written once, 8 dk dv
// bytes, which is all the time there is.  One CTA per (batch, head, 32 * VEC value columns); its
// 8 warps share the dk rows, lane l holds VEC columns, and the warps' partial sums of the output
// join in shared memory.  A warp has kRows rows on their way at once: 128 x 16 states of 128 x 128 take
// 42 us, 6.3 TB/s (row by row, the store of one before the load of the next, 55 us).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) step_kernel(const StepParams p) {
  constexpr int kRows = 8;
  const int h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int e = (blockIdx.x * 32 + lane) * VEC;
  const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + h * p.sq[1];
  const T* k = static_cast<const T*>(p.k) + b * p.sk[0] + h * p.sk[1];
  const T* v = static_cast<const T*>(p.v) + b * p.sv[0] + h * p.sv[1];
  float* s = p.s + b * p.ss[0] + h * p.ss[1] + e;
  __shared__ float part[8][32 * VEC];
  float acc[VEC] = {};
  if (e < p.dv) {
    for (int d0 = warp; d0 < p.dk; d0 += 8 * kRows) {
      float x[kRows][VEC], kd[kRows], qd[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (d0 + 8 * r < p.dk) {
          const float* row = s + (d0 + 8 * r) * p.ss[2];
          if (VEC == 4) *reinterpret_cast<float4*>(x[r]) = __ldcs(reinterpret_cast<const float4*>(row));
          else x[r][0] = row[0];
        }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const bool in = d0 + 8 * r < p.dk;
        kd[r] = in ? to_f32<T>(k[d0 + 8 * r]) : 0.f;
        qd[r] = in ? to_f32<T>(q[d0 + 8 * r]) : 0.f;
      }
      const float g = (float)exp2((double)p.log_decay[h] * 1.4426950408889634);
      float vv[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) vv[i] = to_f32<T>(v[e + i]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (d0 + 8 * r >= p.dk) continue;
        float* row = s + (d0 + 8 * r) * p.ss[2];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          x[r][i] = fmaf(g, x[r][i], kd[r] * vv[i]);
          acc[i] = fmaf(qd[r], x[r][i], acc[i]);
        }
        if (VEC == 4) __stcs(reinterpret_cast<float4*>(row), *reinterpret_cast<float4*>(x[r]));
        else row[0] = x[r][0];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[warp][lane * VEC + i] = acc[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const int c = blockIdx.x * 32 * VEC + i;
    if (c < p.dv) {
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) y += part[w][i];
      static_cast<T*>(p.o)[b * p.so[0] + h * p.so[1] + c] = from_f32<T>(p.scale * y);
    }
  }
}

template <typename T>
static hxm_status launch_step(const StepParams& p, int batch, cudaStream_t st) {
  // 16-byte state accesses where every row allows them
  const bool vec = p.dv % 4 == 0 && reinterpret_cast<uintptr_t>(p.s) % 16 == 0 && p.ss[0] % 4 == 0 && p.ss[1] % 4 == 0 && p.ss[2] % 4 == 0;
  if (vec) step_kernel<T, 4><<<dim3((p.dv + 127) / 128, p.heads, batch), 256, 0, st>>>(p);
  else step_kernel<T, 1><<<dim3((p.dv + 31) / 32, p.heads, batch), 256, 0, st>>>(p);
  return check_launch("hxm_linear_attn_step");
}

}  // namespace lattn
}  // namespace hxm

using namespace hxm;
using namespace hxm::lattn;

extern "C" size_t hxm_linear_attn_workspace_size(const hxm_linear_attn_args* a) {
  if (check_args(a, "hxm_linear_attn_workspace_size") != HXM_OK) return 0;
  Common c = make_common(a);
  const Problem p = fwd_problem(a);
  plan(c, &p, 1, a->io_dtype);
  return ws_floats(c, p) * sizeof(float);
}

extern "C" hxm_status hxm_linear_attn_fwd(const hxm_linear_attn_args* a, void* stream) {
  clear_error();
  const hxm_status s = check_args(a, "hxm_linear_attn_fwd");
  if (s != HXM_OK) return s;
  if (a->batch == 0 || a->heads == 0) return HXM_OK;
  HXM_REQUIRE(a->log_decay && (a->seqlen == 0 || (a->q && a->k && a->v && a->out)), "hxm_linear_attn_fwd: NULL tensor pointer");
  Problem p = fwd_problem(a);
  return run(make_common(a), &p, 1, a->io_dtype, static_cast<float*>(a->workspace), a->workspace_bytes,
             static_cast<cudaStream_t>(stream), "hxm_linear_attn_fwd");
}

static hxm_status check_bwd(const hxm_linear_attn_bwd_args* a, const char* who) {
  HXM_REQUIRE(a != nullptr, "%s: args is NULL", who);
  HXM_REQUIRE(a->struct_size == sizeof(hxm_linear_attn_bwd_args), "%s: struct_size %zu != %zu", who, a->struct_size,
              sizeof(hxm_linear_attn_bwd_args));
  const hxm_status s = check_args(&a->fwd, who);
  if (s != HXM_OK) return s;
  HXM_REQUIRE_SUPPORTED(a->fwd.dv <= 512, "%s: dv %d (at most 512)", who, a->fwd.dv);
  return HXM_OK;
}

extern "C" size_t hxm_linear_attn_bwd_workspace_size(const hxm_linear_attn_bwd_args* a) {
  if (check_bwd(a, "hxm_linear_attn_bwd_workspace_size") != HXM_OK) return 0;
  Common c = make_common(&a->fwd);
  Problem p[3];
  bwd_problems(a, p);
  plan(c, p, 3, a->fwd.io_dtype);
  return (ws_floats(c, p[0]) + ws_floats(c, p[1]) + ws_floats(c, p[2])) * sizeof(float);
}

extern "C" hxm_status hxm_linear_attn_bwd(const hxm_linear_attn_bwd_args* a, void* stream) {
  clear_error();
  const hxm_status s = check_bwd(a, "hxm_linear_attn_bwd");
  if (s != HXM_OK) return s;
  const hxm_linear_attn_args& f = a->fwd;
  if (f.batch == 0 || f.heads == 0) return HXM_OK;
  HXM_REQUIRE(f.log_decay && (f.seqlen == 0 || (f.q && f.k && f.v && a->dout && a->dq && a->dk && a->dv)),
              "hxm_linear_attn_bwd: NULL tensor pointer");
  Problem p[3];
  bwd_problems(a, p);
  return run(make_common(&f), p, 3, f.io_dtype, static_cast<float*>(a->workspace), a->workspace_bytes,
             static_cast<cudaStream_t>(stream), "hxm_linear_attn_bwd");
}

extern "C" hxm_status hxm_linear_attn_step(const hxm_linear_attn_step_args* a, void* stream) {
  clear_error();
  HXM_REQUIRE(a != nullptr, "hxm_linear_attn_step: args is NULL");
  HXM_REQUIRE(a->struct_size == sizeof(hxm_linear_attn_step_args), "hxm_linear_attn_step: struct_size %zu != %zu",
              a->struct_size, sizeof(hxm_linear_attn_step_args));
  HXM_REQUIRE(a->batch >= 0 && a->heads >= 0 && a->dk >= 1 && a->dv >= 1, "hxm_linear_attn_step: bad dims B=%d H=%d dk=%d dv=%d",
              a->batch, a->heads, a->dk, a->dv);
  HXM_REQUIRE(a->io_dtype == HXM_F32 || a->io_dtype == HXM_BF16, "hxm_linear_attn_step: io_dtype must be f32 or bf16");
  HXM_REQUIRE_SUPPORTED(a->batch <= 65535 && a->heads <= 65535, "hxm_linear_attn_step: batch %d or heads %d above 65535", a->batch, a->heads);
  if (a->batch == 0 || a->heads == 0) return HXM_OK;
  HXM_REQUIRE(a->q && a->k && a->v && a->out && a->state && a->log_decay, "hxm_linear_attn_step: NULL tensor pointer");
  StepParams p{};
  p.heads = a->heads; p.dk = a->dk; p.dv = a->dv;
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->out;
  for (int i = 0; i < 2; ++i) { p.sq[i] = a->q_stride[i]; p.sk[i] = a->k_stride[i]; p.sv[i] = a->v_stride[i]; p.so[i] = a->out_stride[i]; }
  p.log_decay = a->log_decay; p.s = a->state;
  for (int i = 0; i < 3; ++i) p.ss[i] = a->state_stride[i];
  p.scale = a->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->io_dtype == HXM_F32 ? launch_step<float>(p, a->batch, st) : launch_step<__nv_bfloat16>(p, a->batch, st);
}
