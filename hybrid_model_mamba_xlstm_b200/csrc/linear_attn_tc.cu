// linear_attn_tc.cu — linear attention with a constant decay per head on the tensor cores (tcgen05).
//
// One CTA per (batch, head, 64 value columns, time segment) walks its steps in chunks of C = 128
// (see linear_attn.h for the algebra; i, j are steps in the chunk, X the carried matrix):
//   S = Q K^T                                   (M = N = 128, K = dk)
//   P = S * g^(64-j) for j <= i, in bf16        (group A; stays in TMEM, the A operand of the next)
//   O = Q bf16(g^64 X) + P V                    (N = 64, one accumulator)
//   out = scale g^(i-64) O                      (group A)
//   U = K^T (V * g^(end-j))                     (M = dk, N = 64 per part of the scaled V)
//   X = g^end X + U                             (group B, in fp32 registers)
// The decay inside a chunk separates into a factor of the column and one of the row.  Those reach
// g^+-64, so heads with 64 |log2 g| > 32 (g < 0.707) weigh P by g^(i-j) itself and keep the two
// products of the output apart, O2 taking its factor g^i at the end.
// Roundings to bf16: P and the copy of X that multiplies Q, one operand of each product of the bf16
// output, as its inputs are.  They bring the norm of the output's error to 1.41 times that of its own rounding
// (2.3e-3 of the output's norm, the rounding alone 1.65e-3).  A second part of X would need 16 KB of shared
// memory, of which less than 1 KB is left for dk <= 128, and the two second parts a fifth more operand
// reads, which bound the kernel.  X itself, which is returned in fp32, comes from products that are exact to
// 32 bits: k is bf16 already, and a scaled V value is carried in three bf16 parts, which leave at most 2^-24 of it
// (two would leave up to 2^-16).
//
// Work is cut by role, so that the tensor core always has something queued while one chunk's
// element-wise work runs: warps 0-7 (group A) turn S into P and write the output; warps 8-23 (group B)
// scale V, keep X and write its bf16 copy; warp 24 issues the MMAs, warp 25 the TMA loads.  S, O and the
// operand stages are double-buffered (dk <= 128), so S of the next chunk is made while this one's P is,
// and group B has the next chunk's scaled V in registers when U of this one is done: the only chain
// from chunk to chunk is U -> X -> bf16(X).
// Reversed time (the gradients) only mirrors a chunk: row r of a tile is step 127 - r, which flips the
// causal mask and the exponents' sign.
#include "capi_internal.h"
#include "linear_attn.h"
#include "tc_sm100.cuh"
#include "tma_host.h"

namespace hxm {
namespace lattn {

constexpr int kC = 128;    // steps per chunk
constexpr int kDV = 64;    // value columns per CTA
constexpr int kParts = 3;  // bf16 parts of a scaled V value: 2^-24 left over
constexpr int kPanel = 16384;  // 128 rows x 128 bytes
// Two warpgroups of group A, four of B, and one for the MMA and TMA warps (its other two warps only
// give up their registers).
constexpr int kThreadsTc = 7 * 128;
constexpr int kWarpsB = 16;
// Registers a thread: the launch gives 72 to all; the last warpgroup goes down to 40 and group A,
// with 32 columns of S at a time, up to 88: 2 * 88 + 4 * 72 + 40 <= 7 * 72.
constexpr int kRegsLaunch = 72, kRegsA = 88, kRegsCtrl = 40;
static_assert(2 * kRegsA + 4 * kRegsLaunch + kRegsCtrl <= 7 * kRegsLaunch, "register split");

struct TcParams {
  CUtensorMap map[9];  // q, k, v of each problem
  Common c;
  Problem p[3];
  int mh[9], mb[9];  // 0 where the tensor repeats along heads / batch, else 1
};

// DK: dk padded to 128 or 256 (TMA fills the rest with zeros).
template <int DK>
struct Layout {
  static constexpr int kNP = DK / 64, kNB = DK / 128;
  static constexpr int kStages = DK == 128 ? 2 : 1;
  static constexpr int kQ = 0, kK = kNP * kPanel, kV = 2 * kNP * kPanel, kStage = kV + kPanel;
  static constexpr int kSnap = kStages * kStage;  // bf16 X: DK rows of 128 bytes
  static constexpr int kVs = kSnap + DK * 128;    // the scaled V's parts
  static constexpr int kPw = kVs + kParts * kPanel;  // float[132]: g^0 .. g^128
  static constexpr int kCf = kPw + 132 * 4;       // float[128]: g^(64 - step) by tile row
  static constexpr int kBar = kCf + 128 * 4;      // 18 mbarriers
  static constexpr int kSlot = kBar + 18 * 8;
  static constexpr int kBytes = kSlot + 16;
  // TMEM columns: two S / P; two O (or O1, O2); U: the first two parts of the scaled V side by side
  // (dk <= 128), or one sum per 128 rows of X
  static constexpr int tS = 0, tO = 256, tU = 384;
  static_assert(kPw % 16 == 0 && kBar % 8 == 0, "alignment");
  static_assert(kBytes + 1024 <= 227 * 1024, "shared memory");
};

// D[tmem] (+)= A[tmem] * B[smem]^T: A is bf16, two of its columns in each 32-bit TMEM column.
template <uint32_t BOFF>
HXM_DEV void mma_bf16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bbase, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "add.s64 b, %2, %5;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bbase), "r"(idesc), "r"((uint32_t)accumulate), "n"(BOFF >> 4)
      : "memory");
}

// One lane of a converged warp.  With this predicate, unlike `lane == 0`, the compiler knows that a
// single lane is active, and takes the MMA descriptors to uniform registers without a loop.
HXM_DEV bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

HXM_DEV float decay_pow_tc(double lg2, int n) { return n == 0 ? 1.f : (float)exp2(lg2 * n); }

template <int DK>
__global__ void __launch_bounds__(kThreadsTc, 1) tc_kernel(const __grid_constant__ TcParams prm, const int tiles,
                                                           const int state_only) {
  using Lt = Layout<DK>;
  constexpr int kNP = Lt::kNP, kNB = Lt::kNB, kStages = Lt::kStages;
  const Common& cm = prm.c;
  const int b = blockIdx.z % cm.batch, ip = blockIdx.z / cm.batch;
  const Problem& p = prm.p[ip];
  const int h = blockIdx.y, e0 = (blockIdx.x % tiles) * kDV, seg = blockIdx.x / tiles;
  if (e0 >= p.dv) return;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* pw = reinterpret_cast<float*>(sm + Lt::kPw);
  float* cf = reinterpret_cast<float*>(sm + Lt::kCf);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + Lt::kBar);  // [2] TMA: a stage's operands
  uint64_t* empty = full + 2;     // [2] MMA: a stage's last reader done
  uint64_t* s_ready = full + 4;   // [2] MMA: S
  uint64_t* p_ready = full + 6;   // [2] group A: P in TMEM
  uint64_t* o_ready = full + 8;   // [2] MMA: O
  uint64_t* o_free = full + 10;   // [2] group A: O read
  uint64_t* x_ready = full + 12;  // group B: bf16 X written
  uint64_t* v_ready = full + 13;  // group B: scaled V written, U of the chunk before read
  uint64_t* u_ready = full + 14;  // MMA: U
  uint64_t* qs_done = full + 15;  // MMA: bf16 X read
  uint64_t* fin = full + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(sm + Lt::kSlot);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + Lt::kSlot + 4);
  volatile int* not_finite = reinterpret_cast<volatile int*>(sm + Lt::kSlot + 8);  // group B: met such a v

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wq = warp & 3, hf = (warp >> 2) & 1;  // TMEM lane quarter, column half
  const int row = wq * 32 + lane, ch = 32 * hf;
  const bool rev = p.reverse != 0;
  const int n = cm.lengths ? min(max(cm.lengths[b], 0), cm.seqlen) : cm.seqlen;
  const int u_lo = seg * cm.seg_len, u_hi = max(u_lo, min(n, u_lo + cm.seg_len));
  const int nch = (u_hi - u_lo + kC - 1) / kC;
  const int is = rev ? 0 : 1, fs = rev ? 1 : 0;
  const double lg2 = (double)cm.log_decay[h] * 1.4426950408889634;
  const long long limit = cm.wait_limit;

  if (warp == 0) tc::tmem_alloc(slot, 512);
  if (tid == 32) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(full + i, 1);
      tc::mbar_init(empty + i, 1);
      tc::mbar_init(s_ready + i, 1);
      tc::mbar_init(p_ready + i, 8);
      tc::mbar_init(o_ready + i, 1);
      tc::mbar_init(o_free + i, 8);
    }
    tc::mbar_init(x_ready, kWarpsB);
    tc::mbar_init(v_ready, kWarpsB);
    tc::mbar_init(u_ready, 1);
    tc::mbar_init(qs_done, 1);
    tc::mbar_init(fin, 1);
    tc::fence_mbar_init();
    *abort_flag = 0;
    *not_finite = 0;
    if (nch > 0)
      for (int i = 0; i < 3; ++i) tc::prefetch_tmap(&prm.map[3 * ip + i]);
  }
  const bool sep = lg2 * -64.0 <= 32.0;  // see the head of the file
  if (tid >= 256 && tid < 256 + kC + 1) pw[tid - 256] = decay_pow_tc(lg2, tid - 256);
  if (tid >= 64 && tid < 64 + kC) cf[tid - 64] = sep ? (float)exp2(lg2 * (64 - (rev ? kC - 1 - (tid - 64) : tid - 64))) : 1.f;
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tb = *slot;
  const uint32_t tm = tb + ((uint32_t)(wq * 32) << 16);

  // steps of chunk k in this segment, and the exponent that its end adds to X
  auto rows_of = [&](int k) { return min(kC, u_hi - u_lo - k * kC); };
  auto end_of = [&](int k) {
    const int nc = rows_of(k);
    return !state_only && u_lo + k * kC + nc == n ? nc - 1 + fs : nc;
  };
  // first time step of chunk k's tile (reversed: may be negative, TMA fills with zeros)
  auto t0_of = [&](int k) { return rev ? n - (u_lo + (k + 1) * kC) : u_lo + k * kC; };
  const int ul = rev ? kC - 1 - row : row;  // this row's step in the chunk
  auto wait = [&](uint64_t* bar, int parity) {  // warp-uniform
    return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity & 1, abort_flag, limit)) != 0;
  };

  if (warp < 8) {
    // ======================= group A: P, outputs =======================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsA));
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.o) + b * p.so[0] + h * p.so[2] + e0;
    if (!state_only) {  // rows past the sequence
      const int lo = max(n, u_lo), hi = min(cm.seqlen, u_lo + cm.seg_len);
      for (int64_t i = tid; i < (int64_t)(hi - lo) * 8; i += 256)
        if (e0 + (i & 7) * 8 < p.dv)
          *reinterpret_cast<uint4*>(o + (lo + (i >> 3)) * p.so[1] + (i & 7) * 8) = make_uint4(0, 0, 0, 0);
    }
    const float rf = p.scale * (sep ? (float)exp2(lg2 * (ul - 64)) : 1.f);  // the output row's factor
    auto weigh = [&](int k) -> bool {
      const int buf = k & 1;
      if (!wait(s_ready + buf, k >> 1)) return false;
      tc::tc_fence_after();
      const uint32_t ts = tm + Lt::tS + 128 * buf + 64 * hf;  // this thread's 64 columns of S
#pragma unroll
      for (int sb = 0; sb < 2; ++sb) {
        const int cb = 2 * hf + sb;  // 32-column block; this warp's rows are block wq
        uint32_t w[16];
        if (rev ? cb >= wq : cb <= wq) {
          float v[32];
          tc::tmem_ld32(ts + 32 * sb, v);
          tc::tmem_wait_ld();
          if (sep) {
            const float4* c4 = reinterpret_cast<const float4*>(cf + 32 * cb);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 c = c4[j];
              const float2 lo = __fmul2_rn(make_float2(v[4 * j], v[4 * j + 1]), make_float2(c.x, c.y));
              const float2 hi = __fmul2_rn(make_float2(v[4 * j + 2], v[4 * j + 3]), make_float2(c.z, c.w));
              v[4 * j] = lo.x;
              v[4 * j + 1] = lo.y;
              v[4 * j + 2] = hi.x;
              v[4 * j + 3] = hi.y;
            }
          } else {
            // masked columns read up to 31 words ahead of the table (the scaled V lies there): dropped below
            const float* d = pw + (rev ? 32 * cb - row : row - 32 * cb);
            const int sg = rev ? 1 : -1;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= d[sg * j];
          }
          if (cb == wq) {
            const uint32_t keep = rev ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = (keep >> j) & 1 ? v[j] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack2<__nv_bfloat16>(v[2 * j], v[2 * j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = 0;
        }
        // over columns of S that this thread has read
        tc::tmem_st16(ts + 16 * sb, reinterpret_cast<const float(&)[16]>(w));
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_ready + buf);
      return true;
    };
    // Zeros stand in V for the values that are not finite (see store_v): these make the outputs of their own and of the
    // later steps NaN.  From the chunk on in which the first one was met; rare, so all v of the chunk up to this
    // row's step are simply read again.
    auto not_finite_rows = [&](int k, float (&a)[32]) {
      const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v) + b * p.sv[0] + h * p.sv[2] + e0 + ch;
#pragma unroll 1
      for (int s = 0; s <= ul; ++s) {
        const int u = u_lo + k * kC + s;
        const __nv_bfloat16* vr = v + (int64_t)(rev ? n - 1 - u : u) * p.sv[1];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (e0 + ch + 8 * q >= p.dv) break;
          const uint4 raw = *reinterpret_cast<const uint4*>(vr + 8 * q);
          const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = __bfloat1622float2(e[j]);
            a[8 * q + 2 * j] = fmaf(0.f, f.x, a[8 * q + 2 * j]);
            a[8 * q + 2 * j + 1] = fmaf(0.f, f.y, a[8 * q + 2 * j + 1]);
          }
        }
      }
    };
    auto output = [&](int k) -> bool {
      if (!wait(o_ready + (k & 1), k >> 1)) return false;
      tc::tc_fence_after();
      float a[32];
      if (sep) {
        tc::tmem_ld32(tm + Lt::tO + 64 * (k & 1) + ch, a);
        tc::tmem_wait_ld();
      } else {
        float x[32];
        tc::tmem_ld32(tm + Lt::tO + ch, a);
        tc::tmem_ld32(tm + Lt::tO + 64 + ch, x);
        tc::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) a[j] = fmaf(pw[ul], x[j], a[j]);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(o_free + (k & 1));
      if (ul < rows_of(k)) {
        if (*not_finite) not_finite_rows(k, a);
        const int64_t t = rev ? n - 1 - (u_lo + k * kC + ul) : u_lo + k * kC + ul;
        __nv_bfloat16* orow = o + t * p.so[1] + ch;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack2<__nv_bfloat16>(rf * a[8 * q + 2 * j], rf * a[8 * q + 2 * j + 1]);
          if (e0 + ch + 8 * q < p.dv) *reinterpret_cast<uint4*>(orow + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      return true;
    };
    if (!state_only) {
      if (kStages == 2) {
        bool ok = nch > 0 && weigh(0);
#pragma unroll 1
        for (int k = 0; ok && k < nch; ++k) {
          if (k + 1 < nch) ok = weigh(k + 1);
          ok = ok && output(k);
        }
      } else {
        bool ok = true;
#pragma unroll 1
        for (int k = 0; ok && k < nch; ++k) ok = weigh(k) && output(k);
      }
    }
  } else if (warp < 8 + kWarpsB) {
    // ======================= group B: scaled V, X =======================
    const int cb = 16 * ((warp - 8) >> 2);  // this thread: a row of V and of X, 16 columns
    float X[kNB][16];
    {  // the state entering the segment
      const int nprev = state_only || n == 0 ? 0 : min(seg, (n + cm.seg_len - 1) / cm.seg_len);
      const float f0 = state_only || !p.s0 ? 0.f : decay_pow_tc(lg2, n == 0 ? 0 : u_lo + is) * p.s0_scale;
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk) {
        const int d = blk * 128 + row;
        const bool first = !state_only && p.s0;
        const float* src = first ? p.s0 + b * p.s0s[0] + h * p.s0s[1] + d * p.s0s[2] + (e0 + cb) * p.s0s[3] : nullptr;
        const bool vec = first && p.s0s[3] == 1 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (first && d < p.dk && e0 + cb + j < p.dv) {  // dv is a multiple of 8
            if (vec) y = *reinterpret_cast<const float4*>(src + j);
            else y = make_float4(src[j * p.s0s[3]], src[(j + 1) * p.s0s[3]], src[(j + 2) * p.s0s[3]], src[(j + 3) * p.s0s[3]]);
          }
          X[blk][j] = f0 * y.x;
          X[blk][j + 1] = f0 * y.y;
          X[blk][j + 2] = f0 * y.z;
          X[blk][j + 3] = f0 * y.w;
        }
      }
      if (u_lo < n)
        for (int r = 0; r < nprev; ++r) {
          const float f = decay_pow_tc(lg2, u_lo - (r + 1) * cm.seg_len);
#pragma unroll
          for (int blk = 0; blk < kNB; ++blk) {
            const int d = blk * 128 + row;
            const float* w = p.ws + ((((int64_t)b * cm.heads + h) * (cm.nseg - 1) + r) * p.dk + d) * p.dv + e0 + cb;
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              if (d < p.dk && e0 + cb + j < p.dv) {
                const float4 y = *reinterpret_cast<const float4*>(w + j);
                X[blk][j] = fmaf(f, y.x, X[blk][j]);
                X[blk][j + 1] = fmaf(f, y.y, X[blk][j + 1]);
                X[blk][j + 2] = fmaf(f, y.z, X[blk][j + 2]);
                X[blk][j + 3] = fmaf(f, y.w, X[blk][j + 3]);
              }
          }
        }
    }
    const float xf = sep ? cf[rev ? kC - 1 : 0] : 1.f;  // g^64
    auto snapshot = [&]() {
      if (!state_only) {
#pragma unroll
        for (int blk = 0; blk < kNB; ++blk)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack2<__nv_bfloat16>(xf * X[blk][8 * q + 2 * j], xf * X[blk][8 * q + 2 * j + 1]);
            *reinterpret_cast<uint4*>(sm + Lt::kSnap + tc::sw128_offset(blk * 128 + row, cb + 8 * q)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(x_ready);
      }
    };
    uint32_t vp[kParts][8];  // this row's 16 scaled values in bf16 parts
    auto scale_v = [&](int k) -> bool {
      const int st = k % kStages;
      unsigned char* stage = sm + st * Lt::kStage;
      const int nc = rows_of(k);
      if (!wait(full + st, k / kStages)) return false;
      // rows past the end of a shorter sequence hold other data: K and V read as zeros there
      if (!rev && nc < kC && t0_of(k) + nc < cm.seqlen) {
        if (!state_only && !wait(s_ready + (k & 1), k >> 1)) return false;
        if (row >= nc) {
#pragma unroll
          for (int i = 0; i < 2 * kNP; ++i) {  // this warp's share of the K row
            const int at = (cb >> 4) * 2 * kNP + i;
            *reinterpret_cast<uint4*>(stage + Lt::kK + (at >> 3) * kPanel + tc::sw128_offset(row, 8 * (at & 7))) = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<uint4*>(stage + Lt::kV + tc::sw128_offset(row, cb + 8 * q)) = make_uint4(0, 0, 0, 0);
        }
      }
      const float w = ul < nc ? pw[end_of(k) - ul] : 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 raw = *reinterpret_cast<const uint4*>(stage + Lt::kV + tc::sw128_offset(row, cb + 8 * q));
        const uint32_t* e = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 f = __fmul2_rn(__bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&e[j])), make_float2(w, w));
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const uint32_t r = pack2<__nv_bfloat16>(f.x, f.y);
            vp[part][4 * q + j] = r;
            const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r));
            f.x -= g.x;
            f.y -= g.y;
          }
        }
      }
      return true;
    };
    auto store_v = [&](int k) {
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<uint4*>(sm + Lt::kVs + part * kPanel + tc::sw128_offset(row, cb + 8 * q)) =
              make_uint4(vp[part][4 * q], vp[part][4 * q + 1], vp[part][4 * q + 2], vp[part][4 * q + 3]);
      // An infinity or NaN in V would go with P V to the steps before it (their weights are 0, and 0 * inf is NaN).  So it
      // leaves V as a zero, and group A brings it to the outputs that it belongs to.  For the state it stays in the
      // first part, and the others are 0 (inf - inf is NaN).  (Looked for here, where it costs no spills for dk <= 128:
      // 8 x 2048 x 16 heads of 128 101.1 -> 103.0 us, 4 x 2048 x 16 of 256 101 -> 105.6; by the two idle warps 108.)
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = __vmaxu2(most, vp[0][j] & 0x7fff7fffu);
      if (__any_sync(0xffffffffu, (most & 0xffffu) >= 0x7f80u || (most >> 16) >= 0x7f80u)) {
        *not_finite = 1;
#pragma unroll 1
        for (int c = 0; c < 16; c += 2) {
          const uint32_t at = tc::sw128_offset(row, cb + (c & 8)) + 2 * (c & 7);
          uint32_t* x = reinterpret_cast<uint32_t*>(sm + (k % kStages) * Lt::kStage + Lt::kV + at);
          const uint32_t keep = ((*x & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((*x & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
          *x &= keep;
          for (int part = 1; part < kParts; ++part) *reinterpret_cast<uint32_t*>(sm + Lt::kVs + part * kPanel + at) &= keep;
        }
      }
    };
    auto v_done = [&]() {
      tc::fence_async_smem();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(v_ready);
    };
    snapshot();
    bool ok = nch == 0 || scale_v(0);
    if (ok && nch) {
      store_v(0);
      v_done();
    }
#pragma unroll 1
    for (int k = 0; ok && k < nch; ++k) {
      const bool more = k + 1 < nch;
      if (kStages == 2 && more && !(ok = scale_v(k + 1))) break;
      if (!(ok = wait(u_ready, k))) break;
      tc::tc_fence_after();
      const float f = pw[end_of(k)];
      if (kStages == 2 && more) store_v(k + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // the parts' two sums (dk <= 128), or the two halves of X
        float u[16];
        tc::tmem_ld16(tm + Lt::tU + 64 * i + cb, u);
        tc::tmem_wait_ld();
        float* x = X[kNB == 2 ? i : 0];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = kNB == 2 || i == 0 ? fmaf(f, x[j], u[j]) : x[j] + u[j];
      }
      if (!more) break;
      if (kStages == 2) v_done();
      if (!state_only && !(ok = wait(qs_done, k))) break;
      snapshot();
      if (kStages == 1) {
        if (!(ok = scale_v(k + 1))) break;
        store_v(k + 1);
        v_done();
      }
    }
    if (ok) {
      float* dst = nullptr;
      int64_t sd = p.dv, se = 1;
      float f = 1.f;
      if (state_only) {
        if (u_lo < n)
          dst = p.ws + (((int64_t)b * cm.heads + h) * (cm.nseg - 1) + seg) * p.dk * p.dv;
      } else if (p.sT && (n == 0 ? seg == 0 : u_lo < n && u_hi == n)) {
        dst = p.sT + b * p.sTs[0] + h * p.sTs[1];
        sd = p.sTs[2];
        se = p.sTs[3];
        f = p.sT_scale;
      }
      if (dst)
#pragma unroll
        for (int blk = 0; blk < kNB; ++blk) {
          const int d = blk * 128 + row;
          float* to = dst + d * sd + (e0 + cb) * se;
          const bool vec = se == 1 && reinterpret_cast<uintptr_t>(to) % 16 == 0;
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            if (d < p.dk && e0 + cb + j < p.dv) {  // dv is a multiple of 8
              if (vec) {
                *reinterpret_cast<float4*>(to + j) = make_float4(f * X[blk][j], f * X[blk][j + 1], f * X[blk][j + 2], f * X[blk][j + 3]);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) to[(j + i) * se] = f * X[blk][j + i];
              }
            }
        }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCtrl));
    if (warp == 8 + kWarpsB) {
    // ======================= MMA issue (one lane) =======================
    if (elect_one()) {
      const uint32_t sb = smem_u32(sm);
      const uint64_t dQ = tc::sdesc_sw128(sb + Lt::kQ, 16, 1024);
      const uint64_t dK = tc::sdesc_sw128(sb + Lt::kK, 16, 1024);
      const uint64_t dKT = tc::sdesc_sw128(sb + Lt::kK, kPanel, 1024);
      const uint64_t dV = tc::sdesc_sw128(sb + Lt::kV, kPanel, 1024);
      const uint64_t dX = tc::sdesc_sw128(sb + Lt::kSnap, kPanel, 1024);
      const uint64_t dVs = tc::sdesc_sw128(sb + Lt::kVs, kPanel, 1024);
      constexpr uint32_t idS = tc::idesc_bf16(128, 128, false, false);
      constexpr uint32_t idO = tc::idesc_bf16(128, kDV, false, true);
      constexpr uint32_t idU = tc::idesc_bf16(128, kDV, true, true);
      constexpr uint32_t idU2 = tc::idesc_bf16(128, 2 * kDV, true, true);
      auto w8 = [&](uint64_t* bar, int parity) { return tc::mbar_wait(bar, parity & 1, abort_flag, limit); };
      auto issue_s = [&](int k) {
        const uint32_t so = (k % kStages) * Lt::kStage;
        const uint64_t q = tc::desc_add(dQ, so), kk = tc::desc_add(dK, so);
        const uint32_t d = tb + Lt::tS + 128 * (k & 1);
        tc::static_for<DK / 16>([&](auto KS) {
          constexpr int ks = decltype(KS)::value;
          constexpr uint32_t off = (ks / 4) * kPanel + (ks % 4) * 32;
          tc::mma_bf16_at<off, off>(d, q, kk, idS, ks > 0);
        });
        tc::mma_commit(s_ready + (k & 1));
      };
      auto issue_u = [&](int k) {
        const uint64_t kt = tc::desc_add(dKT, (k % kStages) * Lt::kStage);
        if (kNB == 1) {  // two parts side by side: N = 128 reads the K tile once for both
          tc::static_for<kC / 16>([&](auto I) {
            constexpr int ks = decltype(I)::value;
            tc::mma_bf16_at<ks * 2048, ks * 2048>(tb + Lt::tU, kt, dVs, idU2, ks > 0);
          });
          tc::static_for<kC / 16>([&](auto I) {
            constexpr int ks = decltype(I)::value;
            tc::mma_bf16_at<ks * 2048, 2 * kPanel + ks * 2048>(tb + Lt::tU + 64, kt, dVs, idU, true);
          });
        } else {
          for (int part = 0; part < kParts; ++part) {
            const uint64_t v = tc::desc_add(dVs, part * kPanel);
            tc::static_for<kNB * (kC / 16)>([&](auto I) {
              constexpr int blk = decltype(I)::value / (kC / 16), ks = decltype(I)::value % (kC / 16);
              tc::mma_bf16_at<2 * blk * kPanel + ks * 2048, ks * 2048>(tb + Lt::tU + 64 * blk, kt, v, idU, ks > 0 || part > 0);
            });
          }
        }
        tc::mma_commit(u_ready);
      };
      bool ok = nch > 0;
      if (!state_only && ok) {
        ok = w8(full, 0);
        if (ok) {
          tc::tc_fence_after();
          issue_s(0);
        }
      }
#pragma unroll 1
      for (int k = 0; ok && k < nch; ++k) {
        const int st = k % kStages;
        if (state_only && !(ok = w8(full + st, k / kStages))) break;
        if (!(ok = w8(v_ready, k))) break;
        tc::tc_fence_after();
        issue_u(k);
        if (state_only) {
          tc::mma_commit(empty + st);
          continue;
        }
        // O of two chunks ago read (apart: O1, O2 of the last one)
        const int back = sep ? 2 : 1;
        if (k >= back && !(ok = w8(o_free + ((k - back) & 1), (k - back) >> 1))) break;
        if (!(ok = w8(x_ready, k))) break;
        tc::tc_fence_after();
        const uint32_t to = tb + Lt::tO + (sep ? 64 * (k & 1) : 0);
        {
          const uint64_t q = tc::desc_add(dQ, st * Lt::kStage);
          tc::static_for<DK / 16>([&](auto KS) {
            constexpr int ks = decltype(KS)::value;
            tc::mma_bf16_at<(ks / 4) * kPanel + (ks % 4) * 32, ks * 2048>(sep ? to : to + 64, q, dX, idO, ks > 0);
          });
          tc::mma_commit(qs_done);
        }
        if (kStages == 2 && k + 1 < nch) {
          if (!(ok = w8(full + ((k + 1) & 1), (k + 1) >> 1))) break;
          tc::tc_fence_after();
          issue_s(k + 1);
        }
        if (!(ok = w8(p_ready + (k & 1), k >> 1))) break;
        tc::tc_fence_after();
        {
          const uint64_t v = tc::desc_add(dV, st * Lt::kStage);
          const uint32_t a = tb + Lt::tS + 128 * (k & 1);
          tc::static_for<kC / 16>([&](auto KS) {
            constexpr int ks = decltype(KS)::value;
            mma_bf16_ta<ks * 2048>(to, a + (ks / 4) * 64 + (ks % 4) * 8, v, idO, ks > 0 || sep);
          });
          tc::mma_commit(o_ready + (k & 1));
          tc::mma_commit(empty + st);
        }
        if (kStages == 1 && k + 1 < nch) {
          if (!(ok = w8(full, k + 1))) break;
          tc::tc_fence_after();
          issue_s(k + 1);
        }
      }
      volatile int none = 0;  // nothing stays in flight, also after a wait that gave up
      tc::mma_commit(fin);
      tc::mbar_wait(fin, 0, &none, 20000000ll);
    }
    __syncwarp();
  } else if (warp == 9 + kWarpsB) {
    // ======================= TMA loads (one lane) =======================
    if (elect_one()) {
      const CUtensorMap* mq = &prm.map[3 * ip];
      const int hq = h * prm.mh[3 * ip], hk = h * prm.mh[3 * ip + 1], hv = h * prm.mh[3 * ip + 2];
      const int bq = b * prm.mb[3 * ip], bk = b * prm.mb[3 * ip + 1], bv = b * prm.mb[3 * ip + 2];
      int issued = 0;
#pragma unroll 1
      for (int k = 0; k < nch; ++k) {
        const int st = k % kStages;
        if (k >= kStages && !tc::mbar_wait(empty + st, (k / kStages - 1) & 1, abort_flag, limit)) break;
        unsigned char* s = sm + st * Lt::kStage;
        const int t0 = t0_of(k);
        tc::mbar_expect_tx(full + st, ((state_only ? 1 : 2) * kNP + 1) * kPanel);
        for (int pn = 0; pn < kNP; ++pn) {
          if (!state_only) tc::tma_load_4d(s + Lt::kQ + pn * kPanel, mq, full + st, pn * 64, t0, hq, bq);
          tc::tma_load_4d(s + Lt::kK + pn * kPanel, mq + 1, full + st, pn * 64, t0, hk, bk);
        }
        tc::tma_load_4d(s + Lt::kV, mq + 2, full + st, e0, t0, hv, bv);
        issued = k + 1;
      }
      volatile int none = 0;  // the loads in flight land before the CTA ends
      for (int k = max(0, issued - kStages); k < issued; ++k)
        tc::mbar_wait(full + k % kStages, (k / kStages) & 1, &none, 20000000ll);
    }
    __syncwarp();
  }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tb, 512);
  }
  if (tid == 0 && *abort_flag && cm.error_flag) atomicExch(cm.error_flag, 1);
}

bool tc_ok(const Problem& p, int seqlen, hxm_dtype io) {
  if (io != HXM_BF16 || p.dk % 8 || p.dv % 8 || p.dk > 256) return false;
  auto rows = [&](const void* t, const int64_t* s) {
    return reinterpret_cast<uintptr_t>(t) % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 &&
           (s[1] > 0 || seqlen <= 1) && s[0] >= 0 && s[2] >= 0;
  };
  return rows(p.q, p.sq) && rows(p.k, p.sk) && rows(p.v, p.sv) && rows(p.o, p.so);
}

template <int DK>
static hxm_status launch_dk(TcParams& t, int np, int tiles, bool state_only, cudaStream_t st) {
  const size_t smem = Layout<DK>::kBytes + 1024;
  // the register split counts on the launch's share (a smaller one would leave setmaxnreg waiting)
  static const int regs = [] {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, tc_kernel<DK>) == cudaSuccess ? at.numRegs : -1;
  }();
  HXM_REQUIRE_SUPPORTED(regs == kRegsLaunch, "hxm_linear_attn: built with %d registers a thread, not %d", regs, kRegsLaunch);
  const hxm_status s = allow_shared_memory<tc_kernel<DK>>();
  if (s != HXM_OK) return s;
  // the last segment's sum is nobody's entering state
  const dim3 grid((unsigned)(tiles * (t.c.nseg - (state_only ? 1 : 0))), (unsigned)t.c.heads, (unsigned)(t.c.batch * np));
  tc_kernel<DK><<<grid, kThreadsTc, smem, st>>>(t, tiles, state_only ? 1 : 0);
  return check_launch("hxm_linear_attn");
}

hxm_status launch_tc(const Common& c, const Problem* p, int np, bool state_only, cudaStream_t st) {
  TcParams t{};
  t.c = c;
  int tiles = 0;
  if (c.seqlen > 0)
    for (int i = 0; i < np; ++i) {
      const void* base[3] = {p[i].q, p[i].k, p[i].v};
      const int64_t* s[3] = {p[i].sq, p[i].sk, p[i].sv};
      const int d[3] = {p[i].dk, p[i].dk, p[i].dv};
      for (int j = 0; j < 3; ++j) {
        const uint64_t any = ((uint64_t)d[j] * 2 + 15) / 16 * 16;  // stride of a dimension of extent 1
        const bool hd = s[j][2] != 0, bt = s[j][0] != 0;
        const uint64_t dims[4] = {(uint64_t)d[j], (uint64_t)c.seqlen, hd ? (uint64_t)c.heads : 1, bt ? (uint64_t)c.batch : 1};
        const uint64_t str[3] = {s[j][1] ? (uint64_t)s[j][1] * 2 : any, hd ? (uint64_t)s[j][2] * 2 : any, bt ? (uint64_t)s[j][0] * 2 : any};
        const hxm_status r = make_map_bf16_4d(&t.map[3 * i + j], base[j], dims, str, "hxm_linear_attn");
        if (r != HXM_OK) return r;
        t.mh[3 * i + j] = hd;
        t.mb[3 * i + j] = bt;
      }
    }
  for (int i = 0; i < np; ++i) {
    t.p[i] = p[i];
    const int n = (p[i].dv + kDV - 1) / kDV;
    tiles = n > tiles ? n : tiles;
  }
  return p[0].dk > 128 ? launch_dk<256>(t, np, tiles, state_only, st) : launch_dk<128>(t, np, tiles, state_only, st);
}

}  // namespace lattn
}  // namespace hxm
