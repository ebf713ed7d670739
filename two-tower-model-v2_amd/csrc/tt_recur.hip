// tt_recur.hip -- gated linear recurrence over event histories (gfx950).
//
//   A_t = sigmoid(g_t)^(w_t) = exp(-w_t softplus(-g_t))      (w absent: 1)
//   h_t = A_t h_{t-1} + (1 - A_t) x_t                        (h_{-1} = h0, or 0)
//
// An event of weight w moves the state exactly as w equal events of weight 1 do.  An event whose
// weight is not above 0 (padding; also NaN) leaves the state as it is, bit for bit, whatever its
// x and g hold, and gets zero gradients.
//
// Backward, with R the gradient that reaches h_t from later events:
//   G_t = dh_t + R ;  dx_t = (1 - A_t) G_t ;  dg_t = w_t A_t sigmoid(-g_t) (h_{t-1} - x_t) G_t
//   R <- A_t G_t   (after event 0: the gradient of h0)
// The state is needed in 32 bits there, so the forward pass saves it (f32) before every 8th
// event, 1/8 of one f32 tensor, and the backward pass recomputes the 8 states between in
// registers: cheaper to read than h itself (0.5 instead of 2 or 4 bytes an element) and the
// rounding of h to bf16 does not reach the gradients.
//
// Bound: HBM.  Forward 3 tensors (x, gate, h), backward 5 (x, gate, dh, dx, dgate).  A lane owns
// VEC neighbouring channels of one history and walks the events; a wave's unit is (history, 64
// VEC channels, chunk of events).  The histories' own count fills the card in training batches
// (one chunk: every tensor is read once).  Few long histories are split along the events: a
// first launch reduces every chunk to (product of A, state reached from 0), a second joins the
// chunks, the third runs the chunks from their true start states.  The split pass reads x and
// gate twice (from the 256 MB last-level cache where they fit).
//
// Measured: 512 histories x 100 events x 768 f32, one chunk: forward without h 91 us, backward 106
// us (4.7 TB/s over both).  8 x 16384 x 768 bf16 with weights, split: sums 118 us, join 8, main pass
// 130 (4.6 TB/s); backward 117, 8, 205 (4.9 TB/s).  The summing passes are bound by the gates'
// arithmetic (exponential, reciprocal, powers of the weights), at 3.4 TB/s: walking them the other
// way in time, so that they end on what the main pass starts with, changed nothing.
#include "tt_common.hpp"

namespace tt {

constexpr int RC_CK = TT_SCAN_CKPT;  // events between saved states
constexpr int RC_U = 8;     // events whose rows are loaded together (forward)
constexpr int RC_SEG = 64, RC_JCH = 16;  // segments and channels of a block of the chunk join

struct ScanArgs {
  const void *x, *gate;
  const float *w, *h0;      // w [B, S] rows wsb apart; h0 [B, D]; either may be null
  void* h;                  // [B, S, D] or null
  float *h_last, *ck;       // [B, D]; [B, ceil(S / RC_CK), D] or null
  const void* dh;           // backward: [B, S, D] or null
  const float* dlast;       // [B, D] or null
  void *dx, *dgate;
  float* dh0;
  int64_t B, S, xsb, xss, gsb, gss, wsb;
  int D, nw, C;             // waves per row, chunks per history
  int64_t T;                // events per chunk (a multiple of RC_CK unless C == 1)
  float *sumA, *sumH, *carry;  // [B, C, D] each (C > 1)
};

template <typename T, int VEC>
struct Pack;
template <>
struct Pack<float, 1> { typedef float type; };
template <>
struct Pack<float, 2> { typedef float type __attribute__((ext_vector_type(2))); };
template <>
struct Pack<uint16_t, 1> { typedef uint16_t type; };
template <>
struct Pack<uint16_t, 2> { typedef uint32_t type; };

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

template <typename T, int VEC>
__device__ __forceinline__ void unpack(typename Pack<T, VEC>::type p, float (&o)[VEC]) {
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (VEC == 1) {
      o[0] = p;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = p[i];
    }
  } else if constexpr (VEC == 1) {
    o[0] = bf_lo(p);
  } else {
    o[0] = bf_lo(p);
    o[1] = bf_hi(p);
  }
}
typedef __bf16 rc_bf16x2 __attribute__((ext_vector_type(2)));
typedef float rc_f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t rc_pack2(float a, float b) {  // round to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(rc_f32x2{a, b}, rc_bf16x2));
}
template <typename T, int VEC>
__device__ __forceinline__ typename Pack<T, VEC>::type pack(const float (&v)[VEC]) {
  typename Pack<T, VEC>::type p;
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (VEC == 1) {
      p = v[0];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = v[i];
    }
  } else if constexpr (VEC == 1) {
    p = (uint16_t)rc_pack2(v[0], 0.0f);
  } else {
    p = rc_pack2(v[0], v[1]);
  }
  return p;
}

// A chunk's product of A as one float: the product P itself, or minus 1 - P where that is below a
// half (bit for bit a sign: P = 1 is -0).  1 - P is summed on its own: taken from a rounded P it
// would be off by the roundings of all its factors, the same in every chunk of equal gates.
__device__ __forceinline__ float enc_prod(float P, float n) { return n < 0.5f ? -n : P; }
__device__ __forceinline__ void dec_prod(float e, float& P, float& n) {
  const bool neg = (int)__float_as_uint(e) < 0;
  P = neg ? 1.0f + e : e;
  n = neg ? -e : 1.0f - e;
}

// exp(-|g|) to about 1 ulp: the product |g| log2(e) in two parts, the low one (< 2^-20) applied
// to first order.
__device__ __forceinline__ float exp_neg_abs(float g) {
  const float n = -fabsf(g);
  const float hi = n * 1.44269504f;
  const float lo = fmaf(n, 1.44269504f, -hi) + n * 1.92596299e-8f;  // log2(e) - f32(log2(e))
  const float e = __builtin_amdgcn_exp2f(hi);
  return hi < -150.0f ? 0.0f : fmaf(e, lo * 0.693147181f, e);
}
struct Gate {
  float a, na;  // A, 1 - A
};
// A s and A h + (1 - A) x.  Near 1 the part that leaves is computed from 1 - A: a rounded A would
// be off 1 - (1 - A) by up to 2^-25, which a memory of 1 / (1 - A) events multiplies.
__device__ __forceinline__ float decay(float a, float na, float s) {
  return na < 0.5f ? fmaf(-na, s, s) : a * s;
}
__device__ __forceinline__ float move(float a, float na, float h, float x) {
  return na < 0.5f ? fmaf(na, x - h, h) : fmaf(a, h, na * x);
}
// e = exp(-|g|), r = 1 / (1 + e): sigmoid(|g|) = r and sigmoid(-|g|) = e r, neither by a
// difference, so 1 - A keeps its relative precision for long memories (A next to 1).  For bf16
// gates the exponent is one product (2^-24 |g| off: far below the gate's own rounding; the
// exponential is a fifth of the kernels' arithmetic, and that is what bounds them next to HBM).
template <typename T>
__device__ __forceinline__ Gate gate_one(float g) {
  const float e = sizeof(T) == 4 ? exp_neg_abs(g) : __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float er = e * r;
  Gate o;
  o.a = g >= 0.0f ? r : er;
  o.na = g >= 0.0f ? er : r;
  return o;
}
// A = exp(-w softplus(-g)).  softplus(-g) = max(-g, 0) + log1p(e), log1p(e) = 2 atanh(e / (2 +
// e)) by its odd series (argument <= 1/3: terms to z^15); expm1 by its series below 0.35, by the
// difference from 1 above (relative error < 2^-22 either way).
__device__ __forceinline__ Gate gate_pow(float g, float w) {
  const float e = exp_neg_abs(g);
  const float z = e * __builtin_amdgcn_rcpf(2.0f + e), z2 = z * z;
  float s = fmaf(z2, 1.0f / 15.0f, 1.0f / 13.0f);
  s = fmaf(s, z2, 1.0f / 11.0f);
  s = fmaf(s, z2, 1.0f / 9.0f);
  s = fmaf(s, z2, 1.0f / 7.0f);
  s = fmaf(s, z2, 0.2f);
  s = fmaf(s, z2, 1.0f / 3.0f);
  s = fmaf(s, z2, 1.0f);
  const float sp = fmaxf(-g, 0.0f) + 2.0f * z * s;
  const float y = sp * w;  // A = exp(-y)
  float q = fmaf(y, -1.0f / 40320.0f, 1.0f / 5040.0f);  // (1 - exp(-y)) / y
  q = fmaf(q, y, -1.0f / 720.0f);
  q = fmaf(q, y, 1.0f / 120.0f);
  q = fmaf(q, y, -1.0f / 24.0f);
  q = fmaf(q, y, 1.0f / 6.0f);
  q = fmaf(q, y, -0.5f);
  q = fmaf(q, y, 1.0f);
  const float nsmall = q * y;
  const float big = exp_neg_abs(y);
  Gate o;
  o.a = y < 0.35f ? 1.0f - nsmall : big;
  o.na = y < 0.35f ? nsmall : 1.0f - big;
  return o;
}

// (A, 1 - A) of weight 1 -> of a whole weight w <= 64 (event weights are counts), by repeated
// squaring of the pair: 1 - A B = (1 - A) + A (1 - B), sums of positive terms only, so both keep
// their relative precision; some 10 operations a channel instead of gate_pow's 50.  w uniform.
template <int VEC>
__device__ __forceinline__ void gate_power(float (&a)[VEC], float (&na)[VEC], int w) {
  float b[VEC], nb[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    b[i] = a[i];
    nb[i] = na[i];
  }
  while (!(w & 1)) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      nb[i] = fmaf(b[i], nb[i], nb[i]);
      b[i] *= b[i];
    }
    w >>= 1;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    a[i] = b[i];
    na[i] = nb[i];
  }
  while (w >>= 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      nb[i] = fmaf(b[i], nb[i], nb[i]);
      b[i] *= b[i];
    }
    if (w & 1) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        na[i] = fmaf(a[i], nb[i], na[i]);
        a[i] *= b[i];
      }
    }
  }
}

// unit = ((b * C) + c) * nw + wave-of-row; uniform over the wave
struct Unit {
  int64_t b;
  int c, ch;  // chunk, first channel of this lane
  bool ok;    // the row has this channel (else the lane reads channel 0 and writes nothing; it
              // stays active, for the weights)
};
template <int VEC>
__device__ __forceinline__ Unit unit_of(const ScanArgs& a, int64_t u, int lane) {
  Unit o;
  const int64_t bc = u / a.nw;
  o.ch = ((int)(u - bc * a.nw) * 64 + lane) * VEC;
  o.ok = o.ch < a.D;
  o.ch = o.ok ? o.ch : 0;
  o.b = bc / a.C;
  o.c = (int)(bc - o.b * a.C);
  return o;
}

// Weights are uniform over a wave (one history): 64 events' weights with one load, lane i's handed
// out as a scalar, so that the choice of the gate's form is a scalar branch.
__device__ __forceinline__ float lane_value(float v, int i) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), i));
}
// The gates of U events: weight 1 for all of them first, without a branch (their exponentials
// overlap), then the other weights event by event.  KQ: also w A sigmoid(-g) (the backward's).
template <typename T, int VEC, int U, bool WT, bool KQ>
__device__ __forceinline__ void gates(const typename Pack<T, VEC>::type (&gp)[U], const float (&w)[U],
                                      float (&a)[U][VEC], float (&na)[U][VEC], float (&kq)[KQ ? U : 1][VEC]) {
#pragma unroll
  for (int j = 0; j < U; ++j) {
    float g[VEC];
    unpack<T, VEC>(gp[j], g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const Gate q = gate_one<T>(g[i]);
      a[j][i] = q.a;
      na[j][i] = q.na;
      if (KQ) kq[j][i] = q.a * q.na;
    }
  }
  if constexpr (WT) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (w[j] == 1.0f || !(w[j] > 0.0f)) continue;
      const float wj = fminf(w[j], 3.0e38f);  // an infinite weight: h becomes x (and w A is 0, no NaN)
      float sn[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) sn[i] = na[j][i];
      if (w[j] <= 64.0f && truncf(w[j]) == w[j]) {
        gate_power<VEC>(a[j], na[j], (int)w[j]);
      } else {
        float g[VEC];
        unpack<T, VEC>(gp[j], g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const Gate q = gate_pow(g[i], wj);
          a[j][i] = q.a;
          na[j][i] = q.na;
        }
      }
      if (KQ) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) kq[j][i] = wj * a[j][i] * sn[i];
      }
    }
  }
}

// SUM: the chunk's (product of A, state from 0) only.  Else the chunk from its start state, with
// h, h_last and the saved states as asked for.
template <typename T, int VEC, bool WT, bool SUM>
__global__ __launch_bounds__(256) void k_scan_fwd(const ScanArgs a) {
  typedef typename Pack<T, VEC>::type P;
  const int lane = threadIdx.x & 63;
  const int64_t nunits = a.B * a.C * a.nw;
  const int64_t nck = (a.S + RC_CK - 1) / RC_CK;
  for (int64_t u0 = (int64_t)blockIdx.x * 4; u0 < nunits; u0 += (int64_t)gridDim.x * 4) {
    const int64_t uu = u0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (uu >= nunits) break;
    const Unit un = unit_of<VEC>(a, uu, lane);
    if (SUM && un.c == a.C - 1) continue;  // the last chunk starts nothing
    const int64_t t0 = (int64_t)un.c * a.T, t1 = t0 + a.T < a.S ? t0 + a.T : a.S;
    const T* xp = (const T*)a.x + un.b * a.xsb + un.ch;
    const T* gp = (const T*)a.gate + un.b * a.gsb + un.ch;
    const float* wp = WT ? a.w + un.b * a.wsb : nullptr;
    float h[VEC], pa[VEC], pn[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      pa[i] = 1.0f;
      pn[i] = 0.0f;
      h[i] = SUM ? 0.0f
             : a.C > 1 ? a.carry[(un.b * a.C + un.c) * a.D + un.ch + i]
             : a.h0    ? a.h0[un.b * a.D + un.ch + i]
                       : 0.0f;
    }
    P xn[RC_U], gn[RC_U];
    float wl = 0.0f;
    auto load = [&](int64_t t) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        const int64_t tt = t + j < t1 ? t + j : t1 - 1;
        xn[j] = *(const P*)(xp + tt * a.xss);
        gn[j] = *(const P*)(gp + tt * a.gss);
      }
    };
    if (t0 < t1) load(t0);
    for (int64_t t = t0; t < t1; t += RC_U) {
      P xc[RC_U], gc[RC_U];
      float wc[RC_U], A[RC_U][VEC], nA[RC_U][VEC], none[1][VEC];
      const int wi = (int)(t - t0) & 63;
      if (WT && wi == 0) wl = t + lane < t1 ? wp[t + lane] : 0.0f;
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        xc[j] = xn[j];
        gc[j] = gn[j];
        wc[j] = WT ? lane_value(wl, wi + j) : 1.0f;
      }
      if (t + RC_U < t1) load(t + RC_U);
      gates<T, VEC, RC_U, WT, false>(gc, wc, A, nA, none);
      if (!SUM && a.ck && un.ok && (t & (RC_CK - 1)) == 0) {
        float* c = a.ck + (un.b * nck + t / RC_CK) * a.D + un.ch;
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = h[i];
      }
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        if (t + j < t1) {
          if (!WT || wc[j] > 0.0f) {
            float xv[VEC];
            unpack<T, VEC>(xc[j], xv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              h[i] = move(A[j][i], nA[j][i], h[i], xv[i]);
              if (SUM) {
                pn[i] = fmaf(pa[i], nA[j][i], pn[i]);
                pa[i] = decay(A[j][i], nA[j][i], pa[i]);
              }
            }
          }
          if (!SUM && a.h && un.ok) *(P*)((T*)a.h + (un.b * a.S + t + j) * a.D + un.ch) = pack<T, VEC>(h);
        }
      }
    }
    if (!un.ok) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (SUM) {
        a.sumA[(un.b * a.C + un.c) * a.D + un.ch + i] = enc_prod(pa[i], pn[i]);
        a.sumH[(un.b * a.C + un.c) * a.D + un.ch + i] = h[i];
      } else if (un.c == a.C - 1) {
        a.h_last[un.b * a.D + un.ch + i] = h[i];
      }
    }
  }
}

// Joins the chunks of one history: carry[c] = the state before chunk c (REV: the gradient that
// reaches the end of chunk c from the chunks after it).  16 channels x 64 segments of chunks per
// block (few histories have many chunks: a thread's walk is short, its loads independent): a
// segment is composed to one (A, H), the segments before it give its start by a scan in 6 steps,
// a second walk writes.  s <- A s + H over chunks c = 0 .. (REV: C - 1 .. 1).
template <bool REV>
__global__ __launch_bounds__(RC_JCH * RC_SEG) void k_scan_join(const float* __restrict__ sumA,
                                                               const float* __restrict__ sumH,
                                                               const float* __restrict__ init,
                                                               float* __restrict__ carry, int64_t B,
                                                               int C, int D) {
  __shared__ float sa[2][RC_SEG][RC_JCH], sn[2][RC_SEG][RC_JCH], sh[2][RC_SEG][RC_JCH];
  const int cl = threadIdx.x % RC_JCH, seg = threadIdx.x / RC_JCH;
  const int nd = (D + RC_JCH - 1) / RC_JCH;
  const int per = (C + RC_SEG - 1) / RC_SEG;
  for (int64_t blk = blockIdx.x; blk < B * nd; blk += gridDim.x) {
    const int64_t b = blk / nd;
    const int ch = (int)(blk - b * nd) * RC_JCH + cl;
    const bool ok = ch < D;
    const int i0 = seg * per < C ? seg * per : C, i1 = i0 + per < C ? i0 + per : C;
    auto at = [&](int i) { return (b * C + (REV ? C - 1 - i : i)) * D + (ok ? ch : 0); };
    // (P, n = 1 - P, H) of the segment's chunks, one after another
    float pa = 1.0f, pn = 0.0f, ph = 0.0f;
    // (the last step's summary starts nothing and is not written: i runs to C - 2)
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
      if (i < C - 1) {
        float P, n;
        dec_prod(sumA[at(i)], P, n);
        ph = decay(P, n, ph) + sumH[at(i)];
        pn = fmaf(pa, n, pn);
        pa = decay(P, n, pa);
      }
    }
    // ... and of all segments up to this one
    int k = 0;
    sa[0][seg][cl] = pa;
    sn[0][seg][cl] = pn;
    sh[0][seg][cl] = ph;
    __syncthreads();
#pragma unroll
    for (int o = 1; o < RC_SEG; o <<= 1, k ^= 1) {
      if (seg >= o) {
        const float P = sa[k][seg - o][cl];
        ph += decay(pa, pn, sh[k][seg - o][cl]);
        pn = fmaf(pa, sn[k][seg - o][cl], pn);
        pa *= P;
      }
      sa[k ^ 1][seg][cl] = pa;
      sn[k ^ 1][seg][cl] = pn;
      sh[k ^ 1][seg][cl] = ph;
      __syncthreads();
    }
    float s = init && ok ? init[b * D + ch] : 0.0f;
    if (seg > 0) s = decay(sa[k][seg - 1][cl], sn[k][seg - 1][cl], s) + sh[k][seg - 1][cl];
    if (ok) {
#pragma unroll 4
      for (int i = i0; i < i1; ++i) {
        carry[at(i)] = s;
        if (i < C - 1) {
          float P, n;
          dec_prod(sumA[at(i)], P, n);
          s = decay(P, n, s) + sumH[at(i)];
        }
      }
    }
    __syncthreads();
  }
}

// Reverse summary of a chunk: product of A, and the gradient that leaves its front when none
// enters its end.
template <typename T, int VEC, bool WT, bool DH>
__global__ __launch_bounds__(256) void k_scan_bwd_sum(const ScanArgs a) {
  typedef typename Pack<T, VEC>::type P;
  const int lane = threadIdx.x & 63;
  const int64_t nunits = a.B * a.C * a.nw;
  for (int64_t u0 = (int64_t)blockIdx.x * 4; u0 < nunits; u0 += (int64_t)gridDim.x * 4) {
    const int64_t uu = u0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (uu >= nunits) break;
    const Unit un = unit_of<VEC>(a, uu, lane);
    if (un.c == 0) continue;
    const int64_t t0 = (int64_t)un.c * a.T, t1 = t0 + a.T < a.S ? t0 + a.T : a.S;
    const T* gp = (const T*)a.gate + un.b * a.gsb + un.ch;
    const T* dp = (const T*)a.dh + un.b * a.S * a.D + un.ch;  // (DH)
    const float* wp = WT ? a.w + un.b * a.wsb : nullptr;
    float R[VEC], pa[VEC], pn[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      pa[i] = 1.0f;
      pn[i] = 0.0f;
      R[i] = 0.0f;
    }
    P gn[RC_U], dn[RC_U];
    float wl = 0.0f;  // lane i: event t1 - 1 - 64 k - i
    auto load = [&](int64_t t) __attribute__((always_inline)) {  // events t, t - 1, ...
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        const int64_t tt = t - j > t0 ? t - j : t0;
        gn[j] = *(const P*)(gp + tt * a.gss);
        if (DH) dn[j] = *(const P*)(dp + tt * a.D);
      }
    };
    load(t1 - 1);
    for (int64_t t = t1 - 1; t >= t0; t -= RC_U) {
      P gc[RC_U], dc[RC_U];
      float wc[RC_U], A[RC_U][VEC], nA[RC_U][VEC], none[1][VEC];
      const int wi = (int)(t1 - 1 - t) & 63;
      if (WT && wi == 0) wl = t - lane >= t0 ? wp[t - lane] : 0.0f;
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        gc[j] = gn[j];
        if (DH) dc[j] = dn[j];
        wc[j] = WT ? lane_value(wl, wi + j) : 1.0f;
      }
      if (t - RC_U >= t0) load(t - RC_U);
      gates<T, VEC, RC_U, WT, false>(gc, wc, A, nA, none);
#pragma unroll
      for (int j = 0; j < RC_U; ++j) {
        if (t - j >= t0) {
          if (DH) {
            float dv[VEC];
            unpack<T, VEC>(dc[j], dv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) R[i] += dv[i];
          }
          if (!WT || wc[j] > 0.0f) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              R[i] = decay(A[j][i], nA[j][i], R[i]);
              pn[i] = fmaf(pa[i], nA[j][i], pn[i]);
              pa[i] = decay(A[j][i], nA[j][i], pa[i]);
            }
          }
        }
      }
    }
    if (!un.ok) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a.sumA[(un.b * a.C + un.c) * a.D + un.ch + i] = enc_prod(pa[i], pn[i]);
      a.sumH[(un.b * a.C + un.c) * a.D + un.ch + i] = R[i];
    }
  }
}

template <typename T, int VEC, bool WT, bool DH>
__global__ __launch_bounds__(256) void k_scan_bwd(const ScanArgs a) {
  typedef typename Pack<T, VEC>::type P;
  const int lane = threadIdx.x & 63;
  const int64_t nunits = a.B * a.C * a.nw;
  const int64_t nck = (a.S + RC_CK - 1) / RC_CK;
  for (int64_t u0 = (int64_t)blockIdx.x * 4; u0 < nunits; u0 += (int64_t)gridDim.x * 4) {
    const int64_t uu = u0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (uu >= nunits) break;
    const Unit un = unit_of<VEC>(a, uu, lane);
    const int64_t t0 = (int64_t)un.c * a.T, t1 = t0 + a.T < a.S ? t0 + a.T : a.S;
    const T* xp = (const T*)a.x + un.b * a.xsb + un.ch;
    const T* gp = (const T*)a.gate + un.b * a.gsb + un.ch;
    const int64_t ob = un.b * a.S * a.D + un.ch;
    const float* wp = WT ? a.w + un.b * a.wsb : nullptr;
    float R[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      R[i] = a.C > 1 ? a.carry[(un.b * a.C + un.c) * a.D + un.ch + i]
             : a.dlast ? a.dlast[un.b * a.D + un.ch + i]
                       : 0.0f;
    // RC_CK events at a time, the last first, the rows of the next ones loaded meanwhile
    P xr[RC_CK], gr[RC_CK], dr[RC_CK];
    float wl = 0.0f, cn[VEC];
    auto load = [&](int64_t s0) __attribute__((always_inline)) {
      const int n = (int)(t1 - s0 < RC_CK ? t1 - s0 : RC_CK);
#pragma unroll
      for (int j = 0; j < RC_CK; ++j) {
        const int64_t tt = s0 + (j < n ? j : n - 1);
        xr[j] = *(const P*)(xp + tt * a.xss);
        gr[j] = *(const P*)(gp + tt * a.gss);
        if (DH) dr[j] = *(const P*)((const T*)a.dh + ob + tt * a.D);
      }
      if (WT) wl = lane < n ? wp[s0 + lane] : 0.0f;
      const float* c = a.ck + (un.b * nck + s0 / RC_CK) * a.D + un.ch;
#pragma unroll
      for (int i = 0; i < VEC; ++i) cn[i] = c[i];
    };
    int64_t s0 = t1 > t0 ? (t1 - 1) / RC_CK * RC_CK : t0 - 1;
    if (s0 >= t0) load(s0);
    for (; s0 >= t0; s0 -= RC_CK) {
      const int n = (int)(t1 - s0 < RC_CK ? t1 - s0 : RC_CK);
      P xc[RC_CK], gc[RC_CK], dc[RC_CK];
      float wc[RC_CK], h[VEC], A[RC_CK][VEC], nA[RC_CK][VEC], q[RC_CK][VEC];
#pragma unroll
      for (int j = 0; j < RC_CK; ++j) {
        xc[j] = xr[j];
        gc[j] = gr[j];
        if (DH) dc[j] = dr[j];
        wc[j] = WT ? lane_value(wl, j) : 1.0f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = cn[i];
      if (s0 - RC_CK >= t0) load(s0 - RC_CK);
      gates<T, VEC, RC_CK, WT, true>(gc, wc, A, nA, q);
#pragma unroll
      for (int j = 0; j < RC_CK; ++j) {
        if (!WT || wc[j] > 0.0f) {
          float xv[VEC];
          unpack<T, VEC>(xc[j], xv);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            q[j][i] *= h[i] - xv[i];
            h[i] = move(A[j][i], nA[j][i], h[i], xv[i]);
          }
        }
      }
#pragma unroll
      for (int j = RC_CK - 1; j >= 0; --j) {
        if (j < n) {
          float G[VEC], dxv[VEC], dgv[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            G[i] = R[i];
            dxv[i] = dgv[i] = 0.0f;
          }
          if (DH) {
            float dv[VEC];
            unpack<T, VEC>(dc[j], dv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) R[i] = G[i] = G[i] + dv[i];
          }
          if (!WT || wc[j] > 0.0f) {  // (else padding: the gradient passes by)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              dxv[i] = nA[j][i] * G[i];
              dgv[i] = q[j][i] * G[i];
              R[i] = decay(A[j][i], nA[j][i], G[i]);
            }
          }
          const int64_t o = ob + (s0 + j) * a.D;
          if (un.ok) {
            *(P*)((T*)a.dx + o) = pack<T, VEC>(dxv);
            *(P*)((T*)a.dgate + o) = pack<T, VEC>(dgv);
          }
        }
      }
    }
    if (a.dh0 && un.c == 0 && un.ok) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a.dh0[un.b * a.D + un.ch + i] = R[i];
    }
  }
}

// ------------------------------------------------------------------------------- host side
struct ScanPlan {
  int vec, nw, C;
  int64_t T;
};
// VEC: two channels a lane where D, the strides and the addresses allow (4- or 8-byte loads),
// else one.  Chunks: as many as give the card about 8192 waves (8 a SIMD), none shorter than 32
// events; one chunk when the histories alone give 640 waves in bf16, 512 in f32 (128 channels, forward
// and backward, us, one chunk : split: bf16 512 x 1000 214 + 265 : 148 + 208, 768 x 1000 205 + 236 :
// 251 + 336, 1000 x 1000 188 + 273 : 317 + 427; f32 256 x 1000 247 + 311 : 135 + 195, 512 x 1000 253 +
// 335 : 302 + 416) or have fewer than 128 events (bf16 256 x 128 27 + 32 : 30 + 31).
static ScanPlan scan_plan(int64_t B, int64_t S, int D, int64_t sz, bool vec_ok) {
  ScanPlan p;
  p.vec = vec_ok && D % 2 == 0 ? 2 : 1;
  p.nw = (D + 64 * p.vec - 1) / (64 * p.vec);
  p.C = 1;
  p.T = S > 0 ? S : 1;
  const int64_t waves = B * p.nw;
  if (waves < (sz == 2 ? 640 : 512) && S >= 128) {
    int64_t c = (8192 + waves - 1) / waves, cmax = (S + 31) / 32;
    c = c < cmax ? c : cmax;
    p.T = ((S + c - 1) / c + RC_CK - 1) / RC_CK * RC_CK;
    p.C = (int)((S + p.T - 1) / p.T);
  }
  return p;
}
// workspace for either type and vector width (the caller of the size does not know the addresses)
static int64_t scan_ws(int64_t B, int64_t S, int D) {
  int64_t need = 0;
  for (int v = 0; v < 4; ++v) {
    const ScanPlan p = scan_plan(B, S, D, v & 2 ? 4 : 2, (v & 1) != 0);
    const int64_t n = p.C > 1 ? 3 * B * p.C * (int64_t)D * 4 : 0;
    need = n > need ? n : need;
  }
  return need;
}

enum { RC_FWD, RC_FWD_SUM, RC_BWD, RC_BWD_SUM };
template <int KIND, typename T, int V, bool W>
static void scan_go(unsigned grid, hipStream_t st, const ScanArgs& a) {
  void (*k)(const ScanArgs);
  if constexpr (KIND == RC_FWD) k = k_scan_fwd<T, V, W, false>;
  else if constexpr (KIND == RC_FWD_SUM) k = k_scan_fwd<T, V, W, true>;
  else if constexpr (KIND == RC_BWD) k = a.dh ? k_scan_bwd<T, V, W, true> : k_scan_bwd<T, V, W, false>;
  else k = a.dh ? k_scan_bwd_sum<T, V, W, true> : k_scan_bwd_sum<T, V, W, false>;
  hipLaunchKernelGGL(k, dim3(grid), dim3(256), 0, st, a);
}
template <int KIND, typename T>
static void scan_vec(int vec, unsigned grid, hipStream_t st, const ScanArgs& a) {
  if (vec == 2) {
    if (a.w) scan_go<KIND, T, 2, true>(grid, st, a); else scan_go<KIND, T, 2, false>(grid, st, a);
  } else {
    if (a.w) scan_go<KIND, T, 1, true>(grid, st, a); else scan_go<KIND, T, 1, false>(grid, st, a);
  }
}
template <int KIND>
static void scan_launch(int dtype, int vec, unsigned grid, hipStream_t st, const ScanArgs& a) {
  if (dtype == TT_DTYPE_F32) scan_vec<KIND, float>(vec, grid, st, a);
  else scan_vec<KIND, uint16_t>(vec, grid, st, a);
}

static bool addr_ok(const void* p, int64_t bytes) { return ((uintptr_t)p % bytes) == 0; }

// shared checks and plan; returns TT_OK with a.C == 0 when there is nothing to do
static int scan_setup(ScanArgs& a, int32_t dtype, ScanPlan& p, void* workspace, int64_t ws_bytes,
                      std::initializer_list<const void*> rows, const char* fn) {
  const int64_t sz = dtype == TT_DTYPE_F32 ? 4 : 2;
  bool vec = a.xsb % 2 == 0 && a.xss % 2 == 0 && a.gsb % 2 == 0 && a.gss % 2 == 0;
  for (const void* r : rows) vec = vec && addr_ok(r, 2 * sz);
  p = scan_plan(a.B, a.S, a.D, sz, vec);
  a.nw = p.nw;
  a.C = p.C;
  a.T = p.T;
  if (p.C > 1) {
    const int64_t one = a.B * p.C * (int64_t)a.D;
    if (!workspace || ws_bytes < 3 * one * 4)
      return fail(TT_ERR_WORKSPACE, std::string(fn) + ": workspace too small");
    a.sumA = (float*)workspace;
    a.sumH = a.sumA + one;
    a.carry = a.sumH + one;
  }
  return TT_OK;
}
static unsigned scan_grid(const ScanArgs& a) {
  const int64_t blocks = (a.B * a.C * a.nw + 3) / 4;
  return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
}
static unsigned join_grid(const ScanArgs& a) {
  const int64_t blocks = a.B * ((a.D + RC_JCH - 1) / RC_JCH);
  return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
}

}  // namespace tt

using namespace tt;

#define RC_SIZES()                                                                              \
  TT_REQUIRE(dtype == TT_DTYPE_F32 || dtype == TT_DTYPE_BF16, "dtype must be f32 or bf16");     \
  TT_REQUIRE(B >= 0 && S >= 0 && D >= 1, "need B >= 0, S >= 0, D >= 1");                        \
  TT_REQUIRE(B < (1LL << 31) && S < (1LL << 40) && D <= (1 << 24), "sizes out of range")

extern "C" int tt_gated_scan_workspace_bytes(int64_t B, int64_t S, int32_t D, int64_t* bytes) {
  TT_REQUIRE(bytes, "null pointer");
  TT_REQUIRE(B >= 0 && S >= 0 && D >= 1, "need B >= 0, S >= 0, D >= 1");
  *bytes = B > 0 ? scan_ws(B, S, D) : 0;
  return TT_OK;
}

extern "C" int tt_gated_scan_fwd(const void* x, const void* gate, int32_t dtype, int64_t B,
                                 int64_t S, int32_t D, int64_t x_sb, int64_t x_ss, int64_t g_sb,
                                 int64_t g_ss, const float* w, int64_t w_sb, const float* h0,
                                 void* h, float* h_last, float* ckpt, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  RC_SIZES();
  if (B == 0) return TT_OK;
  TT_REQUIRE(h_last, "null pointer");
  TT_REQUIRE(S == 0 || (x && gate), "null pointer");
  ScanArgs a{};
  a.x = x; a.gate = gate; a.w = w; a.h0 = h0; a.h = h; a.h_last = h_last; a.ck = ckpt;
  a.B = B; a.S = S; a.D = D;
  a.xsb = x_sb; a.xss = x_ss; a.gsb = g_sb; a.gss = g_ss; a.wsb = w_sb;
  ScanPlan p;
  if (int rc = scan_setup(a, dtype, p, workspace, workspace_bytes, {x, gate, h}, __func__)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (p.C > 1) {
    scan_launch<RC_FWD_SUM>(dtype, p.vec, scan_grid(a), st, a);
    hipLaunchKernelGGL(k_scan_join<false>, dim3(join_grid(a)), dim3(RC_JCH * RC_SEG), 0, st, a.sumA,
                       a.sumH, a.h0, a.carry, B, a.C, D);
  }
  scan_launch<RC_FWD>(dtype, p.vec, scan_grid(a), st, a);
  return check_launch("tt_gated_scan_fwd");
}

extern "C" int tt_gated_scan_bwd(const void* x, const void* gate, int32_t dtype, int64_t B,
                                 int64_t S, int32_t D, int64_t x_sb, int64_t x_ss, int64_t g_sb,
                                 int64_t g_ss, const float* w, int64_t w_sb, const float* ckpt,
                                 const void* dh, const float* dh_last, void* dx, void* dgate,
                                 float* dh0, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  RC_SIZES();
  if (B == 0) return TT_OK;
  TT_REQUIRE(S == 0 || (x && gate && ckpt && dx && dgate), "null pointer");
  ScanArgs a{};
  a.x = x; a.gate = gate; a.w = w; a.ck = const_cast<float*>(ckpt);
  a.dh = dh; a.dlast = dh_last; a.dx = dx; a.dgate = dgate; a.dh0 = dh0;
  a.B = B; a.S = S; a.D = D;
  a.xsb = x_sb; a.xss = x_ss; a.gsb = g_sb; a.gss = g_ss; a.wsb = w_sb;
  ScanPlan p;
  if (int rc = scan_setup(a, dtype, p, workspace, workspace_bytes, {x, gate, dh, dx, dgate}, __func__))
    return rc;
  hipStream_t st = (hipStream_t)stream;
  if (p.C > 1) {
    scan_launch<RC_BWD_SUM>(dtype, p.vec, scan_grid(a), st, a);
    hipLaunchKernelGGL(k_scan_join<true>, dim3(join_grid(a)), dim3(RC_JCH * RC_SEG), 0, st, a.sumA,
                       a.sumH, a.dlast, a.carry, B, a.C, D);
  }
  scan_launch<RC_BWD>(dtype, p.vec, scan_grid(a), st, a);
  return check_launch("tt_gated_scan_bwd");
}
