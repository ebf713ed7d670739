// tt_adamw.hip -- AdamW step over many tensors in one launch, moments in 32 or 8 bits (gfx950).
//
//   m = b1 m + (1 - b1) g ;  v = b2 v + (1 - b2) g g ;  t = t + 1
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  f32: p, g, m, v read and p, m, v written, 28 bytes an element; 8-bit moments: 16.
// Measured: a 1M x 384 f32 table 2.10 ms (5.1 TB/s), an encoder's 117M parameters with 8-bit moments
// 440 - 510 us (3.7 - 4.3 TB/s) and 247 us (4.8 TB/s) to decode them, a tower's ten tensors 12 us.
// A small set of tensors (a tower's ten) is bound by latency (a block's entry, its tensor's, the step
// count and the factors from it, then the data: one after another), not by launches: all tensors go in
// one, a block per chunk of one tensor, tensors and chunks from a table on the device.  Only the gradients'
// addresses change from step to step: they travel in the kernel's arguments.
//
// The step count lives on the device, one per tensor (a tensor without a gradient keeps its
// count), so a captured step advances on every replay.  Every block reads it before it takes a
// ticket; the block with the tensor's last ticket writes t + 1, so no block can see the new
// count in the same launch.  No block waits for another.
//
// 8-bit moments: blocks of 256 elements of the flattened tensor, one wave each, one f32 scale
// (the block's largest magnitude) per moment.
//   m: sign and 127 square-root levels    code = rint(127 sqrt(|m| / s)),    stands for s (code / 127)^2
//   v: 255 fourth-root levels             code = rint(255 (v / s)^(1/4)),    stands for s (code / 255)^4
// Roots, because one block's moments spread over decades: linear levels would send all but the
// largest to 0, and an update divides by sqrt(v).  v > 0 is never coded 0 (code 1 at least), so the
// coding never makes an update larger by more than half a level does.  The new moment is formed in
// 64 bits from the code it had, and the code is the nearest of the 64-bit value: found in 32
// bits, and again in 64 where the 32-bit value lies within its error of a border between two
// codes (1e-4 of a level: some 2 lanes in 10000).  The update itself uses the moments before
// coding, rounded to f32.
#include "tt_common.hpp"

namespace tt {

constexpr int AW_MAXT = 416;  // gradients' addresses in one launch's arguments (3.3 KB)

struct AwGrads {
  const void* g[AW_MAXT];
};
struct AwHyper {
  double lr, b1, b2, wd;
  float eps;
};

__device__ __forceinline__ double ipow(double b, int64_t e) {  // b^e by squaring
  double r = 1.0;
  while (e > 0) {
    if (e & 1) r *= b;
    b *= b;
    e >>= 1;
  }
  return r;
}

typedef uint32_t aw_u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 aw_bf16x2 __attribute__((ext_vector_type(2)));
typedef float aw_f32x2 __attribute__((ext_vector_type(2)));

// 4 elements of a row of n at e, vector access where vec (aligned) and whole
template <typename T>
__device__ __forceinline__ void aw_load(const T* p, int64_t e, int64_t n, bool vec, float (&o)[4]) {
  if (vec && e + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 v = *(const f32x4*)(p + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = v[i];
    } else {
      const aw_u32x2 v = *(const aw_u32x2*)(p + e);
      o[0] = __uint_as_float(v[0] << 16);
      o[1] = __uint_as_float(v[0] & 0xffff0000u);
      o[2] = __uint_as_float(v[1] << 16);
      o[3] = __uint_as_float(v[1] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) o[i] = e + i < n ? p[e + i] : 0.0f;
      else o[i] = e + i < n ? __uint_as_float((uint32_t)p[e + i] << 16) : 0.0f;
    }
  }
}
template <typename T>
__device__ __forceinline__ void aw_store(T* p, int64_t e, int64_t n, bool vec, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    if (vec && e + 4 <= n) {
      *(f32x4*)(p + e) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < n) p[e + i] = v[i];
    }
  } else {  // a bf16 parameter: rounded once, to the nearest
    aw_u32x2 u;
    u[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(aw_f32x2{v[0], v[1]}, aw_bf16x2));
    u[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(aw_f32x2{v[2], v[3]}, aw_bf16x2));
    if (vec && e + 4 <= n) {
      *(aw_u32x2*)(p + e) = u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < n) p[e + i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
  }
}

constexpr double AW_KM = 1.0 / (127.0 * 127.0), AW_KV = 1.0 / (255.0 * 255.0 * 255.0 * 255.0);
__device__ __forceinline__ double aw_dec_m(int q, double s) {
  return (double)(q < 0 ? -q * q : q * q) * AW_KM * s;  // (code 127: s itself, to the bit)
}
__device__ __forceinline__ double aw_dec_v(uint32_t q, double s) {
  return (double)(q * q * (q * q)) * AW_KV * s;  // 255^4 < 2^32
}
// nearest code of |m| (127 square-root levels) / v (255 fourth-root levels), scale s
__device__ __forceinline__ int aw_code_m(double a, float s, float inv) {
  const float r = __builtin_amdgcn_sqrtf((float)a * inv) * 127.0f;
  const float q = rintf(r);
  // inv and the root are off by about an ulp each: 3e-5 of a level at most
  if (s >= 1e-30f && fabsf(r - q) < 0.4999f) return (int)q;
  const double d = rint(127.0 * sqrt(a / (s > 0.0f ? (double)s : 1.0)));
  return d < 127.0 ? (int)d : 127;
}
__device__ __forceinline__ uint32_t aw_code_v(double v, float s, float inv) {
  if (!(v > 0.0)) return 0u;
  const float r = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)v * inv)) * 255.0f;
  float q = rintf(r);
  if (!(s >= 1e-30f && fabsf(r - q) < 0.4998f)) {
    const double d = rint(255.0 * sqrt(sqrt(v / (s > 0.0f ? (double)s : 1.0))));
    q = d < 255.0 ? (float)d : 255.0f;
  }
  return q > 1.0f ? (uint32_t)q : 1u;
}

struct AwFactors {
  float step, rs, decay, eps;
};

// m32, v32 -> p (f32 arithmetic: one rounding per operation, IEEE root and quotient)
__device__ __forceinline__ float aw_update(float p, float m, float v, const AwFactors& f) {
  const float den = __fmul_rn(sqrtf(v), f.rs) + f.eps;
  const float u = __fdiv_rn(m, den);
  return __fmul_rn(p, f.decay) - __fmul_rn(u, f.step);
}

// codes of one 256-element block from its moments (64 bits), 4 elements a lane
__device__ __forceinline__ void aw_encode(const double (&m)[4], const double (&v)[4], int64_t e,
                                          int64_t n, int lane, int8_t* qm, uint8_t* qv, float* sm,
                                          float* sv, int64_t blk) {
  // the block's maxima, by their bits (non-negative floats order as integers; a NaN above all)
  uint32_t bm = 0, bv = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t um = __float_as_uint(fabsf((float)m[i])), uv = __float_as_uint((float)v[i]) & 0x7fffffffu;
    bm = um > bm ? um : bm;
    bv = uv > bv ? uv : bv;
  }
  const float s = __uint_as_float(wave_max_u32(bm)), z = __uint_as_float(wave_max_u32(bv));
  const float is = 1.0f / s, iz = 1.0f / z;
  uint32_t cm = 0, cv = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = aw_code_m(fabs(m[i]), s, is);
    cm |= ((uint32_t)(m[i] < 0.0 ? -q : q) & 0xffu) << (8 * i);
    cv |= aw_code_v(v[i], z, iz) << (8 * i);
  }
  if (e < n) {  // (the state rows are padded to whole blocks)
    *(uint32_t*)(qm + e) = cm;
    *(uint32_t*)(qv + e) = cv;
  }
  if (lane == 0) {
    sm[blk] = s;
    sv[blk] = z;
  }
}

template <int BITS, typename T>
__device__ __forceinline__ void aw_chunk(const tt_adamw_tensor& t, const T* g, int64_t c0, int64_t c1,
                                         const AwHyper& hp, const AwFactors& f, int tid) {
  const int lane = tid & 63;
  T* p = (T*)t.p;
  const bool vp = ((uintptr_t)p % (4 * sizeof(T))) == 0, vg = ((uintptr_t)g % (4 * sizeof(T))) == 0;
  const float b1 = (float)hp.b1, c1f = (float)(1.0 - hp.b1), b2 = (float)hp.b2, c2f = (float)(1.0 - hp.b2);
  for (int64_t e0 = c0 + (tid >> 6) * 256; e0 < c1; e0 += 1024) {
    const int64_t e = e0 + 4 * lane;
    float pv[4], gv[4], mv[4], vv[4];
    aw_load(p, e, t.n, vp, pv);
    aw_load(g, e, t.n, vg, gv);
    if constexpr (BITS == 32) {
      float* m = (float*)t.exp_avg;
      float* v = (float*)t.exp_avg_sq;
      const bool in = e < t.n;  // (the state rows are padded to whole vectors)
      f32x4 ml = in ? *(const f32x4*)(m + e) : f32x4{0.f, 0.f, 0.f, 0.f};
      f32x4 vl = in ? *(const f32x4*)(v + e) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i] = mv[i] = __fmul_rn(ml[i], b1) + __fmul_rn(gv[i], c1f);
        vl[i] = vv[i] = __fmul_rn(vl[i], b2) + __fmul_rn(__fmul_rn(gv[i], c2f), gv[i]);
      }
      if (in) {
        *(f32x4*)(m + e) = ml;
        *(f32x4*)(v + e) = vl;
      }
    } else {
      int8_t* qm = (int8_t*)t.exp_avg;
      uint8_t* qv = (uint8_t*)t.exp_avg_sq;
      const int64_t blk = e0 / 256;
      const uint32_t cm = e < t.n ? *(const uint32_t*)(qm + e) : 0u;
      const uint32_t cv = e < t.n ? *(const uint32_t*)(qv + e) : 0u;
      const double km = (double)t.scale_m[blk], kv = (double)t.scale_v[blk];
      double m64[4], v64[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double gd = e + i < t.n ? (double)gv[i] : 0.0;
        const double M = aw_dec_m((int)(int8_t)(cm >> (8 * i)), km), V = aw_dec_v((cv >> (8 * i)) & 0xffu, kv);
        m64[i] = hp.b1 * M + (1.0 - hp.b1) * gd;
        v64[i] = hp.b2 * V + (1.0 - hp.b2) * gd * gd;
        mv[i] = (float)m64[i];
        vv[i] = (float)v64[i];
      }
      aw_encode(m64, v64, e, t.n, lane, qm, qv, t.scale_m, t.scale_v, blk);
    }
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = aw_update(pv[i], mv[i], vv[i], f);
    aw_store(p, e, t.n, vp, o);
  }
}

template <int BITS>
__global__ __launch_bounds__(256) void k_adamw(const tt_adamw_tensor* __restrict__ tab,
                                               const int32_t* __restrict__ items, int first,
                                               int64_t chunk, const AwGrads gr, const AwHyper hp) {
  const int ti = items[2 * (int64_t)blockIdx.x], ci = items[2 * (int64_t)blockIdx.x + 1];
  const void* g = gr.g[ti - first];
  if (!g) return;  // no gradient: nothing of this tensor moves, its count neither
  const tt_adamw_tensor t = tab[ti];
  __shared__ AwFactors fs;
  __shared__ int64_t s_step;
  const int tid = threadIdx.x;
  if (tid == 0) {
    const int64_t step = *t.step + 1;
    const double bc1 = 1.0 - ipow(hp.b1, step), bc2 = 1.0 - ipow(hp.b2, step);
    fs.step = (float)(hp.lr / bc1);
    fs.rs = (float)(1.0 / sqrt(bc2));
    fs.decay = (float)(1.0 - hp.lr * hp.wd);
    fs.eps = hp.eps;
    s_step = step;
  }
  __syncthreads();
  const AwFactors f = fs;
  const int64_t c0 = (int64_t)ci * chunk, c1 = c0 + chunk < t.n ? c0 + chunk : t.n;
  if (t.dtype == TT_DTYPE_F32) aw_chunk<BITS, float>(t, (const float*)g, c0, c1, hp, f, tid);
  else aw_chunk<BITS, uint16_t>(t, (const uint16_t*)g, c0, c1, hp, f, tid);
  if (tid == 0) {
    // the count was read above; the last of the tensor's blocks advances it
    const uint32_t k = atomicAdd(t.ticket, 1u);
    if (k == (uint32_t)t.blocks - 1u) {
      *t.ticket = 0u;
      *t.step = s_step;
    }
  }
}

// 8-bit moments <-> f32 (ENC: f32 rows at out_off -> codes and scales; else codes -> f32 rows)
template <bool ENC>
__global__ __launch_bounds__(256) void k_adamw_codes(const tt_adamw_tensor* __restrict__ tab,
                                                     const int32_t* __restrict__ items, int64_t chunk,
                                                     const int64_t* __restrict__ off, float* fm,
                                                     float* fv) {
  const int ti = items[2 * (int64_t)blockIdx.x], ci = items[2 * (int64_t)blockIdx.x + 1];
  const tt_adamw_tensor t = tab[ti];
  const int lane = threadIdx.x & 63;
  const int64_t c0 = (int64_t)ci * chunk, c1 = c0 + chunk < t.n ? c0 + chunk : t.n;
  float* m = fm + off[ti];
  float* v = fv + off[ti];
  int8_t* qm = (int8_t*)t.exp_avg;
  uint8_t* qv = (uint8_t*)t.exp_avg_sq;
  for (int64_t e0 = c0 + (threadIdx.x >> 6) * 256; e0 < c1; e0 += 1024) {
    const int64_t e = e0 + 4 * lane, blk = e0 / 256;
    if constexpr (ENC) {
      double m64[4], v64[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m64[i] = e + i < t.n ? (double)m[e + i] : 0.0;
        v64[i] = e + i < t.n ? (double)v[e + i] : 0.0;
      }
      aw_encode(m64, v64, e, t.n, lane, qm, qv, t.scale_m, t.scale_v, blk);
    } else {
      if (e >= t.n) continue;
      const double km = (double)t.scale_m[blk], kv = (double)t.scale_v[blk];
      const uint32_t cm = *(const uint32_t*)(qm + e), cv = *(const uint32_t*)(qv + e);
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = (float)aw_dec_m((int)(int8_t)(cm >> (8 * i)), km);
        b[i] = (float)aw_dec_v((cv >> (8 * i)) & 0xffu, kv);
      }
      aw_store(m, e, t.n, true, a);
      aw_store(v, e, t.n, true, b);
    }
  }
}

}  // namespace tt

using namespace tt;

extern "C" int tt_adamw_step(const tt_adamw_tensor* tensors, const int32_t* items, int64_t n_items,
                             int32_t first, const void* const* grads, int32_t n_grads,
                             int64_t chunk, int32_t state_bits, double lr, double beta1,
                             double beta2, double eps, double weight_decay, void* stream) {
  TT_REQUIRE(state_bits == 32 || state_bits == 8, "state_bits must be 32 or 8");
  TT_REQUIRE(n_items >= 0 && n_items < (1LL << 23), "need 0 <= n_items < 2^23");
  TT_REQUIRE(n_grads >= 0 && n_grads <= AW_MAXT, "at most 416 tensors a launch");
  TT_REQUIRE(chunk >= 1024 && chunk % 1024 == 0, "chunk must be a multiple of 1024");
  TT_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "betas must be in [0, 1)");
  if (n_items == 0) return TT_OK;
  TT_REQUIRE(tensors && items && grads, "null pointer");
  AwGrads g;
  for (int i = 0; i < AW_MAXT; ++i) g.g[i] = i < n_grads ? grads[i] : nullptr;
  const AwHyper hp{lr, beta1, beta2, weight_decay, (float)eps};
  auto k = state_bits == 32 ? k_adamw<32> : k_adamw<8>;
  hipLaunchKernelGGL(k, dim3((unsigned)n_items), dim3(256), 0, (hipStream_t)stream, tensors, items,
                     first, chunk, g, hp);
  return check_launch("tt_adamw_step");
}

static int aw_codes(bool enc, const tt_adamw_tensor* tensors, const int32_t* items, int64_t n_items,
                    int64_t chunk, const int64_t* offsets, float* m, float* v, void* stream,
                    const char* what) {
  if (n_items < 0 || n_items >= (1LL << 23) || chunk < 1024 || chunk % 1024 != 0)
    return fail(TT_ERR_INVALID, std::string(what) + ": bad sizes");
  if (n_items == 0) return TT_OK;
  if (!(tensors && items && offsets && m && v))
    return fail(TT_ERR_INVALID, std::string(what) + ": null pointer");
  auto k = enc ? k_adamw_codes<true> : k_adamw_codes<false>;
  hipLaunchKernelGGL(k, dim3((unsigned)n_items), dim3(256), 0, (hipStream_t)stream, tensors, items,
                     chunk, offsets, m, v);
  return check_launch(what);
}
extern "C" int tt_adamw_decode(const tt_adamw_tensor* tensors, const int32_t* items, int64_t n_items,
                               int64_t chunk, const int64_t* offsets, float* exp_avg,
                               float* exp_avg_sq, void* stream) {
  return aw_codes(false, tensors, items, n_items, chunk, offsets, exp_avg, exp_avg_sq, stream,
                  "tt_adamw_decode");
}
extern "C" int tt_adamw_encode(const tt_adamw_tensor* tensors, const int32_t* items, int64_t n_items,
                               int64_t chunk, const int64_t* offsets, const float* exp_avg,
                               const float* exp_avg_sq, void* stream) {
  return aw_codes(true, tensors, items, n_items, chunk, offsets, const_cast<float*>(exp_avg),
                  const_cast<float*>(exp_avg_sq), stream, "tt_adamw_encode");
}
