// tt_catalog.hip -- log-probabilities of given items over a catalog, with the entropy and the top
// alternatives of every row, and their gradient (gfx950).
//
//   l_nv = s x_n.w_v + bias_v         x [N, E], w [V, E] f32 or bf16;  s = 1 / temperature
//   lse_n = log sum_v exp l_nv ;  p_nv = exp(l_nv - lse_n)
//   log_prob_n = l_{n,id} - lse_n ;  entropy_n = lse_n - sum_v p_nv l_nv ;  top: the k largest l_nv
//   backward (g, e: gradients of log_prob, entropy; H the entropy):
//   c_nv = g_n ([v = id_n] - p_nv) - e_n p_nv (l_nv - lse_n + H_n) ;  dx = s C w ;  dw = s C^T x
//
// The N x V logits never exist in memory.  Everything is done in powers of two (z = l log2 e).
//
// k_logits<STAT>  tiles of 128 items x 128 rows (64 x 64 where that leaves CUs idle, 256 x 256 where
//     those fill them) on MFMA (bf16 16x16x32 or f32 16x16x4); a block walks its share of the catalog
//     for its rows.  The product is formed as w . x^T, so a lane holds a few items of 4 rows: the
//     running maximum m, L = sum 2^(z - m) and T = sum 2^(z - m) (z - m) of a row stay in the lane,
//     with no exchange between lanes until the share's end.
//     Entropy = ln 2 (log2 L - T / L): relative to the maximum, nothing cancels against lse.
// k_combine       joins the shares; the given item's own logit in 64 bits, also in the joined sums.
// top             the STAT pass also writes the maximum of every 16 items a lane saw (N V / 16
//     floats).  The k largest logits lie in the k groups with the largest maxima; k + 8 groups are
//     taken (32-bit maxima may swap near-equal ones), their items scored again in 64 bits, and
//     ordered by that, ties by the lower id.  What 32-bit logits are off by at most is known: see
//     logit_error; the STAT pass also takes the largest item norm that this needs.  A row where groups
//     that were not taken lie within it (a crowd of nearly equal items) is searched again, over all of
//     its groups that do (k_top_wide).
// k_logits<COEF>  the same product again, its epilogue writing C for a chunk of the catalog, in x's type:
//     the products take it as an operand of their matrix instructions.  In bf16 a coefficient is then off
//     by up to 2^-8 of itself.  The given item's, which is most of its row's gradient, keeps what the
//     rounding left (k_lost), and the products begin with that: the gradients of 4096 x 32768 x 768 are
//     1.66e-3 off, their own rounding (2.02e-3 without; 3 in 100 of the call).  The others' roundings
//     are many and small.  Up to 64 rows, where any coefficient may be all of a sum, all are kept in two
//     parts.
// k_product       dx += C w (C rows, w as it lies) and dw = C^T x: operands whose rows run along the
//     sum are read from LDS transposed (ds_read_b64_tr_b16; 4-byte reads in f32), so neither C nor
//     w nor x is ever stored transposed.  What the output's tiles leave of the last round of blocks is
//     filled by splitting their sums (f32 partial sums, added in a fixed order: the result does not
//     depend on timing).
//
// Bound: small N by reading w (1 x 1M x 384 bf16: 150 - 158 us, 4.9 - 5.1 TB/s), large N by the matrix
// pipes with the loads that feed them (4096 x 65537 x 768 bf16: statistics 465 us, 0.89 PFLOP/s;
// coefficients 196 us and the products 154, 159 us per 21888 items, 0.70, 0.90, 0.87 PFLOP/s).
//
// Items with a bias at or below -1e30 (-inf, the type's lowest) are taken out: probability 0 and
// gradient 0 whatever their vectors hold.  Rows whose gradients are both 0 do not reach dw.  A row whose
// lse is no number (a NaN in it or in an item, a logit past the range) has gradients that are none.
#include "tt_common.hpp"

namespace tt {

typedef __bf16 ct_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 ct_bf16x2 __attribute__((ext_vector_type(2)));
typedef float ct_f32x2 __attribute__((ext_vector_type(2)));
typedef short ct_s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t ct_u32x2 __attribute__((ext_vector_type(2)));

constexpr float CT_OUT = -1.0e30f;   // z of an item that is taken out
constexpr float CT_NONE = -2.0e30f;  // maximum of nothing
constexpr float CT_LOG2E = 1.4426950408889634f, CT_LN2 = 0.6931471805599453f;
constexpr int CT_TILE = 128;  // tile edge (items, rows, columns), or half of it
constexpr int CT_TOP_MAX = 32, CT_TOP_EXTRA = 8;

__device__ __forceinline__ void ct_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ct_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ct_dma(const void* g, char* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// ---- operand stages, of 32 NB rows or columns (NB = 4: 128, or 2: 64; a wave's quarter of the tile
// is 16 NB square).  Row form ("K along the row"): rows of 128 B, 16-B chunks XOR-swizzled by
// (row >> 1) & 7.  Wave w of NWV loads pieces w, w + NWV, ...: 8 rows each.
template <typename T, int NB, int NWV = 4>
struct RowStage {
  static constexpr int PW = 4 * NB / NWV;  // 1-KB pieces a wave loads
  int64_t off[PW];
  __device__ __forceinline__ void init(int64_t ld, int64_t row0, int64_t rows, int w, int lane) {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int r = 8 * (w + NWV * j) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
      int64_t row = row0 + r;
      row = row < rows ? row : rows - 1;  // past the end: loaded again, never used
      off[j] = row * ld + c * (16 / (int)sizeof(T));
    }
  }
  __device__ __forceinline__ void issue(const T* p, int64_t k0, char* lds, int w) const {
#pragma unroll
    for (int j = 0; j < PW; ++j) ct_dma(p + off[j] + k0, lds + 1024 * (w + NWV * j));
  }
};
// fragments of NB x 16 rows from row r0: f[s][i] = 16 B at chunk 4 (s0 + s) + g of row r0 + 16 i + rl
template <int NB, int NS>
__device__ __forceinline__ void row_frags(const char* lds, int r0, int lane, u32x4_t (&f)[NS][NB], int s0 = 0) {
  const int g = lane >> 4, rl = lane & 15, sw = (rl >> 1) & 7;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < NB; ++i)
      f[s][i] = *(const u32x4_t*)(lds + (r0 + 16 * i + rl) * 128 + 16 * ((4 * (s0 + s) + g) ^ sw));
}

// Column form ("the sum runs down the rows"): BK rows x 32 NB elements, the operand as it lies.
template <typename T, int NB, int NWV = 4>
struct ColStage {
  static constexpr int PW = 4 * NB / NWV;
  static constexpr int EPC = 16 / (int)sizeof(T), CPR = 32 * NB / EPC;  // elements a chunk, chunks a row
  static constexpr int RPP = 64 / CPR;                                  // rows per 1-KB piece
  // swizzle of a row's chunks: the rows that one fragment read touches together lie in different
  // banks (bf16: 8 rows of two chunks; f32: 4 rows of four)
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (sizeof(T) == 2) return NB >= 4 ? ((r & 3) | ((r >> 1) & 4)) << 1 : (((r >> 1) & 1) | ((r >> 2) & 2)) << 1;
    else return ((r >> 2) & 3) << 2;
  }
  int64_t off[PW];
  int row[PW];
  // cols: valid columns from c0 (a multiple of the chunk); past the end: loaded again, never used
  __device__ __forceinline__ void init(int64_t c0, int64_t cols, int w, int lane) {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int r = RPP * (w + NWV * j) + lane / CPR, pc = lane % CPR;
      int64_t c = c0 + (int64_t)(pc ^ swz(r)) * EPC;
      c = c < cols ? c : cols - EPC;
      row[j] = r;
      off[j] = c;
    }
  }
  __device__ __forceinline__ void issue(const T* p, int64_t ld, int64_t k0, int64_t rows, char* lds,
                                        int w) const {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      int64_t k = k0 + row[j];
      k = k < rows ? k : rows - 1;  // past the end: the other operand is zero there
      ct_dma(p + k * ld + off[j], lds + 1024 * (w + NWV * j));
    }
  }
};
// the same fragments as row_frags gives (16 B of the sum's index for column c0 + 16 i + rl)
template <typename T, int NB, int NF, int NS>
__device__ __forceinline__ void col_frags(const char* lds, int c0, int lane, u32x4_t (&f)[NS][NF], int s0 = 0) {
  const int g = lane >> 4, rl = lane & 15;
  constexpr int ROW_B = 32 * NB * (int)sizeof(T);
  if constexpr (sizeof(T) == 2) {
    // a 16-lane group reads 4 rows x 16 columns: lane 4 q + c supplies row q, columns 4 c .. + 3 and
    // receives column (its index)'s 4 rows
    const int q = rl >> 2, c = rl & 3;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        ct_u32x2 h[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 32 * (s0 + s) + 8 * g + 4 * u + q;
          const int chunk = (2 * (c0 / 16 + i) + (c >> 1)) ^ ColStage<T, NB>::swz(row);
          const char* p = lds + row * ROW_B + chunk * 16 + 8 * (c & 1);
          h[u] = __builtin_bit_cast(ct_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) ct_s16x4*)p));
        }
        f[s][i] = u32x4_t{h[0][0], h[0][1], h[1][0], h[1][1]};
      }
  } else {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = 16 * (s0 + s) + 4 * g + u;
          const int chunk = (4 * (c0 / 16 + i) + (rl >> 2)) ^ ColStage<T, NB>::swz(row);
          f[s][i][u] = *(const uint32_t*)(lds + row * ROW_B + chunk * 16 + 4 * (rl & 3));
        }
  }
}

// acc[i][j] += first[j] . second[i]: lane (g, rl) of block (i, j) holds first-index 16 j + 4 g + r,
// second-index 16 i + rl
template <typename T, int NJ, int NI, int NS>
__device__ __forceinline__ void ct_mfma(const u32x4_t (&first)[NS][NJ], const u32x4_t (&second)[NS][NI],
                                        f32x4 (&acc)[NI][NJ]) {
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (sizeof(T) == 2) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(ct_bf16x8, first[s][j]), __builtin_bit_cast(ct_bf16x8, second[s][i]),
              acc[i][j], 0, 0, 0);
        } else {
          const f32x4 a = __builtin_bit_cast(f32x4, first[s][j]), b = __builtin_bit_cast(f32x4, second[s][i]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u], b[u], acc[i][j], 0, 0, 0);
        }
      }
}

// The same for one stage.  In f32 a stage's products are summed on their own and added as a whole: one
// chain over all of a row's products would be off by some sqrt(E / 3) roundings of the sum (16 at E =
// 768), this way by 3 (23 x 536 x 448: gradients 9.6e-7 -> 3.3e-7 off, 512 x 2560 x 768: 1 us a launch).
// The bf16 instructions sum 32 products at a time already.
template <typename T, int NJ, int NI, int NS>
__device__ __forceinline__ void ct_stage(const u32x4_t (&first)[NS][NJ], const u32x4_t (&second)[NS][NI],
                                         f32x4 (&acc)[NI][NJ]) {
  if constexpr (sizeof(T) == 2) {
    ct_mfma<T>(first, second, acc);
  } else {
    f32x4 part[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) part[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    ct_mfma<T>(first, second, part);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = acc[i][j] + part[i][j];
  }
}

__device__ __forceinline__ uint32_t ct_pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(ct_f32x2{a, b}, ct_bf16x2));
}
// 4 consecutive outputs
template <typename T>
__device__ __forceinline__ void ct_store4(T* p, const f32x4& v) {
  if constexpr (sizeof(T) == 2) *(ct_u32x2*)p = ct_u32x2{ct_pack2(v[0], v[1]), ct_pack2(v[2], v[3])};
  else *(f32x4*)p = v;
}

// d + the sum of the squares of 16 bytes of a vector
template <typename T>
__device__ __forceinline__ float sumsq16(const u32x4_t& v, float d) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      d = fmaf(__uint_as_float(v[i]), __uint_as_float(v[i]), d);
    } else {
      const ct_bf16x2 b = __builtin_bit_cast(ct_bf16x2, v[i]);
      d = __builtin_amdgcn_fdot2_f32_bf16(b, b, d, false);
    }
  }
  return d;
}

// (m, L, T) of two disjoint sets of items
__device__ __forceinline__ void stat_join(float& m, float& L, float& T, float m2, float L2, float T2) {
  const float M = fmaxf(m, m2);
  const float a = __builtin_amdgcn_exp2f(m - M), b = __builtin_amdgcn_exp2f(m2 - M);
  T = a * fmaf(m - M, L, T) + b * fmaf(m2 - M, L2, T2);
  L = fmaf(a, L, b * L2);
  m = M;
}

struct LogitArgs {
  const void *x, *w;
  int64_t ldx, ldw;
  const float* bias;   // may be null
  float s2;            // log2(e) / temperature
  int N, V, E;
  int n_tiles, splits, v_tiles;  // tiles of rows, shares of the catalog, tiles of items
  float4* part;        // STAT [splits, N] (m, L, T, -)
  float* tmax;         // STAT: [N, 4 ceil(V / 64)] or null
  float* wsq;          // STAT with tmax: [blocks] what no |w_v|^2 that the block looked at exceeds
  // COEF [N] (lse in powers of two, rounded; g, e with what its rounding takes out of p put back; H so too);
  // g and e both 0: the row is dead
  const float4* rowc;
  const float* rowg;   // COEF [N] g itself: the given item's
  const int64_t* ids;  // COEF
  void* C;             // COEF [Npad, ldc]: items v_base .. of this chunk
  int64_t ldc;
  int v_base, v_count, Npad;  // v_count: items from v_base on
  bool two;            // COEF in bf16: row n + N of C takes what the rounding of row n leaves
};
// what the rounding of c to bf16 leaves
__device__ __forceinline__ float ct_lost(float c) { return c - __uint_as_float(ct_pack2(c, 0.0f) << 16); }

// A tile of 32 NB rows x 32 NB items: 4 waves of 16 NB x 16 NB, or (NB = 8, bf16) 8 waves of 64 rows x
// 128 items: half the loads per product, and 3/8 of a fragment read from LDS per matrix instruction
// (NB = 4: 1/2).
template <int NB>
struct Tile {
  static constexpr int EDGE = 32 * NB, NWV = NB == 8 ? 8 : 4, NT = 64 * NWV;
  static constexpr int ROW_WV = NB == 8 ? 4 : 2;       // waves along the rows; 2 along the items (columns)
  static constexpr int FI = NB == 8 ? 4 : NB, FJ = NB;  // 16-blocks of a wave: rows, items
  static constexpr int OP_B = EDGE * 128, PER_EU = NB == 2 ? 3 : 2;
};
__device__ __forceinline__ void ct_turn() {  // a barrier that no matrix instruction moves across
  __builtin_amdgcn_sched_barrier(0);
  ct_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// (TOP: with the groups' maxima and the norms; without their registers and branches 457 us for 469)
template <typename T, bool COEF, bool ENT, int NB, bool TOP>
__global__ __launch_bounds__(Tile<NB>::NT, Tile<NB>::PER_EU) void k_logits(const LogitArgs a) {
  using TL = Tile<NB>;
  constexpr int BK = 128 / (int)sizeof(T), FI = TL::FI, FJ = TL::FJ, HJ = FJ < 4 ? FJ : 4;
  __shared__ __attribute__((aligned(16))) char smem[4 * TL::OP_B];
  __shared__ float half[NB == 2 && TOP ? TL::EDGE : 1][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = w % TL::ROW_WV, wv = w / TL::ROW_WV, g = lane >> 4, rl = lane & 15;
  // blocks of one share of the catalog next to each other (one XCD's L2)
  const int lb = xcd_remap(blockIdx.x, gridDim.x);
  const int sp = lb / a.n_tiles, tn = lb % a.n_tiles;
  const int per = (a.v_tiles + a.splits - 1) / a.splits;
  const int vt0 = sp * per, vt1 = vt0 + per < a.v_tiles ? vt0 + per : a.v_tiles;
  const int nw = 16 * FI * wn, n0 = tn * TL::EDGE + nw, v_end = a.v_base + a.v_count;
  const T* x = (const T*)a.x;
  const T* wt = (const T*)a.w;
  const int nk = a.E / BK;

  RowStage<T, NB, TL::NWV> sx, sw;
  sx.init(a.ldx, (int64_t)tn * TL::EDGE, a.N, w, lane);
  float m[FI], L[FI], TT[FI];
  float4 rc[FI];
  int id[FI];
  // (g itself for the given item; in the 256 tile, whose bf16 coefficients k_lost corrects, there are no
  // registers for it)
  constexpr bool OWN_G = NB < 8;
  float go[FI];
  // the items' norms (with tmax): a tile's by the block of the row tile that its number falls to, the
  // blocks of 16 items shared out among the waves that hold them.  A lane has a quarter of an item's
  // elements; the largest quarters of any items, added at the end, exceed no norm by much.  (1 x 1M x
  // 384: the same from reads of their own from LDS took 214 us a call instead of 172.)  The 256 tile has
  // no registers for holding on to the fragments: there every wave reads what it loaded once more (8
  // lanes a row).
  constexpr bool OWN_READ = NB == 8;
  constexpr int JP = OWN_READ ? decltype(sw)::PW : FJ / TL::ROW_WV;
  float sq[JP], wmx = 0.0f;
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    m[i] = CT_NONE;
    L[i] = TT[i] = 0.0f;
    if constexpr (COEF) {
      const int n = n0 + 16 * i + rl;
      rc[i] = n < a.N ? a.rowc[n] : float4{1.0e30f, 0.f, 0.f, 0.f};
      const int64_t q = n < a.N && a.ids ? a.ids[n] : -1;
      id[i] = q >= 0 && q < a.V ? (int)q : -1;
      if constexpr (OWN_G) go[i] = n < a.N ? a.rowg[n] : 0.0f;
    }
  }
  // loads run one stage ahead over (tile, k) as one sequence
  int vt_i = vt0, k_i = 0, g_i = 0;
  auto issue_next = [&]() __attribute__((always_inline)) {
    if (vt_i >= vt1) return;
    if (k_i == 0) sw.init(a.ldw, (int64_t)a.v_base + (int64_t)vt_i * TL::EDGE, v_end, w, lane);
    char* st = smem + (g_i & 1) * 2 * TL::OP_B;
    sw.issue(wt, (int64_t)k_i * BK, st, w);
    sx.issue(x, (int64_t)k_i * BK, st + TL::OP_B, w);
    ++g_i;
    if (++k_i == nk) {
      k_i = 0;
      ++vt_i;
    }
  };
  issue_next();
  int gs = 0;
  for (int vt = vt0; vt < vt1; ++vt) {
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool nrm = TOP && vt % a.n_tiles == tn;
#pragma unroll
    for (int j = 0; j < JP; ++j) sq[j] = 0.0f;
    for (int kt = 0; kt < nk; ++kt, ++gs) {
      ct_wait_vm<0>();
      ct_barrier();  // stage gs complete; every wave is done with the slot refilled next
      issue_next();
      const char* st = smem + (gs & 1) * 2 * TL::OP_B;
      if constexpr (TOP && OWN_READ) {
        if (nrm) {
#pragma unroll
          for (int j = 0; j < JP; ++j)
            sq[j] = sumsq16<T>(*(const u32x4_t*)(st + 1024 * (w + TL::NWV * j) + 16 * lane), sq[j]);
        }
      }
      u32x4_t fw[2][FJ], fx[2][FI];
      row_frags(st, 16 * FJ * wv, lane, fw);
      row_frags(st + TL::OP_B, nw, lane, fx);
      ct_stage<T>(fw, fx, acc);
      if constexpr (TOP && !OWN_READ) {
        if (nrm) {
#pragma unroll
          for (int q = 0; q < TL::ROW_WV; ++q)
            if (wn == q) {
#pragma unroll
              for (int j = 0; j < JP; ++j) sq[j] = sumsq16<T>(fw[1][q * JP + j], sumsq16<T>(fw[0][q * JP + j], sq[j]));
            }
        }
      }
    }
    if constexpr (TOP) {
      if (nrm) {
#pragma unroll
        for (int j = 0; j < JP; ++j) {
          if constexpr (OWN_READ) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) sq[j] += __shfl_xor(sq[j], o, 64);
          }
          const int v = a.v_base + vt * TL::EDGE +
                        (OWN_READ ? 8 * (w + TL::NWV * j) + (lane >> 3) : 16 * (FJ * wv + wn * JP + j) + rl);
          if (v < v_end && !(a.bias && a.bias[v] <= CT_OUT)) wmx = fmaxf(wmx, sq[j]);  // (a NaN: left out)
        }
      }
    }
    // up to 64 of the wave's items at a time
#pragma unroll
    for (int h = 0; h < FJ / HJ; ++h) {
      const int c0 = vt * TL::EDGE + 16 * FJ * wv + 64 * h, v0 = a.v_base + c0;
      const bool edge = v0 + 16 * HJ > v_end;
      const bool sel = a.bias || edge;
      f32x4 b2[HJ];
      if (sel) {
#pragma unroll
        for (int j = 0; j < HJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int v = v0 + 16 * j + 4 * g + r;
            const float b = v < v_end ? (a.bias ? a.bias[v] : 0.0f) : -__builtin_huge_valf();
            b2[j][r] = b > CT_OUT || b != b ? b * CT_LOG2E : CT_NONE;
          }
      }
      const float s2 = sel ? 1.0f : a.s2;
      float tmx[FI];
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int n = n0 + 16 * i + rl;
        f32x4* z = acc[i] + HJ * h;
        if (sel) {
#pragma unroll
          for (int j = 0; j < HJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)  // (taken out: whatever the product is)
              z[j][r] = b2[j][r] == CT_NONE ? CT_OUT : fmaf(z[j][r], a.s2, b2[j][r]);
        }
        if constexpr (!COEF) {
          float mx = fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3]));
#pragma unroll
          for (int j = 1; j < HJ; ++j)
            mx = fmaxf(fmaxf(fmaxf(z[j][0], z[j][1]), fmaxf(z[j][2], z[j][3])), mx);
          const float tm = fmaxf(mx * s2, CT_OUT);
          if constexpr (TOP) {
            if constexpr (NB >= 4) {
              if (n < a.N && v0 < v_end)
                a.tmax[(int64_t)n * (4 * (((int64_t)a.V + 63) / 64)) + (v0 >> 6) * 4 + g] = tm;
            } else {  // (the tile's 64 items lie in two waves)
              if (wv == 1) half[nw + 16 * i + rl][g] = tm;
              tmx[i] = tm;
            }
          }
          // the maximum is moved only where a logit exceeds it twofold
          if (__any(tm > m[i] + 1.0f)) {
            const float mn = fmaxf(m[i], tm), d = m[i] - mn, sc = __builtin_amdgcn_exp2f(d);
            if constexpr (ENT) TT[i] = sc * fmaf(d, L[i], TT[i]);
            L[i] *= sc;
            m[i] = mn;
          }
#pragma unroll
          for (int j = 0; j < HJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float d = fmaf(z[j][r], s2, -m[i]);
              const float e = __builtin_amdgcn_exp2f(d);
              L[i] += e;
              if constexpr (ENT) TT[i] = fmaf(e, d, TT[i]);
            }
        } else {
          const bool live = rc[i].y != 0.0f || rc[i].z != 0.0f;  // (a lse that is no number: NaN)
          const bool two = NB <= 4 && sizeof(T) == 2 && a.two;
          const bool store = n < (two ? a.N : a.Npad) && c0 < a.ldc;
          T* o = (T*)a.C + (int64_t)n * a.ldc + c0;
          f32x4 c[HJ];
#pragma unroll
          for (int j = 0; j < HJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float lp = fmaf(z[j][r], s2, -rc[i].x);  // log2 p
              const float p = __builtin_amdgcn_exp2f(lp);
              const float k = ENT ? fmaf(rc[i].z, fmaf(lp, CT_LN2, rc[i].w), rc[i].y) : rc[i].y;
              const float q = fmaf(-p, k, id[i] == v0 + 16 * j + 4 * g + r ? (OWN_G ? go[i] : rc[i].y) : 0.0f);
              c[j][r] = live && !(sel && z[j][r] == CT_OUT) ? q : 0.0f;
            }
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < HJ; ++j)
              if (store) *(f32x4*)(o + 16 * j + 4 * g) = c[j];
          } else {
            // v_permlane16_swap pairs two 16-item blocks: 8 consecutive items a lane, 16-byte stores
            auto put = [&](T* row, bool in) __attribute__((always_inline)) {
#pragma unroll
              for (int j = 0; j < HJ; j += 2) {
                const auto s0 = __builtin_amdgcn_permlane16_swap(ct_pack2(c[j][0], c[j][1]),
                                                                 ct_pack2(c[j + 1][0], c[j + 1][1]), false, false);
                const auto s1 = __builtin_amdgcn_permlane16_swap(ct_pack2(c[j][2], c[j][3]),
                                                                 ct_pack2(c[j + 1][2], c[j + 1][3]), false, false);
                if (in)
                  *(u32x4_t*)(row + 16 * j + 16 * (g & 1) + 8 * (g >> 1)) = u32x4_t{s0[0], s1[0], s0[1], s1[1]};
              }
            };
            put(o, store);
            if (two) {  // (rows from N on are 0: they fill C up to Npad)
#pragma unroll
              for (int j = 0; j < HJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  c[j][r] = ct_lost(c[j][r]);
              put(o + (int64_t)a.N * a.ldc, n + a.N < a.Npad && c0 < a.ldc);
            }
          }
        }
      }
      if constexpr (TOP && NB == 2) {
        ct_barrier();
        if (wv == 0) {
#pragma unroll
          for (int i = 0; i < FI; ++i) {
            const int n = n0 + 16 * i + rl;
            if (n < a.N) a.tmax[(int64_t)n * (4 * (((int64_t)a.V + 63) / 64)) + (v0 >> 6) * 4 + g] =
                             fmaxf(tmx[i], half[nw + 16 * i + rl][g]);
          }
        }
      }
    }
  }
  if constexpr (!COEF) {
    ct_barrier();  // the last stage's reads are over: its memory takes the waves' statistics
    float* red = (float*)smem;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m[i], o, 64), L2 = __shfl_xor(L[i], o, 64), T2 = __shfl_xor(TT[i], o, 64);
        stat_join(m[i], L[i], TT[i], m2, L2, T2);
      }
      if (wv == 1 && g == 0) {
        float* r = red + (nw + 16 * i + rl) * 3;
        r[0] = m[i];
        r[1] = L[i];
        r[2] = TT[i];
      }
    }
    if constexpr (TOP) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) wmx = fmaxf(wmx, __shfl_xor(wmx, o, 64));
      if (rl == 0) red[TL::EDGE * 3 + 4 * w + g] = wmx;
    }
    ct_barrier();
    if (TOP && tid == 0) {
      float t = 0.0f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float mq = 0.0f;
#pragma unroll
        for (int i = 0; i < TL::NWV; ++i) mq = fmaxf(mq, red[TL::EDGE * 3 + 4 * i + q]);
        t = OWN_READ ? fmaxf(t, mq) : t + mq;  // (whole norms, or quarters)
      }
      a.wsq[blockIdx.x] = t;
    }
    if (wv == 0 && g == 0) {
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const float* r = red + (nw + 16 * i + rl) * 3;
        stat_join(m[i], L[i], TT[i], r[0], r[1], r[2]);
        const int n = n0 + 16 * i + rl;
        if (n < a.N) a.part[(int64_t)sp * a.N + n] = float4{m[i], L[i], TT[i], 0.0f};
      }
    }
  }
}

// ---- bf16, E = 384, many rows: k_ring.  The rows' vectors stay in registers (3 blocks of 16 rows a
// wave, 8 waves: 384 rows a block; no longer E leaves room for that, and at a shorter one k_logits
// re-reads less), the catalog streams through LDS in tiles of 32 items, SLOTS - 1 tiles ahead, one
// barrier a tile, and the previous tile's exponentials run between this tile's MFMAs.  Bound by the
// two together: 2049 x 100003 with entropy and alternatives 223 us (0.71 PFLOP/s).
constexpr int CR_NT = 512;
template <int KS>
struct RingCfg {
  static constexpr int QB = 3;
  static constexpr int TB = KS * 2048;             // bytes of a tile: 32 rows x KS x 64
  static constexpr int SLOTS = 4;
  static constexpr int PW = KS / 4;                // 1-KB pieces a wave loads of a tile
  static constexpr int ROWS = 128 * QB;
};

template <int KS, bool COEF, bool ENT, bool BIAS>
__global__ __launch_bounds__(CR_NT, 2) void k_ring(const LogitArgs a) {
  using C = RingCfg<KS>;
  constexpr int QB = C::QB, TB = C::TB, SLOTS = C::SLOTS, PW = C::PW;
  constexpr int OPS = PW + (BIAS ? 1 : 0);  // DMA instructions a wave issues per tile
  __shared__ __attribute__((aligned(16))) char smem[SLOTS * TB];
  __shared__ __attribute__((aligned(16))) float sbias[SLOTS + 1][64];
  // the items' norms (with tmax; a tile's by the block of the row tile that its number falls to): every
  // lane the squares of the 16 bytes of a row that it loaded, the largest over all tiles for each place
  // in the row, and the sum of these at the end.  No norm exceeds it (of like vectors it is some 2 times
  // the squares), and no register is held for it, of which there are none to spare.
  __shared__ uint32_t place[4 * KS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, rl = lane & 15;
  const int lb = xcd_remap(blockIdx.x, gridDim.x);
  const int sp = lb / a.n_tiles, tn = lb % a.n_tiles;
  // shares in pairs of tiles (64 items: the groups of 16 that the top alternatives use)
  const int per = (a.v_tiles + a.splits - 1) / a.splits;
  const int v_end = a.v_base + a.v_count;
  const int t0 = 2 * sp * per;
  // (COEF: whole pairs, so that the products' 64-item steps find every coefficient written)
  const int nt = COEF ? 2 * ((a.v_count + 63) / 64) : (a.v_count + 31) / 32;
  const int t1 = t0 + 2 * per < nt ? t0 + 2 * per : nt;
  const int nb = tn * C::ROWS + w * 16 * QB;  // this wave's first row
  const uint16_t* x = (const uint16_t*)a.x;
  const uint16_t* wt = (const uint16_t*)a.w;

  // tile bytes [1024 p, +1024) = 64 chunks of 16 B in row order; row r's chunk c lies at c ^ (r & 15)
  int off[PW], row[PW];
#pragma unroll
  for (int j = 0; j < PW; ++j) {
    const int c = (w + 8 * j) * 64 + lane;
    row[j] = c / (4 * KS);
    off[j] = ((c % (4 * KS)) ^ (row[j] & 15)) * 8;
  }
  auto issue = [&](int t) __attribute__((always_inline)) {
    char* st = smem + (t % SLOTS) * TB;
    const int v0 = a.v_base + 32 * t;
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      int v = v0 + row[j];
      v = v < v_end ? v : v_end - 1;  // past the end: loaded again, never used
      ct_dma(wt + (int64_t)v * a.ldw + off[j], st + 1024 * (w + 8 * j));
    }
    if constexpr (BIAS) {
      int v = v0 + lane;
      v = v < v_end ? v : v_end - 1;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.bias + v),
                                       (__attribute__((address_space(3))) void*)sbias[t % (SLOTS + 1)], 4, 0, 0);
    }
  };
  if constexpr (!COEF) {
    if (tid < 4 * KS) place[tid] = 0u;  // (used after a tile's barrier)
  }
  if (t0 >= t1) {  // (no share is empty)
    if (!COEF && a.tmax && tid == 0) a.wsq[blockIdx.x] = 0.0f;
    return;
  }

  u32x4_t xf[KS][QB];
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    int n = nb + 16 * q + rl;
    n = n < a.N ? n : a.N - 1;
#pragma unroll
    for (int k = 0; k < KS; ++k) xf[k][q] = *(const u32x4_t*)(x + (int64_t)n * a.ldx + 32 * k + 8 * g);
  }
  float m[QB], L[QB], TT[QB], tm[QB];
  float4 rc[QB];
  int id[QB];
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    m[q] = CT_NONE;
    L[q] = TT[q] = 0.0f;
    tm[q] = CT_OUT;
    const int n = nb + 16 * q + rl;
    if constexpr (COEF) {
      rc[q] = n < a.N ? a.rowc[n] : float4{1.0e30f, 0.f, 0.f, 0.f};
      const int64_t i = n < a.N && a.ids ? a.ids[n] : -1;
      id[q] = i >= 0 && i < a.V ? (int)i : -1;
    }
  }
  // the loads above are complete before the first counted wait: the DMA sequence starts clean
  ct_wait_vm<0>();
#pragma unroll
  for (int p = 0; p < SLOTS - 1; ++p)
    if (t0 + p < t1) issue(t0 + p);

  uint32_t fo[4];  // fragment offsets in a tile: chunk (4 k + g) ^ rl, k = 0 .. 3 (+ 256 B every 4)
#pragma unroll
  for (int k = 0; k < 4; ++k) fo[k] = (uint32_t)(rl * KS * 64 + 16 * ((4 * k + g) ^ rl));

  // logits of the previous tile's block (q, rows 16 rb + 4 g ..)
  auto bias4 = [&](int t, int rb) __attribute__((always_inline)) {
    f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (BIAS) {
      const f32x4 raw = *(const f32x4*)(sbias[t % (SLOTS + 1)] + 16 * rb + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) b[r] = raw[r] > CT_OUT || raw[r] != raw[r] ? raw[r] * CT_LOG2E : CT_NONE;
    }
    return b;
  };
  // z: in place of the products; edge: items past the end are taken out
  auto to_z = [&](f32x4 (&acc)[QB][2], int t, bool edge) __attribute__((always_inline)) {
    if (!BIAS && !edge) return;  // (scaled where used)
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const f32x4 b = bias4(t, rb);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool out = (BIAS && b[r] == CT_NONE) || (edge && a.v_base + 32 * t + 16 * rb + 4 * g + r >= v_end);
#pragma unroll
        for (int q = 0; q < QB; ++q) {
          const float z = fmaf(acc[q][rb][r], a.s2, b[r]);
          acc[q][rb][r] = out ? CT_OUT : z;
        }
      }
    }
  };
  // the tile's maximum per row; the running maximum moved where it has to be
  auto head = [&](f32x4 (&acc)[QB][2], int t, float s2) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      const f32x4 &u = acc[q][0], &v = acc[q][1];
      const float mx = fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))) * s2;
      const float zm = fmaxf(mx, CT_OUT);
      if (a.tmax) {
        tm[q] = (t & 1) ? fmaxf(tm[q], zm) : zm;
        const int n = nb + 16 * q + rl;
        if (((t & 1) || t + 1 >= nt) && n < a.N)
          a.tmax[(int64_t)n * (4 * (((int64_t)a.V + 63) / 64)) + (t >> 1) * 4 + g] = tm[q];
      }
      if (__any(zm > m[q] + 1.0f)) {
        const float mn = fmaxf(m[q], zm), d = m[q] - mn, sc = __builtin_amdgcn_exp2f(d);
        if constexpr (ENT) TT[q] = sc * fmaf(d, L[q], TT[q]);
        L[q] *= sc;
        m[q] = mn;
      }
    }
  };
  auto body = [&](const f32x4& v, int q, int rb, int t, float s2, bool zform) __attribute__((always_inline)) {
    if constexpr (!COEF) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float d = fmaf(v[r], s2, -m[q]);
        const float e = __builtin_amdgcn_exp2f(d);
        L[q] += e;
        if constexpr (ENT) TT[q] = fmaf(e, d, TT[q]);
      }
    } else {
      const int n = nb + 16 * q + rl, vi = a.v_base + 32 * t + 16 * rb + 4 * g;
      const bool live = rc[q].y != 0.0f || rc[q].z != 0.0f;
      f32x4 c;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float lp = fmaf(v[r], s2, -rc[q].x);
        const float p = __builtin_amdgcn_exp2f(lp);
        const float k = ENT ? fmaf(rc[q].z, fmaf(lp, CT_LN2, rc[q].w), rc[q].y) : rc[q].y;
        const float o = fmaf(-p, k, id[q] == vi + r ? rc[q].y : 0.0f);
        c[r] = live && !(zform && v[r] == CT_OUT) ? o : 0.0f;
      }
      if (n < a.Npad) ct_store4<uint16_t>((uint16_t*)a.C + (int64_t)n * a.ldc + 32 * t + 16 * rb + 4 * g, c);
    }
  };

  f32x4 A[QB][2], B[QB][2];
  // tile t into cur, with the previous tile's epilogue between its steps
  auto tile = [&](int t, f32x4 (&cur)[QB][2], f32x4 (&prev)[QB][2], bool has_prev) __attribute__((always_inline)) {
    if (t + SLOTS - 1 <= t1) ct_wait_vm<(SLOTS - 2) * OPS>();
    else ct_wait_vm<0>();
    ct_barrier();  // tile t is complete; every wave is done with the slot refilled next
    if (t + SLOTS - 1 < t1) issue(t + SLOTS - 1);
    const char* st = smem + (t % SLOTS) * TB;
    if constexpr (!COEF) {
      if (a.tmax && t % a.n_tiles == tn) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
        for (int j = 0; j < PW; ++j) {
          const float q = sumsq16<uint16_t>(*(const u32x4_t*)(st + 1024 * (w + 8 * j) + 16 * lane), 0.0f);
          const int c = (w + 8 * j) * 64 + lane, r = c / (4 * KS);
          if (a.v_base + 32 * t + r < v_end && !(BIAS && sbias[t % (SLOTS + 1)][r] <= CT_OUT))
            atomicMax(&place[(c % (4 * KS)) ^ (r & 15)], __float_as_uint(fmaxf(q, 0.0f)));  // (a NaN: left out)
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const bool edge = COEF && has_prev && a.v_base + 32 * t > v_end;  // (the previous tile's)
    float s2 = a.s2;
    if (has_prev) {
      to_z(prev, t - 1, edge);
      if (BIAS || edge) s2 = 1.0f;
      if constexpr (!COEF) head(prev, t - 1, s2);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) cur[q][rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      u32x4_t f[2];
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
        f[rb] = *(const u32x4_t*)(st + fo[k & 3] + (k >> 2) * 256 + rb * 16 * KS * 64);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int q = 0; q < QB; ++q)
          cur[q][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ct_bf16x8, f[rb]),
                                                               __builtin_bit_cast(ct_bf16x8, xf[k][q]), cur[q][rb], 0, 0, 0);
      if (has_prev) {  // the 2 QB blocks of the epilogue spread over the KS steps
#pragma unroll
        for (int e = 0; e < 2 * QB; ++e)
          if (e * KS / (2 * QB) == k) body(prev[e >> 1][e & 1], e >> 1, e & 1, t - 1, s2, BIAS || edge);
      }
    }
  };
  tile(t0, A, B, false);
  int t = t0 + 1;
  for (; t + 1 < t1; t += 2) {
    tile(t, B, A, true);
    tile(t + 1, A, B, true);
  }
  auto finish = [&](f32x4 (&acc)[QB][2]) __attribute__((always_inline)) {  // the last tile's epilogue
    const bool edge = a.v_base + 32 * t1 > v_end;
    to_z(acc, t1 - 1, edge);
    const float s2 = BIAS || edge ? 1.0f : a.s2;
    if constexpr (!COEF) head(acc, t1 - 1, s2);
#pragma unroll
    for (int e = 0; e < 2 * QB; ++e) body(acc[e >> 1][e & 1], e >> 1, e & 1, t1 - 1, s2, BIAS || edge);
  };
  if (t < t1) {
    tile(t, B, A, true);
    finish(B);
  } else {
    finish(A);
  }
  if constexpr (!COEF) {
    if (a.tmax) {
      ct_barrier();
      if (tid == 0) {
        float t = 0.0f;
        for (int i = 0; i < 4 * KS; ++i) t += __uint_as_float(place[i]);
        a.wsq[blockIdx.x] = t;
      }
    }
    // a row's four lanes
#pragma unroll
    for (int q = 0; q < QB; ++q) {
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m[q], o, 64), L2 = __shfl_xor(L[q], o, 64), T2 = __shfl_xor(TT[q], o, 64);
        stat_join(m[q], L[q], TT[q], m2, L2, T2);
      }
      const int n = nb + 16 * q + rl;
      if (g == 0 && n < a.N) a.part[(int64_t)sp * a.N + n] = float4{m[q], L[q], TT[q], 0.0f};
    }
  }
}

template <typename T>
__device__ __forceinline__ float ct_elt(const T* p, int64_t i) {
  if constexpr (sizeof(T) == 4) return p[i];
  else return __uint_as_float((uint32_t)p[i] << 16);
}
// 16 bytes of x and w -> sum of products in 64 bits
template <typename T>
__device__ __forceinline__ double dot16(const u32x4_t& a, const u32x4_t& b, double d) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      d = fma((double)__uint_as_float(a[i]), (double)__uint_as_float(b[i]), d);
    } else {
      d = fma((double)__uint_as_float(a[i] << 16), (double)__uint_as_float(b[i] << 16), d);
      d = fma((double)__uint_as_float(a[i] & 0xffff0000u), (double)__uint_as_float(b[i] & 0xffff0000u), d);
    }
  }
  return d;
}

// x . w in 64 bits (E a multiple of 64, rows 16-byte aligned)
template <typename T>
__device__ __forceinline__ double wave_dot64(const T* x, const T* w, int E, int lane) {
  constexpr int PC = 16 / (int)sizeof(T);
  double d = 0.0;
  for (int e = lane * PC; e < E; e += 64 * PC) d = dot16<T>(*(const u32x4_t*)(x + e), *(const u32x4_t*)(w + e), d);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
  return d;
}

// x . w as k_logits and k_ring form it, to the bit: the same instructions in the same order (every
// row and column of the block is the same); Q stages' loads on their way
template <typename T, int Q>
__device__ __forceinline__ float mfma_dot(const T* x, const T* w, int E, int lane) {
  const int g = lane >> 4;
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  constexpr int BK = 128 / (int)sizeof(T), PC = 16 / (int)sizeof(T);
  for (int k0 = 0; k0 < E; k0 += Q * BK) {
    u32x4_t fw[Q][2][1], fx[Q][2][1];
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = (k0 + q * BK < E ? k0 + q * BK : k0) + PC * (4 * s + g);
        fw[q][s][0] = *(const u32x4_t*)(w + k);
        fx[q][s][0] = *(const u32x4_t*)(x + k);
      }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (k0 + q * BK < E) ct_stage<T>(fw[q], fx[q], acc);
  }
  return acc[0][0][0];
}
// What the statistics' sums change by when one item's logit z (as they have it) is put right: dz =
// exact - z, in powers of two, d = z - m.  log p of an item that has nearly all the probability is a
// difference of two logits that both hold its own: they have to be the same one (4 x 50 x 768, p next to
// 1: log p 2.9e-5 -> 1.1e-6 of itself off; 3 - 7 us of latency a call).  Below a sixteenth of the probability
// it is left out: the other items' logits are off by as much, with fifteen times its weight.
__device__ __forceinline__ void put_right(double dz, double d, double& L, double& TT) {
  const double e = exp2(d);
  if (!(fabs(dz) < 0.125) || !(16.0 * e > L)) return;  // (not finite, or of little weight)
  const double q = e * expm1(dz * 0.6931471805599453);
  TT += q * (d + dz) + e * dz;
  L += q;
}

// log p is at most 0: what rounding puts above is 0 (a NaN stays)
__device__ __forceinline__ float at_most_0(float v) { return v > 0.0f ? 0.0f : v; }

// What a row's 32-bit logits (in powers of two) are off by at most, 4 u |z| besides: every one of the
// E products and sums (and the few operations after them) rounds or cuts off at most 2^-23 of sum |x_e
// w_e| <= |x| |w|, whatever the order; elements, products and sums below the least normal number may
// count as 0.  xsq, wsq: squares in f32, off by less than 1 in 100; those that the squaring loses are
// of elements below 2^-63.
__device__ __forceinline__ float logit_error(float s2, int E, float xsq, float wsq) {
  const float r = sqrtf((float)E), tiny = 1.2e-19f * r;
  const float X = 1.01f * sqrtf(xsq) + tiny, W = 1.01f * sqrtf(wsq) + tiny;
  return s2 * (X * W) * ((float)(E + 24) * 1.2e-7f) + s2 * (1.2e-38f * (float)E) * (2.0f + X + W);
}

struct CombineArgs {
  const float4* part;
  int splits, N, V, E;
  const void *x, *w;
  int64_t ldx, ldw;
  const int64_t* ids;
  const float* bias;
  double s;
  float s2;   // log2(e) s, as the statistics' kernel has it
  int group;  // items of a wave there: a group that ends past V has its logits rounded on their own
  float *logp, *ent;
  double* lse;
  const float* wsq;  // with alternatives: [n_wsq] of the statistics' blocks
  int n_wsq;
  float* err;        // [N] logit_error
  float2* stat;      // [N] m, L
};
// An item's logit as the statistics have it, from its product in 32 bits.
__device__ __forceinline__ double stat_logit(float dot32, float s2, bool bias, float b, int v, int group, int V) {
  const bool own = bias || (v / group + 1) * group > V;
  return own ? (double)fmaf(dot32, s2, b * CT_LOG2E) : (double)dot32 * (double)s2;
}
// log p = l - lse (natural; m and log2 of the sum in powers of two)
__device__ __forceinline__ float log_p(double l, double m, double l2) {
  return at_most_0((float)(l - (m + l2) * 0.6931471805599453));
}
// One wave per row: the shares' statistics joined, the given item's logit.
template <typename T>
__device__ __forceinline__ void combine_row(const CombineArgs& a, int64_t n, int lane) {
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;
  const float4* part = a.part;
  const int splits = a.splits, N = a.N, V = a.V, E = a.E;
  const int64_t ldx = a.ldx, ldw = a.ldw;
  const int64_t* ids = a.ids;
  const float* bias = a.bias;
  const double s = a.s;
  float *logp = a.logp, *ent = a.ent;
  float m = CT_NONE, L = 0.0f, TT = 0.0f;
  const int64_t id = logp ? ids[n] : -1;
  const bool has = id >= 0 && id < V;
  const float b = has && bias ? bias[id] : 0.0f;
  const double dot = has ? wave_dot64(x + n * ldx, w + id * ldw, E, lane) : 0.0;
  const float dot32 = has ? mfma_dot<T, 4>(x + n * ldx, w + id * ldw, E, lane) : 0.0f;
  for (int i0 = lane; i0 < splits; i0 += 256) {  // 4 loads on their way
    float4 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = i0 + 64 * i < splits ? part[(int64_t)(i0 + 64 * i) * N + n] : float4{CT_NONE, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) stat_join(m, L, TT, p[i].x, p[i].y, p[i].z);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(m, o, 64), L2 = __shfl_xor(L, o, 64), T2 = __shfl_xor(TT, o, 64);
    stat_join(m, L, TT, m2, L2, T2);
  }
  if (a.err) {
    float xsq = 0.0f, wsq = 0.0f;
    constexpr int PC = 16 / (int)sizeof(T);
    for (int e = lane * PC; e < E; e += 64 * PC) xsq = sumsq16<T>(*(const u32x4_t*)(x + n * ldx + e), xsq);
    for (int i = lane; i < a.n_wsq; i += 64) wsq = fmaxf(wsq, a.wsq[i]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      xsq += __shfl_xor(xsq, o, 64);
      wsq = fmaxf(wsq, __shfl_xor(wsq, o, 64));
    }
    if (lane == 0) {
      a.err[n] = logit_error(a.s2, E, xsq, wsq);
      a.stat[n] = float2{m, L};
    }
  }
  const float inf = __builtin_huge_valf();
  const bool empty = m <= CT_OUT && L == L;  // every item taken out (and no NaN)
  const double ls = ((double)m + log2((double)L)) * 0.6931471805599453;
  const double l = s * dot + (double)b;
  double L2 = (double)L, T2 = (double)TT;
  if (has && !(b <= CT_OUT)) {
    const double z = stat_logit(dot32, a.s2, bias != nullptr, b, (int)id, a.group, V);
    put_right(l * 1.4426950408889634 - z, z - (double)m, L2, T2);
  }
  const double l2 = log2(L2);
  if (logp) {
    const float o = !has ? 0.0f : empty || b <= CT_OUT ? -inf
                    : log_p(l, (double)m, l2);
    if (lane == 0) logp[n] = o;
  }
  if (lane == 0) {
    const float h = (float)((l2 - T2 / L2) * 0.6931471805599453);
    if (ent) ent[n] = empty || h < 0.0f ? 0.0f : h;
    a.lse[n] = empty ? -(double)inf : ls;
  }
}
template <typename T>
__global__ __launch_bounds__(256) void k_combine(const CombineArgs a) {
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n < a.N) combine_row<T>(a, n, threadIdx.x & 63);
}

// ------------------------------------------------------------------- top alternatives
// The keep largest keys (unique, above 0) of a wave's 64 x PER, written to out[0 .. count) in no
// order; returns the count (uniform).  The keep-th largest high word is built bit by bit (32 rounds of
// ballots: scalar work), ties at it by the same search over the low words.
template <int PER>
__device__ __forceinline__ int wave_select(const uint64_t (&key)[PER], int keep, uint64_t* out, int lane) {
  int total = 0;
#pragma unroll
  for (int r = 0; r < PER; ++r) total += __popcll(__ballot(key[r] != 0ull));
  uint32_t x = 0u, xl = 0u;  // taken: high > x, or high == x and low >= xl
  if (total > keep) {
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = x | (1u << bit);
      int c = 0;
#pragma unroll
      for (int r = 0; r < PER; ++r) c += __popcll(__ballot((uint32_t)(key[r] >> 32) >= cand));
      if (c >= keep) x = cand;
    }
    int gt = 0, eq = 0;
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      gt += __popcll(__ballot((uint32_t)(key[r] >> 32) > x));
      eq += __popcll(__ballot((uint32_t)(key[r] >> 32) == x && key[r] != 0ull));
    }
    if (eq > keep - gt) {
#pragma unroll 1
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = xl | (1u << bit);
        int c = 0;
#pragma unroll
        for (int r = 0; r < PER; ++r)
          c += __popcll(__ballot((uint32_t)(key[r] >> 32) == x && (uint32_t)key[r] >= cand));
        if (c >= keep - gt) xl = cand;
      }
    }
  }
  int base = 0;
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const uint32_t h = (uint32_t)(key[r] >> 32);
    const bool sel = key[r] != 0ull && (h > x || (h == x && (uint32_t)key[r] >= xl));
    const uint64_t bm = __ballot(sel);
    const int pos = base + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bm >> 32),
                                                          __builtin_amdgcn_mbcnt_lo((uint32_t)bm, 0u));
    if (sel && pos < keep) out[pos] = key[r];
    base += __popcll(bm);
  }
  return base < keep ? base : keep;
}

// how many of n keys in LDS are above `mine` (n even; every lane reads the same two at a time)
__device__ __forceinline__ int key_rank(const uint64_t* keys, int n, uint64_t mine) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  int r = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const u64x2 k = *(const u64x2*)(keys + i);
    r += (k[0] > mine ? 1 : 0) + (k[1] > mine ? 1 : 0);
  }
  return r;
}

// Groups of 16 items (tmax entries) of one row: the keep largest of every segment, key = (maximum,
// ~group).  The launch's last blocks join the statistics (k_combine's work, which nothing here waits
// for: one launch less).  Block = (segment, row): each of its 4 waves keeps the best of its 1024 entries at a
// time, with those it has; of the four lists every key's rank is counted.  Unused places are 0.
template <typename T>
__global__ __launch_bounds__(256) void k_top_groups(const float* __restrict__ tmax, int64_t M, int seg_len,
                                                    int nseg, int keep, uint64_t* __restrict__ out,
                                                    unsigned n_seg_blocks, const CombineArgs ca,
                                                    uint32_t* __restrict__ n_rows) {
  __shared__ uint64_t red[4][64];
  __shared__ __attribute__((aligned(16))) uint64_t all[258];
  __shared__ uint64_t fin[64];
  __shared__ int cnt[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (n_rows && blockIdx.x == 0 && threadIdx.x == 0) *n_rows = 0u;  // (for the next kernel)
  if (blockIdx.x >= n_seg_blocks) {
    const int64_t r = (int64_t)(blockIdx.x - n_seg_blocks) * 4 + w;
    if (r < ca.N) combine_row<T>(ca, r, lane);
    return;
  }
  const int64_t n = blockIdx.x / nseg;
  const int sg = (int)(blockIdx.x % nseg);
  const int64_t i0 = (int64_t)sg * seg_len, i1 = i0 + seg_len < M ? i0 + seg_len : M;
  const float* row = tmax + n * M;
  int have = 0;
  for (int64_t b = i0 + w * 1024; b < i1; b += 4096) {
    uint64_t key[17];
    key[16] = lane < have ? red[w][lane] : 0ull;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t e = b + i * 64 + lane;
      key[i] = e < i1 ? make_key(row[e], (uint32_t)e) : 0ull;
    }
    wave_sync();
    // a bound first: of the largest keys of the lanes' halves the keep-th largest (the upper 20 bits:
    // 2^-11 of it), which at least keep keys reach; few others do
    uint64_t l0 = key[0], l1 = key[8];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      l0 = key[i] > l0 ? key[i] : l0;
      l1 = key[8 + i] > l1 ? key[8 + i] : l1;
    }
    l1 = key[16] > l1 ? key[16] : l1;
    const uint32_t h0 = (uint32_t)(l0 >> 32), h1 = (uint32_t)(l1 >> 32);
    uint32_t bound = 0u;
#pragma unroll 1
    for (int bit = 30; bit >= 12; bit -= 2) {
      int k = 0;
#pragma unroll
      for (uint32_t q = 1; q < 4; ++q) {
        const uint32_t cand = bound | (q << bit);
        k += __popcll(__ballot(h0 >= cand)) + __popcll(__ballot(h1 >= cand)) >= keep;
      }
      bound |= (uint32_t)k << bit;
    }
    int c = 0;
#pragma unroll
    for (int i = 0; i < 17; ++i) {
      const bool in = key[i] != 0ull && (uint32_t)(key[i] >> 32) >= bound;
      const uint64_t bm = __ballot(in);
      const int pos = c + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bm >> 32),
                                                         __builtin_amdgcn_mbcnt_lo((uint32_t)bm, 0u));
      if (in && pos < 64) red[w][pos] = key[i];
      c += __popcll(bm);
    }
    wave_sync();
    if (c <= 64) {
      have = c;  // (some more than keep: sorted out at the end)
    } else {  // (many equal maxima)
      have = wave_select<17>(key, keep, red[w], lane);
    }
    wave_sync();
  }
  if (lane == 0) cnt[w] = have;
  if (threadIdx.x < 64) fin[threadIdx.x] = 0ull;
  __syncthreads();
  int base = 0, nk = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    base += i < w ? cnt[i] : 0;
    nk += cnt[i];
  }
  if (lane < have) all[base + lane] = red[w][lane];
  if (threadIdx.x == 0) all[nk] = 0ull;
  __syncthreads();
  if ((int)threadIdx.x < nk) {
    const uint64_t mine = all[threadIdx.x];
    const int r = key_rank(all, (nk + 1) & ~1, mine);
    if (r < keep) fin[r] = mine;
  }
  __syncthreads();
  if (w == 0 && lane < keep) out[(n * nseg + sg) * keep + lane] = fin[lane];
}

struct TopEntry {
  double l;
  int64_t v;
};
struct TopArgs {
  const uint64_t* segs;
  int nseg, keep, top;
  const void *x, *w;
  int64_t ldx, ldw;
  int N, E, V;
  const float* bias;
  double s;
  float s2;
  int group;  // as in CombineArgs
  const float* err;
  const float2* stat;
  int64_t* ids_out;
  float* lp_out;
  // the second search: n_rows rows [N] of it, in parts of part_len groups
  const float* tmax;
  int64_t M;
  int parts, part_len;
  uint32_t *n_rows, *rows;
  float* floor;     // [N] of the groups' maxima
  TopEntry* kth;    // [N] the top-th item of the groups kept: a later one is none of the top
  uint32_t* done;   // [N] parts that are searched
  TopEntry* found;  // [N, parts, top]
};
constexpr int CT_GROUPS = CT_TOP_MAX + CT_TOP_EXTRA;  // groups scored at a time
struct TopList {
  double l[CT_GROUPS * 16 + CT_TOP_MAX];  // candidates, in any order (ranks do not depend on it)
  int v[CT_GROUPS * 16 + CT_TOP_MAX];
  double bl[CT_TOP_MAX];  // the best of them, the first first
  int bv[CT_TOP_MAX];
  int n;
};

// after k in the order (score, lower id)
__device__ __forceinline__ bool top_after(const TopEntry& k, double l, int v) {
  return l < k.l || (l == k.l && v > (int)k.v);
}
// The items of n_grp groups, scored in 64 bits (16 lanes an item, 16-byte loads, NT / 4 items in
// flight); those not below cut (powers of two) and not after kth join the list.
template <typename T, int NT>
__device__ __forceinline__ void top_score(const TopArgs& a, const T* xr, const uint32_t* grp, int n_grp, double cut,
                                          const TopEntry& kth, TopList& o) {
  constexpr int PC = 16 / (int)sizeof(T), NG = NT / 16;
  const T* w = (const T*)a.w;
  const int sub = threadIdx.x >> 4, l16 = threadIdx.x & 15, cand = n_grp * 16, V = a.V, E = a.E;
  for (int i0 = sub; i0 < cand; i0 += 4 * NG) {
    int v[4];
    double d[4];
    const T* wr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i0 + i * NG < cand ? i0 + i * NG : i0, it = c & 15;
      const uint32_t q = grp[c >> 4];
      v[i] = (int)(q >> 2) * 64 + 16 * (it >> 2) + 4 * (int)(q & 3) + (it & 3);
      wr[i] = w + (int64_t)(v[i] < V ? v[i] : V - 1) * a.ldw;
      d[i] = 0.0;
    }
#pragma unroll 2
    for (int e = l16 * PC; e < E; e += 16 * PC) {
      const u32x4_t xv = *(const u32x4_t*)(xr + e);
      u32x4_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = *(const u32x4_t*)(wr[i] + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = dot16<T>(xv, y[i], d[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int m = 1; m < 16; m <<= 1) d[i] += __shfl_xor(d[i], m, 64);
      if (l16 == 0 && i0 + i * NG < cand && v[i] < V) {
        const float b = a.bias ? a.bias[v[i]] : 0.0f;
        const double l = b <= CT_OUT ? -__builtin_huge_val() : a.s * d[i] + (double)b;
        // (-inf, NaN: only where the cut lets them)
        if (!(l * 1.4426950408889634 < cut) && !top_after(kth, l, v[i])) {
          const int k = atomicAdd(&o.n, 1);
          o.l[k] = l;
          o.v[k] = v[i];
        }
      }
    }
  }
}
// The best of the list, by (score, lower id); NaN scores by id among themselves, below all others.
template <int NT>
__device__ __forceinline__ void top_rank(TopList& o, int top) {
  const int m = o.n;
  for (int i = threadIdx.x; i < m; i += NT) {
    const double l = o.l[i];
    const int v = o.v[i];
    int rank = 0;
    for (int q = 0; q < m; ++q) {
      const double t = o.l[q];
      const bool gt = t > l || (l != l && t == t);
      const bool eq = t == l || (t != t && l != l);
      rank += gt || (eq && o.v[q] < v) ? 1 : 0;
    }
    if (rank < top) {
      o.bl[rank] = l;
      o.bv[rank] = v;
    }
  }
}
// A wave an alternative: the value that log_prob has for it, its own part of the sums put right too.
template <typename T, int NT>
__device__ __forceinline__ void top_write(const TopArgs& a, const TopList& o, int64_t n) {
  const int lane = threadIdx.x & 63;
  const float2 st = a.stat[n];
  const double m = (double)st.x, l20 = log2((double)st.y);
  for (int i = threadIdx.x >> 6; i < a.top; i += NT / 64) {
    const double l = o.bl[i];
    const int v = __builtin_amdgcn_readfirstlane(o.bv[i]);
    double L2 = (double)st.y, T2 = 0.0, l2 = l20;
    if (l * 1.4426950408889634 - m > l20 - 4.25) {  // (else put_right leaves it)
      const float dot32 = mfma_dot<T, 1>((const T*)a.x + n * a.ldx, (const T*)a.w + (int64_t)v * a.ldw, a.E, lane);
      const double z = stat_logit(dot32, a.s2, a.bias != nullptr, a.bias ? a.bias[v] : 0.0f, v, a.group, a.V);
      put_right(l * 1.4426950408889634 - z, z - m, L2, T2);
      l2 = log2(L2);
    }
    if (lane == 0) {
      a.ids_out[n * a.top + i] = v;
      a.lp_out[n * a.top + i] = l == -__builtin_huge_val() ? -__builtin_huge_valf() : log_p(l, m, l2);
    }
  }
}

// One block per row: the keep largest groups of all segments, their items scored in 64 bits, the top of
// them by (score, lower id).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_top_items(const TopArgs a) {
  constexpr int NW = NT / 64;
  __shared__ __attribute__((aligned(16))) uint64_t red[NW][64];
  __shared__ uint64_t fin[64];
  __shared__ uint32_t grp[64];
  __shared__ int s_groups;
  __shared__ float s_floor;
  __shared__ TopList o;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, keep = a.keep, top = a.top;
  const int64_t n = blockIdx.x;
  const int total = a.nseg * keep;
  const uint64_t* src = a.segs + n * total;
  if (total <= NT) {
    red[wv][lane] = tid < total ? src[tid] : 0ull;
  } else {
    int have = 0;
    for (int b = wv * 256; b < total; b += NW * 256) {
      uint64_t key[5];
      key[4] = lane < have ? red[wv][lane] : 0ull;
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i] = b + i * 64 + lane < total ? src[b + i * 64 + lane] : 0ull;
      wave_sync();
      have = wave_select<5>(key, keep, red[wv], lane);
      wave_sync();
    }
    if (lane >= have) red[wv][lane] = 0ull;
  }
  if (tid < 64) fin[tid] = 0ull;
  __syncthreads();
  {
    const int used = total <= NT ? (total + 1) & ~1 : NT;
    if (wv * 64 < used) {
      const uint64_t mine = red[wv][lane];
      const int r = key_rank(&red[0][0], used, mine);
      if (mine != 0ull && r < keep) fin[r] = mine;
    }
  }
  __syncthreads();
  const float e0 = a.err[n];
  const T* xr = (const T*)a.x + n * a.ldx;
  bool more = false;  // (wave 0) groups that were not taken may hold some of the top
  for (bool all = false;; all = true) {
    if (wv == 0) {
      const uint64_t k1 = lane < keep ? fin[lane] : 0ull;
      // the top-th largest maximum: top groups hold an item each that is not below it in 32 bits, so the
      // top-th largest exact logit is not below it by more than a 32-bit logit is off.  A group whose
      // maximum is clearly below that holds none of the top, nor is one of the top below it in 64 bits.
      const uint64_t last = fin[top - 1], end = fin[keep - 1];
      const float kth = key_score(last);
      float fl = kth - (2.01f * e0 + 2.0e-6f * fabsf(kth));
      // (fewer than top groups, taken-out items among the top, values past 32 bits or not numbers, or
      // fewer than top items found: every item of the groups kept takes part)
      const bool few = last == 0ull || kth < 0.9f * CT_OUT;
      if (all || few || !(fabsf(fl) < 3.0e38f)) fl = -__builtin_huge_valf();
      // (few: the groups kept are all that hold anything, and those of the lowest ids besides)
      more = end != 0ull && !few && e0 == e0 && !(key_score(end) < fl);
      const bool use = k1 != 0ull && !(key_score(k1) < fl);
      const uint64_t bm = __ballot(use);
      if (use) grp[__popcll(bm & ((1ull << lane) - 1))] = key_row(k1);
      if (lane == 0) {
        s_groups = __popcll(bm);
        s_floor = fl;
        o.n = 0;
      }
    }
    __syncthreads();
    top_score<T, NT>(a, xr, grp, s_groups, (double)s_floor, TopEntry{-__builtin_huge_val(), 0x7fffffff}, o);
    __syncthreads();
    // (a second round only where sums in 32 bits went past their range: all the groups kept hold at
    // least top items)
    if (all || o.n >= top) break;
    __syncthreads();
  }
  top_rank<NT>(o, top);
  __syncthreads();
  top_write<T, NT>(a, o, n);
  if (a.n_rows && tid == 0 && more) {
    a.floor[n] = s_floor;
    a.kth[n] = TopEntry{o.bl[top - 1], o.bv[top - 1]};
    a.done[n] = 0u;
    a.rows[atomicAdd(a.n_rows, 1u)] = (uint32_t)n;
  }
}

// The second search: rows whose groups above the floor were more than are kept.  Block = (row, part): the
// part's groups above the floor, 40 at a time, are scored in 64 bits, the best of them kept; the row's
// last block joins the parts (no block waits for another).  Without such rows 3 us.
template <typename T>
__global__ __launch_bounds__(256) void k_top_wide(const TopArgs a) {
  __shared__ TopList o;
  __shared__ uint32_t pend[256];
  __shared__ int n_pend, s_last;
  const int tid = threadIdx.x, top = a.top;
  TopEntry kth;
  auto carry = [&]() __attribute__((always_inline)) {  // the list becomes its best
    __syncthreads();
    top_rank<256>(o, top);
    __syncthreads();
    const int k = o.n < top ? o.n : top;
    if (tid < k) {
      o.l[tid] = o.bl[tid];
      o.v[tid] = o.bv[tid];
    }
    __syncthreads();
    if (tid == 0) o.n = k;
    __syncthreads();
    if (o.n == top && !top_after(kth, o.l[top - 1], o.v[top - 1])) kth = TopEntry{o.l[top - 1], o.v[top - 1]};
  };
  const int64_t units = (int64_t)*a.n_rows * a.parts;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t n = a.rows[u / a.parts];
    const int part = (int)(u % a.parts);
    const T* xr = (const T*)a.x + n * a.ldx;
    const float* row = a.tmax + n * a.M;
    const float floor = a.floor[n];
    const int64_t i0 = (int64_t)part * a.part_len, i1 = i0 + a.part_len < a.M ? i0 + a.part_len : a.M;
    const TopEntry kth0 = a.kth[n];
    kth = kth0;
    if (tid == 0) o.n = 0;
    for (int64_t b = i0; b < i1; b += 256) {
      if (tid == 0) n_pend = 0;
      __syncthreads();
      const int64_t e = b + tid;
      if (e < i1 && !(row[e] < floor)) pend[atomicAdd(&n_pend, 1)] = (uint32_t)e;
      __syncthreads();
      const int np = n_pend;
      for (int p = 0; p < np; p += CT_GROUPS) {
        top_score<T, 256>(a, xr, pend + p, np - p < CT_GROUPS ? np - p : CT_GROUPS, (double)floor, kth, o);
        carry();
      }
      __syncthreads();
    }
    __syncthreads();
    TopEntry* f = a.found + n * a.parts * top;
    if (tid < top) f[part * top + tid] = tid < o.n ? TopEntry{o.l[tid], o.v[tid]} : TopEntry{0.0, -1};
    __threadfence();  // visible before the block counts itself in
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(&a.done[n], 1u) == (uint32_t)a.parts - 1u;
    __syncthreads();
    if (s_last) {
      __threadfence();
      const int total = a.parts * top;
      kth = kth0;
      if (tid == 0) o.n = 0;
      __syncthreads();
      for (int b = 0; b < total; b += 512) {
        for (int i = b + tid; i < total && i < b + 512; i += 256) {
          const TopEntry q = f[i];
          if (q.v >= 0 && !top_after(kth, q.l, (int)q.v)) {
            const int k = atomicAdd(&o.n, 1);
            o.l[k] = q.l;
            o.v[k] = (int)q.v;
          }
        }
        carry();
      }
      if (o.n == top) top_write<T, 256>(a, o, n);  // (always: what the first search found is among it)
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------- backward
// Row constants, x with its dead rows (no gradient, or nothing to choose from) set to zero (two: once
// more, for the second rows of C).
template <typename T>
__global__ __launch_bounds__(256) void k_rows(const T* __restrict__ x, int64_t ldx, int N, int E,
                                              const double* __restrict__ lse, const float* __restrict__ ent,
                                              const float* __restrict__ g, const float* __restrict__ e,
                                              const int64_t* __restrict__ ids, int V,
                                              float4* __restrict__ rowc, float* __restrict__ rowg,
                                              T* __restrict__ xo, bool two) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  const int64_t id = ids ? ids[n] : -1;
  const float gn = g && id >= 0 && id < V ? g[n] : 0.0f, en = e ? e[n] : 0.0f;
  const bool live = (gn != 0.0f || en != 0.0f) && !(lse[n] == -__builtin_huge_val());
  if (lane == 0) {
    // a coefficient is g [v = id] - p k: with lse rounded to 32 bits p would be off by up to 2^-25 |lse| of
    // itself, which next to 1 is most of 1 - p.  What is lost of it goes into the factors.
    const double z = lse[n] * 1.4426950408889634, lo = z - (double)(float)z, f = exp2(-lo);
    rowc[n] = live ? float4{(float)z, (float)((double)gn * f), (float)((double)en * f),
                            (float)((ent ? (double)ent[n] : 0.0) - lo * 0.6931471805599453)}
                   : float4{1.0e30f, 0.f, 0.f, 0.f};
    rowg[n] = live ? gn : 0.0f;
  }
  constexpr int PC = 16 / (int)sizeof(T);
  for (int c = lane * PC; c < E; c += 64 * PC)
  {
    const u32x4_t v = live ? *(const u32x4_t*)(x + n * ldx + c) : u32x4_t{0, 0, 0, 0};
    *(u32x4_t*)(xo + n * E + c) = v;
    if (two) *(u32x4_t*)(xo + (n + N) * E + c) = v;
  }
}
// w with the rows of items that are taken out set to zero (they may hold anything)
template <typename T>
__global__ __launch_bounds__(256) void k_items(const T* __restrict__ w, int64_t ldw, int V, int E,
                                               const float* __restrict__ bias, T* __restrict__ wo) {
  constexpr int PC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < V; v += (int64_t)gridDim.x * 4) {
    const bool out = bias[v] <= CT_OUT;
    for (int c = lane * PC; c < E; c += 64 * PC)
      *(u32x4_t*)(wo + v * E + c) = out ? u32x4_t{0, 0, 0, 0} : *(const u32x4_t*)(w + v * ldw + c);
  }
}

// What the rounding of the given items' coefficients to bf16 left of them (the items of this chunk of C):
// the coefficient once more, in f32, from the same 32-bit logit that the row's lse holds, less what C has.
// A wave a row.
__global__ __launch_bounds__(256) void k_lost(const LogitArgs a, float* __restrict__ delta) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= a.N) return;
  const int64_t id = a.ids[n];
  if (id < a.v_base || id >= a.v_base + a.v_count) return;  // (read by the products for this chunk's items alone)
  const float4 rc = a.rowc[n];
  const float b = a.bias ? a.bias[id] : 0.0f;
  float d = 0.0f;
  if (rc.y != 0.0f && !(b <= CT_OUT)) {
    const float z = mfma_dot<uint16_t, 4>((const uint16_t*)a.x + (int64_t)n * a.ldx,
                                          (const uint16_t*)a.w + id * a.ldw, a.E, lane);
    const float lp = a.bias ? fmaf(z, a.s2, b * CT_LOG2E) - rc.x : fmaf(z, a.s2, -rc.x);
    const float k = rc.z != 0.0f ? fmaf(rc.z, fmaf(lp, CT_LN2, rc.w), rc.y) : rc.y;
    const float c = fmaf(-__builtin_amdgcn_exp2f(lp), k, a.rowg[n]);
    d = c - __uint_as_float((uint32_t)((const uint16_t*)a.C)[(int64_t)n * a.ldc + (id - a.v_base)] << 16);
  }
  if (lane == 0) delta[n] = d;
}

// out[m][c] = scale sum_k A[m, k] B[k, c]; B [K rows, cols] as it lies; A rows [m][k] (ACOL false) or
// as it lies [k][m] (ACOL).  K a multiple of BK (rows past a's or b's end are zero in A).  Tiles whose
// sums are split (or all, acc: added to what is there) write f32 partial sums, a square of the tile's
// edge a block; the others write out.
struct ProductArgs {
  const void *A, *B;
  int64_t lda, ldb, a_rows, b_rows;
  int M, cols, K;
  int whole, splits;  // tiles from `whole` on have their sums split over that many blocks
  bool all, acc;      // all: also the whole tiles go to part; acc: part is added to
  float scale;
  void* out;
  int64_t ldo;
  float* part;        // [block from the first that writes here, tile edge^2]
  // bf16, or null: what the given items' coefficients of A lost by their rounding ([rows], items ids),
  // v_base the first item of A; the sums begin with it
  const float* delta;
  const int64_t* ids;
  int v_base;
};
__device__ __forceinline__ f32x4 ct_floats(const ct_u32x2& u) {  // 4 bf16 elements
  return f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
               __uint_as_float(u[1] & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 ct_fma4(float d, const f32x4& x, const f32x4& acc) {
  return f32x4{fmaf(d, x[0], acc[0]), fmaf(d, x[1], acc[1]), fmaf(d, x[2], acc[2]), fmaf(d, x[3], acc[3])};
}
template <typename T, bool ACOL, int NB>
__global__ __launch_bounds__(Tile<NB>::NT, Tile<NB>::PER_EU) void k_product(const ProductArgs a) {
  using TL = Tile<NB>;
  constexpr int BK = 128 / (int)sizeof(T), FI = TL::FI, FJ = TL::FJ, EDGE = TL::EDGE;
  // 8 waves, two on a SIMD: one of them reads fragments while the other multiplies, half a stage at a
  // time, a turn apart all along (4096 x 21888 x 768: dx 176 -> 150 us, dw 172 -> 146.  k_logits, whose
  // tiles end in long vector work that both should do at once, lost by it: 465 -> 524)
  constexpr bool TURNS = NB == 8;
  __shared__ __attribute__((aligned(16))) char smem[4 * TL::OP_B];
  constexpr int FOUND = 256 * TL::NWV;  // (dw in bf16) rows that are looked at together for the tile's items
  __shared__ __attribute__((aligned(16))) uint32_t found[ACOL && sizeof(T) == 2 ? FOUND : 1];  // row << 8 | item
  __shared__ float lost[ACOL && sizeof(T) == 2 ? FOUND : 1];
  __shared__ int n_found[TL::NWV];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w % TL::ROW_WV, wc = w / TL::ROW_WV, g = lane >> 4, rl = lane & 15;
  const int tc = (a.cols + EDGE - 1) / EDGE, tiles = tc * ((a.M + EDGE - 1) / EDGE);
  const int nk = a.K / BK;
  int t, k0 = 0, k1 = nk, slot = -1;
  if ((int)blockIdx.x < a.whole) {
    t = xcd_remap(blockIdx.x, a.whole);
    if (a.all) slot = t;
  } else {
    const int u = xcd_remap(blockIdx.x - a.whole, gridDim.x - a.whole), r = tiles - a.whole;
    const int per = (nk + a.splits - 1) / a.splits;
    t = a.whole + u % r;
    k0 = u / r * per;
    k1 = k0 + per < nk ? k0 + per : nk;
    slot = u + (a.all ? a.whole : 0);
  }
  const int m0 = t / tc * EDGE, c0 = t % tc * EDGE;
  const T* A = (const T*)a.A;
  const T* B = (const T*)a.B;
  RowStage<T, NB, TL::NWV> ra;
  ColStage<T, NB, TL::NWV> ca, cb;
  if constexpr (ACOL) ca.init(m0, a.lda, w, lane);  // (lda: whole tiles, all written)
  else ra.init(a.lda, m0, a.a_rows, w, lane);
  cb.init(c0, a.cols, w, lane);
  auto issue = [&](int kt) __attribute__((always_inline)) {
    char* st = smem + (kt & 1) * 2 * TL::OP_B;
    if constexpr (ACOL) ca.issue(A, a.lda, (int64_t)kt * BK, a.a_rows, st, w);
    else ra.issue(A, (int64_t)kt * BK, st, w);
    cb.issue(B, a.ldb, (int64_t)kt * BK, a.b_rows, st + TL::OP_B, w);
  };
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto frags = [&](const char* st, auto& fa, auto& fb, int s) __attribute__((always_inline)) {
    if constexpr (ACOL) col_frags<T, NB>(st, 16 * FI * wm, lane, fa, s);
    else row_frags(st, 16 * FI * wm, lane, fa, s);
    col_frags<T, NB>(st + TL::OP_B, 16 * FJ * wc, lane, fb, s);
  };
  const int late = TURNS ? w >> 2 : 0;
  if (k0 < k1) issue(k0);
  if constexpr (sizeof(T) == 2) {
    if (a.delta) {
      // (before the loop, whose registers are not taken yet; after it the 256 tile would spill.)  The
      // block's part of the sum runs over [kb, ke): items (dx), rows (dw)
      const int64_t kb = (int64_t)k0 * BK, ke = (int64_t)k1 * BK < a.b_rows ? (int64_t)k1 * BK : a.b_rows;
      const int cb = c0 + 16 * FJ * wc + 4 * g, cl = a.cols - 4;  // (columns past the end: loaded again)
      if constexpr (!ACOL) {
#pragma unroll
        for (int i = 0; i < FI; ++i) {
          const int n = m0 + 16 * FI * wm + 16 * i + rl;
          const int64_t k = n < a.M ? a.ids[n] - a.v_base : -1;
          if (k >= kb && k < ke) {
            const float d = a.delta[n];
            if (d != 0.0f) {
#pragma unroll
              for (int j = 0; j < FJ; ++j) {
                const int c = cb + 16 * j < cl ? cb + 16 * j : cl;
                acc[i][j] = ct_fma4(d, ct_floats(*(const ct_u32x2*)(B + k * a.ldb + c)), acc[i][j]);
              }
            }
          }
        }
      } else {
        // the rows whose item is one of the tile's, FOUND rows looked at at a time (256 a wave), listed in
        // their order (the sums do not depend on timing) and multiplied 32 at a time: 4096 rows, 65537
        // items: 16 a tile, 10 us of 155; a popular item costs 0.1 us a row
        for (int64_t s0 = kb; s0 < ke; s0 += FOUND) {
          const int64_t n0 = s0 + (FOUND / TL::NWV) * w;
          int q[FOUND / TL::NT], np = 0;
#pragma unroll
          for (int u = 0; u < FOUND / TL::NT; ++u) {
            const int64_t n = n0 + 64 * u + lane, v = n < ke ? a.ids[n] - a.v_base - m0 : -1;
            q[u] = v >= 0 && v < EDGE ? (int)v : -1;
            np += __popcll(__ballot(q[u] >= 0));
          }
          if (lane == 0) n_found[w] = np;
          __syncthreads();
          int at = 0, total = 0;
#pragma unroll
          for (int i = 0; i < TL::NWV; ++i) {
            at += i < w ? n_found[i] : 0;
            total += n_found[i];
          }
#pragma unroll
          for (int u = 0; u < FOUND / TL::NT; ++u) {
            const uint64_t bm = __ballot(q[u] >= 0);
            if (q[u] >= 0) {
              const int k = at + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bm >> 32),
                                                                __builtin_amdgcn_mbcnt_lo((uint32_t)bm, 0u));
              found[k] = (uint32_t)(n0 - s0 + 64 * u + lane) << 8 | (uint32_t)q[u];
              lost[k] = a.delta[n0 + 64 * u + lane];
            }
            at += __popcll(bm);
          }
          __syncthreads();
          for (int p = 0; p < total; p += 32) {
            uint32_t e[8];
            float d[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int o = p + 8 * g + k, in = o < total ? o : p;
              e[k] = found[in];
              d[k] = o < total ? lost[in] : 0.0f;
            }
            u32x4_t fa[1][FI], fb[1][FJ];
#pragma unroll
            for (int j = 0; j < FJ; ++j) {
              const int c = c0 + 16 * (FJ * wc + j) + rl;
              const uint16_t* xc = B + s0 * a.ldb + (c < a.cols ? c : 0);  // (columns past the end are not stored)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                fb[0][j][k] = (uint32_t)xc[(int64_t)(e[2 * k] >> 8) * a.ldb] |
                              (uint32_t)xc[(int64_t)(e[2 * k + 1] >> 8) * a.ldb] << 16;
            }
#pragma unroll
            for (int i = 0; i < FI; ++i) {
              const uint32_t r = (uint32_t)(16 * (FI * wm + i) + rl);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                fa[0][i][k] = ct_pack2((e[2 * k] & 255u) == r ? d[2 * k] : 0.0f,
                                       (e[2 * k + 1] & 255u) == r ? d[2 * k + 1] : 0.0f);
            }
            ct_mfma<T>(fb, fa, acc);
          }
          __syncthreads();
        }
      }
    }
  }
  if constexpr (TURNS) {
    ct_wait_vm<0>();
    ct_turn();
    if (late) {
      if (k0 + 1 < k1) issue(k0 + 1);
      ct_turn();
    }
  }
  for (int kt = k0; kt < k1; ++kt) {
    const char* st = smem + (kt & 1) * 2 * TL::OP_B;
    if constexpr (TURNS) {
      // (the slot's last reads ended with the last turn)
      if (!late && kt + 1 < k1) issue(kt + 1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4_t fa[1][FI], fb[1][FJ];
        frags(st, fa, fb, s);
        if (s == 1 && late) ct_wait_vm<0>();
        ct_turn();
        if (s == 1 && late && kt + 2 < k1) issue(kt + 2);
        ct_mfma<T>(fb, fa, acc);
        if (s == 1 && !late) ct_wait_vm<0>();
        ct_turn();
      }
    } else {
      ct_wait_vm<0>();
      ct_barrier();
      if (kt + 1 < k1) issue(kt + 1);
      u32x4_t fa[2][FI], fb[2][FJ];
      frags(st, fa, fb, 0);
      ct_stage<T>(fb, fa, acc);
    }
  }
  if constexpr (TURNS) {
    if (!late) ct_turn();
  }
  float* part = slot >= 0 ? a.part + (int64_t)slot * (EDGE * EDGE) : nullptr;
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int mr = 16 * FI * wm + 16 * i + rl;
    if (m0 + mr >= a.M) continue;
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int cr = 16 * FJ * wc + 16 * j + 4 * g;
      if (c0 + cr >= a.cols) continue;
      if (part) {
        f32x4* p = (f32x4*)(part + mr * EDGE + cr);
        *p = a.acc ? *p + acc[i][j] : acc[i][j];
      } else {
        ct_store4<T>((T*)a.out + (int64_t)(m0 + mr) * a.ldo + c0 + cr, acc[i][j] * a.scale);
      }
    }
  }
}
// out = scale * (sum over a tile's blocks, in order); edge^2 / 1024 blocks for each tile in part
template <typename T>
__global__ __launch_bounds__(256) void k_product_sum(const ProductArgs a, int edge) {
  const int tc = (a.cols + edge - 1) / edge, tiles = tc * ((a.M + edge - 1) / edge);
  const int bt = edge * edge / 1024, i = blockIdx.x / bt;
  const int t = i + (a.all ? 0 : a.whole), r = tiles - a.whole;
  const int e = (blockIdx.x % bt * 256 + threadIdx.x) * 4;
  const int mm = t / tc * edge + e / edge, c = t % tc * edge + e % edge;
  if (mm >= a.M || c >= a.cols) return;
  const int64_t sq = edge * edge;
  const float* p = a.part + (int64_t)i * sq + e;
  f32x4 s = *(const f32x4*)p;
  if (t >= a.whole)
    for (int k = 1; k < a.splits; ++k) s = s + *(const f32x4*)(p + k * r * sq);
  ct_store4<T>((T*)a.out + (int64_t)mm * a.ldo + c, s * a.scale);
}

// ------------------------------------------------------------------------------- host side
static int64_t up(int64_t n, int64_t q) { return (n + q - 1) / q * q; }
static int64_t cdiv(int64_t n, int64_t q) { return (n + q - 1) / q; }

// k_ring against k_logits' 256 x 256 tiles, us: 4096 x 30000 102 : 113 (coefficients 118 : 136), 1024 x
// 100000 93 : 98 (111 : 122), 2049 x 100003 with entropy 214 : 248 (before the norms); not where blocks of 384 rows leave
// more empty, nor in small problems (200 x 3000 13 : 6).  E = 256: 47 : 46, E = 128: 99 : 107 (108 : 97).
constexpr int CR_E = 384, CR_ROWS = 384;
static bool ring_ok(int64_t N, int64_t V, int E, int64_t sz) {
  return sz == 2 && E == CR_E && 100 * up(N, CR_ROWS) <= 115 * up(N, 256) && N * V >= (1ll << 25);
}
template <bool COEF>
static void ring_launch(const LogitArgs& a, bool ent, hipStream_t st) {
  constexpr int KS = CR_E / 32;
  static_assert(RingCfg<KS>::ROWS == CR_ROWS, "");
  const dim3 grid((unsigned)(a.n_tiles * (int64_t)a.splits));
  if (a.bias) {
    if (ent) hipLaunchKernelGGL((k_ring<KS, COEF, true, true>), grid, dim3(CR_NT), 0, st, a);
    else hipLaunchKernelGGL((k_ring<KS, COEF, false, true>), grid, dim3(CR_NT), 0, st, a);
  } else {
    if (ent) hipLaunchKernelGGL((k_ring<KS, COEF, true, false>), grid, dim3(CR_NT), 0, st, a);
    else hipLaunchKernelGGL((k_ring<KS, COEF, false, false>), grid, dim3(CR_NT), 0, st, a);
  }
}
// shares of `pairs` (64 items each) for about one block a CU
static void ring_shape(int64_t N, int64_t V, int& n_tiles, int& pairs, int& splits) {
  n_tiles = (int)cdiv(N, CR_ROWS);
  pairs = (int)cdiv(V, 64);
  int64_t s = 256 / n_tiles;
  s = s < 1 ? 1 : s > pairs ? pairs : s;
  splits = (int)cdiv(pairs, cdiv(pairs, s));
}

// Tile edge of the logits' kernels: 128; 64 where 128 would give the 256 CUs less than a block each
// (512 x 2560 x 768 f32: 57 us with 80 blocks of 128, 32 us with 320 of 64); 256 in bf16 where that
// gives each CU one (4096 x 65537 x 768: 559 us with 128, 465 with 256).
static int logits_edge(int64_t N, int64_t V, int64_t sz) {
  if (sz == 2 && N > 128 && cdiv(N, 256) * cdiv(V, 256) >= 256) return 256;
  return cdiv(N, 128) * cdiv(V, 128) < 256 ? 64 : 128;
}
// shares of the catalog: as many as there are block slots for
static void logits_shape(int64_t N, int64_t V, int edge, int& n_tiles, int& v_tiles, int& splits) {
  n_tiles = (int)cdiv(N, edge);
  v_tiles = (int)cdiv(V, edge);
  int64_t s = (edge == 64 ? 768 : edge == 128 ? 512 : 256) / n_tiles;
  s = s < 1 ? 1 : s > v_tiles ? v_tiles : s;
  splits = (int)cdiv(v_tiles, cdiv(v_tiles, s));
}

struct StatPlan {
  bool ring;
  int edge, n_tiles, v_tiles, splits, keep, nseg, seg_len;
  int64_t M, off_tmax, off_seg, off_wsq, off_err, off_stat, off_floor, off_rows, off_done, off_kth, off_found, bytes;
  int parts, part_len;
};
// Shares: about 512 blocks (two a CU; three of the small tiles).
static StatPlan stat_plan(int64_t N, int64_t V, int E, int64_t sz, int top) {
  StatPlan p{};
  p.ring = ring_ok(N, V, E, sz);
  if (p.ring) {
    ring_shape(N, V, p.n_tiles, p.v_tiles, p.splits);
  } else {
    p.edge = logits_edge(N, V, sz);
    logits_shape(N, V, p.edge, p.n_tiles, p.v_tiles, p.splits);
  }
  p.bytes = up((int64_t)p.splits * N * 16, 256);
  if (top > 0) {
    p.keep = top + CT_TOP_EXTRA;
    p.M = 4 * cdiv(V, 64);
    // segments of 4096 groups, longer ones past 64 segments a row
    p.seg_len = (int)(4096 * cdiv(p.M, 4096 * 64));
    p.nseg = (int)cdiv(p.M, p.seg_len);
    p.off_tmax = p.bytes;
    p.off_seg = p.off_tmax + up(N * p.M * 4, 256);
    p.off_wsq = p.off_seg + up(N * p.nseg * p.keep * 8, 256);
    p.off_err = p.off_wsq + up((int64_t)p.n_tiles * p.splits * 4, 256);
    p.off_stat = p.off_err + up(N * 4, 256);
    p.off_floor = p.off_stat + up(N * 8, 256);
    // the second search: parts of 256 groups, longer ones past 1024 parts a row
    const int64_t nw = p.M > p.keep ? N : 0;
    p.part_len = (int)(256 * cdiv(p.M, 256 * 1024));
    p.parts = (int)cdiv(p.M, p.part_len);
    p.off_rows = p.off_floor + up(nw * 4, 256);
    p.off_done = p.off_rows + up((nw + 1) * 4, 256);  // (their number first)
    p.off_kth = p.off_done + up(nw * 4, 256);
    p.off_found = p.off_kth + up(nw * 16, 256);
    p.bytes = p.off_found + up(nw * p.parts * top * 16, 256);
  }
  return p;
}

constexpr int64_t CT_C_BYTES = 256ll << 20;  // one chunk of C stays in the last-level cache
// A product's tiles: their edge, how many are summed by one block each, and over how many blocks the
// sums of the others are split.
struct ProductPlan {
  int edge, whole, splits;
  int64_t part;  // floats of partial sums (all: of whole tiles too)
};
// The cards' slots are filled with whole tiles first; what is left over, or all where that is less than
// a round, is split.  Chosen: the least of (steps of 128 bytes that a slot walks, and 6 more a block for
// its start and end) x (a step's time), and 1 us per M floats of partial sums.  Step times, us, with all
// slots busy (bf16, measured on 4096 x 21888 x 768 and 2048 x 20096 x 384): 64 0.6, 128 1.1, 256 1.75
// (1.25 PFLOP/s).
static ProductPlan product_plan(int64_t M, int64_t cols, int64_t K, int64_t sz, bool all) {
  static const int edges[3] = {64, 128, 256}, slots[3] = {768, 512, 256};
  static const double step[3] = {0.6, 1.1, 1.75};
  const int64_t nk = K / (128 / sz);
  ProductPlan b{};
  double best = 0;
  for (int i = 0; i < (sz == 2 ? 3 : 2); ++i) {
    const int64_t tiles = cdiv(M, edges[i]) * cdiv(cols, edges[i]), sq = edges[i] * edges[i];
    const int64_t full = tiles / slots[i], rest = tiles % slots[i];
    for (int64_t s = 1; s <= 64 && (s == 1 || s * 4 <= nk); ++s) {
      if (s > 1 && (rest == 0 || rest * s > 4 * slots[i])) break;
      const int64_t ks = cdiv(nk, s), sr = cdiv(nk, ks);  // no empty split
      const bool split = sr > 1;
      const int64_t part = sq * ((split ? rest * sr : all ? rest : 0) + (all ? full * slots[i] : 0));
      const double c = step[i] * (double)(full * (nk + 6) + cdiv(rest * sr, slots[i]) * (ks + 6)) +
                       1.0e-6 * (double)part + (split && !all ? 4.0 : 0.0);
      if (b.edge == 0 || c < best) {
        best = c;
        b = ProductPlan{edges[i], (int)(split ? full * slots[i] : tiles), (int)sr, part};
      }
    }
  }
  return b;
}
struct BwdPlan {
  int64_t Npad, Vc, n_chunks, off_g, off_x, off_d, off_w, off_c, off_px, off_pw, bytes;
  bool two;  // C in two bf16 rows a row
  ProductPlan px, pw, pw_last;  // dx; dw of a chunk, of the last chunk
};
static BwdPlan bwd_plan(int64_t N, int64_t V, int64_t E, int64_t sz, bool bias, bool dx, bool dw) {
  BwdPlan p{};
  // few bf16 rows: coefficients in two parts, 16 bits of them (one part's rounding, 2^-8, would be as
  // large as the result's own; the calls are bound by reading w and by their launches)
  p.two = sz == 2 && N <= 64;
  p.Npad = up(p.two ? 2 * N : N, 64);
  int64_t vc = CT_C_BYTES / (p.Npad * sz) / CT_TILE * CT_TILE;
  vc = vc < CT_TILE ? CT_TILE : vc;
  p.Vc = up(cdiv(V, cdiv(V, vc)), CT_TILE);  // chunks of like size
  p.n_chunks = cdiv(V, p.Vc);
  int64_t o = up(N * 16, 256);
  p.off_g = o;
  o += up(N * 4, 256);
  p.off_x = o;
  o += up((p.two ? 2 * N : N) * E * sz, 256);
  p.off_d = o;
  if (sz == 2 && !p.two) o += up(N * 4, 256);
  p.off_w = o;
  if (bias) o += up(V * E * sz, 256);
  p.off_c = o;
  o += up(p.Npad * p.Vc * sz, 256);
  p.off_px = o;
  if (dx) {
    p.px = product_plan(N, E, p.Vc, sz, p.n_chunks > 1 || p.two);
    o += p.px.part * 4;
  }
  p.off_pw = o;
  if (dw) {
    const int64_t last = V - (p.n_chunks - 1) * p.Vc;
    p.pw_last = product_plan(last, E, p.Npad, sz, false);
    p.pw = p.n_chunks > 1 ? product_plan(p.Vc, E, p.Npad, sz, false) : p.pw_last;
    o += (p.pw.part > p.pw_last.part ? p.pw.part : p.pw_last.part) * 4;
  }
  p.bytes = o;
  return p;
}
template <typename T, bool ACOL>
static void product_launch(ProductArgs& q, const ProductPlan& p, hipStream_t st) {
  q.whole = p.whole;
  q.splits = p.splits;
  const int64_t tiles = cdiv(q.M, p.edge) * cdiv(q.cols, p.edge);
  const dim3 grid((unsigned)(p.whole + (tiles - p.whole) * p.splits));
  if constexpr (sizeof(T) == 2) {
    if (p.edge == 256) {
      hipLaunchKernelGGL((k_product<T, ACOL, 8>), grid, dim3(512), 0, st, q);
      return;
    }
  }
  if (p.edge == 64) hipLaunchKernelGGL((k_product<T, ACOL, 2>), grid, dim3(256), 0, st, q);
  else hipLaunchKernelGGL((k_product<T, ACOL, 4>), grid, dim3(256), 0, st, q);
}
template <typename T>
static void product_sum(const ProductArgs& q, const ProductPlan& p, hipStream_t st) {
  const int64_t tiles = cdiv(q.M, p.edge) * cdiv(q.cols, p.edge) - (q.all ? 0 : p.whole);
  if (tiles == 0) return;
  const dim3 grid((unsigned)(p.edge * p.edge / 1024 * tiles));
  hipLaunchKernelGGL(k_product_sum<T>, grid, dim3(256), 0, st, q, p.edge);
}
template <typename T, bool COEF, int NB>
static void logits_go(const LogitArgs& a, bool ent, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_tiles * (int64_t)a.splits)), block(Tile<NB>::NT);
  if constexpr (!COEF) {
    if (a.tmax) {
      if (ent) hipLaunchKernelGGL((k_logits<T, COEF, true, NB, true>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((k_logits<T, COEF, false, NB, true>), grid, block, 0, st, a);
      return;
    }
  }
  if (ent) hipLaunchKernelGGL((k_logits<T, COEF, true, NB, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_logits<T, COEF, false, NB, false>), grid, block, 0, st, a);
}
template <typename T, bool COEF>
static void logits_launch(const LogitArgs& a, int edge, bool ent, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (edge == 256) return logits_go<T, COEF, 8>(a, ent, st);
  }
  if (edge == 64) logits_go<T, COEF, 2>(a, ent, st);
  else logits_go<T, COEF, 4>(a, ent, st);
}

static int ct_check(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t dtype, int64_t N,
                    int64_t V, int32_t E, float temperature, const char* fn) {
  auto bad = [&](const char* m) { return fail(TT_ERR_INVALID, std::string(fn) + ": " + m); };
  if (dtype != TT_DTYPE_F32 && dtype != TT_DTYPE_BF16) return bad("dtype must be f32 or bf16");
  if (N < 0 || V < 1 || E < 64 || E % 64 != 0) return bad("need N >= 0, V >= 1, E a multiple of 64");
  if (N >= (1ll << 24) || V >= (1ll << 30) || E > (1 << 20)) return bad("sizes out of range");
  if (!(temperature >= 1.0e-30f)) return bad("temperature must be above 0 (at least 1e-30)");
  if (N == 0) return TT_OK;
  if (!x || !w) return bad("null pointer");
  const int64_t sz = dtype == TT_DTYPE_F32 ? 4 : 2;
  if (((uintptr_t)x | (uintptr_t)w) % 16 || (ldx * sz) % 16 || (ldw * sz) % 16 || ldx < E || ldw < E)
    return bad("rows must be 16-byte aligned and at least E long");
  return TT_OK;
}

template <typename T>
static int logprobs_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int64_t V, int E,
                        const int64_t* ids, const float* bias, float temperature, float* logp, float* ent,
                        double* lse, int top, int64_t* top_ids, float* top_lp, char* ws, const StatPlan& p,
                        hipStream_t st) {
  const double s = 1.0 / (double)temperature;
  LogitArgs a{};
  a.x = x; a.w = w; a.ldx = ldx; a.ldw = ldw; a.bias = bias;
  a.s2 = (float)(s * 1.4426950408889634);
  a.N = (int)N; a.V = (int)V; a.E = E;
  a.n_tiles = p.n_tiles; a.splits = p.splits; a.v_tiles = p.v_tiles;
  a.part = (float4*)ws;
  a.tmax = top ? (float*)(ws + p.off_tmax) : nullptr;
  a.wsq = top ? (float*)(ws + p.off_wsq) : nullptr;
  a.v_count = (int)V;
  if (p.ring) ring_launch<false>(a, ent != nullptr, st);
  else logits_launch<T, false>(a, p.edge, ent != nullptr, st);
  const CombineArgs ca{a.part, p.splits, (int)N, (int)V, E, x, w, ldx, ldw, ids, bias, s, a.s2,
                       p.ring || p.edge == 64 ? 32 : 64, logp, ent, lse, a.wsq, p.n_tiles * p.splits,
                       top ? (float*)(ws + p.off_err) : nullptr, top ? (float2*)(ws + p.off_stat) : nullptr};
  const unsigned cb = (unsigned)cdiv(N, 4);
  if (top) {
    uint64_t* seg = (uint64_t*)(ws + p.off_seg);
    const unsigned sb = (unsigned)(N * p.nseg);
    TopArgs ta{};
    ta.segs = seg; ta.nseg = p.nseg; ta.keep = p.keep; ta.top = top;
    ta.x = x; ta.w = w; ta.ldx = ldx; ta.ldw = ldw; ta.N = (int)N; ta.E = E; ta.V = (int)V;
    ta.bias = bias; ta.s = s; ta.s2 = a.s2; ta.group = ca.group; ta.err = ca.err; ta.stat = ca.stat;
    ta.ids_out = top_ids; ta.lp_out = top_lp;
    const bool wide = p.M > p.keep;  // (else no group is left out)
    if (wide) {
      ta.tmax = a.tmax; ta.M = p.M; ta.parts = p.parts; ta.part_len = p.part_len;
      ta.n_rows = (uint32_t*)(ws + p.off_rows);
      ta.rows = ta.n_rows + 1;
      ta.floor = (float*)(ws + p.off_floor);
      ta.kth = (TopEntry*)(ws + p.off_kth);
      ta.done = (uint32_t*)(ws + p.off_done);
      ta.found = (TopEntry*)(ws + p.off_found);
    }
    hipLaunchKernelGGL(k_top_groups<T>, dim3(sb + cb), dim3(256), 0, st, a.tmax, p.M, p.seg_len, p.nseg,
                       p.keep, seg, sb, ca, ta.n_rows);
    // more threads a row while rows are few: 33 rows 26 us with 1024 (31 with 512); 2049 rows 56 us with
    // 256 (90 with 512)
    if (N <= 128) hipLaunchKernelGGL((k_top_items<T, 1024>), dim3((unsigned)N), dim3(1024), 0, st, ta);
    else if (N <= 512) hipLaunchKernelGGL((k_top_items<T, 512>), dim3((unsigned)N), dim3(512), 0, st, ta);
    else hipLaunchKernelGGL((k_top_items<T, 256>), dim3((unsigned)N), dim3(256), 0, st, ta);
    if (wide) {
      const int64_t units = N * p.parts;
      hipLaunchKernelGGL(k_top_wide<T>, dim3((unsigned)(units < 768 ? units : 768)), dim3(256), 0, st, ta);
    }
  } else {
    hipLaunchKernelGGL(k_combine<T>, dim3(cb), dim3(256), 0, st, ca);
  }
  return check_launch("tt_catalog_logprobs");
}

template <typename T>
static int logprobs_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int64_t V, int E,
                        const int64_t* ids, const float* bias, float temperature, const double* lse,
                        const float* ent, const float* g, const float* e, void* dx, void* dw, char* ws,
                        const BwdPlan& p, hipStream_t st) {
  const double s = 1.0 / (double)temperature;
  float4* rowc = (float4*)ws;
  float* rowg = (float*)(ws + p.off_g);
  T* xz = (T*)(ws + p.off_x);
  float* delta = sizeof(T) == 2 && !p.two && ids && g ? (float*)(ws + p.off_d) : nullptr;
  hipLaunchKernelGGL(k_rows<T>, dim3((unsigned)cdiv(N, 4)), dim3(256), 0, st, (const T*)x, ldx, (int)N, E, lse,
                     ent, g, e, ids, (int)V, rowc, rowg, xz, p.two);
  const T* wz = (const T*)w;
  int64_t ldwz = ldw;
  if (bias) {
    const int64_t nb = cdiv(V, 4);
    hipLaunchKernelGGL(k_items<T>, dim3((unsigned)(nb < 8192 ? nb : 8192)), dim3(256), 0, st, (const T*)w, ldw,
                       (int)V, E, bias, (T*)(ws + p.off_w));
    wz = (const T*)(ws + p.off_w);
    ldwz = E;
  }
  T* C = (T*)(ws + p.off_c);
  float* px = (float*)(ws + p.off_px);
  ProductArgs qx{};
  for (int64_t c = 0; c < p.n_chunks; ++c) {
    const int64_t vb = c * p.Vc, vn = V - vb < p.Vc ? V - vb : p.Vc;
    LogitArgs a{};
    a.x = xz; a.w = wz; a.ldx = E; a.ldw = ldwz; a.bias = bias;
    a.s2 = (float)(s * 1.4426950408889634);
    a.N = (int)N; a.V = (int)V; a.E = E;
    a.rowc = rowc; a.rowg = rowg; a.ids = ids; a.C = C; a.ldc = p.Vc; a.v_base = (int)vb; a.Npad = (int)p.Npad;
    a.v_count = (int)vn;
    a.two = p.two;
    if (ring_ok(N, vn, E, sizeof(T))) {
      ring_shape(N, vn, a.n_tiles, a.v_tiles, a.splits);
      ring_launch<true>(a, e != nullptr, st);
    } else {
      const int edge = logits_edge(N, vn, sizeof(T));
      logits_shape(p.two ? p.Npad - N : N, vn, edge, a.n_tiles, a.v_tiles, a.splits);
      logits_launch<T, true>(a, edge, e != nullptr, st);
    }
    if constexpr (sizeof(T) == 2) {
      if (delta) hipLaunchKernelGGL(k_lost, dim3((unsigned)cdiv(N, 4)), dim3(256), 0, st, a, delta);
    }
    const int64_t vk = up(vn, 64);
    if (dx) {
      qx.A = C; qx.lda = p.Vc; qx.a_rows = p.Npad;
      qx.B = wz + vb * ldwz; qx.ldb = ldwz; qx.b_rows = V - vb;
      qx.M = (int)N; qx.cols = E; qx.K = (int)vk;
      qx.all = p.n_chunks > 1 || p.two; qx.acc = c > 0;
      qx.scale = (float)s; qx.out = dx; qx.ldo = E;
      qx.part = px;
      qx.delta = delta; qx.ids = ids; qx.v_base = (int)vb;
      product_launch<T, false>(qx, p.px, st);
      if (p.two) {
        qx.A = C + N * p.Vc; qx.a_rows = p.Npad - N;
        qx.acc = true;
        product_launch<T, false>(qx, p.px, st);
      }
    }
    if (dw) {
      ProductArgs q{};
      q.A = C; q.lda = p.Vc; q.a_rows = p.Npad;
      q.B = xz; q.ldb = E; q.b_rows = p.two ? 2 * N : N;
      q.M = (int)vn; q.cols = E; q.K = (int)p.Npad;
      q.scale = (float)s; q.out = (T*)dw + vb * E; q.ldo = E;
      q.part = (float*)(ws + p.off_pw);
      q.delta = delta; q.ids = ids; q.v_base = (int)vb;
      const ProductPlan& pw = c + 1 < p.n_chunks ? p.pw : p.pw_last;
      product_launch<T, true>(q, pw, st);
      product_sum<T>(q, pw, st);
    }
  }
  if (dx) product_sum<T>(qx, p.px, st);
  return check_launch("tt_catalog_logprobs_bwd");
}

}  // namespace tt

using namespace tt;

#define CT_SIZES_ONLY()                                                                            \
  TT_REQUIRE(bytes, "null pointer");                                                               \
  TT_REQUIRE(dtype == TT_DTYPE_F32 || dtype == TT_DTYPE_BF16, "dtype must be f32 or bf16");        \
  TT_REQUIRE(N >= 0 && V >= 1 && E >= 64 && E % 64 == 0 && N < (1ll << 24) && V < (1ll << 30),     \
             "sizes out of range")

extern "C" int tt_catalog_logprobs_workspace_bytes(int64_t N, int64_t V, int32_t E, int32_t dtype, int32_t top,
                                                   int64_t* bytes) {
  CT_SIZES_ONLY();
  TT_REQUIRE(top >= 0 && top <= CT_TOP_MAX && top <= V, "need 0 <= top <= min(V, 32)");
  *bytes = N > 0 ? stat_plan(N, V, E, dtype == TT_DTYPE_F32 ? 4 : 2, top).bytes : 0;
  return TT_OK;
}

extern "C" int tt_catalog_logprobs(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t dtype,
                                   int64_t N, int64_t V, int32_t E, const int64_t* ids, const float* bias,
                                   float temperature, float* log_prob, float* entropy, double* lse, int32_t top,
                                   int64_t* top_ids, float* top_log_prob, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (int rc = ct_check(x, ldx, w, ldw, dtype, N, V, E, temperature, __func__)) return rc;
  TT_REQUIRE(top >= 0 && top <= CT_TOP_MAX && top <= V, "need 0 <= top <= min(V, 32)");
  if (N == 0) return TT_OK;
  TT_REQUIRE(lse && (!log_prob || ids) && (top == 0 || (top_ids && top_log_prob)), "null pointer");
  const StatPlan p = stat_plan(N, V, E, dtype == TT_DTYPE_F32 ? 4 : 2, top);
  TT_REQUIRE(N * (int64_t)p.nseg < (1ll << 24), "too many rows for this many items: pass fewer at a time");
  if (!workspace || workspace_bytes < p.bytes)
    return fail(TT_ERR_WORKSPACE, "tt_catalog_logprobs: workspace too small");
  auto f = dtype == TT_DTYPE_F32 ? logprobs_fwd<float> : logprobs_fwd<uint16_t>;
  return f(x, ldx, w, ldw, N, V, E, ids, bias, temperature, log_prob, entropy, lse, top, top_ids, top_log_prob,
           (char*)workspace, p, (hipStream_t)stream);
}

extern "C" int tt_catalog_logprobs_bwd_workspace_bytes(int64_t N, int64_t V, int32_t E, int32_t dtype,
                                                       int32_t has_bias, int32_t want_dx, int32_t want_dw,
                                                       int64_t* bytes) {
  CT_SIZES_ONLY();
  *bytes = N > 0 ? bwd_plan(N, V, E, dtype == TT_DTYPE_F32 ? 4 : 2, has_bias != 0, want_dx != 0, want_dw != 0).bytes
                 : 0;
  return TT_OK;
}

extern "C" int tt_catalog_logprobs_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t dtype,
                                       int64_t N, int64_t V, int32_t E, const int64_t* ids, const float* bias,
                                       float temperature, const double* lse, const float* entropy,
                                       const float* g_log_prob, const float* g_entropy, void* dx, void* dw,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = ct_check(x, ldx, w, ldw, dtype, N, V, E, temperature, __func__)) return rc;
  if (N == 0) {
    TT_REQUIRE(!dw, "dw without rows: fill it with zeros");
    return TT_OK;
  }
  TT_REQUIRE(lse && (!g_log_prob || ids) && (!g_entropy || entropy), "null pointer");
  TT_REQUIRE(((uintptr_t)dx | (uintptr_t)dw) % 16 == 0, "dx and dw must be 16-byte aligned");
  const BwdPlan p = bwd_plan(N, V, E, dtype == TT_DTYPE_F32 ? 4 : 2, bias != nullptr, dx != nullptr, dw != nullptr);
  if (!workspace || workspace_bytes < p.bytes)
    return fail(TT_ERR_WORKSPACE, "tt_catalog_logprobs_bwd: workspace too small");
  auto f = dtype == TT_DTYPE_F32 ? logprobs_bwd<float> : logprobs_bwd<uint16_t>;
  return f(x, ldx, w, ldw, N, V, E, ids, bias, temperature, lse, entropy, g_log_prob, g_entropy, dx, dw,
           (char*)workspace, p, (hipStream_t)stream);
}
