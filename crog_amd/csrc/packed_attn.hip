// Attention over packed sequences (crog_packed_attn_*): rows of sequences of different lengths one behind the other, grouped heads, causal or not,
// queries and keys of one sequence or of two.  The padded form beside it (attn.hip) wants rectangles, head dim 64 and one key head per query head.
//
//   o_i = sum_j P_ij v_j,  P = softmax_j(scale q_i . k_j) over the keys the mask leaves (causal: j <= i + Lk - Lq, both ends aligned)
//   dV = P^T dO,  D_i = dO_i . o_i,  dS = P (dO V^T - D) scale,  dQ = dS K,  dK = dS^T Q, the last two sums over the query heads of a group
//
// Rows.  The `group` query heads that share a key head are rows of ONE product: row r of a sequence is (query r / group, head r % group), so a
// key tile is fetched once for the whole group, and a single new token of 8 heads fills 8 rows of a matrix tile instead of one.
// Layout.  As in attn.hip: the 32x32 MFMA returns lane = column, 16 rows in registers, so computing S^T = K Q^T (lane = query row) makes the
// row statistics per-lane scalars and the probabilities an operand of the next product without a shuffle.  float: v_mfma_f32_32x32x2_f32, exact
// products; its k index is the lane's half, so the registers are that operand as they stand.
// One LDS image serves both ways of reading a tile - rows (16 bytes a lane, lane = row) and columns (ds_read_b64_tr_b16, four rows x 64 bytes a
// half wave): the 16-byte slot of a row is XORed with the row's low bits, the lowest two moved to the slot's high bits.
#include "common.h"

namespace {

constexpr int NT = 256;      // 4 waves, 32 rows (forward, dQ) or 32 keys (dK / dV) each
constexpr int BR = 128;      // rows (keys) of a block

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

struct PackedArgs {
  const void *Q, *K, *V, *O, *dO;
  void *Out, *dQ, *dK, *dV;
  float *lse, *D;      // [kv_heads][rows_q * group], lse in log2 units (-inf: no key)
  float *part_o, *part_ml;
  long ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso, lddo, hsdo, lddq, hsdq, lddk, hsdk, lddv, hsdv;
  const int *cu_q, *cu_k, *tiles;
  int seqs, rows_q, rows_k, kv_heads, group, dim, causal, split_keys;
  float scale;
};

// one sequence: its first row and length on both sides (the tables are the caller's device memory: clamped, so that no table reads out of range)
struct Seq { int q0, lq, k0, lk; };
__device__ inline Seq seq_of(const PackedArgs& a, int s) {
  s = min(max(s, 0), a.seqs - 1);
  Seq e;
  e.q0 = min(max(a.cu_q[s], 0), a.rows_q);
  e.lq = min(max(a.cu_q[s + 1], e.q0), a.rows_q) - e.q0;
  e.k0 = min(max(a.cu_k[s], 0), a.rows_k);
  e.lk = min(max(a.cu_k[s + 1], e.k0), a.rows_k) - e.k0;
  return e;
}

// ---- LDS tiles of rows of DP elements ----------------------------------------------------------------------------------------
template <typename T, int DP> struct Tile {
  static constexpr int VEC = Elem<T>::VEC, CPR = DP / VEC;      // 16-byte chunks per row
  static constexpr int NS = CPR / 2;                            // 16-byte operand steps of a lane (its half takes every other chunk)
  static constexpr int NC = DP / 32;                            // 32-column blocks
  __device__ static inline int off(int row, int chunk) {
    const int f = CPR == 8 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
    return row * DP + ((chunk ^ f) * VEC);
  }
};

__device__ inline int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }      // row of accumulator register r of half h
constexpr float LOG2E = 1.4426950408889634f;
__device__ inline float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// acc (32 rows of the tile x 32 columns = lanes) += tile rows . frag (the lane's row of the other operand)
template <typename T, int DP>
__device__ inline void mma_rows(f32x16& acc, const T* tile, int row, int h, const Vec16<T>* frag) {
  using L = Tile<T, DP>;
#pragma unroll
  for (int ks = 0; ks < L::NS; ks++) {
    const Vec16<T> a = ldg16(tile + L::off(row, 2 * ks + h));
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, frag[ks]), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32((float)a.v[e], (float)frag[ks].v[e], acc, 0, 0, 0);
    }
  }
}

// out[c] (columns 32 c .. 32 c + 31 of the tile x lanes) += tile^T . p, p = 32 tile rows (registers, acc_row order) x lanes
template <typename T, int DP>
__device__ inline void mma_cols(f32x16* out, const T* tile, const f32x16& p, int lane) {
  using L = Tile<T, DP>;
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int i = lane & 15, q = i >> 2, pp = i & 3;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      bf16x8 b;      // (the probabilities are rounded to the operand type of the matrix unit: half a bf16 step each, as the inputs are)
#pragma unroll
      for (int j = 0; j < 8; j++) b[j] = (bf16)p[8 * t + j];
#pragma unroll
      for (int c = 0; c < L::NC; c++) {
        const int col = c * 32 + 16 * ((lane >> 4) & 1) + 4 * pp, chunk = col >> 3, inb = col & 7;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + L::off(16 * t + 4 * h + q, chunk) + inb));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + L::off(16 * t + 8 + 4 * h + q, chunk) + inb));
        out[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), b, out[c], 0, 0, 0);
      }
    }
  } else {
    const int ln = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; r++)
#pragma unroll
      for (int c = 0; c < L::NC; c++) {
        const int col = c * 32 + ln;
        out[c] = __builtin_amdgcn_mfma_f32_32x32x2f32((float)tile[L::off(acc_row(r, h), col >> 2) + (col & 3)], p[r], out[c], 0, 0, 0);
      }
  }
}

// a lane's row of a resident operand, zeros behind the head dimension
template <typename T, int DP>
__device__ inline void load_frag(Vec16<T>* frag, const T* row, int h, int dim, bool valid) {
  using L = Tile<T, DP>;
#pragma unroll
  for (int ks = 0; ks < L::NS; ks++) {
    const int at = (2 * ks + h) * L::VEC;
    frag[ks] = (valid && at < dim) ? ldg16(row + at) : zero16<T>();
  }
}

// lane = row, registers = 32-column blocks: a row's D values as pieces of four
template <typename T, int DP>
__device__ inline void store_row(T* row, const f32x16* acc, int h, int dim, float f) {
#pragma unroll
  for (int c = 0; c < DP / 32; c++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int at = c * 32 + 8 * g + 4 * h;
      if (at >= dim) continue;
      if constexpr (sizeof(T) == 2) {
        bf16x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (bf16)(acc[c][4 * g + j] * f);
        *reinterpret_cast<bf16x4*>(row + at) = w;
      } else {
        f32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = acc[c][4 * g + j] * f;
        *reinterpret_cast<f32x4*>(row + at) = w;
      }
    }
}

// R rows on their way from memory to an LDS tile through registers: thread -> (row, chunk), rows >= n and columns >= dim become zeros
// (a row of another sequence may hold infinities or NaN: zero times those is NaN, so it must not reach a product even with probability zero)
template <typename T, int DP, int R> struct Stage {
  using L = Tile<T, DP>;
  static constexpr int NP = R * L::CPR / NT, RPP = NT / L::CPR;
  Vec16<T> v[NP];
  template <typename RowPtr>
  __device__ inline void load(RowPtr rowptr, int r0, int n, int dim, int tid) {
    const int chunk = tid % L::CPR, row = tid / L::CPR;
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int r = r0 + row + p * RPP;
      v[p] = (r < n && chunk * L::VEC < dim) ? ldg16(rowptr(r) + chunk * L::VEC) : zero16<T>();
    }
  }
  __device__ inline void store(T* tile, int tid) const {
    const int chunk = tid % L::CPR, row = tid / L::CPR;
#pragma unroll
    for (int p = 0; p < NP; p++) stg16(tile + L::off(row + p * RPP, chunk), v[p]);
  }
};

// =====================================================================================================================
// forward.  grid (kv_heads * tiles, key splits); a block owns 128 rows of one sequence and key head, keys stream through LDS.
// =====================================================================================================================
template <typename T, int DP, int NB>
__global__ void __launch_bounds__(NT, 2) packed_fwd_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int KT = 32 * NB;
  __shared__ __attribute__((aligned(16))) T sK[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T sV[2][KT * DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, ln = lane & 31;
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  const int rows = e.lq * a.group, dim = a.dim;
  const int r0 = tile * BR + wave * 32, r = r0 + ln;
  if (tile < 0 || tile * BR >= rows) return;      // (uniform)
  const int off = e.lk - e.lq;
  const int rc = min(r, rows - 1), qi = rc / a.group;
  const int lim = a.causal ? min(max(qi + 1 + off, 0), e.lk) : e.lk;      // the lane's row sees keys [0, lim)
  const auto limit = [&](int row) { return a.causal ? min(max(min(row, rows - 1) / a.group + 1 + off, 0), e.lk) : e.lk; };
  const int lim_lo = limit(r0), lim_hi = r0 < rows ? limit(r0 + 31) : 0;
  const int kbeg = blockIdx.y * a.split_keys;
  const int kend = min(limit(tile * BR + BR - 1), kbeg + a.split_keys);

  Vec16<T> qf[L::NS];
  load_frag<T, DP>(qf, (const T*)a.Q + (long)(e.q0 + qi) * a.ldq + (long)(kh * a.group + rc % a.group) * a.hsq, h, dim, r < rows);
  f32x16 o[L::NC];
#pragma unroll
  for (int c = 0; c < L::NC; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[c][i] = 0.f;
  float m = -INFINITY, mu = 0.f, l = 0.f;      // running maximum (log2 units), the same with 0 for -inf, the lane's share of the sum
  const float c2 = a.scale * LOG2E;
  const T* kg = (const T*)a.K + (long)e.k0 * a.ldk + (long)kh * a.hsk;
  const T* vg = (const T*)a.V + (long)e.k0 * a.ldv + (long)kh * a.hsv;
  const auto krow = [&](int key) { return kg + (long)key * a.ldk; };
  const auto vrow = [&](int key) { return vg + (long)key * a.ldv; };
  Stage<T, DP, KT> st_k, st_v;
  if (kbeg < kend) {
    st_k.load(krow, kbeg, e.lk, dim, tid);
    st_v.load(vrow, kbeg, e.lk, dim, tid);
    st_k.store(sK[0], tid);
    st_v.store(sV[0], tid);
  }
  __syncthreads();
  int buf = 0;
  for (int kb = kbeg; kb < kend; kb += KT, buf ^= 1) {
    const bool more = kb + KT < kend;
    if (more) {
      st_k.load(krow, kb + KT, e.lk, dim, tid);
      st_v.load(vrow, kb + KT, e.lk, dim, tid);
    }
    if (kb < lim_hi) {      // (wave-uniform)
      f32x16 s[NB];
      float mt = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[n][i] = 0.f;
        mma_rows<T, DP>(s[n], sK[buf] + n * 32 * DP, ln, h, qf);
      }
      if (kb + KT <= lim_lo) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 16; i++) { s[n][i] *= c2; mt = fmaxf(mt, s[n][i]); }
      } else {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            s[n][i] = kb + n * 32 + acc_row(i, h) < lim ? s[n][i] * c2 : -INFINITY;
            mt = fmaxf(mt, s[n][i]);
          }
      }
      mt = xor32_max(mt);
      if (__any(mt > m + 8.f)) {
        // the accumulators follow the maximum only when it grew by more than 8 (log2 units): until then the probabilities are at most 2^8
        const float mn = fmaxf(m, mt);
        const float alpha = mn == -INFINITY ? 1.f : ex2(m - mn);
        m = mn;
        mu = mn == -INFINITY ? 0.f : mn;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < L::NC; c++)
#pragma unroll
          for (int i = 0; i < 16; i++) o[c][i] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int i = 0; i < 16; i++) { s[n][i] = ex2(s[n][i] - mu); l += s[n][i]; }
        mma_cols<T, DP>(o, sV[buf] + n * 32 * DP, s[n], lane);
      }
    }
    if (more) {
      st_k.store(sK[buf ^ 1], tid);
      st_v.store(sV[buf ^ 1], tid);
    }
    __syncthreads();
  }
  l = xor32_sum(l);
  if (r >= rows) return;
  const long at = (long)kh * a.rows_q * a.group + (long)e.q0 * a.group + r;
  if (a.part_o) {
    const long pr = (long)blockIdx.y * a.kv_heads * a.rows_q * a.group + at;
    store_row<float, DP>(a.part_o + pr * dim, o, h, dim, 1.f);
    if (h == 0) { a.part_ml[2 * pr] = m; a.part_ml[2 * pr + 1] = l; }
    return;
  }
  store_row<T, DP>((T*)a.Out + (long)(e.q0 + qi) * a.ldo + (long)(kh * a.group + rc % a.group) * a.hso, o, h, dim, l == 0.f ? 0.f : 1.f / l);
  if (h == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : m + __log2f(l);
}

// the splits of a row meet: o = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z.  One wave per row.
template <typename T>
__global__ void __launch_bounds__(NT) packed_combine_kernel(const PackedArgs a, int splits) {
  const int lane = threadIdx.x & 63;
  const long total = (long)a.kv_heads * a.rows_q * a.group, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  // rows behind the last sequence have no partial result and stay as they are
  if (row >= total || (row % ((long)a.rows_q * a.group)) >= (long)min(a.cu_q[a.seqs], a.rows_q) * a.group) return;
  const int kh = (int)(row / ((long)a.rows_q * a.group));
  const long rr = row % ((long)a.rows_q * a.group);
  float M = -INFINITY;
  for (int z = 0; z < splits; z++) M = fmaxf(M, a.part_ml[2 * (z * total + row)]);
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int z = 0; z < splits; z++) {
    const float mz = a.part_ml[2 * (z * total + row)], lz = a.part_ml[2 * (z * total + row) + 1];
    const float f = mz == -INFINITY ? (lz == 0.f ? 0.f : 1.f) : ex2(mz - M);
    const float* p = a.part_o + (z * total + row) * a.dim;
    l += f * lz;
    if (f != 0.f) {
      if (lane < a.dim) o0 += f * p[lane];
      if (lane + 64 < a.dim) o1 += f * p[lane + 64];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.Out + (rr / a.group) * a.ldo + (long)(kh * a.group + rr % a.group) * a.hso;
  if (lane < a.dim) op[lane] = Elem<T>::from_f(o0 * inv);
  if (lane + 64 < a.dim) op[lane + 64] = Elem<T>::from_f(o1 * inv);
  if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : M + __log2f(l);
}

// =====================================================================================================================
// backward 1: D and dQ, blocked as the forward.
// =====================================================================================================================
template <typename T, int DP, int NB>
__global__ void __launch_bounds__(NT, 2) packed_bwd_dq_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int KT = 32 * NB;
  __shared__ __attribute__((aligned(16))) T sK[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T sV[2][KT * DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, ln = lane & 31;
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  const int rows = e.lq * a.group, dim = a.dim;
  const int r0 = tile * BR + wave * 32, r = r0 + ln;
  if (tile < 0 || tile * BR >= rows) return;
  const int off = e.lk - e.lq;
  const int rc = min(r, rows - 1), qi = rc / a.group;
  const int lim = a.causal ? min(max(qi + 1 + off, 0), e.lk) : e.lk;
  const auto limit = [&](int row) { return a.causal ? min(max(min(row, rows - 1) / a.group + 1 + off, 0), e.lk) : e.lk; };
  const int lim_lo = limit(r0), lim_hi = r0 < rows ? limit(r0 + 31) : 0;
  const int kend = limit(tile * BR + BR - 1);
  const long row_g = e.q0 + qi, head = (long)kh * a.group + rc % a.group;
  const long at = (long)kh * a.rows_q * a.group + (long)e.q0 * a.group + rc;

  Vec16<T> qf[L::NS], gf[L::NS];
  load_frag<T, DP>(qf, (const T*)a.Q + row_g * a.ldq + head * a.hsq, h, dim, r < rows);
  load_frag<T, DP>(gf, (const T*)a.dO + row_g * a.lddo + head * a.hsdo, h, dim, r < rows);
  // one key tile: D = sum_j P_ij dP_ij from the tile itself, unrounded (the stored o is off by half a step, which few keys do not average out)
  const bool one_tile = kend <= KT;
  float Dr = 0.f;
  if (!one_tile) {
    const T* op = (const T*)a.O + row_g * a.ldo + head * a.hso;
#pragma unroll
    for (int ks = 0; ks < L::NS; ks++) {
      const int c = (2 * ks + h) * L::VEC;
      if (c < dim) {
        const Vec16<T> of = ldg16(op + c);
#pragma unroll
        for (int j = 0; j < L::VEC; j++) Dr += Elem<T>::to_f(gf[ks].v[j]) * Elem<T>::to_f(of.v[j]);
      }
    }
    Dr = xor32_sum(Dr);
    if (h == 0 && r < rows) a.D[at] = Dr;
  }
  const float lse = a.lse[at], c2 = a.scale * LOG2E;
  f32x16 dq[L::NC];
#pragma unroll
  for (int c = 0; c < L::NC; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) dq[c][i] = 0.f;
  const T* kg = (const T*)a.K + (long)e.k0 * a.ldk + (long)kh * a.hsk;
  const T* vg = (const T*)a.V + (long)e.k0 * a.ldv + (long)kh * a.hsv;
  const auto krow = [&](int key) { return kg + (long)key * a.ldk; };
  const auto vrow = [&](int key) { return vg + (long)key * a.ldv; };
  Stage<T, DP, KT> st_k, st_v;
  if (kend > 0) {
    st_k.load(krow, 0, e.lk, dim, tid);
    st_v.load(vrow, 0, e.lk, dim, tid);
    st_k.store(sK[0], tid);
    st_v.store(sV[0], tid);
  }
  __syncthreads();
  int buf = 0;
  for (int kb = 0; kb < kend; kb += KT, buf ^= 1) {
    const bool more = kb + KT < kend;
    if (more) {
      st_k.load(krow, kb + KT, e.lk, dim, tid);
      st_v.load(vrow, kb + KT, e.lk, dim, tid);
    }
    if (kb < lim_hi) {
      f32x16 s[NB], dp[NB];
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[n][i] = dp[n][i] = 0.f;
        mma_rows<T, DP>(s[n], sK[buf] + n * 32 * DP, ln, h, qf);
        mma_rows<T, DP>(dp[n], sV[buf] + n * 32 * DP, ln, h, gf);
      }
      const bool whole = kb + KT <= lim_lo;
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          // (the exponential of a selected argument, so that the compiler makes no branch per score)
          const float x = s[n][i] * c2 - lse;
          s[n][i] = ex2((whole | (kb + n * 32 + acc_row(i, h) < lim)) ? x : -INFINITY);
        }
      if (one_tile) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 16; i++) Dr += s[n][i] * dp[n][i];
        Dr = xor32_sum(Dr);
      }
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[n][i] = s[n][i] * (dp[n][i] - Dr) * a.scale;
        mma_cols<T, DP>(dq, sK[buf] + n * 32 * DP, s[n], lane);
      }
    }
    if (more) {
      st_k.store(sK[buf ^ 1], tid);
      st_v.store(sV[buf ^ 1], tid);
    }
    __syncthreads();
  }
  if (r >= rows) return;
  if (one_tile && h == 0) a.D[at] = Dr;
  store_row<T, DP>((T*)a.dQ + row_g * a.lddq + head * a.hsdq, dq, h, dim, 1.f);
}

// =====================================================================================================================
// backward 2: dK, dV.  grid (kv_heads * key tiles); a block owns 128 keys, 32 a wave; the group's query rows stream through LDS.
// =====================================================================================================================
template <typename T, int DP>
__global__ void __launch_bounds__(NT, sizeof(T) == 2 ? 2 : 1) packed_bwd_dkdv_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int RT = 32;
  __shared__ __attribute__((aligned(16))) T sQ[2][RT * DP];
  __shared__ __attribute__((aligned(16))) T sG[2][RT * DP];
  __shared__ __attribute__((aligned(16))) float sL[2][RT];
  __shared__ __attribute__((aligned(16))) float sD[2][RT];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, ln = lane & 31;
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  const int rows = e.lq * a.group, dim = a.dim;
  const int k0 = tile * BR + wave * 32, key = k0 + ln, kc = min(key, e.lk - 1);
  if (tile < 0 || tile * BR >= e.lk) return;
  const int off = e.lk - e.lq;
  // rows >= first(key) see the key: query >= key - off, row = query * group
  const auto first = [&](int k) { return a.causal ? max(k - off, 0) * a.group : 0; };
  const int rmin = first(key), rbeg = first(tile * BR) / RT * RT;
  const int wbeg = first(k0), wall = first(k0 + 31);      // the wave's first row at all, its first row that sees all its keys
  const T* qg = (const T*)a.Q + (long)e.q0 * a.ldq + (long)kh * a.group * a.hsq;
  const T* gg = (const T*)a.dO + (long)e.q0 * a.lddo + (long)kh * a.group * a.hsdo;
  const auto qrow = [&](int r) { const int q = r / a.group; return qg + (long)q * a.ldq + (long)(r - q * a.group) * a.hsq; };
  const auto grow = [&](int r) { const int q = r / a.group; return gg + (long)q * a.lddo + (long)(r - q * a.group) * a.hsdo; };
  const float* lg = a.lse + (long)kh * a.rows_q * a.group + (long)e.q0 * a.group;
  const float* dg = a.D + (long)kh * a.rows_q * a.group + (long)e.q0 * a.group;
  // rows that do not exist, and rows without a key, take no probability: 2^(s - inf) = 0
  const auto stat = [&](int r) {
    if (tid < RT) { const float v = r + tid < rows ? lg[r + tid] : INFINITY; return v == -INFINITY ? INFINITY : v; }
    return (tid < 2 * RT && r + tid - RT < rows) ? dg[r + tid - RT] : 0.f;
  };
  const auto stat_put = [&](int b, float v) { if (tid < RT) sL[b][tid] = v; else if (tid < 2 * RT) sD[b][tid - RT] = v; };

  Vec16<T> kf[L::NS], vf[L::NS];
  load_frag<T, DP>(kf, (const T*)a.K + (long)(e.k0 + kc) * a.ldk + (long)kh * a.hsk, h, dim, key < e.lk);
  load_frag<T, DP>(vf, (const T*)a.V + (long)(e.k0 + kc) * a.ldv + (long)kh * a.hsv, h, dim, key < e.lk);
  f32x16 dk[L::NC], dv[L::NC];
#pragma unroll
  for (int c = 0; c < L::NC; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) dk[c][i] = dv[c][i] = 0.f;
  const float c2 = a.scale * LOG2E;
  Stage<T, DP, RT> st_q, st_g;
  float rs = 0.f;
  if (rbeg < rows) {
    st_q.load(qrow, rbeg, rows, dim, tid);
    st_g.load(grow, rbeg, rows, dim, tid);
    st_q.store(sQ[0], tid);
    st_g.store(sG[0], tid);
    stat_put(0, stat(rbeg));
  }
  __syncthreads();
  int buf = 0;
  for (int rb = rbeg; rb < rows; rb += RT, buf ^= 1) {
    const bool more = rb + RT < rows;
    if (more) {
      st_q.load(qrow, rb + RT, rows, dim, tid);
      st_g.load(grow, rb + RT, rows, dim, tid);
      rs = stat(rb + RT);
    }
    if (k0 < e.lk && rb + RT > wbeg) {
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = dp[i] = 0.f;
      mma_rows<T, DP>(s, sQ[buf], ln, h, kf);
      mma_rows<T, DP>(dp, sG[buf], ln, h, vf);
      float lr[16], dr[16];
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(&sL[buf][8 * g + 4 * h]), d4 = *reinterpret_cast<const f32x4*>(&sD[buf][8 * g + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; j++) { lr[4 * g + j] = l4[j]; dr[4 * g + j] = d4[j]; }
      }
      const bool whole = rb >= wall;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float x = s[i] * c2 - lr[i];
        s[i] = ex2((whole | (rb + acc_row(i, h) >= rmin)) ? x : -INFINITY);
        dp[i] = s[i] * (dp[i] - dr[i]) * a.scale;
      }
      mma_cols<T, DP>(dv, sG[buf], s, lane);
      mma_cols<T, DP>(dk, sQ[buf], dp, lane);
    }
    if (more) {
      st_q.store(sQ[buf ^ 1], tid);
      st_g.store(sG[buf ^ 1], tid);
      stat_put(buf ^ 1, rs);
    }
    __syncthreads();
  }
  if (key >= e.lk) return;
  store_row<T, DP>((T*)a.dK + (long)(e.k0 + key) * a.lddk + (long)kh * a.hsdk, dk, h, dim, 1.f);
  store_row<T, DP>((T*)a.dV + (long)(e.k0 + key) * a.lddv + (long)kh * a.hsdv, dv, h, dim, 1.f);
}

bool rows16(const void* p, int64_t ld, int64_t hs, int vec) { return ((uintptr_t)p % 16) == 0 && ld % vec == 0 && hs % vec == 0; }

int check_common(const char* what, int dtype, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim, int n_tiles, const int* cu_q,
                 const int* cu_k, const int* tiles) {
  CROG_CHECK_ARG(dtype == CROG_F32 || dtype == CROG_BF16, "%s: dtype must be CROG_F32 or CROG_BF16 (got %d)", what, dtype);
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(head_dim > 0 && head_dim <= 128 && head_dim % vec == 0, "%s: head_dim must be a multiple of %d up to 128 (got %d)", what, vec, head_dim);
  CROG_CHECK_ARG(seqs > 0 && rows_q > 0 && rows_k > 0 && kv_heads > 0 && group > 0 && n_tiles >= 0, "%s: bad sizes", what);
  CROG_CHECK_ARG((int64_t)rows_q * group <= 0x7fffff00 && (int64_t)n_tiles * kv_heads <= 0x7fffffff && rows_k <= 0x7fffff00, "%s: too many rows", what);
  CROG_CHECK_ARG(cu_q && cu_k && tiles, "%s: the sequence tables are missing", what);
  return CROG_OK;
}

}  // namespace

extern "C" int crog_packed_attn_fwd(int dtype, const void* Q, int64_t ldq, int64_t hsq, const void* K, int64_t ldk, int64_t hsk, const void* V,
                                    int64_t ldv, int64_t hsv, void* O, int64_t ldo, int64_t hso, float* lse, const int* cu_q, const int* cu_k,
                                    const int* tiles, int n_tiles, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim, float scale,
                                    int causal, int splits, int split_keys, float* partial, crog_stream_t stream) {
  if (int rc = check_common("packed_attn_fwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, n_tiles, cu_q, cu_k, tiles)) return rc;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(rows16(Q, ldq, hsq, vec) && rows16(K, ldk, hsk, vec) && rows16(V, ldv, hsv, vec) && rows16(O, ldo, hso, vec) && Q && K && V && O,
                 "packed_attn_fwd: heads of Q / K / V / O must start at 16-byte boundaries");
  CROG_CHECK_ARG(splits >= 1 && splits <= 65535 && (splits == 1 || (partial && split_keys > 0 && split_keys % 64 == 0)),
                 "packed_attn_fwd: %d splits need a workspace and a multiple of 64 keys each (got %d)", splits, split_keys);
  if (n_tiles == 0) return CROG_OK;
  PackedArgs a{};
  a.Q = Q; a.K = K; a.V = V; a.Out = O; a.lse = lse;
  a.ldq = ldq; a.hsq = hsq; a.ldk = ldk; a.hsk = hsk; a.ldv = ldv; a.hsv = hsv; a.ldo = ldo; a.hso = hso;
  a.cu_q = cu_q; a.cu_k = cu_k; a.tiles = tiles;
  a.seqs = seqs; a.rows_q = rows_q; a.rows_k = rows_k; a.kv_heads = kv_heads; a.group = group; a.dim = head_dim; a.scale = scale; a.causal = causal != 0;
  const int64_t total = (int64_t)kv_heads * rows_q * group;
  a.split_keys = splits > 1 ? split_keys : 0x7fffff00;
  if (splits > 1) { a.part_o = partial; a.part_ml = partial + (int64_t)splits * total * head_dim; }
  const dim3 grid((unsigned)(n_tiles * kv_heads), splits);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == CROG_BF16) {
    if (head_dim <= 64) packed_fwd_kernel<bf16, 64, 2><<<grid, NT, 0, s>>>(a);
    else packed_fwd_kernel<bf16, 128, 2><<<grid, NT, 0, s>>>(a);
  } else {
    if (head_dim <= 64) packed_fwd_kernel<float, 64, 1><<<grid, NT, 0, s>>>(a);
    else packed_fwd_kernel<float, 128, 1><<<grid, NT, 0, s>>>(a);
  }
  CROG_LAUNCH_CHECK();
  if (splits > 1) {
    if (dtype == CROG_BF16) packed_combine_kernel<bf16><<<cdiv(total, 4), NT, 0, s>>>(a, splits);
    else packed_combine_kernel<float><<<cdiv(total, 4), NT, 0, s>>>(a, splits);
    CROG_LAUNCH_CHECK();
  }
  return CROG_OK;
}

extern "C" int crog_packed_attn_bwd(int dtype, const void* Q, int64_t ldq, int64_t hsq, const void* K, int64_t ldk, int64_t hsk, const void* V,
                                    int64_t ldv, int64_t hsv, const void* O, int64_t ldo, int64_t hso, const void* dO, int64_t lddo, int64_t hsdo,
                                    const float* lse, float* D, void* dQ, int64_t lddq, int64_t hsdq, void* dK, int64_t lddk, int64_t hsdk, void* dV,
                                    int64_t lddv, int64_t hsdv, const int* cu_q, const int* cu_k, const int* row_tiles, int n_row_tiles,
                                    const int* key_tiles, int n_key_tiles, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim,
                                    float scale, int causal, crog_stream_t stream) {
  if (int rc = check_common("packed_attn_bwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, n_row_tiles, cu_q, cu_k, row_tiles)) return rc;
  if (int rc = check_common("packed_attn_bwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, n_key_tiles, cu_q, cu_k, key_tiles)) return rc;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(rows16(Q, ldq, hsq, vec) && rows16(K, ldk, hsk, vec) && rows16(V, ldv, hsv, vec) && rows16(O, ldo, hso, vec) && rows16(dO, lddo, hsdo, vec) &&
                 rows16(dQ, lddq, hsdq, vec) && rows16(dK, lddk, hsdk, vec) && rows16(dV, lddv, hsdv, vec) && Q && K && V && O && dO && lse && D && dQ && dK && dV,
                 "packed_attn_bwd: heads of Q / K / V / O / dO and the gradients must start at 16-byte boundaries");
  PackedArgs a{};
  a.Q = Q; a.K = K; a.V = V; a.O = O; a.dO = dO; a.lse = const_cast<float*>(lse); a.D = D; a.dQ = dQ; a.dK = dK; a.dV = dV;
  a.ldq = ldq; a.hsq = hsq; a.ldk = ldk; a.hsk = hsk; a.ldv = ldv; a.hsv = hsv; a.ldo = ldo; a.hso = hso; a.lddo = lddo; a.hsdo = hsdo;
  a.lddq = lddq; a.hsdq = hsdq; a.lddk = lddk; a.hsdk = hsdk; a.lddv = lddv; a.hsdv = hsdv;
  a.cu_q = cu_q; a.cu_k = cu_k;
  a.seqs = seqs; a.rows_q = rows_q; a.rows_k = rows_k; a.kv_heads = kv_heads; a.group = group; a.dim = head_dim; a.scale = scale; a.causal = causal != 0;
  hipStream_t s = (hipStream_t)stream;
  if (n_row_tiles > 0) {
    a.tiles = row_tiles;
    const unsigned n = (unsigned)(n_row_tiles * kv_heads);
    if (dtype == CROG_BF16) {
      if (head_dim <= 64) packed_bwd_dq_kernel<bf16, 64, 2><<<n, NT, 0, s>>>(a);
      else packed_bwd_dq_kernel<bf16, 128, 2><<<n, NT, 0, s>>>(a);
    } else {
      if (head_dim <= 64) packed_bwd_dq_kernel<float, 64, 1><<<n, NT, 0, s>>>(a);
      else packed_bwd_dq_kernel<float, 128, 1><<<n, NT, 0, s>>>(a);
    }
    CROG_LAUNCH_CHECK();
  }
  if (n_key_tiles > 0) {
    a.tiles = key_tiles;
    const unsigned n = (unsigned)(n_key_tiles * kv_heads);
    if (dtype == CROG_BF16) {
      if (head_dim <= 64) packed_bwd_dkdv_kernel<bf16, 64><<<n, NT, 0, s>>>(a);
      else packed_bwd_dkdv_kernel<bf16, 128><<<n, NT, 0, s>>>(a);
    } else {
      if (head_dim <= 64) packed_bwd_dkdv_kernel<float, 64><<<n, NT, 0, s>>>(a);
      else packed_bwd_dkdv_kernel<float, 128><<<n, NT, 0, s>>>(a);
    }
    CROG_LAUNCH_CHECK();
  }
  return CROG_OK;
}
