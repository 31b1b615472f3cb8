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
// Requests into LDS and their waits are assembly, so the compiler does not know when the resident operands (ordinary loads: qf, gf, kf, vf) have arrived.
// It guards their first use with a wait of its own, and that use stands inside each main loop, behind the request for a tile ahead: as compiled, every
// loop waits for what it has just requested (forward vmcnt(0), dQ vmcnt(1), dK / dV vmcnt(0), at 128 bf16 columns vmcnt(5)) before its first product.
#include "gemm_dma.h"
#include "packed_share.h"
#include <cmath>
#include <type_traits>

namespace {

constexpr int NT = 256;      // 4 waves
constexpr int BR = 128;      // rows of a block (forward, dQ)
constexpr int BK = 128;      // keys of a block (dK / dV)
constexpr int RT = 32;       // query rows of a dK / dV step

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

struct PackedArgs {
  const void *Q, *K, *V, *O, *dO;
  void *Out, *dQ, *dK, *dV;
  float *lse, *D;      // [heads][rows_q], lse in log2 units (+inf: no key, so that 2^(s - lse) is 0)
  float *part_o, *part_ml;
  long ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso, lddo, hsdo, lddq, hsdq, lddk, hsdk, lddv, hsdv;
  const int *cu_q, *cu_k, *tiles, *units;
  int seqs, rows_q, rows_k, kv_heads, group, dim, causal, split_keys, n_tiles, share, total;
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
// gemm_dma.h's request (its wait state after M0 too), to an LDS byte address and with a scalar offset besides the lane's (both below 2^31: their sum is out of range exactly where
// the lane's is DMA_OOB)
__device__ __attribute__((always_inline)) inline void dma_piece_at(const void* base, unsigned lds, unsigned off, unsigned soff) {
  const unsigned long long b = (unsigned long long)base;
  dma_i32x4 r;
  r.x = __builtin_amdgcn_readfirstlane((int)(unsigned)b);
  r.y = __builtin_amdgcn_readfirstlane((int)((unsigned)(b >> 32) & 0xffffu));
  r.z = 0x7fffffff;
  r.w = 0x00020000;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(r), "s"(soff) : "memory", "m0");
}
// the same with 4 bytes a lane
__device__ __attribute__((always_inline)) inline void dma_word_at(const void* base, unsigned lds, unsigned off) {
  const unsigned long long b = (unsigned long long)base;
  dma_i32x4 r;
  r.x = __builtin_amdgcn_readfirstlane((int)(unsigned)b);
  r.y = __builtin_amdgcn_readfirstlane((int)((unsigned)(b >> 32) & 0xffffu));
  r.z = 0x7fffffff;
  r.w = 0x00020000;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
__device__ inline unsigned lds_of(const void* p) {      // the LDS byte address of a shared array
  typedef __attribute__((address_space(3))) const char lds_char;
  return __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(lds_char*)p);
}
__device__ inline void opaque(int& x) { asm volatile("" : "+v"(x)); }      // keeps what is computed from x inside the loop it stands in

// (DP: elements of a row in LDS, 64 or 128; DC <= DP: the columns that enter the products, a multiple of 32)
template <typename T, int DP, int DC> struct Tile {
  static constexpr int VEC = Elem<T>::VEC, CPR = DP / VEC;      // 16-byte chunks per row
  static constexpr int NS = DC / VEC / 2;                       // 16-byte operand steps of a lane (its half takes every other chunk)
  static constexpr int NC = DC / 32;                            // 32-column blocks
  __device__ static constexpr int slot(int row) { return CPR == 8 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3)); }
  static constexpr int RB = DP * (int)sizeof(T);      // bytes of a row
  // Byte offsets of a lane in a tile.  Its other operands of the tile differ from these by XORs with constants and by whole rows (an instruction's
  // immediate), so a kernel keeps one register of each kind and XORs as it reads; all of them kept in registers made the backward kernels spill.
  // rows: row `ln`, 16-byte step 0.  (step ks: ^ 32 ks)
  __device__ static inline int rows_at(int lane) { return (lane & 31) * RB + (((lane >> 5) ^ slot(lane & 31)) << 4); }
  // columns: bf16, 4 rows x 4 columns of the transposed read (column block c: ^ 64 c, the rows 8 further down: ^ 32); float, one column
  __device__ static inline int cols_at(int lane) {
    const int h = lane >> 5, ln = lane & 31;
    if constexpr (sizeof(T) == 2) {
      const int q = (lane & 15) >> 2, pp = lane & 3, row = 4 * h + q;
      return row * RB + (((2 * ((lane >> 4) & 1) + (pp >> 1)) ^ slot(row)) << 4) + (pp & 1) * 8;
    } else {
      return 4 * h * RB + (((ln >> 2) ^ h) << 4) + (ln & 3) * 4;
    }
  }
};

__device__ inline int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }      // row of accumulator register r of half h
constexpr float LOG2E = 1.4426950408889634f;
__device__ inline float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// acc (32 rows of the tile x 32 columns = lanes) += tile rows . frag (the lane's row of the other operand).  at: rows_at + the buffer's offset
template <typename T, int DP, int DC>
__device__ inline void mma_rows(f32x16& acc, const T* tile, int at, int tile_row, const Vec16<T>* frag) {
  using L = Tile<T, DP, DC>;
#pragma unroll
  for (int ks = 0; ks < L::NS; ks++) {
    const Vec16<T> a = ldg16((const T*)((const char*)tile + (at ^ (ks << 5)) + tile_row * L::RB));
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, frag[ks]), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32((float)a.v[e], (float)frag[ks].v[e], acc, 0, 0, 0);
    }
  }
}

// out[c] (columns 32 c .. 32 c + 31 of the tile x lanes) += tile^T . p, p = 32 tile rows (registers, acc_row order) x lanes.  at: cols_at + ...
template <typename T, int DP, int DC>
__device__ inline void mma_cols(f32x16* out, const T* tile, int at, int tile_row, const f32x16& p) {
  using L = Tile<T, DP, DC>;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      bf16x8 b;      // (the probabilities are rounded to the operand type of the matrix unit: half a bf16 step each, as the inputs are)
#pragma unroll
      for (int j = 0; j < 8; j++) b[j] = (bf16)p[8 * t + j];
#pragma unroll
      for (int c = 0; c < L::NC; c++) {
        const char* base = (const char*)tile + (tile_row + 16 * t) * L::RB;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(base + (at ^ (c << 6))));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(base + 8 * L::RB + (at ^ (c << 6) ^ 32)));
        out[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), b, out[c], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; r++)
#pragma unroll
      for (int c = 0; c < L::NC; c++) {
        const int flip = ((8 * c) ^ ((r & 3) << 2) ^ (((r >> 2) & 1) << 1)) << 4;
        const float v = *(const float*)((const char*)tile + (at ^ flip) + (tile_row + (r & 3) + 8 * (r >> 2)) * L::RB);
        out[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[r], out[c], 0, 0, 0);
      }
  }
}

// p becomes what the rounding of mma_cols leaves of it.  With few keys or few rows these roundings do not average out (two keys: dQ off by twice its
// own rounding), so there, where a pass is launches and latency in any case, the rest goes through the matrix unit too.
constexpr int FEW = 128;
__device__ inline void leave_rest(f32x16& p) {
#pragma unroll
  for (int i = 0; i < 16; i++) p[i] -= (float)(bf16)p[i];
}

// the transposed operands of 16 tile rows from tile_row on, for all column blocks
template <typename T, int DP, int DC>
__device__ inline void load_cols(bf16x8* v, const T* tile, int at, int tile_row) {
  using L = Tile<T, DP, DC>;
#pragma unroll
  for (int c = 0; c < L::NC; c++) {
    const char* base = (const char*)tile + tile_row * L::RB;
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(base + (at ^ (c << 6))));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(base + 8 * L::RB + (at ^ (c << 6) ^ 32)));
    v[c] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// a lane's row of a resident operand, zeros behind the head dimension
template <typename T, int DP, int DC>
__device__ inline void load_frag(Vec16<T>* frag, const T* row, int h, int dim, bool valid) {
  using L = Tile<T, DP, DC>;
#pragma unroll
  for (int ks = 0; ks < L::NS; ks++) {
    const int at = (2 * ks + h) * L::VEC;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (valid && at < dim) v = *reinterpret_cast<const f32x4*>(row + at);
    frag[ks] = __builtin_bit_cast(Vec16<T>, v);
  }
}

// lane = row, registers = 32-column blocks: a row's D values as pieces of four
template <typename T, int DC>
__device__ inline void store_row(T* row, const f32x16* acc, int h, int dim, float f) {
#pragma unroll
  for (int c = 0; c < DC / 32; c++)
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

// R rows of a tile, fetched straight into LDS (gemm_dma.h: 1 KiB a request, 64 lanes x 16 bytes in LDS order; the swizzle is applied to the
// source address).  Rows that do not exist and columns behind the head dimension are requested out of range: the hardware writes zeros.  (A row
// of another sequence may hold infinities or NaN, and zero times those is NaN: it must not reach a product even with probability zero.)
// The lane's slot of a row is linear in the bits of the row's number, so request i differs from request 0 by an XOR and by whole rows, which go
// into the instruction's scalar offset: one v_xad a request.
template <typename T, int DP, int R> struct Fetch {
  using L = Tile<T, DP, DP>;
  static constexpr int NR = R * L::CPR / NT, RPR = 64 / L::CPR;      // requests of a wave, rows of a request
  int wave, lrow;
  int col;
  unsigned rows, ldb;      // col: byte offset in the row (request 0), of the row, of a row step
  __device__ inline void init(int wave_, int lane, long ld) {
    wave = wave_;
    lrow = wave * NR * RPR + lane / L::CPR;
    ldb = (unsigned)(ld * (long)sizeof(T));
    col = ((lane % L::CPR) ^ L::slot(lrow)) << 4;
    rows = (unsigned)lrow * ldb;
  }
  __device__ inline void get(unsigned tile, const T* base, int n, int dim) const {      // tile: LDS address, n: rows that exist
    const unsigned dst = tile + wave * NR * 1024;
    int col = this->col;
    opaque(col);
    if (n >= R && dim == DP) {
#pragma unroll
      for (int i = 0; i < NR; i++) dma_piece_at(base, dst + i * 1024, (unsigned)(col ^ (L::slot(i * RPR) << 4)) + rows, i * RPR * ldb);
    } else {
#pragma unroll
      for (int i = 0; i < NR; i++) {
        const unsigned c = (unsigned)(col ^ (L::slot(i * RPR) << 4));
        dma_piece_at(base, dst + i * 1024, (lrow + i * RPR < n && c < dim * sizeof(T)) ? c + rows + i * RPR * ldb : DMA_OOB, 0);
      }
    }
  }
};

// =====================================================================================================================
// forward.  grid (kv_heads * tiles, key splits); a block owns 128 rows of one sequence and key head, keys stream through LDS in two buffers of 64.
// Measured: one causal sequence of 16384 rows, 16 / 2 heads of 128: 1060 us, 1.04 PFLOP/s (a large library product reaches 1.24 here), at 1.9 GHz the matrix
// units busy 50 % of the clocks, the vector units 46 %; 32 sequences of 676 tokens, 8 heads of 64: 51 us, 0.6 PFLOP/s, matrix 25 %, vector 48 % (a maximum,
// a fused step, an exponential, a sum and a conversion an element).  Bound by neither unit alone but by one waiting for the other and both for the tile
// that each step has just requested (the waves wait 29 and 37 % of their time).  Single tokens (16 sequences of 200 to 8192 keys, 32 / 8 heads of 128:
// 71 + 5 us, 4.0 TB/s) wait for memory with nothing else in flight; with at most 32 rows one wave of four has products, the others fetch only.  64 rows a
// wave instead of 32, one wave a SIMD: 1370 us for the long sequence.  P is rounded to bf16 for the second product (mma_cols), the sum is of the float P.
// =====================================================================================================================
template <typename T, int DP, int DC, int NB>
__global__ void __launch_bounds__(NT, 2) packed_fwd_kernel(const PackedArgs a) {
  using L = Tile<T, DP, DC>;
  constexpr int KT = 32 * NB;
  __shared__ __attribute__((aligned(16))) T sK[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T sV[2][KT * DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, ln = lane & 31;
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  const int rows = e.lq * a.group, dim = a.dim;
  if (tile < 0 || (long)tile * BR >= rows) return;      // (uniform)
  const int r0 = tile * BR + wave * 32, r = r0 + ln;
  const int off = e.lk - e.lq;
  const int rc = min(r, rows - 1), qi = rc / a.group;
  const int lim = a.causal ? min(max(qi + 1 + off, 0), e.lk) : e.lk;      // the lane's row sees keys [0, lim)
  const auto limit = [&](int row) { return a.causal ? min(max(min(row, rows - 1) / a.group + 1 + off, 0), e.lk) : e.lk; };
  const int lim_lo = limit(r0), lim_hi = r0 < rows ? limit(r0 + 31) : 0;
  const int kbeg = (int)min((long)blockIdx.y * a.split_keys, (long)0x7fffff00);
  const int klast = limit(tile * BR + BR - 1), kend = blockIdx.y + 1 == gridDim.y ? klast : (int)min((long)klast, (long)kbeg + a.split_keys);

  Vec16<T> qf[L::NS];
  load_frag<T, DP, DC>(qf, (const T*)a.Q + (long)(e.q0 + qi) * a.ldq + (long)(kh * a.group + rc % a.group) * a.hsq, h, dim, r < rows);
  f32x16 o[L::NC];
#pragma unroll
  for (int c = 0; c < L::NC; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[c][i] = 0.f;
  float m = -INFINITY, mu = 0.f, l = 0.f;      // running maximum (log2 units), the same with 0 for -inf, the lane's share of the sum
  // the maximum is taken over the unscaled products: a negative scale goes to the queries' signs.  (A scale of zero becomes a tiny one: zero times
  // the -inf of a masked score would be NaN)
  const float c2 = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f);
  if (a.scale < 0.f)
#pragma unroll
    for (int ks = 0; ks < L::NS; ks++)
#pragma unroll
      for (int j = 0; j < L::VEC; j++) qf[ks].v[j] = -qf[ks].v[j];
  const int rows_at = L::rows_at(lane), cols_at = L::cols_at(lane);
  const T* kg = (const T*)a.K + (long)e.k0 * a.ldk + (long)kh * a.hsk;
  const T* vg = (const T*)a.V + (long)e.k0 * a.ldv + (long)kh * a.hsv;
  const unsigned lds_k = lds_of(sK), lds_v = lds_of(sV);
  Fetch<T, DP, KT> fk, fv;
  fk.init(wave, lane, a.ldk);
  fv.init(wave, lane, a.ldv);
  kg += (long)kbeg * a.ldk;
  vg += (long)kbeg * a.ldv;
  if (kbeg < kend) {
    fk.get(lds_k, kg, e.lk - kbeg, dim);
    fv.get(lds_v, vg, e.lk - kbeg, dim);
  }
  wait_vmcnt<0>();
  __syncthreads();
  int buf = 0;
  for (int kb = kbeg; kb < kend; kb += KT, buf ^= 1) {
    const bool more = kb + KT < kend;
    if (more) {      // (the barrier below: every wave is done with the other buffer)
      kg += KT * a.ldk;
      vg += KT * a.ldv;
      fk.get(lds_k + (buf ^ 1) * KT * L::RB, kg, e.lk - kb - KT, dim);
      fv.get(lds_v + (buf ^ 1) * KT * L::RB, vg, e.lk - kb - KT, dim);
    }
    if (kb < lim_hi) {      // (wave-uniform)
      int at_r = rows_at + buf * KT * L::RB, at_c = cols_at + buf * KT * L::RB;
      opaque(at_r);
      opaque(at_c);
      f32x16 s[NB];
      float mt = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[n][i] = 0.f;
        mma_rows<T, DP, DC>(s[n], sK[0], at_r, n * 32, qf);
      }
      if (kb + KT > lim_lo)
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 16; i++) s[n][i] = kb + n * 32 + acc_row(i, h) < lim ? s[n][i] : -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) mt = fmaxf(mt, s[n][i]);
      mt = xor32_max(mt) * c2;
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
      if constexpr (sizeof(T) == 2) {
        // 16 keys a group: the products of a group run while the next one's exponentials are formed
        constexpr int G = 2 * NB;
        bf16x8 v[2][L::NC], pb[2];
        const auto probs = [&](int g) {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float x = ex2(s[g / 2][8 * (g & 1) + j] * c2 - mu);
            l += x;
            pb[g & 1][j] = (bf16)x;
          }
        };
        load_cols<T, DP, DC>(v[0], sV[0], at_c, 0);
        probs(0);
#pragma unroll
        for (int g = 0; g < G; g++) {
          if (g + 1 < G) load_cols<T, DP, DC>(v[(g + 1) & 1], sV[0], at_c, (g + 1) * 16);
#pragma unroll
          for (int c = 0; c < L::NC; c++) o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[g & 1][c], pb[g & 1], o[c], 0, 0, 0);
          if (g + 1 < G) probs(g + 1);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NB; n++) {
#pragma unroll
          for (int i = 0; i < 16; i++) { s[n][i] = ex2(s[n][i] * c2 - mu); l += s[n][i]; }
          mma_cols<T, DP, DC>(o, sV[0], at_c, n * 32, s[n]);
        }
      }
    }
    wait_vmcnt<0>();
    __syncthreads();
  }
  l = xor32_sum(l);
  if (r >= rows) return;
  const int hd = rc - qi * a.group;
  if (a.part_o) {
    const long pr = ((long)blockIdx.y * a.kv_heads + kh) * a.rows_q * a.group + (long)e.q0 * a.group + r;
    store_row<float, DC>(a.part_o + pr * dim, o, h, dim, 1.f);
    if (h == 0) { a.part_ml[2 * pr] = m; a.part_ml[2 * pr + 1] = l; }
    return;
  }
  store_row<T, DC>((T*)a.Out + (long)(e.q0 + qi) * a.ldo + (long)(kh * a.group + hd) * a.hso, o, h, dim, l == 0.f ? 0.f : 1.f / l);
  if (h == 0 && a.lse) a.lse[(long)(kh * a.group + hd) * a.rows_q + e.q0 + qi] = l == 0.f ? INFINITY : m + __log2f(l);
}

// the splits of a row meet: o = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z.  W waves of a row take every W-th split each (W = 4 from 8 splits on: one
// row of 63 splits took 21.7 us on one wave); a lane takes the statistics of one of its wave's splits, so that their loads are in flight together.  The
// partial rows come one behind the other (the compiler does not unroll a loop of unknown length around a read of another lane).
template <typename T, int W>
__global__ void __launch_bounds__(NT) packed_combine_kernel(const PackedArgs a, int splits) {
  constexpr int ROWS = 4 / W;
  __shared__ float sm[4], part[4][3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave % W;
  const long per = (long)a.rows_q * a.group, total = a.kv_heads * per, row = (long)blockIdx.x * ROWS + wave / W;
  const int kh = (int)(min(row, total - 1) / per);
  const long rr = min(row, total - 1) - kh * per;
  // rows behind the last sequence have no partial result and stay as they are
  const bool live = row < total && rr < (long)min(a.cu_q[a.seqs], a.rows_q) * a.group;
  const auto stat = [&](int z, float& m, float& l) {
    const float2 v = live && z < splits ? *reinterpret_cast<const float2*>(a.part_ml + 2 * (z * total + row)) : make_float2(-INFINITY, 0.f);
    m = v.x;
    l = v.y;
  };
  float m, l, M = -INFINITY;
  for (int z0 = w; z0 < splits; z0 += 64 * W) {
    stat(z0 + lane * W, m, l);
    M = fmaxf(M, m);
  }
  M = wave_max(M);
  if constexpr (W > 1) {
    if (lane == 0) sm[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  }
  float sum = 0.f, o0 = 0.f, o1 = 0.f;
  const int c0 = min(lane, a.dim - 1), c1 = min(lane + 64, a.dim - 1);
  for (int z0 = w; z0 < splits; z0 += 64 * W) {
    stat(z0 + lane * W, m, l);
    // (a split without a key: m = -inf, l = 0, o = 0; one whose scores were all NaN: m = -inf, l NaN, which has to come through)
    const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - M);
    sum += f * l;
    const int n = live ? min(64, (splits - z0 + W - 1) / W) : 0;
    const float* p = a.part_o + (z0 * total + row) * a.dim;
    for (int z = 0; z < n; z++) {
      const float fz = readlane_f(f, z);
      o0 += fz * p[z * W * total * a.dim + c0];
      o1 += fz * p[z * W * total * a.dim + c1];
    }
  }
  sum = wave_sum(sum);
  if constexpr (W > 1) {
    part[wave][0][lane] = sum;
    part[wave][1][lane] = o0;
    part[wave][2][lane] = o1;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int k = 1; k < W; k++) {
      sum += part[k][0][lane];
      o0 += part[k][1][lane];
      o1 += part[k][2][lane];
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* op = (T*)a.Out + (rr / a.group) * a.ldo + (long)(kh * a.group + rr % a.group) * a.hso;
  if (lane < a.dim) op[lane] = Elem<T>::from_f(o0 * inv);
  if (lane + 64 < a.dim) op[lane + 64] = Elem<T>::from_f(o1 * inv);
  if (lane == 0 && a.lse) a.lse[(kh * a.group + rr % a.group) * a.rows_q + rr / a.group] = sum == 0.f ? INFINITY : M + __log2f(sum);
}
template <typename T>
void launch_combine(const PackedArgs& a, int splits, int64_t total, hipStream_t s) {
  if (splits < 8) packed_combine_kernel<T, 1><<<cdiv(total, 4), NT, 0, s>>>(a, splits);
  else packed_combine_kernel<T, 4><<<(unsigned)total, NT, 0, s>>>(a, splits);
}

// =====================================================================================================================
// backward 1: D and dQ, blocked as the forward, its few rows over long keys cut in the same way (the float sums meet in packed_dq_sum_kernel).  Three
// products a tile, of which S and dP are formed again by the next kernel (nine in all with the forward's, where seven are needed): counting all three,
// 1.1 PFLOP/s at 128 columns (four sequences of 4096 rows, 16 / 4 heads: 730 us), 0.66 at 64 (32 of 676 tokens, 8 heads: 69 us; matrix units busy 29 %,
// vector units 41 % of the clocks).  P and dS are rounded to bf16 for their products.  float: 17 registers spilled at 128 columns, two at 96.
// =====================================================================================================================
template <typename T, int DP, int DC, int NB>
__global__ void __launch_bounds__(NT, sizeof(T) == 2 && DC <= 32 ? 4 : 2) packed_bwd_dq_kernel(const PackedArgs a) {
  using L = Tile<T, DP, DC>;
  constexpr int KT = 32 * NB;
  __shared__ __attribute__((aligned(16))) T sK[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T sV[2][KT * DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, ln = lane & 31;
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  const int rows = e.lq * a.group, dim = a.dim;
  if (tile < 0 || (long)tile * BR >= rows) return;
  const int r0 = tile * BR + wave * 32, r = r0 + ln;
  const int off = e.lk - e.lq;
  const int rc = min(r, rows - 1), qi = rc / a.group;
  const int lim = a.causal ? min(max(qi + 1 + off, 0), e.lk) : e.lk;
  const auto limit = [&](int row) { return a.causal ? min(max(min(row, rows - 1) / a.group + 1 + off, 0), e.lk) : e.lk; };
  const int lim_lo = limit(r0), lim_hi = r0 < rows ? limit(r0 + 31) : 0;
  const int klast = limit(tile * BR + BR - 1), kbeg = (int)min((long)blockIdx.y * a.split_keys, (long)0x7fffff00);
  const int kend = blockIdx.y + 1 == gridDim.y ? klast : (int)min((long)klast, (long)kbeg + a.split_keys);
  const long row_g = e.q0 + qi, head = (long)kh * a.group + rc % a.group;
  const long at = head * a.rows_q + row_g;

  Vec16<T> qf[L::NS], gf[L::NS];
  load_frag<T, DP, DC>(qf, (const T*)a.Q + row_g * a.ldq + head * a.hsq, h, dim, r < rows);
  load_frag<T, DP, DC>(gf, (const T*)a.dO + row_g * a.lddo + head * a.hsdo, h, dim, r < rows);
  // D = dO . o; of a row that sees the first key tile alone, sum_j P_ij dP_ij from the tile itself, unrounded (the stored o is off by half a step,
  // which few keys do not average out: sequences of up to 147 causal rows had dQ off by 0.0026 of its norm, 0.0024 with this)
  float Dr = 0.f;
  if (lim_hi > KT) {
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
  }
  const float lse = a.lse[at], c2 = a.scale * LOG2E;
  const int rows_at = L::rows_at(lane), cols_at = L::cols_at(lane);
  f32x16 dq[L::NC];
#pragma unroll
  for (int c = 0; c < L::NC; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) dq[c][i] = 0.f;
  const T* kg = (const T*)a.K + (long)e.k0 * a.ldk + (long)kh * a.hsk;
  const T* vg = (const T*)a.V + (long)e.k0 * a.ldv + (long)kh * a.hsv;
  const unsigned lds_k = lds_of(sK), lds_v = lds_of(sV);
  Fetch<T, DP, KT> fk, fv;
  fk.init(wave, lane, a.ldk);
  fv.init(wave, lane, a.ldv);
  kg += (long)kbeg * a.ldk;
  vg += (long)kbeg * a.ldv;
  if (kbeg < kend) {
    fk.get(lds_k, kg, e.lk - kbeg, dim);
    fv.get(lds_v, vg, e.lk - kbeg, dim);
  }
  const auto probs = [&](int kb, int at_r, int n, f32x16& s, f32x16& dp) {      // P and dP of 32 keys
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = dp[i] = 0.f;
    __builtin_amdgcn_s_setprio(1);
    mma_rows<T, DP, DC>(s, sK[0], at_r, n * 32, qf);
    mma_rows<T, DP, DC>(dp, sV[0], at_r, n * 32, gf);
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = s[i] * c2 - lse;
    if (kb + KT > lim_lo)
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = kb + n * 32 + acc_row(i, h) < lim ? s[i] : -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = ex2(s[i]);
  };
  wait_vmcnt<0>();
  __syncthreads();
  if (kbeg == 0 && lim_lo <= KT && lim_hi > 0) {
    float d = 0.f;
#pragma unroll 1
    for (int n = 0; n < NB; n++) {
      f32x16 s, dp;
      probs(0, rows_at, n, s, dp);
#pragma unroll
      for (int i = 0; i < 16; i++) d += s[i] * dp[i];
    }
    d = xor32_sum(d);
    Dr = lim <= KT ? d : Dr;
  }
  int buf = 0;
  for (int kb = kbeg; kb < kend; kb += KT, buf ^= 1) {
    const bool more = kb + KT < kend;
    if (more) {      // (the barrier below: every wave is done with the other buffer)
      kg += KT * a.ldk;
      vg += KT * a.ldv;
      fk.get(lds_k + (buf ^ 1) * KT * L::RB, kg, e.lk - kb - KT, dim);
      fv.get(lds_v + (buf ^ 1) * KT * L::RB, vg, e.lk - kb - KT, dim);
    }
    if (kb < lim_hi) {
      int at_r = rows_at + buf * KT * L::RB, at_c = cols_at + buf * KT * L::RB;
      opaque(at_r);
      opaque(at_c);
      f32x16 s, dp;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        probs(kb, at_r, n, s, dp);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = s[i] * (dp[i] - Dr);      // (the scale follows at the end)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll 1
        for (int again = sizeof(T) == 2 && min(rows, lim_hi) <= FEW;; again--) {
          mma_cols<T, DP, DC>(dq, sK[0], at_c, n * 32, s);
          if (!again) break;
          leave_rest(s);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
    wait_vmcnt<0>();
    __syncthreads();
  }
  if (r >= rows) return;
  if (h == 0 && blockIdx.y == 0) a.D[at] = -Dr;      // (dK / dV begins its product with it)
  if (a.part_o) {
    store_row<float, DC>(a.part_o + ((long)blockIdx.y * a.kv_heads * a.group * a.rows_q + at) * dim, dq, h, dim, a.scale);
    return;
  }
  store_row<T, DC>((T*)a.dQ + row_g * a.lddq + head * a.hsdq, dq, h, dim, a.scale);
}

// dQ = the splits' sums in order.  16 threads a row of four columns each, twice
template <typename T>
__global__ void __launch_bounds__(NT) packed_dq_sum_kernel(const PackedArgs a, int splits) {
  const long total = (long)a.kv_heads * a.group * a.rows_q, at = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const long head = at / a.rows_q, row = at - head * a.rows_q;
  // rows behind the last sequence have no partial result and stay as they are
  if (at >= total || row >= min(a.cu_q[a.seqs], a.rows_q)) return;
  for (int c = (threadIdx.x & 15) * 4; c < a.dim; c += 64) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int z = 0; z < splits; z++) v += *reinterpret_cast<const f32x4*>(a.part_o + (z * total + at) * a.dim + c);
    T* p = (T*)a.dQ + row * a.lddq + head * a.hsdq + c;
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = Elem<T>::from_f(v[j]);
  }
}

// =====================================================================================================================
// backward 2: dK, dV.  A block takes 128 keys at a time, 32 a wave, and the group's query rows stream past them through a ring of four LDS tiles of
// 32 rows, requested three steps ahead (of which the compiler's wait, see the top, leaves the step's own request: the counted waits below never bind).
// bf16 at 128 columns: seven registers spilled, two of them read back in the partial form of the request, which head dimensions 104 to 120 take each step.
// A key tile's steps are 32 queries (of a grid from the sequence's first) of one head each, from the LAST queries backwards, the group's heads
// inside: every key tile of a sequence starts with the same step.
// The steps of all tiles lie one behind the other on one axis, each tile's with OPERANDS units more for its operands and results, and every block takes an
// equal share of that axis (share > 0): causal or ragged tiles have anything between one step and thousands, and in pieces of equal length left CUs
// idle for a quarter of the time (six causal sequences of up to 5000 rows, 16 / 4 heads of 128: 796 + 16 us to meet, in shares 632 + 26, 0.99
// PFLOP/s counting all four products; where every block has as many steps in any case 1.1; matrix units busy 46 % of the clocks at 2.07 GHz).  A tile that lies in several shares leaves a float sum in each, two places a block, which meet in
// packed_meet_kernel in order.  share 0: a block a tile.
// =====================================================================================================================
__device__ inline int steps_of(const PackedArgs& a, const Seq& e, int tile) {
  const int first = a.causal ? min(max(tile * BK - (e.lk - e.lq), 0), e.lq) : 0;
  return ((e.lq + RT - 1) / RT - first / RT) * a.group;
}

// the kernel's argument, loaded where it is used again: kept in registers through a loop of segments, its 60 words did not fit beside the loop's own
__device__ inline PackedArgs args_again() {
#ifdef __HIP_DEVICE_COMPILE__
  auto p = (const __attribute__((address_space(4))) PackedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
#else
  return {};      // (the host's pass has no address spaces)
#endif
}

template <typename T, int DP, int DC>
__global__ void __launch_bounds__(NT, sizeof(T) == 2 ? DC <= 32 ? 4 : DC <= 64 ? 3 : 2 : 1) packed_bwd_dkdv_kernel(const PackedArgs args) {
  using L = Tile<T, DP, DC>;
  using F = Fetch<T, DP, RT>;
  constexpr int RING = 4, REQ = 2 * F::NR + 2;      // tiles of the ring, requests of a wave and step
  __shared__ __attribute__((aligned(16))) T sQ[RING][RT * DP];
  __shared__ __attribute__((aligned(16))) T sG[RING][RT * DP];
  __shared__ __attribute__((aligned(16))) float sS[RING][4][2][64];      // every wave fetches its own lse and D (32 of the 64): all have as many requests
  int kh, ti, block = blockIdx.x;
  long pos = 0, end = 1;
  if (args.share == 0) {
    kh = block % args.kv_heads;
    ti = block / args.kv_heads;
  } else {
    // neighbouring shares on one XCD: they read the same rows (workgroups go round the 8 XCDs; the grid is a multiple of 8)
    block = block % 8 * (gridDim.x / 8) + block / 8;
    const Place p = place_of(args.units, args.n_tiles, args.total, args.kv_heads, args.share, block);
    if (p.pos >= p.end) return;
    pos = p.pos;
    end = p.end;
    kh = p.kh;
    ti = p.ti;
  }
  while (pos < end) {
    const PackedArgs a = args_again();
    int tid = threadIdx.x;
    opaque(tid);      // (what depends on the lane alone is formed again for each segment too)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, ln = lane & 31;
    const int dim = a.dim;
    const int tile = a.tiles[2 * ti + 1];
    const Seq e = seq_of(a, a.tiles[2 * ti]);
    const int all = steps_of(a, e, tile);
    int first = 0, last = all, slot = -1;      // steps of this segment; place of its float sum (-1: the whole tile)
    const int hn = kh;
    if (a.share == 0) {
      pos = end;
    } else {
      // (the heads' axes from the total in the table, which is a.total: held through the loop that one spilled, six causal sequences to 5000 rows, backward 885 -> 898 us)
      const Segment seg = segment_of(pos, end, block, (long)kh * a.units[a.n_tiles] + a.units[ti], units_of(a.units, ti), all);
      first = seg.first;
      last = seg.last;
      slot = seg.slot;
      pos = seg.next;
      if (++ti == a.n_tiles) {
        ti = 0;
        kh = min(kh + 1, a.kv_heads - 1);
      }
    }
    if (tile < 0 || (long)tile * BK >= e.lk) continue;      // (uniform)
    const int k0 = tile * BK + wave * 32, key = k0 + ln, kc = min(key, e.lk - 1);
    const int off = e.lk - e.lq;
    const int qmin = a.causal ? key - off : 0;      // the lane's key is seen by queries >= qmin
    const int wbeg = a.causal ? k0 - off : 0, wall = a.causal ? k0 + 31 - off : 0;      // the wave's first query at all, its first that sees all its keys
    const long hd0 = (long)hn * a.group;

    Vec16<T> kf[L::NS], vf[L::NS];
    load_frag<T, DP, DC>(kf, (const T*)a.K + (long)(e.k0 + kc) * a.ldk + (long)hn * a.hsk, h, dim, key < e.lk);
    load_frag<T, DP, DC>(vf, (const T*)a.V + (long)(e.k0 + kc) * a.ldv + (long)hn * a.hsv, h, dim, key < e.lk);
    f32x16 dk[L::NC], dv[L::NC];
#pragma unroll
    for (int c = 0; c < L::NC; c++)
#pragma unroll
      for (int i = 0; i < 16; i++) dk[c][i] = dv[c][i] = 0.f;
    const float c2 = fabsf(a.scale) * LOG2E < 1e-30f ? 1e-30f : a.scale * LOG2E;      // (0 times a masked score's infinity would be NaN)
    const float masked = c2 > 0.f ? -INFINITY : INFINITY;
    F fq, fg;
    fq.init(wave, lane, a.ldq);
    fg.init(wave, lane, a.lddo);
    const unsigned lds_q = lds_of(sQ), lds_g = lds_of(sG), lds_s = lds_of(sS) + wave * 2 * 64 * 4;
    const int rows_at = L::rows_at(lane), cols_at = L::cols_at(lane);

    // the next step to be requested: its head and first query, and running pointers to its rows
    int hd = first % a.group, q = ((e.lq + RT - 1) / RT - 1 - first / a.group) * RT;
    const T* qp = (const T*)a.Q + (long)(e.q0 + q) * a.ldq + (hd0 + hd) * a.hsq;
    const T* gp = (const T*)a.dO + (long)(e.q0 + q) * a.lddo + (hd0 + hd) * a.hsdo;
    const float *lp = a.lse + (hd0 + hd) * a.rows_q + e.q0 + q, *Dp = a.D + (hd0 + hd) * a.rows_q + e.q0 + q;
    const long next_q = RT * a.ldq + (a.group - 1) * a.hsq, next_g = RT * a.lddo + (a.group - 1) * a.hsdo, next_s = RT + (a.group - 1) * (long)a.rows_q;
    const auto request = [&](int slot) {      // (rows that do not exist are zeros throughout: their dS is 0 and their dO is)
      fq.get(lds_q + slot * RT * L::RB, qp, e.lq - q, dim);
      fg.get(lds_g + slot * RT * L::RB, gp, e.lq - q, dim);
      const unsigned so = lane < RT && q + lane < e.lq ? lane * 4 : DMA_OOB;
      dma_word_at(lp, lds_s + slot * 4 * 2 * 64 * 4, so);
      dma_word_at(Dp, lds_s + slot * 4 * 2 * 64 * 4 + 64 * 4, so);
      if (++hd < a.group) {
        qp += a.hsq;
        gp += a.hsdo;
        lp += a.rows_q;
        Dp += a.rows_q;
      } else {      // the first head of the queries before
        hd = 0;
        q -= RT;
        qp -= next_q;
        gp -= next_g;
        lp -= next_s;
        Dp -= next_s;
      }
    };
    wait_vmcnt<0>();      // (the operands above: from here on only requests are counted)
    __syncthreads();      // (every wave is done with the segment before)
    const int steps = last - first;
#pragma unroll
    for (int i = 0; i < RING - 1; i++)
      if (i < steps) request(i);
    int hd_now = first % a.group, q_now = ((e.lq + RT - 1) / RT - 1 - first / a.group) * RT;
    for (int st = 0; st < steps; st++) {
      // this step's tile is there, and (the barrier) every wave is done with the one before, whose place the step three ahead takes
      if (st + 2 < steps) wait_vmcnt<2 * REQ>();
      else if (st + 1 < steps) wait_vmcnt<REQ>();
      else wait_vmcnt<0>();
      __syncthreads();
      if (st + RING - 1 < steps) request((st + RING - 1) % RING);
      const int r0 = q_now;
      if (++hd_now == a.group) {
        hd_now = 0;
        q_now -= RT;
      }
      if (k0 >= e.lk || r0 + RT <= wbeg) continue;
      const int buf = st % RING;
      int at_r = rows_at + buf * RT * L::RB, at_c = cols_at + buf * RT * L::RB;
      opaque(at_r);
      opaque(at_c);
      f32x16 s, dp;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(&sS[buf][wave][1][8 * g + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[4 * g + j] = 0.f;
          dp[4 * g + j] = d4[j];      // (-D: the product adds dO . v)
        }
      }
      __builtin_amdgcn_s_setprio(1);      // (products first, where the waves of a SIMD compete: 32 sequences of 676 tokens, a training pass 246 -> 221 us)
      mma_rows<T, DP, DC>(s, sQ[0], at_r, 0, kf);
      mma_rows<T, DP, DC>(dp, sG[0], at_r, 0, vf);
      __builtin_amdgcn_s_setprio(0);
      if (r0 < wall)
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = r0 + acc_row(i, h) >= qmin ? s[i] : masked;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(&sS[buf][wave][0][8 * g + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int i = 4 * g + j;
          s[i] = ex2(s[i] * c2 - l4[j]);
          dp[i] *= s[i];      // (the scale follows at the end)
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll 1
      for (int again = sizeof(T) == 2 && e.lq <= FEW;; again--) {
        mma_cols<T, DP, DC>(dv, sG[0], at_c, 0, s);
        mma_cols<T, DP, DC>(dk, sQ[0], at_c, 0, dp);
        if (!again) break;
        leave_rest(s);
        leave_rest(dp);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (key < e.lk && slot >= 0) {
      float* p = a.part_o + ((long)slot * BK + wave * 32 + ln) * 2 * dim;
      store_row<float, DC>(p, dk, h, dim, a.scale);
      store_row<float, DC>(p + dim, dv, h, dim, 1.f);
    } else if (key < e.lk) {
      store_row<T, DC>((T*)a.dK + (long)(e.k0 + key) * a.lddk + (long)hn * a.hsdk, dk, h, dim, a.scale);
      store_row<T, DC>((T*)a.dV + (long)(e.k0 + key) * a.lddv + (long)hn * a.hsdv, dv, h, dim, 1.f);
    }
  }
}

// dK, dV of the key tiles in several shares, summed in order.  grid (kv_heads * key tiles, chunks of 16 keys)
template <typename T>
__global__ void __launch_bounds__(NT) packed_meet_kernel(const PackedArgs a, int blocks) {
  const int kh = blockIdx.x % a.kv_heads, ti = blockIdx.x / a.kv_heads;
  const int tile = a.tiles[2 * ti + 1];
  const Seq e = seq_of(a, a.tiles[2 * ti]);
  if (tile < 0 || (long)tile * BK + blockIdx.y * 16 >= e.lk) return;
  const Meeting meet = meeting_of((long)kh * a.units[a.n_tiles] + a.units[ti], units_of(a.units, ti), a.share, blocks);
  const int b0 = meet.first, b1 = meet.last;
  if (b0 >= b1) return;
  const int k0 = blockIdx.y * 16, keys = min(16, e.lk - tile * BK - k0), per = 2 * a.dim / 4;
  for (int i = threadIdx.x; i < keys * per; i += NT) {
    const int k = k0 + i / per, c = (i % per) * 4;
    const auto sum_of = [&](int slot) { return *reinterpret_cast<const f32x4*>(a.part_o + ((long)slot * BK + k) * 2 * a.dim + c); };
    f32x4 v = sum_of(2 * b0 + 1);
#pragma unroll 4
    for (int b = b0 + 1; b <= b1; b++) v += sum_of(2 * b);
    const long key = e.k0 + tile * BK + k;
    T* p = c < a.dim ? (T*)a.dK + key * a.lddk + (long)kh * a.hsdk + c : (T*)a.dV + key * a.lddv + (long)kh * a.hsdv + c - a.dim;
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = Elem<T>::from_f(v[j]);
  }
}

// calls f(T{}, columns of a tile row, columns of the products) for a type and head dimension
template <typename F>
void for_dim(int dtype, int head_dim, F f) {
  using std::integral_constant;
  const auto pick = [&](auto t) {
    if (head_dim <= 32) f(t, integral_constant<int, 64>{}, integral_constant<int, 32>{});
    else if (head_dim <= 64) f(t, integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else if (head_dim <= 96) f(t, integral_constant<int, 128>{}, integral_constant<int, 96>{});
    else f(t, integral_constant<int, 128>{}, integral_constant<int, 128>{});
  };
  if (dtype == CROG_BF16) pick(bf16{});
  else pick(float{});
}

bool rows16(const void* p, int64_t ld, int64_t hs, int vec) { return ((uintptr_t)p % 16) == 0 && ld % vec == 0 && hs % vec == 0; }

// the rows of one tile lie within 2^31 bytes (32-bit offsets of the LDS requests)
bool near(int64_t ld, int dtype) { return ld >= 0 && ld * 64 * (dtype == CROG_BF16 ? 2 : 4) < 0x7fff0000; }

int check_common(const char* what, int dtype, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim, float scale, int n_tiles,
                 const int* cu_q, const int* cu_k, const int* tiles) {
  CROG_CHECK_ARG(dtype == CROG_F32 || dtype == CROG_BF16, "%s: dtype must be CROG_F32 or CROG_BF16 (got %d)", what, dtype);
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(head_dim > 0 && head_dim <= 128 && head_dim % vec == 0, "%s: head_dim must be a multiple of %d up to 128 (got %d)", what, vec, head_dim);
  CROG_CHECK_ARG(seqs > 0 && rows_q > 0 && rows_k > 0 && kv_heads > 0 && group > 0 && n_tiles >= 0, "%s: bad sizes", what);
  CROG_CHECK_ARG((int64_t)rows_q * group <= 0x7fffff00 && (int64_t)n_tiles * kv_heads <= 0x7fffffff && rows_k <= 0x7fffff00, "%s: too many rows", what);
  CROG_CHECK_ARG(std::isfinite(scale * LOG2E), "%s: scale times log2(e) must be finite (got %g)", what, scale);
  CROG_CHECK_ARG(cu_q && cu_k && tiles, "%s: the sequence tables are missing", what);
  return CROG_OK;
}

}  // namespace

extern "C" int crog_packed_attn_fwd(int dtype, const void* Q, int64_t ldq, int64_t hsq, const void* K, int64_t ldk, int64_t hsk, const void* V,
                                    int64_t ldv, int64_t hsv, void* O, int64_t ldo, int64_t hso, float* lse, const int* cu_q, const int* cu_k,
                                    const int* tiles, int n_tiles, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim, float scale,
                                    int causal, int splits, int split_keys, float* partial, crog_stream_t stream) {
  if (int rc = check_common("packed_attn_fwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, scale, n_tiles, cu_q, cu_k, tiles)) return rc;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(rows16(Q, ldq, hsq, vec) && rows16(K, ldk, hsk, vec) && rows16(V, ldv, hsv, vec) && rows16(O, ldo, hso, vec) && Q && K && V && O,
                 "packed_attn_fwd: heads of Q / K / V / O must start at 16-byte boundaries");
  CROG_CHECK_ARG(near(ldk, dtype) && near(ldv, dtype), "packed_attn_fwd: 64 key rows must lie within 2 GiB");
  CROG_CHECK_ARG(splits == 1 || (int64_t)kv_heads * rows_q * group <= 0x7fffffff, "packed_attn_fwd: too many rows for splits");
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
  for_dim(dtype, head_dim, [&](auto t, auto dp, auto dc) {
    using T = decltype(t);
    packed_fwd_kernel<T, dp(), dc(), sizeof(T) == 2 ? 2 : 1><<<grid, NT, 0, s>>>(a);
  });
  CROG_LAUNCH_CHECK();
  if (splits > 1) {
    if (dtype == CROG_BF16) launch_combine<bf16>(a, splits, total, s);
    else launch_combine<float>(a, splits, total, s);
    CROG_LAUNCH_CHECK();
  }
  return CROG_OK;
}

extern "C" int crog_packed_attn_bwd(int dtype, const void* Q, int64_t ldq, int64_t hsq, const void* K, int64_t ldk, int64_t hsk, const void* V,
                                    int64_t ldv, int64_t hsv, const void* O, int64_t ldo, int64_t hso, const void* dO, int64_t lddo, int64_t hsdo,
                                    const float* lse, float* D, void* dQ, int64_t lddq, int64_t hsdq, void* dK, int64_t lddk, int64_t hsdk, void* dV,
                                    int64_t lddv, int64_t hsdv, const int* cu_q, const int* cu_k, const int* row_tiles, int n_row_tiles,
                                    const int* key_tiles, int n_key_tiles, int seqs, int rows_q, int rows_k, int kv_heads, int group, int head_dim,
                                    float scale, int causal, int splits, int split_keys, const int* key_units,
                                    int total_units, int share, float* partial, crog_stream_t stream) {
  if (int rc = check_common("packed_attn_bwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, scale, n_row_tiles, cu_q, cu_k, row_tiles)) return rc;
  if (int rc = check_common("packed_attn_bwd", dtype, seqs, rows_q, rows_k, kv_heads, group, head_dim, scale, n_key_tiles, cu_q, cu_k, key_tiles)) return rc;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  CROG_CHECK_ARG(rows16(Q, ldq, hsq, vec) && rows16(K, ldk, hsk, vec) && rows16(V, ldv, hsv, vec) && rows16(O, ldo, hso, vec) && rows16(dO, lddo, hsdo, vec) &&
                 rows16(dQ, lddq, hsdq, vec) && rows16(dK, lddk, hsdk, vec) && rows16(dV, lddv, hsdv, vec) && Q && K && V && O && dO && lse && D && dQ && dK && dV,
                 "packed_attn_bwd: heads of Q / K / V / O / dO and the gradients must start at 16-byte boundaries");
  CROG_CHECK_ARG(splits >= 1 && splits <= 65535 && (splits == 1 || (partial && split_keys > 0 && split_keys % 64 == 0)),
                 "packed_attn_bwd: %d splits need a workspace and a multiple of 64 keys each (got %d)", splits, split_keys);
  CROG_CHECK_ARG(share >= 0 && (share == 0 || (key_units && total_units >= n_key_tiles && partial && cdiv((int64_t)total_units * kv_heads, share) < (1 << 24))),
                 "packed_attn_bwd: shares of %d units need their table (%d units) and a workspace", share, total_units);
  CROG_CHECK_ARG(near(ldk, dtype) && near(ldv, dtype) && near(ldq, dtype) && near(lddo, dtype),
                 "packed_attn_bwd: 64 rows must lie within 2 GiB");
  PackedArgs a{};
  a.Q = Q; a.K = K; a.V = V; a.O = O; a.dO = dO; a.lse = const_cast<float*>(lse); a.D = D; a.dQ = dQ; a.dK = dK; a.dV = dV;
  a.ldq = ldq; a.hsq = hsq; a.ldk = ldk; a.hsk = hsk; a.ldv = ldv; a.hsv = hsv; a.ldo = ldo; a.hso = hso; a.lddo = lddo; a.hsdo = hsdo;
  a.lddq = lddq; a.hsdq = hsdq; a.lddk = lddk; a.hsdk = hsdk; a.lddv = lddv; a.hsdv = hsdv;
  a.cu_q = cu_q; a.cu_k = cu_k;
  a.seqs = seqs; a.rows_q = rows_q; a.rows_k = rows_k; a.kv_heads = kv_heads; a.group = group; a.dim = head_dim; a.scale = scale; a.causal = causal != 0;
  hipStream_t s = (hipStream_t)stream;
  if (n_row_tiles > 0) {
    a.tiles = row_tiles;
    a.split_keys = splits > 1 ? split_keys : 0x7fffff00;
    a.part_o = splits > 1 ? partial : nullptr;
    const dim3 n((unsigned)(n_row_tiles * kv_heads), splits);
    for_dim(dtype, head_dim, [&](auto t, auto dp, auto dc) {
      using T = decltype(t);
      packed_bwd_dq_kernel<T, dp(), dc(), sizeof(T) == 2 ? 2 : 1><<<n, NT, 0, s>>>(a);
    });
    CROG_LAUNCH_CHECK();
    if (splits > 1) {
      const unsigned blocks = (unsigned)cdiv((int64_t)kv_heads * group * rows_q, 16);
      if (dtype == CROG_BF16) packed_dq_sum_kernel<bf16><<<blocks, NT, 0, s>>>(a, splits);
      else packed_dq_sum_kernel<float><<<blocks, NT, 0, s>>>(a, splits);
      CROG_LAUNCH_CHECK();
    }
  }
  if (n_key_tiles > 0) {
    a.tiles = key_tiles;
    a.n_tiles = n_key_tiles;
    a.units = key_units;
    a.share = share;
    a.part_o = partial;
    const unsigned n = (unsigned)(n_key_tiles * kv_heads), blocks = share > 0 ? (unsigned)cdiv((int64_t)total_units * kv_heads, share) : n;
    a.total = total_units;
    const unsigned grid = share > 0 ? (blocks + 7) / 8 * 8 : n;
    for_dim(dtype, head_dim, [&](auto t, auto dp, auto dc) { packed_bwd_dkdv_kernel<decltype(t), dp(), dc()><<<grid, NT, 0, s>>>(a); });
    CROG_LAUNCH_CHECK();
    if (share > 0) {
      if (dtype == CROG_BF16) packed_meet_kernel<bf16><<<dim3(n, BK / 16), NT, 0, s>>>(a, (int)blocks);
      else packed_meet_kernel<float><<<dim3(n, BK / 16), NT, 0, s>>>(a, (int)blocks);
      CROG_LAUNCH_CHECK();
    }
  }
  return CROG_OK;
}
