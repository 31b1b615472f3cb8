// Rotary positions with several axes (crog_rotary): the first 2 * pairs columns of each head are pairs (a, b), and pair i of a row turns by
//   angle = positions[row][axis(i)] * theta^(-place of i in its axis / pairs of its axis):   (a, b) -> (a cos - b sin, b cos + a sin)
// so that the product of a query and a key depends on the DIFFERENCE of their positions along every axis (time, height, width of a video token;
// one axis for text).  The columns behind the pairs are copied.  The backward pass is the same rotation by minus the angle.
//
// Angles.  A far position turns a fast pair thousands of times, so the product is formed in 64 bits, in revolutions; what is left of it after
// the whole turns (|x| <= 1/2) is rounded once to 32 bits (2^-25 of a half turn) before the sine and cosine.
// Bound: memory, each element read and written once (16384 rows of 16 + 4 heads x 128, bf16, 168 MB: 33.2 us, 5.0 TB/s, what a large copy reaches).  A
// block takes TOK rows and computes their pairs' sines and cosines ONCE, into LDS, for all query and key heads of the row (40 heads x 64 pairs share 64
// angles).  Not at that rate: columns behind the pairs, which are copied element by element, and calls whose pairs are no whole vectors (20 pairs of a head
// of 80, bf16) or whose heads are not aligned, which go element by element throughout.
#include "common.h"

namespace {

constexpr int NT = 256, MAXP = 128;      // pairs of a head at most

struct RotArgs {
  const void *Q, *K;
  void *Qo, *Ko;
  long ldq, hsq, ldk, hsk, ldqo, hsqo, ldko, hsko;
  const void* pos;
  const double* rev;      // [pairs] revolutions per unit of position
  const int* axis;        // [pairs]
  long ldpos;
  int rows, heads_q, heads_k, dim, pairs, axes, pos64, inverse;
};

// The fused steps are written out: left to the compiler, the variants below fused different ones of the two products, and the same pair came out
// one fp32 step apart (now and then a bf16 one) with another alignment.
__device__ inline void turn(float& x, float& y, float c, float s) {
  const float x1 = fmaf(-y, s, x * c);
  y = fmaf(x, s, y * c);
  x = x1;
}

// PV: pairs of one work item (16 bytes of each half, or PV interleaved pairs)
template <typename T, int PV, bool INTER, int TOK>
__global__ void __launch_bounds__(NT) rotary_kernel(const RotArgs a) {
  __shared__ float sc[TOK][MAXP][2];
  const int tid = threadIdx.x;
  const int row0 = blockIdx.x * TOK, nrow = min(TOK, a.rows - row0);
  for (int i = tid; i < nrow * a.pairs; i += NT) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const long at = (long)(row0 + t) * a.ldpos + min(max(a.axis[p], 0), a.axes - 1);
    const double pos = a.pos64 ? (double)((const long long*)a.pos)[at] : (double)((const int*)a.pos)[at];
    const double turns = pos * a.rev[p];
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    sc[t][p][0] = c;
    sc[t][p][1] = a.inverse ? -s : s;
  }
  __syncthreads();
  const int units = a.pairs / PV, rest = a.dim - 2 * a.pairs;      // (units * PV == pairs: checked on the host)
  const int rest_units = PV == 1 ? rest : (rest + 2 * PV - 1) / (2 * PV);
  const int per_head = units + rest_units, heads = a.heads_q + a.heads_k;
  const int n = nrow * heads * per_head;
  for (int i = tid; i < n; i += NT) {
    const int u = i % per_head, j = i / per_head, hd = j % heads, t = j / heads;
    const bool isq = hd < a.heads_q;
    const long row = row0 + t;
    const T* src = isq ? (const T*)a.Q + row * a.ldq + (long)hd * a.hsq : (const T*)a.K + row * a.ldk + (long)(hd - a.heads_q) * a.hsk;
    T* dst = isq ? (T*)a.Qo + row * a.ldqo + (long)hd * a.hsqo : (T*)a.Ko + row * a.ldko + (long)(hd - a.heads_q) * a.hsko;
    if (u >= units) {      // columns behind the pairs
      if constexpr (PV == 1) {
        dst[2 * a.pairs + u - units] = src[2 * a.pairs + u - units];
      } else {
        const int c0 = 2 * a.pairs + (u - units) * 2 * PV;
#pragma unroll
        for (int e = 0; e < 2 * PV; e++)
          if (c0 + e < a.dim) dst[c0 + e] = src[c0 + e];
      }
      continue;
    }
    const int p0 = u * PV;
    if constexpr (INTER) {
      T v[2 * PV];
      __builtin_memcpy(v, __builtin_assume_aligned(src + 2 * p0, PV == 1 ? sizeof(T) : 16), sizeof(v));
#pragma unroll
      for (int e = 0; e < PV; e++) {
        const float c = sc[t][p0 + e][0], s = sc[t][p0 + e][1];
        float x = Elem<T>::to_f(v[2 * e]), y = Elem<T>::to_f(v[2 * e + 1]);
        turn(x, y, c, s);
        v[2 * e] = Elem<T>::from_f(x);
        v[2 * e + 1] = Elem<T>::from_f(y);
      }
      __builtin_memcpy(__builtin_assume_aligned(dst + 2 * p0, PV == 1 ? sizeof(T) : 16), v, sizeof(v));
    } else {
      T x[PV], y[PV];
      constexpr int AL = PV == 1 ? sizeof(T) : 16;
      __builtin_memcpy(x, __builtin_assume_aligned(src + p0, AL), sizeof(x));
      __builtin_memcpy(y, __builtin_assume_aligned(src + a.pairs + p0, AL), sizeof(y));
#pragma unroll
      for (int e = 0; e < PV; e++) {
        const float c = sc[t][p0 + e][0], s = sc[t][p0 + e][1];
        float xf = Elem<T>::to_f(x[e]), yf = Elem<T>::to_f(y[e]);
        turn(xf, yf, c, s);
        x[e] = Elem<T>::from_f(xf);
        y[e] = Elem<T>::from_f(yf);
      }
      __builtin_memcpy(__builtin_assume_aligned(dst + p0, AL), x, sizeof(x));
      __builtin_memcpy(__builtin_assume_aligned(dst + a.pairs + p0, AL), y, sizeof(y));
    }
  }
}

template <typename T, bool INTER>
void launch(const RotArgs& a, bool wide, hipStream_t s) {
  constexpr int PV = INTER ? 8 / (int)sizeof(T) : 16 / (int)sizeof(T);
  constexpr int TOK = 4;
  const int grid = cdiv(a.rows, TOK);
  if (wide) rotary_kernel<T, PV, INTER, TOK><<<grid, NT, 0, s>>>(a);
  else rotary_kernel<T, 1, INTER, TOK><<<grid, NT, 0, s>>>(a);
}

}  // namespace

extern "C" int crog_rotary(int dtype, const void* Q, int64_t ldq, int64_t hsq, const void* K, int64_t ldk, int64_t hsk, void* Qout, int64_t ldqo,
                           int64_t hsqo, void* Kout, int64_t ldko, int64_t hsko, const void* positions, int64_t ldpos, int pos_bytes, const void* revs,
                           const int* axis, int rows, int heads_q, int heads_k, int head_dim, int pairs, int axes, int interleaved, int inverse,
                           crog_stream_t stream) {
  CROG_CHECK_ARG(dtype == CROG_F32 || dtype == CROG_BF16, "rotary: dtype must be CROG_F32 or CROG_BF16 (got %d)", dtype);
  CROG_CHECK_ARG(rows >= 0 && rows <= 0x7fff0000 && heads_q >= 0 && heads_k >= 0 && (int64_t)(heads_q + heads_k) * head_dim <= (1 << 24), "rotary: bad sizes");
  CROG_CHECK_ARG(pairs > 0 && pairs <= MAXP && 2 * pairs <= head_dim, "rotary: 2 * pairs must fit the head and pairs be at most %d (pairs %d, head_dim %d)",
                 MAXP, pairs, head_dim);
  if (rows == 0 || heads_q + heads_k == 0) return CROG_OK;
  CROG_CHECK_ARG(axes > 0 && axes <= ldpos && (pos_bytes == 4 || pos_bytes == 8) && positions && revs && axis, "rotary: positions [rows][axes] of 4 or 8 bytes each");
  CROG_CHECK_ARG((heads_q == 0 || (Q && Qout)) && (heads_k == 0 || (K && Kout)), "rotary: a tensor is missing");
  RotArgs a{};
  a.Q = Q; a.K = K; a.Qo = Qout; a.Ko = Kout;
  a.ldq = ldq; a.hsq = hsq; a.ldk = ldk; a.hsk = hsk; a.ldqo = ldqo; a.hsqo = hsqo; a.ldko = ldko; a.hsko = hsko;
  a.pos = positions; a.ldpos = ldpos; a.pos64 = pos_bytes == 8; a.rev = (const double*)revs; a.axis = axis;
  a.rows = rows; a.heads_q = heads_q; a.heads_k = heads_k; a.dim = head_dim; a.pairs = pairs; a.axes = axes; a.inverse = inverse;
  // 16-byte items where every head starts on a 16-byte boundary and the pairs are whole items; element by element otherwise
  const int es = dtype == CROG_BF16 ? 2 : 4, vec = 16 / es, pv = interleaved ? vec / 2 : vec;
  const auto ok = [&](const void* p, int64_t ld, int64_t hs, int heads) { return heads == 0 || ((uintptr_t)p % 16 == 0 && ld % vec == 0 && hs % vec == 0); };
  const bool wide = pairs % pv == 0 && ok(Q, ldq, hsq, heads_q) && ok(K, ldk, hsk, heads_k) && ok(Qout, ldqo, hsqo, heads_q) && ok(Kout, ldko, hsko, heads_k);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == CROG_BF16) { if (interleaved) launch<bf16, true>(a, wide, s); else launch<bf16, false>(a, wide, s); }
  else { if (interleaved) launch<float, true>(a, wide, s); else launch<float, false>(a, wide, s); }
  CROG_LAUNCH_CHECK();
  return CROG_OK;
}
