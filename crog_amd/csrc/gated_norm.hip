// The residual between two blocks in one pass (crog_gated_norm_*): the norm behind a block (post), its gate, the scaled residual, and the norm
// in front of the next block (pre):
//   z = N(y) * post_w + post_b   (z = y without a post norm),   u = alpha x + gate * z,   h = N(u) * pre_w + pre_b
// N is LayerNorm's (t - mean) / sqrt(var + eps) or, rms, t / sqrt(mean(t^2) + eps).  The second norm reads the float sum, before it is rounded
// to be stored as u: both outputs are rounded once, and the backward pass, which forms u again from x and y, sees the same values.
// Backward, with U = N(u), Y = N(y):
//   dU = du + N'(dh * pre_w),  dx = alpha dU,  dy = N'(dU * gate * post_w),   N'(d) = (d - mean(d) - t mean(d t)) / deviation  (rms: no mean(d))
//   dpre_w = sum dh U, dpre_b = sum dh, dgate = sum dU z, dpost_w = gate sum dU Y, dpost_b = gate sum dU   - sums over the rows
// so four column sums (dU Y, dU, dh U, dh) give all five.
//
// Bound: memory.  Forward reads x, y and writes u, h (the next row is fetched during this one: 77 -> 46 us at 32768 x 1024 bf16, 268 MB, 5.8 TB/s);
// backward reads x, y, du, dh and writes dx, dy (403 MB, 91 us, 4.4 TB/s).  The weights stay in registers or LDS while a group of TPR threads walks
// over rows.  A thread holds at most 16 columns (four sums and four weights each are 128 registers): a row takes 16, 64, 256 or 512 threads.  Column sums: registers, then the block's groups through LDS, then one slab row per block, added up in block order by a
// second launch - no atomics, the same bits every time.
#include "common.h"
#include <cmath>

namespace {

struct GnArgs {
  const void *x, *y, *du, *dh;
  void *u, *h, *dx, *dy;
  const float *gate, *post_w, *post_b, *pre_w, *pre_b;
  float* stats;      // [rows][4]: mean and 1 / deviation of y, of u
  float* slab;       // [blocks][4][cols]
  long ldx, ldy, ldu, ldh, lddu, lddh, lddx, lddy;
  int rows, cols, rms, has_post, has_pre;
  float alpha, eps;
};

// Rows whose length is a whole number of 16-byte vectors and whose tensors are 16-byte aligned (WHOLE) are read vector by vector, and a thread's
// vector is there or it is not; of other rows the whole vectors by unaligned accesses, which the memory path takes (16000 x 1021 bf16, forward: 80 us
// element by element, 52 so), the end element by element.
template <typename T, bool WHOLE>
__device__ inline Vec16<T> load_vec(const T* row, int c0, int cols) {
  constexpr int V = Elem<T>::VEC;
  Vec16<T> v = zero16<T>();
  if constexpr (WHOLE) {
    f32x4 q = {0.f, 0.f, 0.f, 0.f};
    if (c0 < cols) q = *reinterpret_cast<const f32x4*>(row + c0);
    v = __builtin_bit_cast(Vec16<T>, q);
  } else if (c0 + V <= cols) {
    __builtin_memcpy(&v, row + c0, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < V; e++)
      if (c0 + e < cols) v.v[e] = row[c0 + e];
  }
  return v;
}
template <typename T, bool WHOLE>
__device__ inline void store_vec(T* row, const float* f, int c0, int cols) {
  constexpr int V = Elem<T>::VEC;
  if constexpr (WHOLE) {
    Vec16<T> v;
#pragma unroll
    for (int e = 0; e < V; e++) v.v[e] = Elem<T>::from_f(f[e]);
    if (c0 < cols) stg16(row + c0, v);
  } else if (c0 + V <= cols) {
    Vec16<T> v;
#pragma unroll
    for (int e = 0; e < V; e++) v.v[e] = Elem<T>::from_f(f[e]);
    __builtin_memcpy(row + c0, &v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < V; e++)
      if (c0 + e < cols) row[c0 + e] = Elem<T>::from_f(f[e]);
  }
}

// sum over the TPR threads of a row, in all of them.  TPR > 64: through LDS, a slot per wave; two sets in turn, so that one barrier a sum is enough
// (a set is written again only behind the barrier of the sum between)
struct Meet {
  float* slots;      // [2][waves of the block]
  int turn;
};
template <int TPR>
__device__ inline float row_sum(float v, Meet& m) {
  if constexpr (TPR <= 64) {
    return group_sum<TPR>(v);
  } else {
    float* set = m.slots + m.turn * (blockDim.x >> 6);
    m.turn ^= 1;
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) set[threadIdx.x >> 6] = v;
    __syncthreads();
    const int first = threadIdx.x / TPR * (TPR / 64);
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; w++) t += set[first + w];
    return t;
  }
}

template <typename T, int TPR, int NV, bool WHOLE> struct Threads {
  static constexpr int V = Elem<T>::VEC, N = NV * V;
  static constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  // column of element i of thread t, and whether the row has it
  __device__ static inline int col(int t, int i) { return (i / V * TPR + t) * V + i % V; }
  __device__ static inline bool has(int t, int i, int cols) { return col(t, WHOLE ? i / V * V : i) < cols; }
};

template <typename T, int NV> struct Row { Vec16<T> v[NV]; };      // a thread's share of a row as it is stored
template <typename T, int TPR, int NV, bool WHOLE>
__device__ inline Row<T, NV> fetch(const void* base, long ld, int row, int t, int cols) {
  Row<T, NV> r;
  const T* p = (const T*)base + (long)row * ld;
#pragma unroll
  for (int k = 0; k < NV; k++) r.v[k] = load_vec<T, WHOLE>(p, (k * TPR + t) * Elem<T>::VEC, cols);
  return r;
}
template <typename T, int NV, int N>
__device__ inline void widen(float (&f)[N], const Row<T, NV>& r) {
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = Elem<T>::to_f(r.v[i / Elem<T>::VEC].v[i % Elem<T>::VEC]);
}
template <typename T, int TPR, bool WHOLE, int N>
__device__ inline void store_row(void* base, long ld, int row, const float (&f)[N], int t, int cols) {
  T* p = (T*)base + (long)row * ld;
#pragma unroll
  for (int k = 0; k < N / Elem<T>::VEC; k++) store_vec<T, WHOLE>(p, f + k * Elem<T>::VEC, (k * TPR + t) * Elem<T>::VEC, cols);
}
template <typename S, int N>
__device__ inline void load_weights(float (&f)[N], const float* w, float otherwise, int t, int cols) {      // (0 behind the row's end)
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = S::has(t, i, cols) ? (w ? w[S::col(t, i)] : otherwise) : 0.f;
}

// f becomes the normalised row; mean and 1 / deviation in two passes over the registers (columns behind the row's end count as nothing)
template <int TPR, typename S, int N>
__device__ inline void normalise(float (&f)[N], int t, int cols, bool rms, float eps, float& mean, float& inv, Meet& red) {
  mean = 0.f;
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) s += f[i];
    mean = row_sum<TPR>(s, red) / (float)cols;
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = S::has(t, i, cols) ? f[i] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) q += f[i] * f[i];
  inv = 1.f / sqrtf(row_sum<TPR>(q, red) / (float)cols + eps);
#pragma unroll
  for (int i = 0; i < N; i++) f[i] *= inv;
}

template <typename T, int TPR, int NV, bool WHOLE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) gated_norm_fwd_kernel(const GnArgs a) {
  using S = Threads<T, TPR, NV, WHOLE>;
  __shared__ float slots[S::THREADS / 32];
  Meet red{slots, 0};
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  float gate[S::N], w1[S::N], b1[S::N], w2[S::N], b2[S::N];
  load_weights<S>(gate, a.gate, 1.f, t, a.cols);
  if (a.has_post) {
    load_weights<S>(w1, a.post_w, 1.f, t, a.cols);
    load_weights<S>(b1, a.post_b, 0.f, t, a.cols);
  }
  if (a.has_pre) {
    load_weights<S>(w2, a.pre_w, 1.f, t, a.cols);
    load_weights<S>(b2, a.pre_b, 0.f, t, a.cols);
  }
  // (a group whose row lies behind the last one joins the cross-lane sums with the last row's values and stores nothing)
  const int step = gridDim.x * S::GROUPS;
  int row = blockIdx.x * S::GROUPS + grp;
  Row<T, NV> nx = fetch<T, TPR, NV, WHOLE>(a.x, a.ldx, min(row, a.rows - 1), t, a.cols), ny = fetch<T, TPR, NV, WHOLE>(a.y, a.ldy, min(row, a.rows - 1), t, a.cols);
  for (int base = blockIdx.x * S::GROUPS; base < a.rows; base += step, row += step) {
    const bool live = row < a.rows;
    float x[S::N], y[S::N];
    widen(x, nx);
    widen(y, ny);
    if (base + step < a.rows) {      // the next row is on its way during this one
      nx = fetch<T, TPR, NV, WHOLE>(a.x, a.ldx, min(row + step, a.rows - 1), t, a.cols);
      ny = fetch<T, TPR, NV, WHOLE>(a.y, a.ldy, min(row + step, a.rows - 1), t, a.cols);
    }
    float mean1 = 0.f, inv1 = 1.f, mean2 = 0.f, inv2 = 1.f;
    if (a.has_post) {
      normalise<TPR, S>(y, t, a.cols, a.rms, a.eps, mean1, inv1, red);
#pragma unroll
      for (int i = 0; i < S::N; i++) y[i] = y[i] * w1[i] + b1[i];
    }
#pragma unroll
    for (int i = 0; i < S::N; i++) x[i] = a.alpha * x[i] + gate[i] * y[i];
    if (live) store_row<T, TPR, WHOLE>(a.u, a.ldu, row, x, t, a.cols);
    if (a.has_pre) {
      normalise<TPR, S>(x, t, a.cols, a.rms, a.eps, mean2, inv2, red);
#pragma unroll
      for (int i = 0; i < S::N; i++) x[i] = x[i] * w2[i] + b2[i];
      if (live) store_row<T, TPR, WHOLE>(a.h, a.ldh, row, x, t, a.cols);
    }
    if (a.stats && live && t == 0) *reinterpret_cast<f32x4*>(a.stats + 4 * (long)row) = f32x4{mean1, inv1, mean2, inv2};
  }
}

// d becomes N'(d) for the normalised row n
template <int TPR, typename S, int N>
__device__ inline void normalise_back(float (&d)[N], const float (&n)[N], int t, int cols, bool rms, float inv, Meet& red) {
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) { s += d[i]; q += d[i] * n[i]; }
  const float md = rms ? 0.f : row_sum<TPR>(s, red) / (float)cols, mq = row_sum<TPR>(q, red) / (float)cols;
#pragma unroll
  for (int i = 0; i < N; i++) d[i] = S::has(t, i, cols) ? (d[i] - md - n[i] * mq) * inv : 0.f;
}

template <typename T, int TPR, int NV, bool WHOLE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, 2) gated_norm_bwd_kernel(const GnArgs a) {
  using S = Threads<T, TPR, NV, WHOLE>;
  __shared__ float slots[S::THREADS / 32];
  Meet red{slots, 0};
  __shared__ float part[S::GROUPS > 1 ? S::THREADS : 1];
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  // The weights (gate, post_w, post_b, pre_w) in registers, where they leave no room for the next row beside the four sums; or in LDS, with the next
  // row on its way: rows with an odd end (16000 x 1021 bf16: 116 us of 154 before) and of at most 256 columns (40000 x 256: 36 of 49), but longer
  // ones lose more to the reads than they gain (32768 x 1024: 91 -> 128).
  constexpr bool AHEAD = TPR == 16 || (!WHOLE && TPR <= 256);
  __shared__ __attribute__((aligned(16))) float wts[4][AHEAD ? TPR * S::N : 1];
  float wreg[4][AHEAD ? 1 : S::N];
  const float* const from[4] = {a.gate, a.post_w, a.post_b, a.pre_w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float otherwise = k == 2 ? 0.f : 1.f;
    if constexpr (AHEAD) {
      for (int c = threadIdx.x; c < TPR * S::N; c += S::THREADS) wts[k][c] = c < a.cols ? (from[k] ? from[k][c] : otherwise) : 0.f;
    } else {
      load_weights<S>(wreg[k], from[k], otherwise, t, a.cols);
    }
  }
  if constexpr (AHEAD) __syncthreads();
  float sum[4][S::N];      // dU Y, dU, dh U, dh
#pragma unroll
  for (int k = 0; k < 4; k++)
#pragma unroll
    for (int i = 0; i < S::N; i++) sum[k][i] = 0.f;
  struct Next {
    f32x4 st;
    Row<T, NV> x, y, du, dh;
  };
  const bool both = a.has_pre && a.dh;
  const auto request = [&](int row) {
    Next next{};
    const int rc = min(row, a.rows - 1);
    next.st = *reinterpret_cast<const f32x4*>(a.stats + 4 * (long)rc);
    next.y = fetch<T, TPR, NV, WHOLE>(a.y, a.ldy, rc, t, a.cols);
    if (both) {
      next.x = fetch<T, TPR, NV, WHOLE>(a.x, a.ldx, rc, t, a.cols);
      next.dh = fetch<T, TPR, NV, WHOLE>(a.dh, a.lddh, rc, t, a.cols);
    }
    if (a.du) next.du = fetch<T, TPR, NV, WHOLE>(a.du, a.lddu, rc, t, a.cols);
    return next;
  };
  const int step = gridDim.x * S::GROUPS;
  Next next;
  if constexpr (AHEAD) next = request(blockIdx.x * S::GROUPS + grp);
  for (int base = blockIdx.x * S::GROUPS; base < a.rows; base += step) {
    const int row = base + grp;
    const bool live = row < a.rows;
    int lane = t;
    if constexpr (AHEAD) asm volatile("" : "+v"(lane));      // (or the weights in LDS would be read once, into registers)
    const auto w = [&](int k, int i) {
      if constexpr (AHEAD) return wts[k][S::col(lane, i)];
      else return wreg[k][i];
    };
    Next now;
    if constexpr (AHEAD) now = next;
    else now = request(row);
    const f32x4 st = now.st;
    float y[S::N], d[S::N];      // Y (y itself without a post norm), dU
    widen(y, now.y);
    if constexpr (AHEAD) {
      if (base + step < a.rows) next = request(row + step);
    }
    if (a.has_post)
#pragma unroll
      for (int i = 0; i < S::N; i++) y[i] = S::has(t, i, a.cols) ? (y[i] - st[0]) * st[1] : 0.f;
    if (both) {
      float u[S::N], g[S::N];
      widen(u, now.x);
      widen(g, now.dh);
#pragma unroll
      for (int i = 0; i < S::N; i++) {
        const float z = a.has_post ? y[i] * w(1, i) + w(2, i) : y[i];
        u[i] = S::has(t, i, a.cols) ? (a.alpha * u[i] + w(0, i) * z - st[2]) * st[3] : 0.f;
        if (live) { sum[2][i] += g[i] * u[i]; sum[3][i] += g[i]; }
        d[i] = g[i] * w(3, i);
      }
      normalise_back<TPR, S>(d, u, t, a.cols, a.rms, st[3], red);
    } else {
#pragma unroll
      for (int i = 0; i < S::N; i++) d[i] = 0.f;
    }
    if (a.du) {
      float g[S::N];
      widen(g, now.du);
#pragma unroll
      for (int i = 0; i < S::N; i++) d[i] += g[i];
    }
    float o[S::N];
#pragma unroll
    for (int i = 0; i < S::N; i++) {
      if (live) { sum[0][i] += d[i] * y[i]; sum[1][i] += d[i]; }
      o[i] = a.alpha * d[i];
      d[i] = a.has_post ? d[i] * w(0, i) * w(1, i) : d[i] * w(0, i);
    }
    if (live && a.dx) store_row<T, TPR, WHOLE>(a.dx, a.lddx, row, o, t, a.cols);
    if (a.has_post) normalise_back<TPR, S>(d, y, t, a.cols, a.rms, st[1], red);
    if (live && a.dy) store_row<T, TPR, WHOLE>(a.dy, a.lddy, row, d, t, a.cols);
  }
  if (!a.slab) return;
#pragma unroll
  for (int k = 0; k < 4; k++)
#pragma unroll
    for (int i = 0; i < S::N; i++) {
      float v = sum[k][i];
      if constexpr (S::GROUPS > 1) {      // the block's groups in order
        __syncthreads();
        part[threadIdx.x] = v;
        __syncthreads();
        v = 0.f;
        if (grp == 0)
#pragma unroll
          for (int g = 0; g < S::GROUPS; g++) v += part[g * TPR + t];
      }
      const int c = S::col(t, i);
      if (grp == 0 && c < a.cols) a.slab[((long)blockIdx.x * 4 + k) * a.cols + c] = v;
    }
}

// the blocks' sums in order -> the five gradients, added onto what the buffers hold.  A block takes 16 columns, 64 runs of slab rows each (latency: 512
// slab rows of 1024 columns are 8 MB, 64 blocks; 16 runs took 13.9 us)
constexpr int RUNS = 64;
__global__ void __launch_bounds__(16 * RUNS) gated_norm_sums_kernel(const float* slab, int blocks, int cols, const float* gate, const float* post_w,
                                                                    const float* post_b, int has_post, float* dgate, float* dpost_w, float* dpost_b,
                                                                    float* dpre_w, float* dpre_b) {
  __shared__ float part[4][RUNS][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
  const int per = (blocks + RUNS - 1) / RUNS, lo = run * per, hi = min(lo + per, blocks);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < cols)
#pragma unroll 4
    for (int b = lo; b < hi; b++)
#pragma unroll
      for (int k = 0; k < 4; k++) s[k] += slab[((long)b * 4 + k) * cols + c];
#pragma unroll
  for (int k = 0; k < 4; k++) part[k][run][threadIdx.x & 15] = s[k];
  __syncthreads();
  __shared__ float total[4][16];
  if (run < 4) {      // (run = which of the four sums)
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < RUNS; r++) t += part[run][r][threadIdx.x & 15];
    total[run][threadIdx.x & 15] = t;
  }
  __syncthreads();
  if (run != 0 || c >= cols) return;
#pragma unroll
  for (int k = 0; k < 4; k++) s[k] = total[k][threadIdx.x];
  const float g = gate ? gate[c] : 1.f;
  if (dgate) dgate[c] += has_post ? (post_w ? post_w[c] : 1.f) * s[0] + (post_b ? post_b[c] : 0.f) * s[1] : s[0];
  if (dpost_w) dpost_w[c] += g * s[0];
  if (dpost_b) dpost_b[c] += g * s[1];
  if (dpre_w) dpre_w[c] += s[2];
  if (dpre_b) dpre_b[c] += s[3];
}

constexpr int MAX_COLS = 8192;
constexpr int MAX_BLOCKS = 512;      // two per CU.  (32768 x 1024 bf16: forward 46.0 us, with 1024 / 2048 blocks 53.7 / 49.2; backward 89.6, with 768 105)

// threads of a row: 16 columns a thread at most.  (8 a thread, a row of 1024 columns on two waves that meet in LDS: 55.6 / 122 us)
int threads_per_row(int cols) { return cols <= 256 ? 16 : cols <= 1024 ? 64 : cols <= 4096 ? 256 : 512; }
int blocks_for(int rows, int cols) {
  const int tpr = threads_per_row(cols), groups = tpr > 256 ? 1 : 256 / tpr;
  const int n = cdiv(rows, groups);
  return n < MAX_BLOCKS ? n : MAX_BLOCKS;
}

template <typename T, int TPR, int NV, bool WHOLE>
void launch(const GnArgs& a, bool fwd, hipStream_t s) {
  const int blocks = blocks_for(a.rows, a.cols);
  if (fwd) gated_norm_fwd_kernel<T, TPR, NV, WHOLE><<<blocks, Threads<T, TPR, NV, WHOLE>::THREADS, 0, s>>>(a);
  else gated_norm_bwd_kernel<T, TPR, NV, WHOLE><<<blocks, Threads<T, TPR, NV, WHOLE>::THREADS, 0, s>>>(a);
}
template <typename T, int TPR>
void launch_nv(const GnArgs& a, bool fwd, bool whole, hipStream_t s) {
  constexpr int MOST = 16 / Elem<T>::VEC;                // 16 columns a thread at most (threads_per_row)
  const int nv = cdiv(a.cols, TPR * Elem<T>::VEC);
  if (!whole) launch<T, TPR, MOST, false>(a, fwd, s);
  else if (nv == 1) launch<T, TPR, 1, true>(a, fwd, s);
  else if (nv == 2 || MOST == 2) launch<T, TPR, 2, true>(a, fwd, s);
  else launch<T, TPR, MOST, true>(a, fwd, s);
}
template <typename T>
void launch_t(const GnArgs& a, bool fwd, bool aligned, hipStream_t s) {
  const bool whole = aligned && a.cols % Elem<T>::VEC == 0;
  switch (threads_per_row(a.cols)) {
    case 16: launch_nv<T, 16>(a, fwd, whole, s); break;
    case 64: launch_nv<T, 64>(a, fwd, whole, s); break;
    case 256: launch_nv<T, 256>(a, fwd, whole, s); break;
    default: launch_nv<T, 512>(a, fwd, whole, s); break;
  }
}

bool vec_rows(const void* p, int64_t ld, int vec) { return p == nullptr || ((uintptr_t)p % 16 == 0 && ld % vec == 0); }

}  // namespace

extern "C" int crog_gated_norm_slab_floats(int rows, int cols) { return rows > 0 && cols > 0 ? blocks_for(rows, cols) * 4 * cols : 0; }

extern "C" int crog_gated_norm_fwd(int dtype, const void* x, int64_t ldx, const void* y, int64_t ldy, const float* gate, const float* post_w,
                                   const float* post_b, const float* pre_w, const float* pre_b, int has_post, int has_pre, int rms, float alpha, float eps,
                                   int rows, int cols, void* u, int64_t ldu, void* h, int64_t ldh, float* stats, crog_stream_t stream) {
  CROG_CHECK_ARG(dtype == CROG_F32 || dtype == CROG_BF16, "gated_norm_fwd: dtype must be CROG_F32 or CROG_BF16 (got %d)", dtype);
  CROG_CHECK_ARG(rows >= 0 && rows <= 0x7fff0000 && cols > 0 && cols <= MAX_COLS, "gated_norm_fwd: rows of 1 .. %d columns (got %d x %d)", MAX_COLS, rows, cols);
  CROG_CHECK_ARG(std::isfinite(alpha), "gated_norm_fwd: alpha must be finite (got %g)", alpha);
  if (rows == 0) return CROG_OK;
  CROG_CHECK_ARG(x && y && u && (!has_pre || h) && ldx >= cols && ldy >= cols && ldu >= cols && (!has_pre || ldh >= cols), "gated_norm_fwd: bad tensors");
  CROG_CHECK_ARG((uintptr_t)stats % 16 == 0, "gated_norm_fwd: stats must be 16-byte aligned");
  GnArgs a{};
  a.x = x; a.y = y; a.u = u; a.h = h; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b; a.stats = stats;
  a.ldx = ldx; a.ldy = ldy; a.ldu = ldu; a.ldh = ldh; a.rows = rows; a.cols = cols; a.rms = rms; a.has_post = has_post; a.has_pre = has_pre;
  a.alpha = alpha; a.eps = eps;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  const int vec16 = vec_rows(x, ldx, vec) && vec_rows(y, ldy, vec) && vec_rows(u, ldu, vec) && (!has_pre || vec_rows(h, ldh, vec));
  if (dtype == CROG_BF16) launch_t<bf16>(a, true, vec16, (hipStream_t)stream);
  else launch_t<float>(a, true, vec16, (hipStream_t)stream);
  CROG_LAUNCH_CHECK();
  return CROG_OK;
}

extern "C" int crog_gated_norm_bwd(int dtype, const void* x, int64_t ldx, const void* y, int64_t ldy, const void* du, int64_t lddu, const void* dh,
                                   int64_t lddh, const float* gate, const float* post_w, const float* post_b, const float* pre_w, int has_post, int has_pre,
                                   int rms, float alpha, int rows, int cols, const float* stats, void* dx, int64_t lddx, void* dy, int64_t lddy, float* slab,
                                   crog_stream_t stream) {
  CROG_CHECK_ARG(dtype == CROG_F32 || dtype == CROG_BF16, "gated_norm_bwd: dtype must be CROG_F32 or CROG_BF16 (got %d)", dtype);
  CROG_CHECK_ARG(rows >= 0 && rows <= 0x7fff0000 && cols > 0 && cols <= MAX_COLS, "gated_norm_bwd: rows of 1 .. %d columns (got %d x %d)", MAX_COLS, rows, cols);
  CROG_CHECK_ARG(std::isfinite(alpha), "gated_norm_bwd: alpha must be finite (got %g)", alpha);
  if (rows == 0) return CROG_OK;
  CROG_CHECK_ARG(x && y && stats && ldx >= cols && ldy >= cols && (!du || lddu >= cols) && (!dh || lddh >= cols) && (!dx || lddx >= cols) && (!dy || lddy >= cols),
                 "gated_norm_bwd: bad tensors");
  CROG_CHECK_ARG((uintptr_t)stats % 16 == 0, "gated_norm_bwd: stats must be 16-byte aligned");
  GnArgs a{};
  a.x = x; a.y = y; a.du = du; a.dh = dh; a.dx = dx; a.dy = dy; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w;
  a.stats = const_cast<float*>(stats); a.slab = slab;
  a.ldx = ldx; a.ldy = ldy; a.lddu = lddu; a.lddh = lddh; a.lddx = lddx; a.lddy = lddy; a.rows = rows; a.cols = cols; a.rms = rms;
  a.has_post = has_post; a.has_pre = has_pre; a.alpha = alpha;
  const int vec = dtype == CROG_BF16 ? 8 : 4;
  const int vec16 = vec_rows(x, ldx, vec) && vec_rows(y, ldy, vec) && vec_rows(du, lddu, vec) && vec_rows(dh, lddh, vec) && vec_rows(dx, lddx, vec) && vec_rows(dy, lddy, vec);
  if (dtype == CROG_BF16) launch_t<bf16>(a, false, vec16, (hipStream_t)stream);
  else launch_t<float>(a, false, vec16, (hipStream_t)stream);
  CROG_LAUNCH_CHECK();
  return CROG_OK;
}

extern "C" int crog_gated_norm_sums(const float* slab, int rows, int cols, const float* gate, const float* post_w, const float* post_b, int has_post,
                                    float* dgate, float* dpost_w, float* dpost_b, float* dpre_w, float* dpre_b, crog_stream_t stream) {
  CROG_CHECK_ARG(rows >= 0 && rows <= 0x7fff0000 && cols > 0 && cols <= MAX_COLS, "gated_norm_sums: rows of 1 .. %d columns (got %d x %d)", MAX_COLS, rows, cols);
  if (rows == 0 || !(dgate || dpost_w || dpost_b || dpre_w || dpre_b)) return CROG_OK;
  CROG_CHECK_ARG(slab, "gated_norm_sums: the slab of crog_gated_norm_bwd is missing");
  gated_norm_sums_kernel<<<cdiv(cols, 16), 16 * RUNS, 0, (hipStream_t)stream>>>(slab, blocks_for(rows, cols), cols, gate, post_w, post_b, has_post, dgate,
                                                                                dpost_w, dpost_b, dpre_w, dpre_b);
  CROG_LAUNCH_CHECK();
  return CROG_OK;
}
