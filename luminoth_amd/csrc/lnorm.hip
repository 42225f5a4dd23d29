// Layer norm over the last dimension, forward and backward (gfx950, HBM-bound).
//
//   y = (x - mu) rstd gamma + beta,   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps)            per row of D
//   t = dy gamma,  xh = (x - mu) rstd,  dx = rstd (t - mean(t) - xh mean(t xh)) (+ addend)
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// A row lies in the registers of the TPR threads that share it (16 columns a thread at most), so x is read once and the
// variance is the mean of the squared DEVIATIONS (no E[x^2] - E[x]^2).  A thread keeps its columns while it walks over rows:
// gamma and beta are loaded once a thread (per row they would be 2 x 4 bytes a column from the L2 against 2 x 2 bytes of
// 16-bit data), and the backward pass sums dgamma / dbeta in registers.  Their sums leave as one partial row per block
// and a second launch adds those up in block order: the same bits every time.
// Measured: 16384 x 4096 bf16 forward 44 us = 6.0 TB/s of x and y, backward with an addend 97 + 5 us = 5.5 TB/s of four arrays (a
// large copy: 4.7; parts still lie in the last-level cache); 5003 x 1001 f16 backward, rows 2016 bytes apart, 15 + 4 us; 512 x 1024
// fp32 forward 4.3 us, a launch's own time.
#include "rowops.h"

#define LN_MAX_REG_COLS 16384     // 1024 threads x 16 columns; longer rows: the kernels that read a row three times

template <typename T, typename P, int TPR, int NC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
k_ln_fwd(const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma, const P* __restrict__ beta, T* __restrict__ y,
         float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int D, float inv_d, float eps) {
  constexpr int VEC = row_type<T>::VEC, BT = TPR > 256 ? TPR : 256, GPB = BT / TPR;
  __shared__ float red[2][TPR > 64 ? TPR / 64 : 1];
  const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR;
  float ga[NC * VEC], be[NC * VEC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    load_params<VEC>(ga + c * VEC, gamma, (c * TPR + lane) * VEC, D, 1.f);
    load_params<VEC>(be + c * VEC, beta, (c * TPR + lane) * VEC, D, 0.f);
  }
  const int64_t step = (int64_t)gridDim.x * GPB;
  int64_t base = (int64_t)blockIdx.x * GPB;
  raw16 cur[NC], nxt[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    cur[c] = raw16{0, 0, 0, 0};
    if (base + grp < rows) cur[c] = load_cols(x + (base + grp) * ldx, (c * TPR + lane) * VEC, D);
  }
  for (; base < rows; base += step) {       // (the same trip count for every thread of the block: there are barriers inside)
    const int64_t row = base + grp;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      nxt[c] = raw16{0, 0, 0, 0};
      if (row + step < rows) nxt[c] = load_cols(x + (row + step) * ldx, (c * TPR + lane) * VEC, D);
    }
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += elem<T>(cur[c], e);            // (zeros behind the end of the row)
    const float mu = reduce_row<TPR>(s, op_add(), red[0]) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = (c * TPR + lane) * VEC + e < D ? elem<T>(cur[c], e) - mu : 0.f;
        q = fmaf(d, d, q);
      }
    const float var = reduce_row<TPR>(q, op_add(), red[1]) * inv_d;
    const float rs = 1.f / sqrtf(var + eps);
    if (row < rows) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = fmaf((elem<T>(cur[c], e) - mu) * rs, ga[c * VEC + e], be[c * VEC + e]);
        store_cols(y + row * (int64_t)D, (c * TPR + lane) * VEC, D, o);
      }
      if (lane == 0) {
        mean[row] = mu;
        rstd[row] = rs;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) cur[c] = nxt[c];
  }
}

// Rows too long for the registers: one block a row, read three times (the second and third time from the caches).
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
k_ln_fwd_long(const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma, const P* __restrict__ beta, T* __restrict__ y,
              float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int D, float inv_d, float eps) {
  constexpr int VEC = row_type<T>::VEC;
  __shared__ float red[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.f;
    for (int64_t col = (int64_t)threadIdx.x * VEC; col < D; col += 1024 * VEC) {
      const raw16 r = load_cols(xr, (int)col, D);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += elem<T>(r, e);
    }
    const float mu = reduce_row<1024>(s, op_add(), red[0]) * inv_d;
    float q = 0.f;
    for (int64_t col = (int64_t)threadIdx.x * VEC; col < D; col += 1024 * VEC) {
      const raw16 r = load_cols(xr, (int)col, D);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = col + e < D ? elem<T>(r, e) - mu : 0.f;
        q = fmaf(d, d, q);
      }
    }
    const float var = reduce_row<1024>(q, op_add(), red[1]) * inv_d;
    const float rs = 1.f / sqrtf(var + eps);
    for (int64_t col = (int64_t)threadIdx.x * VEC; col < D; col += 1024 * VEC) {
      const raw16 r = load_cols(xr, (int)col, D);
      float o[VEC];
      float ga[VEC], be[VEC];
      load_params<VEC>(ga, gamma, (int)col, D, 1.f);
      load_params<VEC>(be, beta, (int)col, D, 0.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = fmaf((elem<T>(r, e) - mu) * rs, ga[e], be[e]);
      store_cols(y + row * (int64_t)D, (int)col, D, o);
    }
    if (threadIdx.x == 0) {
      mean[row] = mu;
      rstd[row] = rs;
    }
  }
}

// part: [gridDim.x][2][E][TPR] partial sums of dgamma / dbeta (NULL: not wanted); dx NULL: not wanted.
template <typename T, typename P, int TPR, int NC, int BT, bool PF>
__global__ void __launch_bounds__(BT)
k_ln_bwd(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const T* __restrict__ addend, int64_t ldadd,
         const float* __restrict__ mean, const float* __restrict__ rstd, const P* __restrict__ gamma, T* __restrict__ dx,
         float* __restrict__ part, int64_t rows, int D, float inv_d) {
  constexpr int VEC = row_type<T>::VEC, GPB = BT / TPR, E = NC * VEC;
  __shared__ float red[2][2][BT / 64];
  extern __shared__ float sums[];       // [GPB / 2][2][E][TPR]
  const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR;
  float ga[E], dg[E], db[E];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    load_params<VEC>(ga + c * VEC, gamma, (c * TPR + lane) * VEC, D, 1.f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dg[c * VEC + e] = db[c * VEC + e] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * GPB;
  int64_t base = (int64_t)blockIdx.x * GPB;
  raw16 cx[NC], cd[NC], ca[NC], nx[NC], nd[NC], na[NC];
  float mu = 0.f, rs = 0.f, nmu = 0.f, nrs = 0.f;
  auto fetch = [&](int64_t row, raw16* fx, raw16* fd, raw16* fa, float& m, float& r) {
    m = r = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) fx[c] = fd[c] = fa[c] = raw16{0, 0, 0, 0};
    if (row < rows) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + lane) * VEC;
        fx[c] = load_cols(x + row * ldx, col, D);
        fd[c] = load_cols(dy + row * lddy, col, D);
        if (addend) fa[c] = load_cols(addend + row * ldadd, col, D);
      }
      m = mean[row];
      r = rstd[row];
    }
  };
  if (PF) fetch(base + grp, cx, cd, ca, mu, rs);
  int par = 0;
  for (; base < rows; base += step, par ^= 1) {
    const int64_t row = base + grp;
    if (PF) fetch(row + step, nx, nd, na, nmu, nrs);
    else fetch(row, cx, cd, ca, mu, rs);
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = c * VEC + e;
        // behind the end of the row dy is zero: nothing is added there whatever xh is
        const float d = elem<T>(cd[c], e), xh = (elem<T>(cx[c], e) - mu) * rs;
        const float t = d * ga[i];
        a += t;
        b = fmaf(t, xh, b);
        db[i] += d;
        dg[i] = fmaf(d, xh, dg[i]);
      }
    if (dx) {
      if constexpr (TPR > 64) {            // both sums behind ONE barrier; the arrays alternate from row to row
        a = reduce64(a, op_add());
        b = reduce64(b, op_add());
        if ((threadIdx.x & 63) == 0) {
          red[par][0][threadIdx.x >> 6] = a;
          red[par][1][threadIdx.x >> 6] = b;
        }
        __syncthreads();
        const int w0 = grp * (TPR / 64);
        a = red[par][0][w0];
        b = red[par][1][w0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) {
          a += red[par][0][w0 + i];
          b += red[par][1][w0 + i];
        }
      } else {
        a = reduce_row<TPR>(a, op_add(), nullptr);
        b = reduce_row<TPR>(b, op_add(), nullptr);
      }
      a *= inv_d;
      b *= inv_d;
      if (row < rows) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float o[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xh = (elem<T>(cx[c], e) - mu) * rs;
            o[e] = rs * (elem<T>(cd[c], e) * ga[c * VEC + e] - a - xh * b) + elem<T>(ca[c], e);
          }
          store_cols(dx + row * (int64_t)D, (c * TPR + lane) * VEC, D, o);
        }
      }
    }
    if (PF) {
#pragma unroll
      for (int c = 0; c < NC; ++c) { cx[c] = nx[c]; cd[c] = nd[c]; ca[c] = na[c]; }
      mu = nmu;
      rs = nrs;
    }
  }
  if (!part) return;
  // the block's groups, halved in turn: a fixed tree.  A thread's column i lies at [i][lane]: lanes side by side in LDS and in
  // the partial row (k_ln_params puts the columns in order)
  if constexpr (GPB > 1) {
    for (int half = GPB / 2; half > 0; half >>= 1) {
      float* s = sums + (size_t)(grp & (half - 1)) * 2 * E * TPR;
      __syncthreads();
      if (grp >= half && grp < 2 * half) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          s[i * TPR + lane] = dg[i];
          s[(E + i) * TPR + lane] = db[i];
        }
      }
      __syncthreads();
      if (grp < half) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          dg[i] += s[i * TPR + lane];
          db[i] += s[(E + i) * TPR + lane];
        }
      }
    }
  }
  if (grp == 0) {
    float* out = part + (size_t)blockIdx.x * 2 * E * TPR;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      out[i * TPR + lane] = dg[i];
      out[(E + i) * TPR + lane] = db[i];
    }
  }
}

// Rows too long for the registers: dx with one block a row (two passes), the column sums by a launch of their own.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
k_ln_bwd_long(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const T* __restrict__ addend, int64_t ldadd,
              const float* __restrict__ mean, const float* __restrict__ rstd, const P* __restrict__ gamma, T* __restrict__ dx,
              int64_t rows, int D, float inv_d) {
  constexpr int VEC = row_type<T>::VEC;
  __shared__ float red[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = mean[row], rs = rstd[row];
    float a = 0.f, b = 0.f;
    for (int64_t col = (int64_t)threadIdx.x * VEC; col < D; col += 1024 * VEC) {
      const raw16 rx = load_cols(x + row * ldx, (int)col, D), rd = load_cols(dy + row * lddy, (int)col, D);
      float ga[VEC];
      load_params<VEC>(ga, gamma, (int)col, D, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float t = elem<T>(rd, e) * ga[e];
        a += t;
        b = fmaf(t, (elem<T>(rx, e) - mu) * rs, b);
      }
    }
    a = reduce_row<1024>(a, op_add(), red[0]) * inv_d;
    b = reduce_row<1024>(b, op_add(), red[1]) * inv_d;
    for (int64_t col = (int64_t)threadIdx.x * VEC; col < D; col += 1024 * VEC) {
      const raw16 rx = load_cols(x + row * ldx, (int)col, D), rd = load_cols(dy + row * lddy, (int)col, D);
      raw16 ra = {0, 0, 0, 0};
      if (addend) ra = load_cols(addend + row * ldadd, (int)col, D);
      float ga[VEC], o[VEC];
      load_params<VEC>(ga, gamma, (int)col, D, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float t = elem<T>(rd, e) * ga[e];
        o[e] = rs * (t - a - (elem<T>(rx, e) - mu) * rs * b) + elem<T>(ra, e);
      }
      store_cols(dx + row * (int64_t)D, (int)col, D, o);
    }
  }
}

// grid (column strips of 64 vectors, row slices): one partial row per slice
template <typename T>
__global__ void __launch_bounds__(64)
k_ln_cols_long(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean,
               const float* __restrict__ rstd, float* __restrict__ part, int64_t rows, int D) {
  constexpr int VEC = row_type<T>::VEC;
  const int64_t col = ((int64_t)blockIdx.x * 64 + threadIdx.x) * VEC;
  if (col >= D) return;
  float dg[VEC], db[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) dg[e] = db[e] = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float mu = mean[row], rs = rstd[row];
    const raw16 rx = load_cols(x + row * ldx, (int)col, D), rd = load_cols(dy + row * lddy, (int)col, D);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      db[e] += elem<T>(rd, e);
      dg[e] = fmaf(elem<T>(rd, e), (elem<T>(rx, e) - mu) * rs, dg[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (col + e < D) {
      part[(size_t)blockIdx.y * 2 * D + col + e] = dg[e];
      part[(size_t)blockIdx.y * 2 * D + D + col + e] = db[e];
    }
}

// dgamma | dbeta from nb partial rows of [2][W] columns: 64 a block, 16 threads a column (slice s takes rows s, s + 16, ...),
// joined in slice order.  tpr: place p of a partial row is column ((p / tpr / vec) tpr + p % tpr) vec + (p / tpr) % vec, 0: column
// p.  nb = 0 (no rows): zeros.
template <typename P>
__global__ void __launch_bounds__(1024)
k_ln_params(const float* __restrict__ part, int nb, int D, int W, int tpr, int vec, P* __restrict__ dgamma, P* __restrict__ dbeta) {
  __shared__ float red[16][65];
  const int s = threadIdx.x >> 6;
  for (int64_t first = (int64_t)blockIdx.x * 64; first < 2 * (int64_t)W; first += (int64_t)gridDim.x * 64) {
    const int64_t i = first + (threadIdx.x & 63);                       // place in [dgamma | dbeta]
    float a = 0.f;
    if (i < 2 * (int64_t)W) {
#pragma unroll 8
      for (int r = s; r < nb; r += 16) a += part[(size_t)r * 2 * W + i];
    }
    red[s][threadIdx.x & 63] = a;
    __syncthreads();
    if (s == 0 && i < 2 * (int64_t)W) {
#pragma unroll
      for (int r = 1; r < 16; ++r) a += red[r][threadIdx.x];
      P* out = i < W ? dgamma : dbeta;
      int p = (int)(i < W ? i : i - W);
      if (tpr) p = (p / tpr / vec * tpr + p % tpr) * vec + p / tpr % vec;
      if (out && p < D) out[p] = from_f32<P>(a);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------- host ----
#define LN_FWD_BLOCKS 1536        // six of 256 threads a compute unit: what its registers hold (1024: 1-14 % slower, 2048: 6-26 %)
struct ln_shape { int tpr, nc; };
// 16 columns a thread at most: 16, 64, 256 or 1024 threads a row; the forward pass of 16-bit rows of 4097 to 8192 columns has 512
// (three blocks a compute unit instead of one: 6000 x 8192 bf16 50 -> 35 us; fp32 60 -> 64, the backward pass 75 -> 78)
static ln_shape ln_pick(int D, int vec, bool fwd = false) {
  ln_shape s;
  s.tpr = D <= 256 ? 16 : D <= 1024 ? 64 : D <= 4096 ? 256 : fwd && vec == 8 && D <= 8192 ? 512 : 1024;
  const int per = (D + s.tpr * vec - 1) / (s.tpr * vec);
  s.nc = vec == 8 ? (per <= 1 ? 1 : 2) : (per <= 1 ? 1 : per <= 2 ? 2 : 4);
  return s;
}

static const int LN_LONG_SLICES = 64;
static int ln_bwd_threads(int tpr) { return tpr == 1024 ? 1024 : 512; }
static int ln_bwd_blocks(int64_t rows, int D, int vec) {
  if (D > LN_MAX_REG_COLS) return (int)(rows < LN_LONG_SLICES ? rows : LN_LONG_SLICES);
  const ln_shape s = ln_pick(D, vec);
  const int bt = ln_bwd_threads(s.tpr), gpb = bt / s.tpr;
  // what the registers hold at a time: 256 blocks with 16 columns a thread (a second one would wait: 5003 x 1001 f16 15.5 us, 18.5 with
  // 512), 512 with 8 (60000 x 500 f16 69 us, 103 with 256), 768 with 4
  const int64_t need = (rows + gpb - 1) / gpb, cap = s.tpr == 1024 || s.nc * vec == 16 ? 256 : s.nc * vec == 8 ? 512 : 768;
  return (int)(need < cap ? need : cap);
}
static int ln_part_cols(int D, int vec) {         // columns of a partial row
  if (D > LN_MAX_REG_COLS) return D;
  const ln_shape s = ln_pick(D, vec);
  return s.tpr * s.nc * vec;
}

static bool ln_dtype_ok(int d) { return d == LMH_F32 || d == LMH_F16 || d == LMH_BF16; }
static int ln_vec(int d) { return d == LMH_F32 ? 4 : 8; }

// CALL(T, P, threads, vectors) for a shape: one or two vectors of 16-bit values, two or four of fp32 (one too for 16 threads).
// LEAST: of a row of 1024 threads in 16 bits
#define LN_PICK_NC(CALL, T, P, TPR, LEAST16)                                    \
  do {                                                                          \
    if constexpr (row_type<T>::VEC == 8) {                                      \
      if (s.nc <= LEAST16) CALL(T, P, TPR, LEAST16); else CALL(T, P, TPR, 2);   \
    } else {                                                                    \
      if (TPR == 16 && s.nc == 1) CALL(T, P, 16, 1); else if (s.nc == 2) CALL(T, P, TPR, 2); else CALL(T, P, TPR, 4); \
    }                                                                           \
  } while (0)
#define LN_PICK(CALL, T, P, LEAST)                                              \
  do {                                                                          \
    switch (s.tpr) {                                                            \
      case 16: LN_PICK_NC(CALL, T, P, 16, 1); break;                            \
      case 64: LN_PICK_NC(CALL, T, P, 64, 1); break;                            \
      case 256: LN_PICK_NC(CALL, T, P, 256, 1); break;                          \
      default: LN_PICK_NC(CALL, T, P, 1024, LEAST);                             \
    }                                                                           \
  } while (0)

template <typename T, typename P>
static void ln_fwd_launch(const void* x, int64_t ldx, const void* gamma, const void* beta, void* y, float* mean, float* rstd,
                          int64_t rows, int D, float eps, hipStream_t st) {
  const float inv_d = 1.f / (float)D;
  if (D > LN_MAX_REG_COLS) {
    lmh_launch((k_ln_fwd_long<T, P>), dim3((unsigned)(rows < 4096 ? rows : 4096)), dim3(1024), 0, st, (const T*)x, ldx, (const P*)gamma,
               (const P*)beta, (T*)y, mean, rstd, rows, D, inv_d, eps);
    return;
  }
  const ln_shape s = ln_pick(D, row_type<T>::VEC, true);
  const int bt = s.tpr > 256 ? s.tpr : 256, gpb = bt / s.tpr;
  const int64_t need = (rows + gpb - 1) / gpb, cap = LN_FWD_BLOCKS * 256 / (bt == 1024 ? 1536 : bt);
  const dim3 grid((unsigned)(need < cap ? need : cap));
#define LN_FWD(T_, P_, TPR_, NC_)                                                                                          \
  lmh_launch((k_ln_fwd<T_, P_, TPR_, NC_>), grid, dim3(bt), 0, st, (const T_*)x, ldx, (const P_*)gamma, (const P_*)beta, (T_*)y, mean, \
             rstd, rows, D, inv_d, eps)
  if constexpr (row_type<T>::VEC == 8) {
    if (s.tpr == 512) {
      LN_FWD(T, P, 512, 2);
      return;
    }
  }
  LN_PICK(LN_FWD, T, P, 2);
#undef LN_FWD
}

template <typename T, typename P>
static void ln_bwd_launch(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* addend, int64_t ldadd, const float* mean,
                          const float* rstd, const void* gamma, void* dx, void* dgamma, void* dbeta, float* part, int64_t rows, int D,
                          hipStream_t st) {
  const float inv_d = 1.f / (float)D;
  const bool params = dgamma || dbeta;
  const int nb = rows ? ln_bwd_blocks(rows, D, row_type<T>::VEC) : 0;
  if (rows && D > LN_MAX_REG_COLS) {
    if (dx)
      lmh_launch((k_ln_bwd_long<T, P>), dim3((unsigned)(rows < 4096 ? rows : 4096)), dim3(1024), 0, st, (const T*)dy, lddy, (const T*)x, ldx,
                 (const T*)addend, ldadd, mean, rstd, (const P*)gamma, (T*)dx, rows, D, inv_d);
    if (params) {
      const int strip = 64 * row_type<T>::VEC;
      lmh_launch((k_ln_cols_long<T>), dim3((unsigned)((D + (int64_t)strip - 1) / strip), (unsigned)nb), dim3(64), 0, st, (const T*)dy, lddy,
                 (const T*)x, ldx, mean, rstd, part, rows, D);
    }
  } else if (rows) {
    const ln_shape s = ln_pick(D, row_type<T>::VEC);
    float* p = params ? part : nullptr;
#define LN_BWD(T_, P_, TPR_, NC_)                                                                                              \
  lmh_launch((k_ln_bwd<T_, P_, TPR_, NC_, (TPR_ == 1024 ? 1024 : 512), (TPR_ < 1024)>), dim3((unsigned)nb), dim3(ln_bwd_threads(TPR_)),     \
             (unsigned)(TPR_ == 1024 ? 0 : 512 / TPR_ / 2 * 2 * sizeof(float) * NC_ * row_type<T_>::VEC * TPR_), st, (const T_*)dy, lddy, (const T_*)x, ldx, (const T_*)addend, ldadd, \
             mean, rstd, (const P_*)gamma, (T_*)dx, p, rows, D, inv_d)
    LN_PICK(LN_BWD, T, P, 1);
#undef LN_BWD
  }
  if (params) {
    const int W = ln_part_cols(D, row_type<T>::VEC), tpr = D > LN_MAX_REG_COLS ? 0 : ln_pick(D, row_type<T>::VEC).tpr;
    const int64_t strips = (2 * (int64_t)W + 63) / 64;
    lmh_launch((k_ln_params<P>), dim3((unsigned)(strips < 65536 ? strips : 65536)), dim3(1024), 0, st, (const float*)part, nb, D, W, tpr,
               row_type<T>::VEC, (P*)dgamma, (P*)dbeta);
  }
}

#define LN_TYPES(FN, ...)                                                                                      \
  do {                                                                                                         \
    if (dtype == LMH_F32) FN<f32_t, f32_t>(__VA_ARGS__);                                                       \
    else if (dtype == LMH_F16) { if (param_dtype == LMH_F32) FN<f16_t, f32_t>(__VA_ARGS__); else FN<f16_t, f16_t>(__VA_ARGS__); }   \
    else { if (param_dtype == LMH_F32) FN<bf16_t, f32_t>(__VA_ARGS__); else FN<bf16_t, bf16_t>(__VA_ARGS__); } \
  } while (0)

extern "C" int lmh_layer_norm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, int dtype, int param_dtype,
                                  int64_t rows, int D, float eps, void* y, float* mean, float* rstd, lmh_stream_t stream) {
  LMH_CHECK_ARG(ln_dtype_ok(dtype) && (param_dtype == LMH_F32 || param_dtype == dtype));
  LMH_CHECK_ARG(rows >= 0 && D > 0 && D <= LMH_ROW_MAX_COLS && ldx >= D && eps >= 0.f);
  if (rows == 0) return LMH_OK;
  LMH_CHECK_ARG(x && y && mean && rstd);
  hipStream_t st = (hipStream_t)stream;
  LN_TYPES(ln_fwd_launch, x, ldx, gamma, beta, y, mean, rstd, rows, D, eps, st);
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}

extern "C" size_t lmh_layer_norm_bwd_workspace_bytes(int64_t rows, int D, int dtype) {
  if (rows <= 0 || D <= 0 || D > LMH_ROW_MAX_COLS || !ln_dtype_ok(dtype)) return 256;
  return lmh_align_up((size_t)ln_bwd_blocks(rows, D, ln_vec(dtype)) * 2 * ln_part_cols(D, ln_vec(dtype)) * sizeof(float), 256);
}

extern "C" int lmh_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* addend, int64_t ldadd,
                                  const float* mean, const float* rstd, const void* gamma, int dtype, int param_dtype, int64_t rows,
                                  int D, void* dx, void* dgamma, void* dbeta, void* ws, size_t ws_bytes, lmh_stream_t stream) {
  LMH_CHECK_ARG(ln_dtype_ok(dtype) && (param_dtype == LMH_F32 || param_dtype == dtype));
  LMH_CHECK_ARG(rows >= 0 && D > 0 && D <= LMH_ROW_MAX_COLS && ldx >= D && lddy >= D && (!addend || ldadd >= D));
  LMH_CHECK_ARG(rows == 0 || (dy && x && mean && rstd));
  LMH_CHECK_ARG(dx || !addend);
  if ((dgamma || dbeta) && rows > 0 && (!ws || ws_bytes < lmh_layer_norm_bwd_workspace_bytes(rows, D, dtype))) {
    lmh_set_error("lmh_layer_norm_bwd: workspace too small");
    return LMH_ERR_WORKSPACE;
  }
  hipStream_t st = (hipStream_t)stream;
  LN_TYPES(ln_bwd_launch, dy, lddy, x, ldx, addend, ldadd, mean, rstd, gamma, dx, dgamma, dbeta, (float*)ws, rows, D, st);
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}
