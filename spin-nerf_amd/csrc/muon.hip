// Orthogonalised updates: Newton-Schulz products on stacks of matrices, and the optimizer step around them (gfx950).
//
//   X_0 = x / max(|x|_F, eps);   A = X X^T;   X <- a X + (b A + c A A) X, `steps` times
//
// acts on the singular values alone (s -> a s + b s^3 + c s^5); x^T gives the transposed result, so every matrix is taken as
// Y [r x c] with r <= c and the Gram matrix A is r x r.
//
// Numbers.  Y, A and B = b A + c A^2 are held as hi + 2^-11 lo, two fp16 planes (22 mantissa bits, as much memory as fp32), each
// scaled by a power of two so that fp16's range covers what a polynomial that stays bounded can reach (orth_bounded below).
// SNR_ORTH_FP32 multiplies hi hi + hi lo + lo hi (three v_mfma_f32_32x32x16_f16; the dropped lo lo is 2^-24 of a product): fp32's
// accuracy at a third of the fp16 rate, 5 x the fp32 matrix rate.  SNR_ORTH_FP16 multiplies the hi planes only, except where the
// shorter side is 64 or less: there the roundings of a direction's few entries do not average out (up to 1 % of a singular value
// over five steps; a tenth of that from some 64 entries on), and the time is latency, not products.  The term a X is
// taken from both planes in either mode: a rounding of X itself would be full-rank noise, which the iteration amplifies by a per
// step (485 x over five) in the directions x is weak in, while a rounding inside B X only turns directions x is strong in.
#include "snr_common.h"

namespace snr {

constexpr int kOrthMax = 24;                // stacks per launch sequence: the kernel arguments hold the table
constexpr int kTile = 64;                   // padding and output tile
constexpr float kYs = 1024.f, kAs = 512.f;  // powers of two that the planes of Y and of A, B are scaled by
constexpr float kLo = 2048.f;               // ... and the lo planes on top

struct OrthGeom {        // a stack of equal matrices
  int r, c, rp, cp;      // sides of Y, and padded to the tile
  int batch, split;      // split: the lo planes take part in the products
  int sym0, full0;       // first workgroup of the stack in the symmetric products / in B Y
  int64_t ws;            // its planes
};
struct OrthIo {
  const void* x;         // the input, or the gradients
  void* out;             // the result, or the parameters
  float* mom;            // momentum (null: plain orthogonalisation)
  int64_t xb, xr, ob, orow;  // element strides: matrix, row (columns are contiguous)
  int m, n, chunk0, split0;  // sizes as stored; first workgroup in the reduction / in the split
  int nchunk;            // workgroups (partial sums) per matrix in the reduction
  int64_t part;          // first partial sum (doubles)
};
struct OrthTable { int n; OrthGeom g[kOrthMax]; };
struct OrthArgs {
  OrthTable t;
  OrthIo io[kOrthMax];
  int dtype;             // of x / out without momentum
  float mu, gscale, eps;
  int nesterov;
  double* part;
  char* ws;
};
struct OrthOut {         // the last product's epilogue
  int dtype, muon, scale_mode;
  float lr, decay;
  const snr_step_state* st;
};

// planes of one matrix, in fp16 elements
struct OrthPlanes { int64_t yh, yl, t0h, t0l, t1h, t1l, ah, al, bh, bl, total; };
__host__ __device__ inline OrthPlanes orth_planes(int rp, int cp) {
  const int64_t y = (int64_t)rp * cp, g = (int64_t)rp * rp;
  OrthPlanes p;
  p.yh = 0; p.yl = y; p.t0h = 2 * y; p.t0l = 3 * y; p.t1h = 4 * y; p.t1l = 5 * y;
  p.ah = 6 * y; p.al = p.ah + g; p.bh = p.al + g; p.bl = p.bh + g; p.total = p.bl + g;
  return p;
}

__device__ __forceinline__ float orth_load(const void* p, int64_t i, int dtype) {
  if (dtype == SNR_F32) return ((const float*)p)[i];
  if (dtype == SNR_F16) return (float)((const _Float16*)p)[i];
  return (float)((const __bf16*)p)[i];
}
__device__ __forceinline__ void orth_store(void* p, int64_t i, int dtype, float v) {
  if (dtype == SNR_F32) ((float*)p)[i] = v;
  else if (dtype == SNR_F16) ((_Float16*)p)[i] = (_Float16)v;
  else ((__bf16*)p)[i] = (__bf16)v;
}
__device__ __forceinline__ void orth_split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)((v - (float)hi) * kLo);
}

// ---- 1. momentum (in place) and the partial sums of squares of the update, in 64 bits and in a fixed order ------------------
__global__ __launch_bounds__(256) void orth_reduce_kernel(OrthArgs a) {
  int s = 0;
  while (s + 1 < a.t.n && (int)blockIdx.x >= a.io[s + 1].chunk0) ++s;
  const OrthIo& io = a.io[s];
  const int k = blockIdx.x - io.chunk0, mat = k / io.nchunk, ch = k % io.nchunk;
  const int64_t count = (int64_t)io.m * io.n;
  const int64_t per = (count + io.nchunk - 1) / io.nchunk, e0 = ch * per, e1 = e0 + per < count ? e0 + per : count;
  double sum = 0.0;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
    float u;
    if (io.mom) {
      const int64_t i = mat * count + e;
      const float g = ((const float*)io.x)[i] * a.gscale, mo = io.mom[i] * a.mu + g;
      io.mom[i] = mo;
      u = a.nesterov ? g + a.mu * mo : mo;
    } else {
      u = orth_load(io.x, mat * io.xb + (e / io.n) * io.xr + e % io.n, a.dtype);
    }
    sum += (double)u * (double)u;
  }
  __shared__ double red[256];
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.part[io.part + mat * io.nchunk + ch] = red[0];
}

// ---- 2. Y = scaled input (transposed where it is tall) and Y^T, as planes, zero in the padding --------------------------------
__global__ __launch_bounds__(256) void orth_split_kernel(OrthArgs a) {
  int s = 0;
  while (s + 1 < a.t.n && (int)blockIdx.x >= a.io[s + 1].split0) ++s;
  const OrthIo& io = a.io[s];
  const OrthGeom& G = a.t.g[s];
  const int nti = G.rp / kTile, ntj = G.cp / kTile;
  const int k = blockIdx.x - io.split0, mat = k / (nti * ntj), t = k % (nti * ntj);
  const int i0 = t / ntj * kTile, j0 = t % ntj * kTile;
  const bool tall = io.m > io.n;
  __shared__ double red[256];
  __shared__ float tile[kTile][kTile + 1];
  double sum = 0.0;
  for (int p = threadIdx.x; p < io.nchunk; p += 256) sum += a.part[io.part + mat * io.nchunk + p];
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  const double norm = sqrt(red[0]);
  const double scale = (double)kYs / (norm < (double)a.eps ? (double)a.eps : norm);   // (a NaN stays one)
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // rows of the input are contiguous: lanes run along them
  for (int q = w; q < kTile; q += 4) {
    const int mi = tall ? j0 + q : i0 + q, nj = (tall ? i0 : j0) + lane;
    float u = 0.f;
    if (mi < io.m && nj < io.n) {
      if (io.mom) {
        const int64_t i = ((int64_t)mat * io.m + mi) * io.n + nj;
        const float mo = io.mom[i];
        u = a.nesterov ? ((const float*)io.x)[i] * a.gscale + a.mu * mo : mo;
      } else {
        u = orth_load(io.x, mat * io.xb + mi * io.xr + nj, a.dtype);
      }
      u = (float)((double)u * scale);
    }
    if (tall) tile[lane][q] = u; else tile[q][lane] = u;
  }
  __syncthreads();
  const OrthPlanes P = orth_planes(G.rp, G.cp);
  _Float16* W = (_Float16*)(a.ws + G.ws) + mat * P.total;
  for (int q = w; q < kTile; q += 4) {
    _Float16 hi, lo;
    orth_split(tile[q][lane], hi, lo);
    const int64_t y = (int64_t)(i0 + q) * G.cp + j0 + lane;
    W[P.yh + y] = hi; W[P.yl + y] = lo;
    orth_split(tile[lane][q], hi, lo);
    const int64_t yt = (int64_t)(j0 + q) * G.rp + i0 + lane;
    W[P.t0h + yt] = hi; W[P.t0l + yt] = lo;
  }
}

// ---- 3. the products: C[i][j] = sum_k P[i][k] Q[j][k], rows contiguous in k ----------------------------------------------------
//   phase 0: A = Y Y^T          (symmetric: tiles i <= j, mirrored)
//   phase 1: B = b A + c A A^T  (symmetric)
//   phase 2: Y <- a Y + B Y, taken as B (Y^T)^T; also Y^T for the next step, or the result
enum { kGram = 0, kPoly = 1, kApply = 2 };
constexpr int kLd = kTile + 8;   // LDS row of 64 + 8 fp16: 144 B, 16-byte reads of 32 rows spread over the banks

template <int PHASE>
__global__ __launch_bounds__(256) void orth_product_kernel(OrthArgs a, OrthOut o, float ca, float cb, float cc, int flip, int last) {
  int s = 0;
  if (PHASE == kApply) { while (s + 1 < a.t.n && (int)blockIdx.x >= a.t.g[s + 1].full0) ++s; }
  else { while (s + 1 < a.t.n && (int)blockIdx.x >= a.t.g[s + 1].sym0) ++s; }
  const OrthGeom& G = a.t.g[s];
  const int nti = G.rp / kTile;
  int mat, ti, tj;
  if (PHASE == kApply) {
    const int ntj = G.cp / kTile, k = blockIdx.x - G.full0;
    mat = k / (nti * ntj); ti = k % (nti * ntj) / ntj; tj = k % ntj;
  } else {
    const int per = nti * (nti + 1) / 2, k = blockIdx.x - G.sym0;
    mat = k / per; tj = 0;
    int t = k % per;                       // column tj holds tj + 1 tiles
    while (t > tj) { t -= tj + 1; ++tj; }
    ti = t;
  }
  const OrthPlanes P = orth_planes(G.rp, G.cp);
  _Float16* W = (_Float16*)(a.ws + G.ws) + mat * P.total;
  const int64_t th = flip ? P.t1h : P.t0h, tl = flip ? P.t1l : P.t0l;
  const _Float16* ph = W + (PHASE == kGram ? P.yh : PHASE == kPoly ? P.ah : P.bh);
  const _Float16* pl = W + (PHASE == kGram ? P.yl : PHASE == kPoly ? P.al : P.bl);
  const _Float16* qh = W + (PHASE == kGram ? P.yh : PHASE == kPoly ? P.ah : th);
  const _Float16* ql = W + (PHASE == kGram ? P.yl : PHASE == kPoly ? P.al : tl);
  const int ld = PHASE == kGram ? G.cp : G.rp, K = ld;
  constexpr int NP = 4;
  const bool split = G.split;
  __shared__ _Float16 lds[NP][kTile * kLd];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  f32x16 acc = {}, acl = {};
  const _Float16* src[4] = {ph + (int64_t)ti * kTile * ld, qh + (int64_t)tj * kTile * ld, pl + (int64_t)ti * kTile * ld,
                            ql + (int64_t)tj * kTile * ld};
  for (int k0 = 0; k0 < K; k0 += kTile) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (p >= 2 && !split) continue;
        const int ck = tid + 256 * h, row = ck >> 3, col = (ck & 7) * 8;
        *(f16x8*)&lds[p][row * kLd + col] = *(const f16x8*)(src[p] + (int64_t)row * ld + k0 + col);
      }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kTile; kk += 16) {
      const int at = (lane & 31) * kLd + kk + 8 * (lane >> 5);
      const f16x8 x = *(const f16x8*)&lds[0][wi * kLd + at], y = *(const f16x8*)&lds[1][wj * kLd + at];
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, acc, 0, 0, 0);
      if (split) {
        const f16x8 xl = *(const f16x8*)&lds[NP - 2][wi * kLd + at], yl = *(const f16x8*)&lds[NP - 1][wj * kLd + at];
        acl = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, yl, acl, 0, 0, 0);
        acl = __builtin_amdgcn_mfma_f32_32x32x16_f16(xl, y, acl, 0, 0, 0);
      }
    }
    __syncthreads();
  }
  float lr_q = 0.f, keep = 1.f;
  if (PHASE == kApply && last && o.muon) {
    const float lr = o.st ? o.st->lr : o.lr;
    const float m = (float)a.io[s].m, n = (float)a.io[s].n;
    const float q = o.scale_mode == SNR_MUON_SPECTRAL ? sqrtf(fmaxf(1.f, m / n)) : o.scale_mode == SNR_MUON_RMS ? 0.2f * sqrtf(fmaxf(m, n)) : 1.f;
    lr_q = lr * q; keep = 1.f - lr * o.decay;
  }
  const int j = tj * kTile + wj + (lane & 31);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = ti * kTile + wi + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    float v = acc[e] + acl[e] * (1.f / kLo);
    _Float16 hi, lo;
    if (PHASE == kGram || PHASE == kPoly) {
      if (PHASE == kGram) v *= kAs / (kYs * kYs);
      else v = cb * ((float)W[P.ah + (int64_t)i * G.rp + j] + (float)W[P.al + (int64_t)i * G.rp + j] * (1.f / kLo)) + cc * (v * (1.f / kAs));
      orth_split(v, hi, lo);
      const int64_t dh = PHASE == kGram ? P.ah : P.bh, dl = PHASE == kGram ? P.al : P.bl;
      W[dh + (int64_t)i * G.rp + j] = hi; W[dl + (int64_t)i * G.rp + j] = lo;
      if (ti != tj) { W[dh + (int64_t)j * G.rp + i] = hi; W[dl + (int64_t)j * G.rp + i] = lo; }
    } else {
      const int64_t y = (int64_t)i * G.cp + j;
      v = ca * ((float)W[P.yh + y] + (float)W[P.yl + y] * (1.f / kLo)) + v * (1.f / kAs);
      if (!last) {
        orth_split(v, hi, lo);
        W[P.yh + y] = hi; W[P.yl + y] = lo;
        const int64_t yt = (int64_t)j * G.rp + i, nh = flip ? P.t0h : P.t1h, nl = flip ? P.t0l : P.t1l;
        W[nh + yt] = hi; W[nl + yt] = lo;
      } else if (i < G.r && j < G.c) {
        const OrthIo& io = a.io[s];
        const bool tall = io.m > io.n;
        const int64_t at = mat * io.ob + (tall ? (int64_t)j * io.orow + i : (int64_t)i * io.orow + j);
        v *= 1.f / kYs;
        if (o.muon) { float* p = (float*)io.out + at; *p = *p * keep - lr_q * v; }
        else orth_store(io.out, at, o.dtype, v);
      }
    }
  }
}

}  // namespace snr

using namespace snr;

// ---- host ------------------------------------------------------------------------------------------------------------------
// The largest |s| that the iteration can reach from [0, 1], and the largest |b l + c l^2| on the way: the planes' scales hold 8 and
// 64.  Extremes of the odd quintic lie at the bound or where a + 3 b t + 5 c t^2 = 0, t = s^2.
static bool orth_bounded(int steps, double a, double b, double c) {
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double t2 = top * top;
    auto p = [&](double t) { return fabs(sqrt(t) * (a + b * t + c * t * t)); };
    auto q = [&](double t) { return fabs(b * t + c * t * t); };
    double next = p(t2), poly = q(t2);
    if (c != 0.0) {
      const double d = 9.0 * b * b - 20.0 * a * c;
      if (d >= 0.0)
        for (int sg = -1; sg <= 1; sg += 2) {
          const double t = (-3.0 * b + sg * sqrt(d)) / (10.0 * c);
          if (t > 0.0 && t < t2) next = fmax(next, p(t));
        }
      const double t = -b / (2.0 * c);
      if (t > 0.0 && t < t2) poly = fmax(poly, q(t));
    } else if (b != 0.0) {
      const double t = -a / (3.0 * b);
      if (t > 0.0 && t < t2) next = fmax(next, p(t));
    }
    if (!(next <= 8.0) || !(poly <= 64.0)) return false;
    top = fmax(next, 1e-30);
  }
  return true;
}

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
static int orth_chunks(int64_t count) {
  const int64_t n = (count + 4095) / 4096;
  return (int)(n < 1 ? 1 : n > 1024 ? 1024 : n);
}
static int64_t matrix_bytes(int64_t m, int64_t n) {
  const int64_t r = m < n ? m : n, c = m < n ? n : m;
  return align256(orth_planes((int)((r + kTile - 1) / kTile * kTile), (int)((c + kTile - 1) / kTile * kTile)).total * 2);
}
static const int64_t kMaxSide = 65536, kMaxBatch = 65536;
static int stack_ok(int64_t batch, int64_t m, int64_t n) {
  if (batch < 1 || m < 1 || n < 1 || m > kMaxSide || n > kMaxSide || batch > kMaxBatch) return SNR_ERR_SHAPE;
  return SNR_OK;
}
static int64_t stack_bytes(int64_t batch, int64_t m, int64_t n) {
  return align256(batch * orth_chunks(m * n) * 8) + batch * matrix_bytes(m, n);
}

// one launch sequence over a.t.n stacks whose io fields x, out, mom, strides, m, n and g.batch are filled in
static int orth_run(OrthArgs& a, OrthOut o, int steps, float ca, float cb, float cc, int precision, char* ws, hipStream_t st) {
  int64_t sym = 0, full = 0, chunk = 0, split = 0, part = 0, off = 0;
  for (int s = 0; s < a.t.n; ++s) part += (int64_t)a.t.g[s].batch * orth_chunks((int64_t)a.io[s].m * a.io[s].n);
  off = align256(part * 8);
  part = 0;
  for (int s = 0; s < a.t.n; ++s) {
    OrthIo& io = a.io[s];
    OrthGeom& g = a.t.g[s];
    g.r = io.m < io.n ? io.m : io.n; g.c = io.m < io.n ? io.n : io.m;
    g.rp = (g.r + kTile - 1) / kTile * kTile; g.cp = (g.c + kTile - 1) / kTile * kTile;
    g.split = precision == SNR_ORTH_FP32 || g.r <= 64;
    const int64_t nti = g.rp / kTile, ntj = g.cp / kTile;
    g.sym0 = (int)sym; g.full0 = (int)full; io.chunk0 = (int)chunk; io.split0 = (int)split;
    io.nchunk = orth_chunks((int64_t)io.m * io.n); io.part = part; g.ws = off;
    sym += g.batch * (nti * (nti + 1) / 2); full += g.batch * nti * ntj; split += g.batch * nti * ntj;
    chunk += (int64_t)g.batch * io.nchunk; part += (int64_t)g.batch * io.nchunk;
    off += (int64_t)g.batch * orth_planes(g.rp, g.cp).total * 2;
    if (sym > INT32_MAX || full > INT32_MAX || chunk > INT32_MAX) return SNR_ERR_SHAPE;
  }
  a.part = (double*)ws; a.ws = ws;
  {
    ProfScope ps(K_ORTH_PREPARE, st);
    orth_reduce_kernel<<<dim3((unsigned)chunk), dim3(256), 0, st>>>(a);
    orth_split_kernel<<<dim3((unsigned)split), dim3(256), 0, st>>>(a);
  }
  for (int k = 0; k < steps; ++k) {
    const int flip = k & 1, last = k + 1 == steps;
    ProfScope ps(K_ORTH_PRODUCT, st);
    orth_product_kernel<kGram><<<dim3((unsigned)sym), dim3(256), 0, st>>>(a, o, ca, cb, cc, flip, last);
    orth_product_kernel<kPoly><<<dim3((unsigned)sym), dim3(256), 0, st>>>(a, o, ca, cb, cc, flip, last);
    orth_product_kernel<kApply><<<dim3((unsigned)full), dim3(256), 0, st>>>(a, o, ca, cb, cc, flip, last);
  }
  return launch_status();
}

extern "C" int64_t snr_orthogonalise_ws_bytes(int64_t batch, int64_t rows, int64_t cols, int precision) {
  if (precision != SNR_ORTH_FP16 && precision != SNR_ORTH_FP32) return SNR_ERR_UNSUPPORTED;
  const int st = stack_ok(batch, rows, cols);
  return st != SNR_OK ? st : stack_bytes(batch, rows, cols);
}

extern "C" int snr_orthogonalise(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int64_t x_batch_stride,
                                 int64_t x_row_stride, void* out, int64_t out_batch_stride, int64_t out_row_stride, int steps,
                                 float a, float b, float c, float eps, int precision, void* ws, snr_stream_t stream) {
  SNR_CHECK_ARG(x && out && ws, SNR_ERR_NULL);
  SNR_CHECK_ARG(stack_ok(batch, rows, cols) == SNR_OK && steps >= 1 && steps <= 100 && eps >= 1e-30f, SNR_ERR_SHAPE);
  SNR_CHECK_ARG(out_row_stride >= cols && (batch == 1 || out_batch_stride >= (rows - 1) * out_row_stride + cols), SNR_ERR_SHAPE);
  SNR_CHECK_ARG(dtype == SNR_F32 || dtype == SNR_F16 || dtype == SNR_BF16, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(precision == SNR_ORTH_FP16 || precision == SNR_ORTH_FP32, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(orth_bounded(steps, a, b, c), SNR_ERR_UNSUPPORTED);
  OrthArgs A{};
  A.t.n = 1; A.t.g[0].batch = (int)batch;
  A.io[0] = OrthIo{x, out, nullptr, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride, (int)rows, (int)cols, 0, 0, 0, 0};
  A.dtype = dtype; A.eps = eps;
  OrthOut o{};
  o.dtype = dtype;
  return orth_run(A, o, steps, a, b, c, precision, (char*)ws, (hipStream_t)stream);
}

extern "C" int64_t snr_muon_ws_bytes(const snr_muon_item* items, int n_items, int precision) {
  if (!items) return SNR_ERR_NULL;
  if (n_items < 1) return SNR_ERR_SHAPE;
  if (precision != SNR_ORTH_FP16 && precision != SNR_ORTH_FP32) return SNR_ERR_UNSUPPORTED;
  int64_t most = 0;
  for (int i = 0; i < n_items; i += kOrthMax) {      // one launch sequence after the other: they share the workspace
    int64_t sum = 0;
    for (int k = i; k < n_items && k < i + kOrthMax; ++k) {
      const int st = stack_ok(items[k].batch, items[k].rows, items[k].cols);
      if (st != SNR_OK) return st;
      sum += stack_bytes(items[k].batch, items[k].rows, items[k].cols);
    }
    most = sum > most ? sum : most;
  }
  return most;
}

extern "C" int snr_muon_step_multi(const snr_muon_item* items, int n_items, float lr, float momentum, int nesterov, float weight_decay,
                                   int scale_mode, int steps, float a, float b, float c, float eps, float grad_scale, int precision,
                                   const snr_step_state* state, void* ws, snr_stream_t stream) {
  SNR_CHECK_ARG(items && ws, SNR_ERR_NULL);
  SNR_CHECK_ARG(n_items >= 1 && steps >= 1 && steps <= 100 && eps >= 1e-30f, SNR_ERR_SHAPE);
  SNR_CHECK_ARG(precision == SNR_ORTH_FP16 || precision == SNR_ORTH_FP32, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(scale_mode == SNR_MUON_NONE || scale_mode == SNR_MUON_SPECTRAL || scale_mode == SNR_MUON_RMS, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(orth_bounded(steps, a, b, c), SNR_ERR_UNSUPPORTED);
  for (int i = 0; i < n_items; ++i) {
    SNR_CHECK_ARG(items[i].params && items[i].grads && items[i].momentum, SNR_ERR_NULL);
    SNR_CHECK_ARG(stack_ok(items[i].batch, items[i].rows, items[i].cols) == SNR_OK, SNR_ERR_SHAPE);
  }
  for (int i = 0; i < n_items; i += kOrthMax) {
    OrthArgs A{};
    OrthOut o{};
    for (int k = i; k < n_items && k < i + kOrthMax; ++k) {
      const snr_muon_item& it = items[k];
      const int64_t mn = it.rows * it.cols;
      A.t.g[k - i].batch = (int)it.batch;
      A.io[k - i] = OrthIo{it.grads, it.params, it.momentum, mn, it.cols, mn, it.cols, (int)it.rows, (int)it.cols, 0, 0, 0, 0};
      A.t.n = k - i + 1;
    }
    A.mu = momentum; A.gscale = grad_scale; A.eps = eps; A.nesterov = nesterov;
    o.muon = 1; o.scale_mode = scale_mode; o.lr = lr; o.decay = weight_decay; o.st = state;
    const int st = orth_run(A, o, steps, a, b, c, precision, (char*)ws, (hipStream_t)stream);
    if (st != SNR_OK) return st;
  }
  return SNR_OK;
}
