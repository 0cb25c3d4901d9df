// Orthogonalised updates: Newton-Schulz products on stacks of matrices, and the optimizer step around them (gfx950).
//
//   X_0 = x / max(|x|_F, eps);   A = X X^T;   X <- a X + (b A + c A A) X, `steps` times
//
// acts on the singular values alone (s -> a s + b s^3 + c s^5); x^T gives the transposed result, so every matrix is taken as
// Y [r x c] with r <= c and the Gram matrix A is r x r.
//
// Numbers.  Y, A and B = b A + c A^2 are held as hi + 2^-11 lo, two fp16 planes (22 mantissa bits, as much memory as fp32), each
// scaled by a power of two so that fp16's range covers what a polynomial that stays bounded can reach (orth_bounded below); at the
// other end an entry of Y below 2^-24 keeps 2^-46 absolutely, fp16's subnormals over both scales.
// SNR_ORTH_FP32 multiplies hi hi + hi lo + lo hi (three v_mfma_f32_32x32x16_f16; the dropped lo lo is 2^-24 of a product): fp32's
// accuracy at a third of the fp16 rate, 5 x the fp32 matrix rate.  SNR_ORTH_FP16 multiplies the hi planes only, except where the
// shorter side is 64 or less: there the roundings of a direction's few entries do not average out (up to 1 % of a singular value
// over five steps; a tenth of that from some 64 entries on), and the time is latency, not products.  The term a X is
// taken from both planes in either mode: a rounding of X itself would be full-rank noise, which the iteration amplifies by a per
// step (485 x over five) in the directions x is weak in, while a rounding inside B X only turns directions x is strong in.
#include "snr_common.h"

namespace snr {

constexpr int kOrthMax = 24;                // items per launch sequence: the first kernel's arguments hold the table
constexpr int kPad = 64;                    // what the planes' sides are padded to
constexpr float kYs = 1024.f, kAs = 512.f;  // powers of two that the planes of Y and of A, B are scaled by
constexpr float kLo = 2048.f;               // ... and the lo planes on top

struct OrthGeom {        // matrices of one size, whatever items they come from
  int r, c, rp, cp;      // sides of Y, and padded
  int batch, pad;
  int64_t ws;            // their planes
};
struct OrthIo {          // an item: a stack of matrices
  const void* x;         // the input, or the gradients
  void* out;             // the result, or the parameters
  float* mom;            // momentum (null: plain orthogonalisation)
  int64_t xb, xr, ob, orow;  // element strides: matrix, row (columns are contiguous)
  int m, n;              // sizes as stored
  int batch, geom, mat0; // its matrices are those of a geometry from mat0 on
  int nchunk;            // workgroups (partial sums) per matrix in the reduction
  int64_t part;          // first partial sum (doubles)
};
// What the launches of a sequence share.  The first one has it as arguments and leaves a copy in the workspace for the others: 3.6 KB of
// arguments make a launch 1.6 us longer, and a miss on them costs another microsecond, so an item is found by one load (find_item).
struct OrthArgs {
  int chunk0[kOrthMax], split0[kOrthMax];   // each item's first workgroup in the reduction and in the split
  int sym0[kOrthMax], full0[kOrthMax];      // each geometry's in the symmetric products and in B Y (small kernel: each item's in sym0)
  int n_geom, n_items;
  OrthGeom g[kOrthMax];
  OrthIo io[kOrthMax];
  int dtype;             // of x / out without momentum
  float mu, gscale, eps;
  int nesterov, split;
  double* part;
  char* ws;
};
// What a product needs of it, as arguments where there are few geometries: no chain of loads before the first slice is asked for.
constexpr int kHead = 4;
struct OrthHead {
  const OrthArgs* args;
  char* ws;
  int n;                 // 0: look them up in args
  int first[kHead];      // of the phase
  int spread;            // every XCD has its part of every geometry
  OrthGeom g[kHead];
};
struct OrthOut {         // the last product's epilogue
  int dtype, muon, scale_mode;
  float lr, decay;
  const snr_step_state* st;
};

// Planes of one matrix, in fp16 elements.  Y has two places, a step reads one and writes the other.  Without the split products the
// lo planes of A and B do not exist (B = b A + c A^2 takes A's rounding in both terms: near s = 1 the two errors cancel in part), and
// Y's lo plane, which only the workgroup of its own tile reads then, has one place.
struct OrthPlanes { int64_t h[2], l[2], ah, al, bh, bl, total; };
__host__ __device__ inline OrthPlanes orth_planes(int rp, int cp, bool split) {
  const int64_t y = (int64_t)rp * cp, g = (int64_t)rp * rp;
  OrthPlanes p;
  p.h[0] = 0; p.h[1] = y; p.l[0] = 2 * y; p.l[1] = split ? 3 * y : 2 * y;
  p.ah = p.l[1] + y; p.bh = p.ah + g; p.al = p.bh + (split ? g : 0); p.bl = p.al + (split ? g : 0);
  p.total = (split ? p.bl : p.bh) + g;
  return p;
}

// the item (geometry) a workgroup belongs to: its lanes look at every one's first workgroup at once
__device__ __forceinline__ int find_item(const int* first, int block) {   // (INT_MAX behind the last)
  const int lane = threadIdx.x & 63;
  const bool mine = lane < kOrthMax && block >= first[lane < kOrthMax ? lane : 0];
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
}

// a parameter p becomes keep p - lr_q x
__device__ __forceinline__ void muon_rate(const OrthOut& o, const OrthIo& io, float& lr_q, float& keep) {
  lr_q = 0.f; keep = 1.f;
  if (!o.muon) return;
  const float lr = o.st ? o.st->lr : o.lr, m = (float)io.m, n = (float)io.n;
  const float q = o.scale_mode == SNR_MUON_SPECTRAL ? sqrtf(fmaxf(1.f, m / n)) : o.scale_mode == SNR_MUON_RMS ? 0.2f * sqrtf(fmaxf(m, n)) : 1.f;
  lr_q = lr * q; keep = 1.f - lr * o.decay;
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

// four consecutive elements; wide: they lie on their own size
__device__ __forceinline__ f32x4 orth_load4(const void* p, int64_t i, int dtype, bool wide) {
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  if (wide) {
    if (dtype == SNR_F32) return *(const f32x4*)((const float*)p + i);
    if (dtype == SNR_F16) return __builtin_convertvector(*(const f16x4*)((const _Float16*)p + i), f32x4);
    return __builtin_convertvector(*(const bf16x4*)((const __bf16*)p + i), f32x4);
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = orth_load(p, i + e, dtype);
  return v;
}
__device__ __forceinline__ bool on_grid(const void* p, int64_t a, int64_t b, int bytes) {   // address and strides are multiples of it
  return (((uintptr_t)p | (uint64_t)a | (uint64_t)b) & (bytes - 1)) == 0;
}
__device__ __forceinline__ int type_bytes(int dtype) { return dtype == SNR_F32 ? 4 : 2; }

// sum over the workgroup's W waves, in a fixed order; everyone gets it
template <int W = 4> __device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[W];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < W; w += 4) sum += (part[w] + part[w + 1]) + (part[w + 2] + part[w + 3]);
  return sum;
}

// ---- 1. momentum (in place) and the partial sums of squares of the update, in 64 bits and in a fixed order ------------------
// A pass over the input, bound by memory: 16 B a lane where its place allows, four of them in flight.  With the split (a pass over the
// update, twice its bytes written): 57 us for 12.6 M parameters, gradients and momentum, 300 MB.
__global__ __launch_bounds__(256) void orth_reduce_kernel(OrthArgs a, OrthArgs* copy) {
  if (blockIdx.x == 0) {
    static_assert(sizeof(OrthArgs) % 8 == 0, "copied as words");
    const uint64_t* from = (const uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();    // (the first argument)
    for (int k = threadIdx.x; k < (int)(sizeof(OrthArgs) / 8); k += 256) ((uint64_t*)copy)[k] = from[k];
  }
  const int s = find_item(a.chunk0, blockIdx.x);
  const OrthIo& io = a.io[s];
  const int k = blockIdx.x - a.chunk0[s], mat = k / io.nchunk, ch = k % io.nchunk;
  const int64_t count = (int64_t)io.m * io.n;
  double sum = 0.0;
  if (io.mom || io.xr == io.n) {                // elements one after the other
    const int64_t per = ((count + io.nchunk - 1) / io.nchunk + 3) / 4 * 4, e0 = ch * per, e1 = e0 + per < count ? e0 + per : count;
    const int64_t base = mat * io.xb;
    const int b = io.mom ? 4 : type_bytes(a.dtype);
    const bool wide = on_grid(io.x, base * b, 0, 4 * b) && (!io.mom || on_grid(io.mom, base * 4, 0, 16));
    int64_t e = e0 + 4 * threadIdx.x;
    constexpr int AHEAD = 4;                    // pieces a thread has in flight: one at a time is a memory latency each
    if (wide)
      for (; e + 1024 * (AHEAD - 1) + 4 <= e1; e += 1024 * AHEAD) {
        f32x4 g[AHEAD], mo[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          g[q] = orth_load4(io.x, base + e + 1024 * q, io.mom ? SNR_F32 : a.dtype, true);
          if (io.mom) mo[q] = *(const f32x4*)(io.mom + base + e + 1024 * q);
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          f32x4 u = g[q];
          if (io.mom) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float gs = g[q][i] * a.gscale;
              mo[q][i] = mo[q][i] * a.mu + gs;
              u[i] = a.nesterov ? gs + a.mu * mo[q][i] : mo[q][i];
            }
            *(f32x4*)(io.mom + base + e + 1024 * q) = mo[q];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += (double)u[i] * (double)u[i];
        }
      }
    for (; e < e1; e += 1024) {
      f32x4 u = {0.f, 0.f, 0.f, 0.f};
      const bool whole = e + 4 <= e1;
      if (io.mom) {
        float* M = io.mom + base + e;
        f32x4 g = {0.f, 0.f, 0.f, 0.f}, mo = g;
        if (whole) { g = orth_load4(io.x, base + e, SNR_F32, wide); mo = orth_load4(M, 0, SNR_F32, wide); }
        else for (int i = 0; i < (int)(e1 - e); ++i) { g[i] = ((const float*)io.x)[base + e + i]; mo[i] = M[i]; }
#pragma unroll
        for (int i = 0; i < 4; ++i) { g[i] *= a.gscale; mo[i] = mo[i] * a.mu + g[i]; u[i] = a.nesterov ? g[i] + a.mu * mo[i] : mo[i]; }
        if (whole && wide) *(f32x4*)M = mo;
        else for (int i = 0; i < 4 && e + i < e1; ++i) M[i] = mo[i];
      } else if (whole) {
        u = orth_load4(io.x, base + e, a.dtype, wide);
      } else {
        for (int i = 0; i < (int)(e1 - e); ++i) u[i] = orth_load(io.x, base + e + i, a.dtype);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += (double)u[i] * (double)u[i];
    }
  } else {                                      // row by row
    const int per = (io.m + io.nchunk - 1) / io.nchunk, r0 = ch * per, r1 = r0 + per < io.m ? r0 + per : io.m;
    for (int r = r0; r < r1; ++r)
      for (int c = threadIdx.x; c < io.n; c += 256) {
        const float u = orth_load(io.x, mat * io.xb + r * io.xr + c, a.dtype);
        sum += (double)u * (double)u;
      }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) a.part[io.part + mat * io.nchunk + ch] = sum;
}

// ---- 2. Y = scaled input (transposed where it is tall) as planes, zero in the padding --------------------------------------------
__global__ __launch_bounds__(256) void orth_split_kernel(const OrthArgs* __restrict__ args) {
  const OrthArgs& a = *args;
  const int s = find_item(a.split0, blockIdx.x);
  const OrthIo& io = a.io[s];
  const OrthGeom& G = a.g[io.geom];
  const int nti = G.rp / kPad, ntj = G.cp / kPad;
  const int k = blockIdx.x - a.split0[s], mat = k / (nti * ntj), t = k % (nti * ntj);
  const int i0 = t / ntj * kPad, j0 = t % ntj * kPad;
  const bool tall = io.m > io.n;
  __shared__ float tile[kPad][kPad + 1];
  double sum = 0.0;
  for (int p = threadIdx.x; p < io.nchunk; p += 256) sum += a.part[io.part + mat * io.nchunk + p];
  const double norm = sqrt(block_sum(sum));
  const double scale = (double)kYs / (norm < (double)a.eps ? (double)a.eps : norm);   // (a NaN stays one)
  const OrthPlanes P = orth_planes(G.rp, G.cp, a.split);
  _Float16* W = (_Float16*)(a.ws + G.ws) + (io.mat0 + mat) * P.total;
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  // four columns a thread, sixteen rows of the input at once
  const int b = io.mom ? 4 : type_bytes(a.dtype);
  const bool wide = on_grid(io.x, mat * io.xb * b, io.xr * b, 4 * b) && (!io.mom || on_grid(io.mom, mat * io.xb * 4, io.xr * 4, 16));
  const int c4 = 4 * (threadIdx.x & 15), r = threadIdx.x >> 4;
#pragma unroll
  for (int q = r; q < kPad; q += 16) {
    const int mi = (tall ? j0 : i0) + q, nj = (tall ? i0 : j0) + c4;
    f32x4 u = {0.f, 0.f, 0.f, 0.f};
    if (mi < io.m && nj < io.n) {
      const int64_t at = mat * io.xb + mi * io.xr + nj;
      const bool whole = nj + 4 <= io.n;
      if (io.mom) {
        f32x4 mo = u;
        if (whole) mo = orth_load4(io.mom, at, SNR_F32, wide);
        else for (int e = 0; e < io.n - nj; ++e) mo[e] = io.mom[at + e];
        u = mo;
        if (a.nesterov) {
          f32x4 g = {0.f, 0.f, 0.f, 0.f};
          if (whole) g = orth_load4(io.x, at, SNR_F32, wide);
          else for (int e = 0; e < io.n - nj; ++e) g[e] = ((const float*)io.x)[at + e];
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = g[e] * a.gscale + a.mu * mo[e];
        }
      } else if (whole) {
        u = orth_load4(io.x, at, a.dtype, wide);
      } else {
        for (int e = 0; e < io.n - nj; ++e) u[e] = orth_load(io.x, at + e, a.dtype);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = (float)((double)u[e] * scale);
    }
    if (tall) {
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[c4 + e][q] = u[e];
    } else {
      f16x4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 x, y; orth_split(u[e], x, y); h[e] = x; l[e] = y; }
      const int64_t y = (int64_t)(i0 + q) * G.cp + j0 + c4;
      *(f16x4*)(W + P.h[0] + y) = h; *(f16x4*)(W + P.l[0] + y) = l;
    }
  }
  if (!tall) return;
  __syncthreads();
#pragma unroll
  for (int q = r; q < kPad; q += 16) {
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 x, y; orth_split(tile[q][c4 + e], x, y); h[e] = x; l[e] = y; }
    const int64_t y = (int64_t)(i0 + q) * G.cp + j0 + c4;
    *(f16x4*)(W + P.h[0] + y) = h; *(f16x4*)(W + P.l[0] + y) = l;
  }
}

// ---- 3. the products -------------------------------------------------------------------------------------------------------------
//   Gram:  A = Y Y^T          (symmetric: tiles i <= j, mirrored)
//   Poly:  B = b A + c A A^T  (symmetric)
//   Apply: Y <- a Y + B Y, or the result
//
// A workgroup makes a T x T tile C[i][j] = sum_k P[i][k] Q[j][k] (Apply: Q[k][j]) from BK-wide slices of K that stream through LDS by DMA
// (16 B a lane), STAGES - 1 of them in flight.  A slice's rows of P are RB bytes, their 16 B chunks permuted so that the 16 rows that
// 16 lanes read at one k fall on different banks; Apply's Q slice has rows of T columns, read transposed (ds_read_b64_tr_b16: four k of
// a column to a lane).  The planes are padded to 64 only: a tile that hangs over reads the last row or column again and drops what
// comes of it.
//
// What bounds them.  A launch costs some 5 us however little it has to do (2 x 128 x 283: 6.5 us a product), plus a tile's first
// slices and its epilogue; then a compute unit takes in about 88 B / ns by DMA (128-wide tiles: 32 KB and 0.37 us a slice), which is
// what larger tiles are for; below that, compute units without a tile (136 of 128 a symmetric product of 2048^2: 120 idle, 0.6 PF); and
// with the whole chip busy, power: 4096^2 runs at 0.92 PF in all, B Y (256 wide) at 1.0, where a library product of the same size and
// data reaches 0.99 and one of zeros 1.5 (fp16; 8192^3: 1.30 and 1.8).  Halving the fragments' reads from LDS changes nothing, nor does
// the order of the tiles.
enum { kGram = 0, kPoly = 1, kApply = 2 };   // template PHASE; LAST: the result instead of planes

template <int T_, int WI_, int WJ_, bool SPLIT_, int STAGES_, int BK_> struct TileCfg {
  static constexpr int BAND = T_ >= 192 ? 4 : 8;                  // tiles side by side that an XCD takes together
  static constexpr int BK = BK_, CH = BK_ / 8, RB = 2 * BK_, RPL = 1024 / RB, STAGES = STAGES_, T = T_, WI = WI_, WJ = WJ_, NW = WI_ * WJ_, NT = 64 * NW;
  static constexpr bool SPLIT = SPLIT_;
  static constexpr int TI = T / WI / 32, TJ = T / WJ / 32;       // 32 x 32 blocks of a wave
  static constexpr int SECT = T * RB;                             // bytes of one operand plane's slice
  static constexpr int STAGE = SECT * (SPLIT ? 4 : 2);
  static constexpr int PER = T / RPL / NW;                        // DMA instructions of a wave per plane: RPL rows each
  static_assert(T % (RPL * NW) == 0 && T % (32 * WI) == 0 && T % (32 * WJ) == 0, "whole blocks");
  static constexpr int LOADS = PER * (SPLIT ? 4 : 2);             // ... per slice
  // where 16-byte chunk c of row r lies in a slice's plane
  static __host__ __device__ constexpr int swz(int r, int c) { return r * RB + ((c ^ (BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3)) << 4); }
  // ... and, in Apply's Q slice, chunk c of row k: the 64 B that a group of 16 lanes reads of four rows fall on different banks
  static __host__ __device__ constexpr int swzt(int k, int c) { return k * 2 * T + ((c ^ (T % 128 == 0 ? (k & 3) << 2 : T > 32 ? (k >> 1 & 1) << 2 : 0)) << 4); }
  static constexpr int EPI = NW * 32 * 36 * 4;                    // epilogue: a 32 x 36 fp32 block a wave
};

__device__ __forceinline__ unsigned lds_at(const char* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

// A slice, 16 bytes a lane and load, from base + off straight to LDS: a wave's pieces lie NW KB apart, plane after plane.  In asm, as
// the compiler cannot tell which LDS reads such a load concerns and waits for all of them; the waits are landed()'s.  There is no
// register to be overwritten, and the loads are counted in order with every other one, so that the compiler's own waits only get
// stricter.  Nor does the compiler see into it for hazards: a VALU write of a base (a readfirstlane, a spilled SGPR read back) has to be
// five wait states away, whatever it puts in front: s_mov and the four of s_nop 3, once for the whole slice (at every load: 4 x 1000 x
// 333 fp16 161 -> 169 us, 2048 x 8192 bf16 834 -> 860); tools/check_lds_asm.py --own holds the listing to it.  m0 needs one.
// A slice past the end is one 16-byte piece again and again: the number of loads in flight stays what the waits count on.
#define SNR_DMA_FIRST "s_mov_b32 m0, %[d]\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %[x0], %[p0]"
#define SNR_DMA(off, base) "\n\ts_add_u32 m0, m0, %[s]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[" off "], %[" base "]"
template <class C>
__device__ __forceinline__ void fetch_slice(unsigned dst, const _Float16* const (&src)[4], const unsigned (&voff)[2][C::PER], int k, int n, int64_t ldq, int wave) {
  static_assert(C::SECT == C::PER * C::NW * 1024, "a plane's pieces and the next one's first are as far apart");
  const int k0 = k < n ? k * C::BK : 0;
  const unsigned keep = k < n ? ~0u : 0u, d = dst + wave * 1024;
  const _Float16 *p0 = src[0] + k0, *q0 = src[1] + k0 * ldq, *p1 = src[2] + k0, *q1 = src[3] + k0 * ldq;   // hi of P and Q, lo
  unsigned x[4], y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) { x[q] = voff[0][q < C::PER ? q : 0] & keep; y[q] = voff[1][q < C::PER ? q : 0] & keep; }
#define SNR_DMA_ARGS(...) [d] "s"(d), [s] "n"(C::NW * 1024), [p0] "s"(p0), [q0] "s"(q0), __VA_ARGS__ : "memory", "m0", "scc"
  if constexpr (C::SPLIT && C::PER == 1)
    asm volatile(SNR_DMA_FIRST SNR_DMA("y0", "q0") SNR_DMA("x0", "p1") SNR_DMA("y0", "q1")
                 ::SNR_DMA_ARGS([p1] "s"(p1), [q1] "s"(q1), [x0] "v"(x[0]), [y0] "v"(y[0])));
  else if constexpr (C::SPLIT && C::PER == 2)
    asm volatile(SNR_DMA_FIRST SNR_DMA("x1", "p0") SNR_DMA("y0", "q0") SNR_DMA("y1", "q0")
                 SNR_DMA("x0", "p1") SNR_DMA("x1", "p1") SNR_DMA("y0", "q1") SNR_DMA("y1", "q1")
                 ::SNR_DMA_ARGS([p1] "s"(p1), [q1] "s"(q1), [x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1])));
  else if constexpr (C::SPLIT && C::PER == 4)
    asm volatile(SNR_DMA_FIRST SNR_DMA("x1", "p0") SNR_DMA("x2", "p0") SNR_DMA("x3", "p0")
                 SNR_DMA("y0", "q0") SNR_DMA("y1", "q0") SNR_DMA("y2", "q0") SNR_DMA("y3", "q0")
                 SNR_DMA("x0", "p1") SNR_DMA("x1", "p1") SNR_DMA("x2", "p1") SNR_DMA("x3", "p1")
                 SNR_DMA("y0", "q1") SNR_DMA("y1", "q1") SNR_DMA("y2", "q1") SNR_DMA("y3", "q1")
                 ::SNR_DMA_ARGS([p1] "s"(p1), [q1] "s"(q1), [x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]),
                                [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3])));
  else if constexpr (C::PER == 2)
    asm volatile(SNR_DMA_FIRST SNR_DMA("x1", "p0") SNR_DMA("y0", "q0") SNR_DMA("y1", "q0")
                 ::SNR_DMA_ARGS([x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1])));
  else {
    static_assert(!C::SPLIT && C::PER == 4, "a slice's loads are written out for these");
    asm volatile(SNR_DMA_FIRST SNR_DMA("x1", "p0") SNR_DMA("x2", "p0") SNR_DMA("x3", "p0")
                 SNR_DMA("y0", "q0") SNR_DMA("y1", "q0") SNR_DMA("y2", "q0") SNR_DMA("y3", "q0")
                 ::SNR_DMA_ARGS([x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]),
                                [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3])));
  }
#undef SNR_DMA_ARGS
}
#undef SNR_DMA_FIRST
#undef SNR_DMA

// one slice: the fragments of the next 16 of K are read while those of this 16 are multiplied (sched_barrier keeps the compiler from
// moving the reads back to their use: a wave alone on its SIMD would wait out LDS's latency eight times a slice)
template <class C> struct Frags { f16x8 x[C::TI], y[C::TJ], xl[C::SPLIT ? C::TI : 1], yl[C::SPLIT ? C::TJ : 1]; };
typedef short s16x4 __attribute__((ext_vector_type(4)));
// eight k of 32 columns from rows of columns: lane l gets column l % 32, k = 8 (l / 32) + 0 .. 7 of the 16 at kk; of a group of 16 lanes
// lane i points at four columns of row i / 4, and receives one column of the four rows
template <class C> __device__ __forceinline__ f16x8 read_turned(const char* src, int kk, int col, int lane) {
  const int k = 16 * kk + 8 * (lane >> 5) + ((lane & 15) >> 2), c = col + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
  auto part = [&](int kq) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(src + C::swzt(kq, c >> 3) + (c & 4) * 2)); };
  union { s16x4 q[2]; f16x8 v; } u;
  u.q[0] = part(k); u.q[1] = part(k + 4);
  return u.v;
}
template <class C, bool TURN> __device__ __forceinline__ void read_frags(Frags<C>& f, const char* src, int kk, int wi, int wj, int lane) {
  const int at = C::swz(lane & 31, 2 * kk + (lane >> 5));
#pragma unroll
  for (int i = 0; i < C::TI; ++i) f.x[i] = *(const f16x8*)(src + (wi + 32 * i) * C::RB + at);
#pragma unroll
  for (int j = 0; j < C::TJ; ++j) {
    if constexpr (TURN) f.y[j] = read_turned<C>(src + C::SECT, kk, wj + 32 * j, lane);
    else f.y[j] = *(const f16x8*)(src + C::SECT + (wj + 32 * j) * C::RB + at);
  }
  if constexpr (C::SPLIT) {
#pragma unroll
    for (int i = 0; i < C::TI; ++i) f.xl[i] = *(const f16x8*)(src + 2 * C::SECT + (wi + 32 * i) * C::RB + at);
#pragma unroll
    for (int j = 0; j < C::TJ; ++j) {
      if constexpr (TURN) f.yl[j] = read_turned<C>(src + 3 * C::SECT, kk, wj + 32 * j, lane);
      else f.yl[j] = *(const f16x8*)(src + 3 * C::SECT + (wj + 32 * j) * C::RB + at);
    }
  }
}
template <class C>
__device__ __forceinline__ void mul_frags(const Frags<C>& g, f32x16 (&acc)[C::TI][C::TJ], f32x16 (&acl)[C::SPLIT ? C::TI : 1][C::SPLIT ? C::TJ : 1]) {
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < C::TI; ++i)
#pragma unroll
    for (int j = 0; j < C::TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.x[i], g.y[j], acc[i][j], 0, 0, 0);
  if constexpr (C::SPLIT) {
#pragma unroll
    for (int i = 0; i < C::TI; ++i)
#pragma unroll
      for (int j = 0; j < C::TJ; ++j) acl[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.x[i], g.yl[j], acl[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < C::TI; ++i)
#pragma unroll
      for (int j = 0; j < C::TJ; ++j) acl[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.xl[i], g.y[j], acl[i][j], 0, 0, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// this wave's DMA has landed but for the last N loads, and its LDS reads are done; then every wave's
template <int N> __device__ __forceinline__ void landed() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4 << 14));   // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// what lanes of this wave wrote to LDS is read by others of it
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 16 consecutive fp16 of a row (32 B) as two vectors
struct Half16 { f16x8 a, b; };
__device__ __forceinline__ Half16 load16(const _Float16* p) { return Half16{*(const f16x8*)p, *(const f16x8*)(p + 8)}; }
template <bool LO> __device__ __forceinline__ void store16(const float (&v)[16], _Float16* hi, _Float16* lo) {
  f16x8 h[2], l[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    _Float16 a, b;
    orth_split(v[e], a, b);
    h[e >> 3][e & 7] = a; l[e >> 3][e & 7] = b;
  }
  *(f16x8*)hi = h[0]; *(f16x8*)(hi + 8) = h[1];
  if constexpr (LO) { *(f16x8*)lo = l[0]; *(f16x8*)(lo + 8) = l[1]; }
}

__device__ __forceinline__ void store16_out(void* p, int64_t i, int dtype, const float (&v)[16]) {
  typedef float f32v __attribute__((ext_vector_type(8)));
#pragma unroll
  for (int e = 0; e < 16; e += 8) {
    f32v x;
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = v[e + q];
    if (dtype == SNR_F32) {
      *(f32x4*)((float*)p + i + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
      *(f32x4*)((float*)p + i + e + 4) = f32x4{v[e + 4], v[e + 5], v[e + 6], v[e + 7]};
    } else if (dtype == SNR_F16) {
      *(f16x8*)((_Float16*)p + i + e) = __builtin_convertvector(x, f16x8);
    } else {
      *(bf16x8*)((__bf16*)p + i + e) = __builtin_convertvector(x, bf16x8);
    }
  }
}

// Workgroups go round the 8 XCDs, each with its own L2: number n of them (a multiple of 8) so that an XCD has a run of neighbours, which
// share operand rows.  Of the whole launch, or, where geometries differ in K, of each: an XCD with all the long ones would be the last
// (us, fp32: 2048^2 with 2048 x 8192 3310 -> 2630, eight of 512^2 with four of 512 x 2048 434 -> 398; but 7 of 256^2 with 256 x 319 and
// 128 x 283 125 -> 131, where a small geometry is better off in one L2).
__device__ __forceinline__ int xcd_block(int k, int n) { return (k & 7) * (n >> 3) + (k >> 3); }
// tile t of the upper triangle (ti <= tj) of n x n tiles, taken in bands of BAND columns, row by row within a band
template <int BAND> __device__ __forceinline__ void sym_tile(int t, int n, int& ti, int& tj) {
  int b = (int)((sqrtf(8.f * t + 1.f) - 1.f) * (0.5f / BAND));     // column c starts at tile c (c + 1) / 2
  while (b > 0 && BAND * b * (BAND * b + 1) / 2 > t) --b;
  while (BAND * (b + 1) < n && BAND * (b + 1) * (BAND * (b + 1) + 1) / 2 <= t) ++b;
  const int c0 = BAND * b, w = n - c0 < BAND ? n - c0 : BAND;
  int q = t - c0 * (c0 + 1) / 2;
  if (q < (c0 + 1) * w) { ti = q / w; tj = c0 + q % w; return; }
  q -= (c0 + 1) * w;
  int r = 1;
  while (q >= w - r) { q -= w - r; ++r; }
  ti = c0 + r; tj = c0 + r + q;
}

template <int PHASE, bool last, class C>
__global__ __launch_bounds__(C::NT) void orth_product_kernel(OrthHead h, OrthOut o, float ca, float cb, float cc, int flip) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (asked for together: one after the other they are a miss each)
  const int blocks = gridDim.x;
  asm volatile("" ::"s"(h.n), "s"(h.spread), "s"(blocks), "s"(h.ws), "s"(h.first[1]), "s"(h.first[2]), "s"(h.first[3]), "s"(h.g[0].rp),
               "s"(h.g[0].cp), "s"(h.g[0].batch), "s"(h.g[0].ws), "s"(h.g[1].rp), "s"(h.g[1].cp), "s"(h.g[1].batch), "s"(h.g[1].ws), "s"(h.g[2].rp),
               "s"(h.g[2].cp), "s"(h.g[2].batch), "s"(h.g[2].ws), "s"(h.g[3].rp), "s"(h.g[3].cp), "s"(h.g[3].batch), "s"(h.g[3].ws));
  const int block = h.spread ? (int)blockIdx.x : xcd_block(blockIdx.x, blocks);
  int s = 0, first = 0, next = h.first[1];
  struct { int r, c, rp, cp, batch; int64_t ws; } G = {h.g[0].r, h.g[0].c, h.g[0].rp, h.g[0].cp, h.g[0].batch, h.g[0].ws};
  if (h.n == 0) {
    const int* const all = PHASE == kApply ? h.args->full0 : h.args->sym0;
    s = find_item(all, block); first = all[s]; next = s + 1 < kOrthMax ? all[s + 1] : INT32_MAX;
    const OrthGeom& g = h.args->g[s];
    G.r = g.r; G.c = g.c; G.rp = g.rp; G.cp = g.cp; G.batch = g.batch; G.ws = g.ws;
  } else {
#pragma unroll
    for (int k = 1; k < kHead; ++k) {
      const bool is = block >= h.first[k];
      s = is ? k : s; first = is ? h.first[k] : first; next = is ? (k + 1 < kHead ? h.first[k + 1] : INT32_MAX) : next;
      G.r = is ? h.g[k].r : G.r; G.c = is ? h.g[k].c : G.c; G.rp = is ? h.g[k].rp : G.rp; G.cp = is ? h.g[k].cp : G.cp;
      G.batch = is ? h.g[k].batch : G.batch; G.ws = is ? h.g[k].ws : G.ws;
    }
  }
  if (next == INT32_MAX) next = blocks;
  const int nti = (G.rp + C::T - 1) / C::T, tile = h.spread ? xcd_block(block - first, next - first) : block - first;
  int mat, ti, tj;
  if (PHASE == kApply) {
    const int ntj = (G.cp + C::T - 1) / C::T, t = tile % (nti * ntj), band = t / (C::BAND * ntj);
    const int h = nti - band * C::BAND < C::BAND ? nti - band * C::BAND : C::BAND, q = t - band * C::BAND * ntj;
    mat = tile / (nti * ntj); ti = band * C::BAND + q % h; tj = q / h;
  } else {
    const int per = nti * (nti + 1) / 2;
    mat = tile / per;
    sym_tile<C::BAND>(tile % per, nti, ti, tj);
  }
  if (mat >= G.batch) return;        // what rounds the geometry's workgroups up
  const OrthPlanes P = orth_planes(G.rp, G.cp, C::SPLIT);
  _Float16* W = (_Float16*)(h.ws + G.ws) + mat * P.total;
  const int64_t yh = flip ? P.h[1] : P.h[0], yl = flip ? P.l[1] : P.l[0];
  const int wi = (wave / C::WJ) * (C::T / C::WI), wj = (wave % C::WJ) * (C::T / C::WJ);
  f32x16 acc[C::TI][C::TJ] = {}, acl[C::SPLIT ? C::TI : 1][C::SPLIT ? C::TJ : 1] = {};
  // one array per stage: no read of one is held up by a write to another
  __shared__ __attribute__((aligned(16))) char s0[C::STAGE > C::EPI ? C::STAGE : C::EPI];
  __shared__ __attribute__((aligned(16))) char s1[C::STAGE];
  __shared__ __attribute__((aligned(16))) char s2[C::STAGES > 2 ? C::STAGE : 16];
  __shared__ __attribute__((aligned(16))) char s3[C::STAGES > 3 ? C::STAGE : 16];
  char* const buf[4] = {s0, s1, s2, s3};
  const unsigned at[4] = {lds_at(s0), lds_at(s1), lds_at(s2), lds_at(s3)};
  const int K = PHASE == kGram ? G.cp : G.rp;
  const int64_t ldq = PHASE == kApply ? G.cp : 1;      // how far apart slices of Q lie, an element of k
  const int64_t ph = PHASE == kGram ? yh : PHASE == kPoly ? P.ah : P.bh, pl = PHASE == kGram ? yl : PHASE == kPoly ? P.al : P.bl;
  const int64_t pi = (int64_t)ti * C::T * K, qj = PHASE == kApply ? (int64_t)tj * C::T : (int64_t)tj * C::T * K;
  const _Float16* src[4] = {W + ph + pi, W + (PHASE == kApply ? yh : ph) + qj, W + pl + pi, W + (PHASE == kApply ? yl : pl) + qj};
  unsigned voff[2][C::PER];         // bytes
#pragma unroll
  for (int q = 0; q < C::PER; ++q) {
    const int blk = wave + q * C::NW, row = blk * C::RPL + lane / C::CH, col = (C::swz(row, lane % C::CH) - row * C::RB) / 2;
    const int lp = G.rp - 1 - ti * C::T;
    voff[0][q] = 2u * ((row < lp ? row : lp) * K + col);
    if constexpr (PHASE == kApply) {
      const int at = blk * 64 + lane, kr = at / (C::T / 8), kc = (C::swzt(kr, at % (C::T / 8)) - kr * 2 * C::T) / 2, lc = G.cp - 8 - tj * C::T;
      voff[1][q] = 2u * (kr * G.cp + (kc < lc ? kc : lc));
    } else {
      const int lq = G.rp - 1 - tj * C::T;
      voff[1][q] = 2u * ((row < lq ? row : lq) * K + col);
    }
  }
  const int n = K / C::BK;
  // (one block a wave: what the epilogue adds to is read ahead of the products)
  constexpr bool EARLY = C::TI * C::TJ == 1 && PHASE != kGram;
  const int64_t ld_out = PHASE == kApply ? G.cp : G.rp;
  Half16 eh = {}, el = {};
  if (EARLY && ti * C::T + wi < G.rp && tj * C::T + wj < ld_out) {
    const int64_t y = (int64_t)(ti * C::T + wi + (lane >> 1)) * ld_out + tj * C::T + wj + (lane & 1) * 16;
    eh = load16(W + (PHASE == kPoly ? P.ah : yh) + y);
    if (PHASE == kApply || C::SPLIT) el = load16(W + (PHASE == kPoly ? P.al : yl) + y);
  }
  // Slice k's last 16 of K are multiplied behind the barrier that frees its buffer and shows slice k + 1, whose first fragments are
  // read under them; slice k + STAGES is fetched into the buffer at once.
  constexpr int KK = C::BK / 16;
  Frags<C> f[2];
#pragma unroll
  for (int u = 0; u < C::STAGES; ++u) fetch_slice<C>(at[u], src, voff, u, n, ldq, wave);
  landed<(C::STAGES - 1) * C::LOADS>();
  read_frags<C, PHASE == kApply>(f[0], s0, 0, wi, wj, lane);
  int k = 0;
  for (; k + C::STAGES <= n; k += C::STAGES) {
#pragma unroll
    for (int u = 0; u < C::STAGES; ++u) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk + 1 < KK) read_frags<C, PHASE == kApply>(f[(kk + 1) & 1], buf[u], kk + 1, wi, wj, lane);
        else {
          landed<(C::STAGES - 2) * C::LOADS>();
          fetch_slice<C>(at[u], src, voff, k + u + C::STAGES, n, ldq, wave);
          read_frags<C, PHASE == kApply>(f[0], buf[(u + 1) % C::STAGES], 0, wi, wj, lane);
        }
        mul_frags<C>(f[kk & 1], acc, acl);
      }
    }
  }
  landed<0>();
#pragma unroll
  for (int u = 0; u < C::STAGES - 1; ++u)
    if (k + u < n) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (u || kk) read_frags<C, PHASE == kApply>(f[kk & 1], buf[u], kk, wi, wj, lane);
        mul_frags<C>(f[kk & 1], acc, acl);
      }
    }
  landed<0>();

  // epilogue: a wave turns its 32 x 32 blocks in LDS, so that rows (and, for the mirrored or transposed copy, columns) are written
  // 32 B a lane
  float (*blk)[36] = (float (*)[36])(s0 + wave * (32 * 36 * 4));
  float lr_q = 0.f, keep = 1.f;
  int item = 0;
  if (last) {                         // the item that the matrix belongs to, and its number there
    const OrthArgs& a = *h.args;
    const int at = lane < kOrthMax ? lane : 0;
    const bool mine = lane < a.n_items && a.io[at].geom == s && mat >= a.io[at].mat0 && mat < a.io[at].mat0 + a.io[at].batch;
    item = __builtin_amdgcn_readfirstlane(__ffsll(__ballot(mine)) - 1);
    mat -= a.io[item].mat0;
    muon_rate(o, a.io[item], lr_q, keep);
  }
  const OrthIo& io = h.args->io[item];
  const int row = lane >> 1, c0 = (lane & 1) * 16;
  bool wide = false;                  // 16-byte pieces of the result
  if (last) { const int b = o.muon ? 4 : type_bytes(o.dtype); wide = on_grid(io.out, mat * io.ob * b, io.orow * b, 16); }
#pragma unroll
  for (int bi = 0; bi < C::TI; ++bi)
#pragma unroll
    for (int bj = 0; bj < C::TJ; ++bj) {
      const int i0 = ti * C::T + wi + 32 * bi, j0 = tj * C::T + wj + 32 * bj;
      if (i0 >= G.rp || j0 >= (PHASE == kApply ? G.cp : G.rp)) continue;
      wave_sync();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = acc[bi][bj][e];
        if constexpr (C::SPLIT) v += acl[bi][bj][e] * (1.f / kLo);
        blk[8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)][lane & 31] = v;
      }
      wave_sync();
      float v[16];
      const int64_t y = (int64_t)(i0 + row) * ld_out + j0 + c0;
      if (PHASE == kGram) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = blk[row][c0 + e] * (kAs / (kYs * kYs));
      } else {
        const Half16 h = EARLY ? eh : load16(W + (PHASE == kPoly ? P.ah : yh) + y);
        Half16 l = el;
        if (!EARLY && (PHASE == kApply || C::SPLIT)) l = load16(W + (PHASE == kPoly ? P.al : yl) + y);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float old = (float)(e < 8 ? h.a[e & 7] : h.b[e & 7]);
          if (PHASE == kApply || C::SPLIT) old += (float)(e < 8 ? l.a[e & 7] : l.b[e & 7]) * (1.f / kLo);
          v[e] = PHASE == kPoly ? cb * old + cc * (blk[row][c0 + e] * (1.f / kAs)) : ca * old + blk[row][c0 + e] * (1.f / kAs);
        }
      }
      const int64_t dh = PHASE == kGram ? P.ah : PHASE == kPoly ? P.bh : flip ? P.h[0] : P.h[1];
      const int64_t dl = PHASE == kGram ? P.al : PHASE == kPoly ? P.bl : flip ? P.l[0] : P.l[1];
      if (!last) store16<PHASE == kApply || C::SPLIT>(v, W + dh + y, W + dl + y);
      if (PHASE == kApply ? !last : ti == tj) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) blk[row][c0 + e] = v[e];
      wave_sync();
      if (PHASE != kApply) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = blk[c0 + e][row];
        const int64_t yt = (int64_t)(j0 + row) * G.rp + i0 + c0;
        store16<C::SPLIT>(v, W + dh + yt, W + dl + yt);
      } else {
        const bool tall = io.m > io.n;
        const int i = i0 + row, j = j0 + row;        // a row of the result: Y's or, where it is tall, Y's column
        const int from = (tall ? i0 : j0) + c0, len = tall ? G.r : G.c;
        const int64_t at = mat * io.ob + (tall ? j : i) * io.orow + from;
        if (wide && (tall ? i0 : j0) + 32 <= len) {
          const bool mine = (tall ? j : i) < (tall ? G.c : G.r);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = (tall ? blk[c0 + e][row] : blk[row][c0 + e]) * (1.f / kYs);
          if (!mine) {
          } else if (o.muon) {
            float* p = (float*)io.out + at;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              f32x4 x = *(const f32x4*)(p + e);
#pragma unroll
              for (int q = 0; q < 4; ++q) x[q] = x[q] * keep - lr_q * v[e + q];
              *(f32x4*)(p + e) = x;
            }
          } else {
            store16_out(io.out, at, o.dtype, v);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {             // lanes along the result's rows
            const int u = 2 * e + (lane >> 5), w = lane & 31;
            const int ei = i0 + (tall ? w : u), ej = j0 + (tall ? u : w);
            if (ei >= G.r || ej >= G.c) continue;
            const float x = (tall ? blk[w][u] : blk[u][w]) * (1.f / kYs);
            const int64_t at1 = mat * io.ob + (tall ? (int64_t)ej * io.orow + ei : (int64_t)ei * io.orow + ej);
            if (o.muon) { float* p = (float*)io.out + at1; *p = *p * keep - lr_q * x; }
            else orth_store(io.out, at1, o.dtype, x);
          }
        }
      }
    }
}

// ---- 4. small matrices: everything in one workgroup ----------------------------------------------------------------------------------
// Where a matrix fits, a workgroup keeps it from its input to its result: 17 launches of a microsecond's work each become one.  Y stays in
// registers in 32 bits, as 32 x 32 blocks in the layout the matrix instructions give them back in (NB a wave; a wave's block never
// moves); LDS holds the planes that all waves multiply from: 32 RB rows, 64 NB columns, hi and lo (SPLIT) or hi alone.  As many columns
// as fit 160 KB beside A, with B in A's place where there is no room for both: 64 x 448 and 128 x 128 split.  128 x 384 of hi planes
// would fit, but not the 256 registers that 8 waves leave each other: 61 of them would be spilled; 128 x 320, and 128 x 128 split, spill 7
// outside the products' loops.  Bound by the latency of a few rounds of LDS reads and products between four barriers a step, then by
// LDS; two matrices use two compute units.  Us a call, here / in tiles: 2 x 128 x 283 fp16 47 / 82, 2 x 128 x 128 fp16 29 / 70,
// fp32 57 / 84; 1024 x 128 x 128 fp16 120 / 538, fp32 242 / 708; 64 x 64: 17 (what calling it takes), 64 x 448: 52.
template <int RB, int NB, bool SPLIT>
__global__ __launch_bounds__(128 * RB) void orth_small_kernel(OrthArgs a, OrthOut o, float ca, float cb, float cc, int steps) {
  constexpr int R = 32 * RB, LD = R + (RB == 2 ? 8 : 16);    // rows in fp16: off a multiple of 128 B, so that rows at one k spread over the banks
  constexpr bool ROOM = (64 * NB + 2 * R) * LD * (SPLIT ? 4 : 2) <= 160 * 1024 - 128;   // ... for B beside A
  __shared__ __attribute__((aligned(16))) _Float16 yh[64 * NB * LD], yl[SPLIT ? 64 * NB * LD : 8], ah[R * LD], al[SPLIT ? R * LD : 8];
  __shared__ __attribute__((aligned(16))) _Float16 own_h[ROOM ? R * LD : 8], own_l[ROOM && SPLIT ? R * LD : 8];
  _Float16 *bh = ROOM ? own_h : ah, *bl = ROOM ? own_l : al;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int s = find_item(a.sym0, blockIdx.x);
  const OrthIo& io = a.io[s];
  const int64_t mat = blockIdx.x - a.sym0[s];
  const bool tall = io.m > io.n;
  int r = tall ? io.n : io.m, c = tall ? io.m : io.n;
  const int lj = lane & 31, li = 4 * (lane >> 5);
  const int y0 = 32 * (wave % RB), x0 = 32 * (wave / RB);     // this wave's blocks of Y: at y0, x0 + 64 b
  // what lies outside the matrix is read at its last row and column, so that no load waits for a branch
  float v[NB][16];
  int64_t at[16];
  const int64_t in_i = tall ? 1 : io.xr, in_j = tall ? io.xr : 1;
  auto where = [&](int b, int64_t base, int64_t pi, int64_t pj) {
    __builtin_amdgcn_sched_barrier(0);               // one block's addresses at a time: seven would not fit the registers
    const int i0 = y0 + li, j = x0 + 64 * b + lj;
#pragma unroll
    for (int e = 0; e < 16; ++e) at[e] = base + min(i0 + 8 * (e >> 2) + (e & 3), r - 1) * pi + min(j, c - 1) * pj;
  };
  auto inside = [&](int b, int e) { return y0 + li + 8 * (e >> 2) + (e & 3) < r && x0 + 64 * b + lj < c; };
  // addresses and the tests of what lies inside are made anew: kept from one loop to the next, they would not fit the registers
  auto again = [&] { asm volatile("" : "+s"(r), "+s"(c)); };
  auto fetch = [&](auto* x) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      where(b, mat * io.xb, in_i, in_j);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[b][e] = (float)x[at[e]];
    }
  };
  if (io.mom) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      where(b, mat * io.xb, in_i, in_j);
      float mo[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) { v[b][e] = ((const float*)io.x)[at[e]]; mo[e] = io.mom[at[e]]; }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float g = v[b][e] * a.gscale;
        mo[e] = mo[e] * a.mu + g;
        v[b][e] = a.nesterov ? g + a.mu * mo[e] : mo[e];
        if (inside(b, e)) io.mom[at[e]] = mo[e];
      }
    }
  } else if (a.dtype == SNR_F32) {
    fetch((const float*)io.x);
  } else if (a.dtype == SNR_F16) {
    fetch((const _Float16*)io.x);
  } else {
    fetch((const __bf16*)io.x);
  }
  again();
  double sum = 0.0;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (!inside(b, e)) v[b][e] = 0.f;
      sum += (double)v[b][e] * (double)v[b][e];
    }
  const double norm = sqrt(block_sum<2 * RB>(sum));
  const double scale = (double)kYs / (norm < (double)a.eps ? (double)a.eps : norm);   // (a NaN stays one)
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[b][e] = (float)((double)v[b][e] * scale);

  // the operand fragments of one matrix instruction: 32 rows of a plane at 16 k, and 32 columns at 16 rows
  auto rows = [&](const _Float16* p, int row, int k) { return *(const f16x8*)(p + (row + lj) * LD + 16 * k + 8 * (lane >> 5)); };
  auto cols = [&](const _Float16* p, int k, int col) {
    const _Float16* q = p + (16 * k + 8 * (lane >> 5) + ((lane & 15) >> 2)) * LD + col + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
    union { s16x4 q[2]; f16x8 v; } u;
    u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q);
    u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q + 4 * LD));
    return u.v;
  };
  // 64 of K of an operand: all fragments ahead of the products, so that LDS's latency is not waited out more than once
  struct Frag64 { f16x8 h[4], l[SPLIT ? 4 : 1]; };
  auto take = [&](Frag64& f, const _Float16* h, const _Float16* l, auto get) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f.h[k] = get(h, k);
      if constexpr (SPLIT) f.l[k] = get(l, k);
    }
  };
  // ... and the products, of hi and lo planes into sums of their own (a third where there are registers for it: the next one that adds to
  // the same sum has to wait)
  auto mul = [&](f32x16& hi, f32x16& lo, const Frag64& x, const Frag64& y) {
    constexpr bool THIRD = SPLIT && RB == 2 && NB < 7;
    f32x16 other = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      hi = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h[k], y.h[k], hi, 0, 0, 0);
      if constexpr (SPLIT) {
        lo = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h[k], y.l[k], lo, 0, 0, 0);
        f32x16& third = THIRD ? other : lo;
        third = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.l[k], y.h[k], third, 0, 0, 0);
      }
    }
    if constexpr (THIRD) lo += other;
  };
  auto both = [&](const f32x16& hi, const f32x16& lo, int e) { return SPLIT ? hi[e] + lo[e] * (1.f / kLo) : hi[e]; };
  // a block's transpose: what a lane holds in a row then, four at a time, is a wide write.  Y lies transposed; A and B are symmetric.
  auto put = [&](_Float16* h, _Float16* l, int i0, int j, const float (&w)[16]) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      f16x4 x, y;
#pragma unroll
      for (int q = 0; q < 4; ++q) { _Float16 a1, b1; orth_split(w[e + q], a1, b1); x[q] = a1; y[q] = b1; }
      *(f16x4*)(h + j * LD + i0 + 2 * e) = x;
      if constexpr (SPLIT) *(f16x4*)(l + j * LD + i0 + 2 * e) = y;
    }
  };
  constexpr int AB = RB / 2;                                  // this wave's blocks of A and B: at a0 + 64 n, a1
  const int a0 = 32 * (wave / RB), a1 = 32 * (wave % RB);
  for (int step = 0;; ++step) {
#pragma unroll
    for (int b = 0; b < NB; ++b) put(yh, yl, y0 + li, x0 + 64 * b + lj, v[b]);
    __syncthreads();
    float w[AB][16];
    f32x16 hi[AB] = {}, lo[AB] = {};
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      Frag64 x[AB], y;
      take(y, yh, yl, [&](const _Float16* p, int k) { return cols(p, 4 * q + k, a1); });
#pragma unroll
      for (int n = 0; n < AB; ++n) take(x[n], yh, yl, [&](const _Float16* p, int k) { return cols(p, 4 * q + k, a0 + 64 * n); });
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < AB; ++n) mul(hi[n], lo[n], x[n], y);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int n = 0; n < AB; ++n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) w[n][e] = both(hi[n], lo[n], e) * (kAs / (kYs * kYs));
      put(ah, al, a0 + 64 * n + li, a1 + lj, w[n]);
      hi[n] = f32x16{}; lo[n] = f32x16{};
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < AB; ++q) {
      Frag64 x[AB], y;
      take(y, ah, al, [&](const _Float16* p, int k) { return rows(p, a1, 4 * q + k); });
#pragma unroll
      for (int n = 0; n < AB; ++n) take(x[n], ah, al, [&](const _Float16* p, int k) { return rows(p, a0 + 64 * n, 4 * q + k); });
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < AB; ++n) mul(hi[n], lo[n], x[n], y);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!ROOM) __syncthreads();
#pragma unroll
    for (int n = 0; n < AB; ++n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) w[n][e] = cb * w[n][e] + cc * (both(hi[n], lo[n], e) * (1.f / kAs));
      put(bh, bl, a0 + 64 * n + li, a1 + lj, w[n]);
    }
    __syncthreads();
    Frag64 x[AB];
#pragma unroll
    for (int q = 0; q < AB; ++q) take(x[q], bh, bl, [&](const _Float16* p, int k) { return rows(p, y0, 4 * q + k); });
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x16 h = {}, l = {};
      Frag64 y[AB];
#pragma unroll
      for (int q = 0; q < AB; ++q) take(y[q], yh, yl, [&](const _Float16* p, int k) { return rows(p, x0 + 64 * b, 4 * q + k); });
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < AB; ++q) mul(h, l, x[q], y[q]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[b][e] = ca * v[b][e] + both(h, l, e) * (1.f / kAs);
    }
    if (step + 1 == steps) break;
    __syncthreads();
  }
  again();
  float lr_q, keep;
  muon_rate(o, io, lr_q, keep);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    where(b, mat * io.ob, tall ? 1 : io.orow, tall ? io.orow : 1);
    if (o.muon) {
      float* p = (float*)io.out;
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = p[at[e]];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (inside(b, e)) p[at[e]] = x[e] * keep - lr_q * (v[b][e] * (1.f / kYs));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (inside(b, e)) orth_store(io.out, at[e], o.dtype, v[b][e] * (1.f / kYs));
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

// Whether matrices of a stack may be overwritten before they are read: where `out` touches x without being it.  A matrix is read before
// its own result is written, whatever its route.
static bool stack_clash(const void* x, const void* out, int bytes, int64_t batch, int64_t m, int64_t n, int64_t xb, int64_t xr, int64_t ob, int64_t orow) {
  if (batch == 1 || (x == out && xb == ob && (m == 1 || xr == orow))) return false;
  const int64_t lo = (xb < 0 ? (batch - 1) * xb : 0) + (xr < 0 ? (m - 1) * xr : 0);
  const int64_t hi = (xb > 0 ? (batch - 1) * xb : 0) + (xr > 0 ? (m - 1) * xr : 0) + n, end = (batch - 1) * ob + (m - 1) * orow + n;
  const int64_t a = (int64_t)(uintptr_t)x, b = (int64_t)(uintptr_t)out;
  return a + lo * bytes < b + end * bytes && b < a + hi * bytes;
}

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
static const int64_t kMaxSide = 65536, kMaxBatch = 65536;
static const int64_t kMaxBlocks = 1 << 22;      // a launch is at most 2^32 threads, 1024 a workgroup
static int stack_ok(int64_t batch, int64_t m, int64_t n) {
  if (batch < 1 || m < 1 || n < 1 || m > kMaxSide || n > kMaxSide || batch > kMaxBatch) return SNR_ERR_SHAPE;
  return SNR_OK;
}
// What a matrix goes through: one workgroup (64 or 128 rows, so many columns, split or hi planes alone), the split products of tiles, or
// fp16 products of tiles.
enum { kSmall64 = SNR_ROUTE_64x64, kSmall128, kSmall256, kSmall448, kMid128, kMid128h, kMid192h, kMid320h, kSplit = SNR_ROUTE_TILES, kHalf, kKinds };
static int kind_of(int precision, int64_t m, int64_t n) {
  const int64_t r = m < n ? m : n, c = m < n ? n : m;
  const bool split = precision == SNR_ORTH_FP32 || r <= 64;
  if (r <= 64 && c <= 448) return c <= 64 ? kSmall64 : c <= 128 ? kSmall128 : c <= 256 ? kSmall256 : kSmall448;
  if (r <= 128 && split && c <= 128) return kMid128;
  if (r <= 128 && !split && c <= 320) return c <= 128 ? kMid128h : c <= 192 ? kMid192h : kMid320h;
  return split ? kSplit : kHalf;
}

using S32 = TileCfg<32, 1, 1, true, 4, 64>;
using H32 = TileCfg<32, 1, 1, false, 4, 64>;
using S64 = TileCfg<64, 2, 2, true, 2, 64>;
using S128 = TileCfg<128, 4, 4, true, 2, 64>;
using H64 = TileCfg<64, 2, 2, false, 3, 64>;
template <int PHASE> struct Half {                     // fp16 products: 128, and the largest
  using T128 = TileCfg<128, 4, 2, false, 4, 64>;       // deep: mostly one round of tiles
  using Most = TileCfg<192, 6, 2, false, 3, 64>;
};
template <> struct Half<kApply> {
  using T128 = TileCfg<128, 2, 4, false, 2, 64>;       // two a compute unit, so that one writes its planes while the other multiplies
  using Most = TileCfg<256, 2, 4, false, 2, 64>;
};

// Everything of a launch sequence that follows from its stacks' sizes; also the bytes of its workspace.
struct OrthPlan { int ts, tf; int64_t sym, full, chunk, split, bytes; OrthArgs* args; };

static int64_t sym_tiles(const OrthGeom& g, int T) { const int64_t t = (g.rp + T - 1) / T; return g.batch * (t * (t + 1) / 2); }
static int64_t full_tiles(const OrthGeom& g, int T) { return (int64_t)g.batch * ((g.rp + T - 1) / T) * ((g.cp + T - 1) / T); }

// Tiles of 32, 64, 128 and, for fp16 products, 192 (symmetric) or 256 (B Y).  A larger one reads less per product, but idle compute units are
// worth more: 64 from 3 / 8 of the chip on, 128, which has a compute unit to itself, from half of it on.  A tile of 32 is one wave's.  Us a
// call with / without 32 (tiles of 64 a symmetric product, B Y): fp32, 256 x 8000 (10, 500) 282 / 452, 256^2 (10, 16) 88 / 103, 512^2 (36, 64)
// 114 / 142, 333 x 1000 (21, 96) x 4 (84, 384) 160 / 175, 2 x 512^2 (72, 128) 132 / 144; fp16 172 / 219, 72 / 80, 82 / 95, 114 / 120, 91 / 97; with
// 32 everywhere 1024^2 (136, 256) and 14 x 256^2 (140, 224) are slower, B Y by a third.  Us a product at 64 / 128, fp16: symmetric, 2048^2
// (136 tiles of 128): 24 / 22, 4 x 1024^2 (144): 16 / 15, 3 x 1024^2 (108): 12 / 14; B Y, 1024 x 4096: 23 / 21, 1400^2: 17 / 20.  fp32 (no
// larger tile fits LDS twice): symmetric, 2048^2: 53 / 44, 1400^2: 21 / 29; B Y, 2048^2: 67 / 59, 3 x 1024^2: 34 / 30.
static int pick_tile(int64_t n64, int64_t n128) { return 8 * n64 <= 3 * cu_count() ? 32 : n128 >= cu_count() / 2 ? 128 : 64; }
// 128 or 192: a round of tiles (one a compute unit) takes as long as a tile's rows take to come in, the products of the whole chip as long
// as its power allows, whichever is more; and every round after the first has an epilogue that nothing hides.  Us at 128 / 192: 4096^2
// (528 / 253 tiles): 105 / 81, 2048^2 (136 / 66): 22 / 32, 13 x 1024^2 (468 / 273): 27 / 38, 2 x 2048 x 3000 (272 / 132): 50 / 42, 3 x 2048^2
// (408 / 198): 40 / 38, 5 x 1500^2 (390 / 180): 32 / 30.
static int pick_sym(int64_t n64, int64_t n128, int64_t n192) {
  const int64_t cus = cu_count();
  auto cost = [&](double T, int64_t n, double slower) {
    const double rounds = (double)((n + cus - 1) / cus);
    return fmax(rounds * T * slower, (double)n * T * T / (99.0 * (double)cus)) * (0.9 + 0.1 * rounds);
  };
  const int T = pick_tile(n64, n128);
  return T == 128 && cost(192, n192, 1.13) < cost(128, n128, 1.0) ? 192 : T;
}
// 128 or 256: 256 where its rounds are more than three quarters full.  Us at 128 / 256: 4096^2 (256 tiles of 256): 144 / 133, 2048 x 7000
// (224): 82 / 77, 3500^2 (196): 120 / 106, 3 x 2048^2 (192): 73 / 77, 12 x 512 x 2048 (192): 34 / 40, 5 x 1500^2 (180): 58 / 61.
static int pick_full(int64_t n64, int64_t n128, int64_t n256) {
  const int64_t cus = cu_count(), room = (n256 + cus - 1) / cus * cus;
  const int T = pick_tile(n64, n128);
  return T == 128 && 4 * n256 > 3 * room ? 256 : T;
}

static int orth_plan(OrthArgs& a, int kind, OrthPlan& p) {
  int64_t off = 0, part = 0;
  const bool split = kind != kHalf;
  p.chunk = p.split = p.sym = p.full = 0;
  for (int s = 0; s < kOrthMax; ++s) a.sym0[s] = a.full0[s] = a.chunk0[s] = a.split0[s] = INT32_MAX;
  if (kind < kSplit) {                       // a workgroup a matrix, no workspace
    for (int s = 0; s < a.n_items; ++s) { a.sym0[s] = (int)p.sym; p.sym += a.io[s].batch; }
    p.bytes = 256;
    return SNR_OK;
  }
  a.n_geom = 0;
  for (int s = 0; s < a.n_items; ++s) {      // the sizes there are, longest K first: what takes longest begins first
    const OrthIo& io = a.io[s];
    const int r = io.m < io.n ? io.m : io.n, c = io.m < io.n ? io.n : io.m;
    int k = 0;
    while (k < a.n_geom && (a.g[k].c > c || (a.g[k].c == c && a.g[k].r > r))) ++k;
    if (k < a.n_geom && a.g[k].c == c && a.g[k].r == r) continue;
    for (int q = a.n_geom++; q > k; --q) a.g[q] = a.g[q - 1];
    a.g[k] = OrthGeom{r, c, (r + kPad - 1) / kPad * kPad, (c + kPad - 1) / kPad * kPad, 0, 0, 0};
  }
  for (int s = 0; s < a.n_items; ++s) {
    OrthIo& io = a.io[s];
    const int r = io.m < io.n ? io.m : io.n, c = io.m < io.n ? io.n : io.m;
    int k = 0;
    while (a.g[k].r != r || a.g[k].c != c) ++k;
    OrthGeom& g = a.g[k];
    io.geom = k; io.mat0 = g.batch; g.batch += io.batch;
    const int64_t n = ((int64_t)io.m * io.n + 8191) / 8192;
    io.nchunk = (int)(n > 1024 ? 1024 : n);
    io.part = part; part += (int64_t)io.batch * io.nchunk;
    a.chunk0[s] = (int)p.chunk; p.chunk += (int64_t)io.batch * io.nchunk;
    a.split0[s] = (int)p.split; p.split += (int64_t)io.batch * (g.rp / kPad) * (g.cp / kPad);
    if (p.chunk > kMaxBlocks || p.split > kMaxBlocks) return SNR_ERR_SHAPE;
  }
  int64_t ns[3] = {}, nf[3] = {};
  for (int s = 0; s < a.n_geom; ++s)
    for (int k = 0; k < 3; ++k) { ns[k] += sym_tiles(a.g[s], k < 2 ? 64 << k : 192); nf[k] += full_tiles(a.g[s], 64 << k); }
  p.ts = split ? pick_tile(ns[0], ns[1]) : pick_sym(ns[0], ns[1], ns[2]);
  p.tf = split ? pick_tile(nf[0], nf[1]) : pick_full(nf[0], nf[1], nf[2]);
  for (int s = 0; s < a.n_geom; ++s) {       // (no more tiles than the split's where there are many: one holds 64 x 64 or more)
    OrthGeom& g = a.g[s];
    g.ws = off; off += (int64_t)g.batch * orth_planes(g.rp, g.cp, split).total * 2;
    a.sym0[s] = (int)p.sym; a.full0[s] = (int)p.full;
    p.sym += (sym_tiles(g, p.ts) + 7) / 8 * 8; p.full += (full_tiles(g, p.tf) + 7) / 8 * 8;
  }
  const int64_t at_part = align256(off);     // the planes come first: on 256 bytes
  a.part = (double*)(a.ws + at_part);
  a.split = split;
  const int64_t at_args = at_part + align256(part * 8);
  p.args = (OrthArgs*)(a.ws + at_args);
  p.bytes = at_args + align256(sizeof(OrthArgs));
  return SNR_OK;
}

static OrthHead orth_head(const OrthArgs& a, const OrthArgs* in_ws, const int* first) {
  OrthHead h{};
  h.args = in_ws; h.ws = a.ws;
  h.n = a.n_geom <= kHead ? a.n_geom : 0;
  h.spread = a.g[0].c >= 2 * a.g[a.n_geom - 1].c;
  for (int k = 0; k < kHead; ++k) { h.first[k] = k < a.n_geom ? first[k] : INT32_MAX; h.g[k] = a.g[k]; }
  return h;
}

template <int PHASE, bool last, class C>
static void launch(const OrthHead& a, const OrthOut& o, int64_t n, float ca, float cb, float cc, int flip, hipStream_t st) {
  orth_product_kernel<PHASE, last, C><<<dim3((unsigned)n), dim3(C::NT), 0, st>>>(a, o, ca, cb, cc, flip);
}
template <int PHASE, bool last>
static void launch_tile(bool split, int T, const OrthHead& a, const OrthOut& o, int64_t n, float ca, float cb, float cc, int flip, hipStream_t st) {
  if (split) {
    if (T == 32) launch<PHASE, last, S32>(a, o, n, ca, cb, cc, flip, st);
    else if (T == 64) launch<PHASE, last, S64>(a, o, n, ca, cb, cc, flip, st);
    else launch<PHASE, last, S128>(a, o, n, ca, cb, cc, flip, st);
  } else if (T == 32) {
    launch<PHASE, last, H32>(a, o, n, ca, cb, cc, flip, st);
  } else if (T == 64) {
    launch<PHASE, last, H64>(a, o, n, ca, cb, cc, flip, st);
  } else if (T == 128) {
    launch<PHASE, last, typename Half<PHASE>::T128>(a, o, n, ca, cb, cc, flip, st);
  } else {
    launch<PHASE, last, typename Half<PHASE>::Most>(a, o, n, ca, cb, cc, flip, st);
  }
}

// one launch sequence over a.n_items items of one kind, whose x, out, mom, strides, m, n and batch are filled in
static int orth_run(OrthArgs& a, const OrthOut& o, int steps, float ca, float cb, float cc, int kind, char* ws, hipStream_t st) {
  a.ws = ws;
  OrthPlan p;
  const int ok = orth_plan(a, kind, p);
  if (ok != SNR_OK) return ok;
  const bool split = kind != kHalf;
  if (kind < kSplit) {
    ProfScope ps(K_ORTH_SMALL, st);
    const dim3 n((unsigned)p.sym);
    switch (kind) {
      case kSmall64: orth_small_kernel<2, 1, true><<<n, dim3(256), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kSmall128: orth_small_kernel<2, 2, true><<<n, dim3(256), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kSmall256: orth_small_kernel<2, 4, true><<<n, dim3(256), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kSmall448: orth_small_kernel<2, 7, true><<<n, dim3(256), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kMid128: orth_small_kernel<4, 2, true><<<n, dim3(512), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kMid128h: orth_small_kernel<4, 2, false><<<n, dim3(512), 0, st>>>(a, o, ca, cb, cc, steps); break;
      case kMid192h: orth_small_kernel<4, 3, false><<<n, dim3(512), 0, st>>>(a, o, ca, cb, cc, steps); break;
      default: orth_small_kernel<4, 5, false><<<n, dim3(512), 0, st>>>(a, o, ca, cb, cc, steps);
    }
    return launch_status();
  }
  {
    ProfScope ps(K_ORTH_PREPARE, st);
    orth_reduce_kernel<<<dim3((unsigned)p.chunk), dim3(256), 0, st>>>(a, p.args);
    orth_split_kernel<<<dim3((unsigned)p.split), dim3(256), 0, st>>>(p.args);
  }
  const OrthHead hs = orth_head(a, p.args, a.sym0), hf = orth_head(a, p.args, a.full0);
  for (int k = 0; k < steps; ++k) {
    {
      ProfScope ps(K_ORTH_GRAM, st);
      launch_tile<kGram, false>(split, p.ts, hs, o, p.sym, ca, cb, cc, k & 1, st);
    }
    {
      ProfScope ps(K_ORTH_POLY, st);
      launch_tile<kPoly, false>(split, p.ts, hs, o, p.sym, ca, cb, cc, k & 1, st);
    }
    ProfScope ps(K_ORTH_APPLY, st);
    if (k + 1 == steps) launch_tile<kApply, true>(split, p.tf, hf, o, p.full, ca, cb, cc, k & 1, st);
    else launch_tile<kApply, false>(split, p.tf, hf, o, p.full, ca, cb, cc, k & 1, st);
  }
  return launch_status();
}

extern "C" int64_t snr_orthogonalise_ws_bytes(int64_t batch, int64_t rows, int64_t cols, int precision) {
  if (precision != SNR_ORTH_FP16 && precision != SNR_ORTH_FP32) return SNR_ERR_UNSUPPORTED;
  const int st = stack_ok(batch, rows, cols);
  if (st != SNR_OK) return st;
  OrthArgs A{};
  OrthPlan p;
  A.n_items = 1; A.io[0].batch = (int)batch; A.io[0].m = (int)rows; A.io[0].n = (int)cols;
  const int ok = orth_plan(A, kind_of(precision, rows, cols), p);
  return ok != SNR_OK ? ok : p.bytes;
}

extern "C" int snr_orthogonalise(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int64_t x_batch_stride,
                                 int64_t x_row_stride, void* out, int64_t out_batch_stride, int64_t out_row_stride, int steps,
                                 float a, float b, float c, float eps, int precision, void* ws, snr_stream_t stream) {
  SNR_CHECK_ARG(x && out && ws, SNR_ERR_NULL);
  SNR_CHECK_ARG(stack_ok(batch, rows, cols) == SNR_OK && steps >= 1 && steps <= 100 && eps >= 1e-30f, SNR_ERR_SHAPE);
  SNR_CHECK_ARG(out_row_stride >= cols && (batch == 1 || out_batch_stride >= (rows - 1) * out_row_stride + cols), SNR_ERR_SHAPE);
  SNR_CHECK_ARG(dtype == SNR_F32 || dtype == SNR_F16 || dtype == SNR_BF16, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(!stack_clash(x, out, dtype == SNR_F32 ? 4 : 2, batch, rows, cols, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride), SNR_ERR_SHAPE);
  SNR_CHECK_ARG(precision == SNR_ORTH_FP16 || precision == SNR_ORTH_FP32, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(orth_bounded(steps, a, b, c), SNR_ERR_UNSUPPORTED);
  OrthArgs A{};
  A.n_items = 1;
  A.io[0] = OrthIo{x, out, nullptr, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride, (int)rows, (int)cols, (int)batch, 0, 0, 0, 0};
  A.dtype = dtype; A.eps = eps;
  OrthOut o{};
  o.dtype = dtype;
  return orth_run(A, o, steps, a, b, c, kind_of(precision, rows, cols), (char*)ws, (hipStream_t)stream);
}

// Where the matrices of each kind go in a call that has several: sequences run one after the other, and one that does little takes its
// latency all the same (us: 17 .. 55 for one workgroup a matrix, 70 .. 125 for tiles).  Those that would fit a workgroup therefore go
// with the tiles if there are any at their precision and their own tiles are one for each compute unit at most, and those of several
// widths go with the widest, up to one matrix for each.  Us together / apart, with 14 x 256^2: 2 x 128 x 128 fp16 90 / 120, fp32
// 115 / 174; 64 x 128 x 128 109 / 121, 152 / 175; 64 x 64 x 448 fp32 209 / 176.  64 x 64, x 100, x 200 and x 400: 54 / 133.
static void merge_kinds(const snr_muon_item* items, int n_items, int precision, int (&to)[kKinds]) {
  int64_t n[kKinds] = {}, tiles[kKinds] = {};
  for (int i = 0; i < n_items; ++i) {
    const snr_muon_item& it = items[i];
    const int k = kind_of(precision, it.rows, it.cols);
    n[k] += it.batch;
    tiles[k] += it.batch * ((it.rows + kPad - 1) / kPad) * ((it.cols + kPad - 1) / kPad);
  }
  for (int k = 0; k < kKinds; ++k) to[k] = k;
  const int cus = cu_count();
  const struct { int first, last, with; } groups[] = {{kSmall64, kSmall448, kSplit}, {kMid128, kMid128, kSplit}, {kMid128h, kMid320h, kHalf}};
  for (const auto& g : groups) {
    int64_t total = 0, work = 0;
    int widest = g.first;
    for (int k = g.first; k <= g.last; ++k) { total += n[k]; work += tiles[k]; widest = n[k] ? k : widest; }
    const bool join = n[g.with] && work <= cus;
    for (int k = g.first; k <= g.last; ++k) to[k] = join ? g.with : total <= cus ? widest : k;
  }
}

// The launch sequences of a list of items: stacks of one kind share one, kOrthMax at a time; they run one after the other and share
// the workspace.  F(OrthArgs&, kind) returns a status.
template <class F> static int for_sequences(const snr_muon_item* items, int n_items, int precision, F f) {
  int to[kKinds];
  merge_kinds(items, n_items, precision, to);
  for (int kind = 0; kind < kKinds; ++kind) {
    OrthArgs A{};
    for (int i = 0; i <= n_items; ++i) {
      if (A.n_items == kOrthMax || (i == n_items && A.n_items)) {
        const int st = f(A, kind);
        if (st != SNR_OK) return st;
        A.n_items = 0;
      }
      if (i == n_items) break;
      const snr_muon_item& it = items[i];
      if (to[kind_of(precision, it.rows, it.cols)] != kind) continue;
      const int64_t mn = it.rows * it.cols;
      A.io[A.n_items++] = OrthIo{it.grads, it.params, it.momentum, mn, it.cols, mn, it.cols, (int)it.rows, (int)it.cols, (int)it.batch, 0, 0, 0, 0};
    }
  }
  return SNR_OK;
}

// F(const OrthPlan&, kind) for each sequence that the items would take
template <class F> static int plan_sequences(const snr_muon_item* items, int n_items, int precision, F f) {
  if (!items) return SNR_ERR_NULL;
  if (n_items < 1) return SNR_ERR_SHAPE;
  if (precision != SNR_ORTH_FP16 && precision != SNR_ORTH_FP32) return SNR_ERR_UNSUPPORTED;
  for (int i = 0; i < n_items; ++i) {
    const int st = stack_ok(items[i].batch, items[i].rows, items[i].cols);
    if (st != SNR_OK) return st;
  }
  return for_sequences(items, n_items, precision, [&](OrthArgs& A, int kind) {
    OrthPlan p;
    const int ok = orth_plan(A, kind, p);
    if (ok == SNR_OK) f(p, kind);
    return ok;
  });
}

extern "C" int64_t snr_muon_ws_bytes(const snr_muon_item* items, int n_items, int precision) {
  int64_t most = 0;
  const int st = plan_sequences(items, n_items, precision, [&](const OrthPlan& p, int) { most = p.bytes > most ? p.bytes : most; });
  return st != SNR_OK ? st : most;
}

extern "C" int snr_muon_routes(const snr_muon_item* items, int n_items, int precision, int* routes, int max_routes) {
  if (max_routes > 0 && !routes) return SNR_ERR_NULL;
  int n = 0;
  const int st = plan_sequences(items, n_items, precision, [&](const OrthPlan& p, int kind) {
    if (n < max_routes) { routes[3 * n] = kind; routes[3 * n + 1] = kind < kSplit ? 0 : p.ts; routes[3 * n + 2] = kind < kSplit ? 0 : p.tf; }
    ++n;
  });
  return st != SNR_OK ? st : n;
}

extern "C" int snr_muon_step_multi(const snr_muon_item* items, int n_items, float lr, float momentum, int nesterov, float weight_decay,
                                   int scale_mode, int steps, float a, float b, float c, float eps, float grad_scale, int precision,
                                   const snr_step_state* state, void* ws, snr_stream_t stream) {
  SNR_CHECK_ARG(items && ws, SNR_ERR_NULL);
  SNR_CHECK_ARG(n_items >= 1 && steps >= 1 && steps <= 100 && eps >= 1e-30f, SNR_ERR_SHAPE);
  SNR_CHECK_ARG(precision == SNR_ORTH_FP16 || precision == SNR_ORTH_FP32, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(scale_mode == SNR_MUON_NONE || scale_mode == SNR_MUON_SPECTRAL || scale_mode == SNR_MUON_RMS, SNR_ERR_UNSUPPORTED);
  SNR_CHECK_ARG(orth_bounded(steps, a, b, c), SNR_ERR_UNSUPPORTED);
  int64_t tiles = 0;
  for (int i = 0; i < n_items; ++i) {
    SNR_CHECK_ARG(items[i].params && items[i].grads && items[i].momentum, SNR_ERR_NULL);
    SNR_CHECK_ARG(stack_ok(items[i].batch, items[i].rows, items[i].cols) == SNR_OK, SNR_ERR_SHAPE);
    tiles += items[i].batch * ((items[i].rows + kPad - 1) / kPad) * ((items[i].cols + kPad - 1) / kPad);
  }
  if (tiles > kMaxBlocks) {                    // a later sequence may be too large: all are planned before the first is launched
    const int64_t bytes = snr_muon_ws_bytes(items, n_items, precision);
    if (bytes < 0) return (int)bytes;
  }
  Span* spans = (Span*)malloc(sizeof(Span) * 3 * (size_t)n_items);
  if (!spans) return (int)hipErrorOutOfMemory;
  for (int i = 0; i < n_items; ++i) {
    const snr_muon_item& it = items[i];
    const void* at[3] = {it.params, it.grads, it.momentum};
    const uintptr_t bytes = 4 * (uintptr_t)(it.batch * it.rows * it.cols);
    for (int k = 0; k < 3; ++k) spans[3 * i + k] = Span{(uintptr_t)at[k], (uintptr_t)at[k] + bytes, k != 1};
  }
  const bool clash = spans_clash(spans, 3 * (size_t)n_items);
  free(spans);
  SNR_CHECK_ARG(!clash, SNR_ERR_SHAPE);
  OrthOut o{};
  o.muon = 1; o.scale_mode = scale_mode; o.lr = lr; o.decay = weight_decay; o.st = state;
  return for_sequences(items, n_items, precision, [&](OrthArgs& A, int kind) {
    A.mu = momentum; A.gscale = grad_scale; A.eps = eps; A.nesterov = nesterov;
    return orth_run(A, o, steps, a, b, c, kind, (char*)ws, (hipStream_t)stream);
  });
}
