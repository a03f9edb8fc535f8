// Orthogonalising a matrix by Newton-Schulz products, and the optimizer step built on it (Muon).
//
// X0 = G / (|G|_F + eps); then `steps` times  A = X X^T,  B = b A + c A A,  X <- a X + B X.
// Every singular value s of X goes through s <- a s + b s^3 + c s^5 and the singular vectors stay: with (a, b, c) = (3.4445, -4.7750, 2.0315)
// five steps bring everything above ~1e-3 of the norm into about 0.7 .. 1.2, i.e. X is near the closest orthogonal matrix U V^T.  A matrix with
// more rows than columns is worked on transposed, so A and B are as small as they can be: m x m with m = min(rows, cols), n = max.
//
// Numbers.  Everything between the products is kept as a PAIR of fp16, hi + lo = 22 bits, scaled by 4096 (|X| <= ~1.2, |A| <= ~1.5, |B| <= ~4:
// nothing overflows, and the low halves of entries down to 1e-5 are still normal fp16).  The matrix cores multiply fp16 pairs exactly and add in fp32.
//   fp32 tensors:  hi hi + hi lo + lo hi  -- three products per product; what is left out is 2^-22 of an entry, as much as an fp32 sum of this
//                  length loses anyway (1e-6 of the result on the sizes tested, the same as fp32 products).
//   bf16 tensors:  hi hi only -- one product -- but X itself advances from its 22 bits (the a X term), because noise put into X is amplified
//                  ~a^5 = 480 times in the directions G hardly has, while noise of the products stays in the row space of X.  The diagonals of A and B, where
//                  most of their weight is once X is nearly orthogonal, are multiplied in fp32 outside the matrix cores.  Together 1 - 2e-3 of the
//                  result; rounding it to bf16 costs 1.7e-3, and bf16 products throughout would cost 1e-2 (well conditioned) to 0.5.
//
// Bound: the matrix cores for large matrices, launches and memory latency for the weights of a small network.
#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "pwr_common.h"
#include "pwr.h"

namespace pwr {

typedef _Float16 half_t;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;

constexpr float kOrthScale = 4096.f;                     // of every stored pair
constexpr float kOrthInv = 1.f / 4096.f;

// One matrix.  In a table on the device (a parameter list), or made from the launch's arguments (a batch of equal ones).
struct OrthItem {
  long long src, dst;       // offsets of its first element in the source and in the result (in elements)
  long long ws;             // offset of its workspace block (in bytes)
  int rows, cols;           // as the caller has it
  int Mp, Np;               // min / max of the two, up to the tile
  float gain;               // of the update
  int pad;
};

// Its workspace block: X in two buffers (a step reads one and writes the other), A, B, the two diagonals, the partial sums of squares.
struct OrthWs {
  long long xplane, aplane;         // halves per plane
  __host__ __device__ OrthWs(int Mp, int Np) : xplane((long long)Mp * Np), aplane((long long)Mp * Mp) {}
  __host__ __device__ long long x(int buf) const { return buf * 4 * xplane; }             // bytes: hi plane, then lo plane
  __host__ __device__ long long a() const { return 8 * xplane; }
  __host__ __device__ long long b() const { return 8 * xplane + 4 * aplane; }
  __host__ __device__ long long diag(int Mp) const { return 8 * xplane + 8 * aplane; }
  __host__ __device__ long long parts(int Mp) const { return diag(Mp) + 8ll * Mp; }
};
struct OrthArgs {
  const OrthItem* items; const int4* tiles;              // table form (items != null): tiles[block] = {item, ti, tj, -}
  OrthItem one; long long src_stride, dst_stride, ws_stride; int per;    // batch form: block = batch * per + tile
  char* ws;
  int buf;                                               // which X buffer is read
  float a, b, c, eps;
};

__device__ __forceinline__ OrthItem orth_item(const OrthArgs& g, int& t, int4& tile) {
  if (g.items) {
    tile = g.tiles[blockIdx.x];
    t = -1;
    return g.items[tile.x];
  }
  const int batch = blockIdx.x / g.per;
  t = blockIdx.x - batch * g.per;
  OrthItem o = g.one;
  o.src += batch * g.src_stride;
  o.dst += batch * g.dst_stride;
  o.ws += batch * g.ws_stride;
  return o;
}

__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
  const float s = v * kOrthScale;
  hi = (half_t)s;
  lo = (half_t)(s - (float)hi);
}

// ---- what is orthogonalised: a tensor of T with a row stride, or u = g + mu buf of an optimizer step.  Indices are offsets from the matrix's first
// element; quad() is four neighbours, at any alignment.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Quad { T v[4]; };

template <typename T> struct OrthTensor {
  const T* x; long long ld;
  __device__ __forceinline__ long long stride(const OrthItem&) const { return ld; }
  __device__ __forceinline__ float one(const OrthItem& o, long long i) const { return Elem<T>::to_f(x[o.src + i]); }
  __device__ __forceinline__ void quad(const OrthItem& o, long long i, float (&v)[4]) const {
    const Quad<T> q = *reinterpret_cast<const Quad<T>*>(x + o.src + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Elem<T>::to_f(q.v[e]);
  }
  __device__ __forceinline__ float first(const OrthItem& o, long long i) const { return one(o, i); }
  __device__ __forceinline__ void first_quad(const OrthItem& o, long long i, float (&v)[4]) const { quad(o, i, v); }
};
struct OrthMomentum {
  const float* g; float* buf; float mu, grad_scale; int nesterov;
  __device__ __forceinline__ long long stride(const OrthItem& o) const { return o.cols; }
  __device__ __forceinline__ float u(float gv, float m) const { return nesterov ? grad_scale * gv + mu * m : m; }
  __device__ __forceinline__ float one(const OrthItem& o, long long i) const { return u(g[o.src + i], buf[o.src + i]); }
  __device__ __forceinline__ void quad(const OrthItem& o, long long i, float (&v)[4]) const {
    const Quad<float> a = *reinterpret_cast<const Quad<float>*>(g + o.src + i), b = *reinterpret_cast<const Quad<float>*>(buf + o.src + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = u(a.v[e], b.v[e]);
  }
  // the first pass over the gradient updates the momentum
  __device__ __forceinline__ float first(const OrthItem& o, long long i) const {
    const float gv = g[o.src + i], m = mu * buf[o.src + i] + grad_scale * gv;
    buf[o.src + i] = m;
    return u(gv, m);
  }
  __device__ __forceinline__ void first_quad(const OrthItem& o, long long i, float (&v)[4]) const {
    const Quad<float> a = *reinterpret_cast<const Quad<float>*>(g + o.src + i);
    Quad<float> b = *reinterpret_cast<const Quad<float>*>(buf + o.src + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) { b.v[e] = mu * b.v[e] + grad_scale * a.v[e]; v[e] = u(a.v[e], b.v[e]); }
    *reinterpret_cast<Quad<float>*>(buf + o.src + i) = b;
  }
};

// A matrix's squares are summed by orth_parts() workgroups of orth_part_rows() rows each: about 4096 elements, more where that would be over 1024
// workgroups (every workgroup of the next launch adds all partial sums).
__host__ __device__ static inline int orth_part_rows(int rows, int cols) {
  const long long per = 4096 * (((long long)rows * cols + 4096 * 1024 - 1) / (4096 * 1024));
  return (int)(per / cols > 1 ? per / cols : 1);
}
__host__ __device__ static inline int orth_parts(int rows, int cols) { const int r = orth_part_rows(rows, cols); return (rows + r - 1) / r; }
static inline long long orth_ws_bytes(int rows, int cols, int Mp, int Np) {
  const OrthWs w(Mp, Np);
  return (w.parts(Mp) + 8ll * orth_parts(rows, cols) + 255) / 256 * 256;
}

__device__ __forceinline__ double orth_block_sum(double s, double* red) {
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// partial sums of squares, in 64 bits: neither 1e30 nor 1e-30 leaves the range, and the norm is exact to its last bit
template <typename SRC>
__global__ __launch_bounds__(256) void orth_norm_kernel(OrthArgs g, SRC src) {
  __shared__ double red[4];
  int t; int4 tile;
  const OrthItem o = orth_item(g, t, tile);
  const int part = t < 0 ? tile.y : t, nr = orth_part_rows(o.rows, o.cols), r0 = part * nr, r1 = min(o.rows, r0 + nr);
  const long long ld = src.stride(o);
  const bool flat = ld == o.cols;                                   // rows without gaps are one run
  double s = 0.0;
  if (!flat && o.cols < 1024) {                                     // short rows with gaps: 16 threads each
    for (int r = r0 + (threadIdx.x >> 4); r < r1; r += 16)
      for (int c = threadIdx.x & 15; c < o.cols; c += 16) {
        const double v = src.first(o, r * ld + c);
        s += v * v;
      }
  }
  const int runs = flat ? 1 : o.cols < 1024 ? 0 : r1 - r0;
  const long long len = flat ? (long long)(r1 - r0) * o.cols : o.cols;
  for (int k = 0; k < runs; ++k) {
    const long long at = (r0 + k) * ld;
    long long i = threadIdx.x * 4;
    for (; i + 3 * 1024 + 4 <= len; i += 4 * 1024) {
      float v[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) src.first_quad(o, at + i + u * 1024, v[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += (double)v[u][e] * v[u][e];
    }
    for (; i < len; i += 1024) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (i + 4 <= len) src.first_quad(o, at + i, v);
      else
        for (int e = 0; i + e < len; ++e) v[e] = src.first(o, at + i + e);
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)v[e] * v[e];
    }
  }
  s = orth_block_sum(s, red);
  if (threadIdx.x == 0) reinterpret_cast<double*>(g.ws + o.ws + OrthWs(o.Mp, o.Np).parts(o.Mp))[part] = s;
}

// X0 = G / (|G| + eps) as pairs, a 64 x 64 tile per workgroup, transposed where the matrix is tall; zero beyond m x n.  A thread has four neighbours
// of a row of the SOURCE in each of four rows 16 apart; its loads are under way while the partial sums are added.
template <typename SRC>
__global__ __launch_bounds__(256) void orth_pack_kernel(OrthArgs g, SRC src) {
  __shared__ double red[4];
  __shared__ float turn[64][65];
  int t; int4 tile;
  const OrthItem o = orth_item(g, t, tile);
  const OrthWs w(o.Mp, o.Np);
  const int tj = t < 0 ? tile.z : t % (o.Np / 64), ti = t < 0 ? tile.y : t / (o.Np / 64);
  const int tid = threadIdx.x, a = tid >> 4, b = (tid & 15) * 4;
  const bool tall = o.rows > o.cols;
  const int r0 = (tall ? tj : ti) * 64, c0 = (tall ? ti : tj) * 64;
  const long long ld = src.stride(o);
  float v[4][4];
  if (r0 + 64 <= o.rows && c0 + 64 <= o.cols) {
#pragma unroll
    for (int k = 0; k < 4; ++k) src.quad(o, (r0 + a + 16 * k) * ld + c0 + b, v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = r0 + a + 16 * k, c = c0 + b + e;
        const float x = src.one(o, min(r, o.rows - 1) * ld + min(c, o.cols - 1));
        v[k][e] = r < o.rows && c < o.cols ? x : 0.f;
      }
  }
  const double* parts = reinterpret_cast<const double*>(g.ws + o.ws + w.parts(o.Mp));
  const int np = orth_parts(o.rows, o.cols);
  double s = 0.0;
  for (int k = tid; k < np; k += 256) s += parts[k];
  const double inv = 1.0 / (sqrt(orth_block_sum(s, red)) + (double)g.eps);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = (float)((double)v[k][e] * inv);
  if (tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) turn[b + e][a + 16 * k] = v[k][e];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = turn[a + 16 * k][b + e];
  }
  half_t* hi = reinterpret_cast<half_t*>(g.ws + o.ws + w.x(0));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) { half_t x, y; split(v[k][e], x, y); h[e] = x; l[e] = y; }
    const long long at = (long long)(ti * 64 + a + 16 * k) * o.Np + tj * 64 + b;
    *reinterpret_cast<half4*>(hi + at) = h;
    *reinterpret_cast<half4*>(hi + w.xplane + at) = l;
  }
}

// ---- what the last step does with a row of four neighbouring entries X[i][j .. j + 3]
template <typename T> struct OrthOut {
  T* out; long long ld;
  __device__ __forceinline__ void put(const OrthItem& o, bool tall, int i, int j, float v) const {
    out[o.dst + (tall ? (long long)j * ld + i : (long long)i * ld + j)] = Elem<T>::from_f(v);
  }
};
struct OrthUpdate {
  float* p; float keep, lr;           // keep = 1 - lr weight_decay
  __device__ __forceinline__ void put(const OrthItem& o, bool tall, int i, int j, float v) const {
    float* q = p + o.dst + (tall ? (long long)j * o.cols + i : (long long)i * o.cols + j);
    *q = *q * keep - lr * o.gain * v;
  }
};
struct OrthNone {
  __device__ __forceinline__ void put(const OrthItem&, bool, int, int, float) const {}
};

enum { kGram = 0, kPoly = 1, kApply = 2 };

// ---- the products: one TILE x TILE tile of the result per workgroup of four waves, each (TILE / 2)^2.
// First MFMA operand P: the entries j (a lane ends up with four neighbouring j of one row i), second operand Q: the rows i.
// A and A A are symmetric: tiles tj >= ti only, written twice.  In B X the columns of X are needed along K: its rows are staged as they are
// and read transposed by the LDS hardware.
// TILE 128: stages of 32 along K, two in LDS, the next one in registers on its way.  TILE 64, for the few workgroups of small matrices, where a stage
// costs its latency: 128 along K in one stage.
template <int TERMS, int KIND, int TILE, typename OUT>
__global__ __launch_bounds__(256) void orth_gemm_kernel(OrthArgs g, OUT fin, int last) {
  constexpr int KS = TILE == 128 ? (TERMS == 3 ? 32 : 64) : 128;        // K per stage
  constexpr int STAGES = TILE == 128 ? 2 : 1;
  constexpr int HALF = TILE / 2, NF = HALF / 16;                        // 16 x 16 fragments per wave and direction
  constexpr int PLANES = TERMS == 3 ? 2 : 1;
  constexpr int OPB = TILE * KS * 2;                                    // bytes of one operand plane of a stage
  constexpr int UNITS = OPB / 16 / 256;                                 // 16-byte units per thread and plane
  constexpr int STAGE = 2 * PLANES * OPB;
  constexpr int CK = KS / 8, CT = TILE / 8;                             // 16-byte units of a row along K, and along the tile
  __shared__ __attribute__((aligned(16))) char lds[STAGES * STAGE];
  int t; int4 tile;
  const OrthItem o = orth_item(g, t, tile);
  const OrthWs w(o.Mp, o.Np);
  int ti, tj;
  if (t < 0) { ti = tile.y; tj = tile.z; }
  else if (KIND == kApply) { const int nj = o.Np / TILE; ti = t / nj; tj = t - ti * nj; }
  else {                                                                // t -> (ti <= tj): column tj starts at tj (tj + 1) / 2
    tj = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > t) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
    ti = t - tj * (tj + 1) / 2;
  }
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wp = (wid & 1) * HALF, wq = (wid >> 1) * HALF;              // this wave's part of the tile: entries j, rows i
  char* base = g.ws + o.ws;
  const half_t* X = reinterpret_cast<const half_t*>(base + w.x(g.buf));
  const half_t* A = reinterpret_cast<const half_t*>(base + w.a());
  const half_t* B = reinterpret_cast<const half_t*>(base + w.b());
  const half_t* Q = KIND == kGram ? X : KIND == kPoly ? A : B;
  const half_t* P = KIND == kPoly ? A : X;
  const long long qplane = KIND == kGram ? w.xplane : w.aplane, pplane = KIND == kPoly ? w.aplane : w.xplane;
  const int ldq = KIND == kGram ? o.Np : o.Mp, ldp = KIND == kPoly ? o.Mp : o.Np;
  const int K = KIND == kGram ? o.Np : o.Mp;                            // a multiple of 64

  // Staging.  A plane is [row][CK units along K], the unit swizzled by the row, or (columns of X) [k][CT units], 32-byte pieces swizzled by k, so
  // that neither kind of read meets its own bank.  Where K ends inside a stage the units beyond are loaded from inside and not used.
  half8 rq[PLANES][UNITS], rp[PLANES][UNITS];
  auto ntf = [](int row) { return CK == 4 ? (row >> 1) & 3 : CK == 8 ? (row >> 1) & 7 : row & 15; };
  auto trf = [](int k) { return TILE == 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1; };
  auto load = [&](int k0) {
    const int left = K - k0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int id = u * 256 + tid, row = id / CK, c = KS > 64 ? min(id % CK, left / 8 - 1) : id % CK;
      const int kr = KS > 64 ? min(id / CT, left - 1) : id / CT;
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        rq[p][u] = *reinterpret_cast<const half8*>(Q + p * qplane + (long long)(ti * TILE + row) * ldq + k0 + c * 8);
        if constexpr (KIND == kApply)
          rp[p][u] = *reinterpret_cast<const half8*>(P + p * pplane + (long long)(k0 + kr) * ldp + tj * TILE + (id % CT) * 8);
        else
          rp[p][u] = *reinterpret_cast<const half8*>(P + p * pplane + (long long)(tj * TILE + row) * ldp + k0 + c * 8);
      }
    }
  };
  auto store = [&](int stage) {
    char* s = lds + stage * STAGE;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int id = u * 256 + tid;
      const int row = id / CK, nt = row * KS * 2 + (((id % CK) ^ ntf(row)) << 4);
      const int k = id / CT, ch = id % CT;
      const int tr = k * TILE * 2 + (((ch >> 1) ^ trf(k)) << 5) + ((ch & 1) << 4);
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        *reinterpret_cast<half8*>(s + p * OPB + nt) = rq[p][u];
        *reinterpret_cast<half8*>(s + (PLANES + p) * OPB + (KIND == kApply ? tr : nt)) = rp[p][u];
      }
    }
  };
  auto frag = [&](const char* plane, int row0, int kk) {
    const int row = row0 + (lane & 15);
    return *reinterpret_cast<const half8*>(plane + row * KS * 2 + (((kk * 4 + (lane >> 4)) ^ ntf(row)) << 4));
  };
  auto frag_tr = [&](const char* plane, int j0, int kk) {
    typedef __attribute__((address_space(3))) bf16x4* lptr;              // (the read moves 16-bit patterns, whatever they mean)
    const int i = lane & 15, k = kk * 32 + 8 * (lane >> 4) + (i >> 2);
    const char* a0 = plane + k * TILE * 2 + (((j0 >> 4) ^ trf(k)) << 5) + ((i & 3) << 3);
    const half4 lo = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(a0)));
    const half4 hi = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(a0 + 4 * TILE * 2)));
    half8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = lo[e]; f[4 + e] = hi[e]; }
    return f;
  };
  f32x4 acc[NF][NF];
#pragma unroll
  for (int p = 0; p < NF; ++p)
#pragma unroll
    for (int q = 0; q < NF; ++q) acc[p][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const char* s, int kk) {
    half8 fq[PLANES][NF], fp[PLANES][NF];
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        fq[p][f] = frag(s + p * OPB, wq + 16 * f, kk);
        if constexpr (KIND == kApply) fp[p][f] = frag_tr(s + (PLANES + p) * OPB, wp + 16 * f, kk);
        else fp[p][f] = frag(s + (PLANES + p) * OPB, wp + 16 * f, kk);
      }
#pragma unroll
    for (int p = 0; p < NF; ++p)
#pragma unroll
      for (int q = 0; q < NF; ++q) {
        if constexpr (TERMS == 3) {
          acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[1][p], fq[0][q], acc[p][q], 0, 0, 0);
          acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][p], fq[1][q], acc[p][q], 0, 0, 0);
        }
        acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][p], fq[0][q], acc[p][q], 0, 0, 0);
      }
  };

  load(0);
  if constexpr (STAGES == 2) {
    store(0);
    __syncthreads();
    int stage = 0;
    for (int k0 = 0; k0 < K; k0 += KS) {
      const bool more = k0 + KS < K;
      if (more) load(k0 + KS);
#pragma unroll
      for (int kk = 0; kk < KS / 32; ++kk) compute(lds + stage * STAGE, kk);
      if (more) store(stage ^ 1);
      __syncthreads();
      stage ^= 1;
    }
  } else {
    for (int k0 = 0; k0 < K; k0 += KS) {
      if (k0) __syncthreads();                                          // (everyone has read the stage before)
      store(0);
      __syncthreads();
      if (k0 + KS < K) load(k0 + KS);
#pragma unroll
      for (int kk = 0; kk < KS / 32; ++kk)
        if (k0 + kk * 32 < K) compute(lds, kk);
    }
  }

  // epilogue: lane (l & 15) has row i, entries j .. j + 3
  const bool tall = o.rows > o.cols;
  const int m = tall ? o.cols : o.rows, n = tall ? o.rows : o.cols;
  float* dA = reinterpret_cast<float*>(base + w.diag(o.Mp));
  float* dB = dA + o.Mp;
#pragma unroll
  for (int q = 0; q < NF; ++q) {
    const int i = ti * TILE + wq + 16 * q + (lane & 15);
#pragma unroll
    for (int p = 0; p < NF; ++p) {
      const int j = tj * TILE + wp + 16 * p + 4 * (lane >> 4);
      half4 h, l;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[p][q][e] * (kOrthInv * kOrthInv);
      if constexpr (KIND == kApply) {
        const long long at = (long long)i * o.Np + j;
        const half4 xh = *reinterpret_cast<const half4*>(X + at), xl = *reinterpret_cast<const half4*>(X + w.xplane + at);
        const float d = TERMS == 1 ? dB[i] : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float xhf = (float)xh[e] * kOrthInv;
          float r = fmaf(g.a, xhf + (float)xl[e] * kOrthInv, v[e]);
          if constexpr (TERMS == 1) r = fmaf(d, xhf, r);
          v[e] = r;
        }
        if (last) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i < m && j + e < n) fin.put(o, tall, i, j + e, v[e]);
        } else {
          half_t* xo = reinterpret_cast<half_t*>(base + w.x(g.buf ^ 1));
#pragma unroll
          for (int e = 0; e < 4; ++e) { half_t a, b; split(v[e], a, b); h[e] = a; l[e] = b; }
          *reinterpret_cast<half4*>(xo + at) = h;
          *reinterpret_cast<half4*>(xo + w.xplane + at) = l;
        }
      } else {
        const long long at = (long long)i * o.Mp + j;
        half_t* dst = reinterpret_cast<half_t*>(base + (KIND == kGram ? w.a() : w.b()));
        if constexpr (KIND == kPoly) {
          const half4 ah = *reinterpret_cast<const half4*>(A + at), al = *reinterpret_cast<const half4*>(A + w.aplane + at);
          const float di = TERMS == 1 ? dA[i] : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float aij = ((float)ah[e] + (float)al[e]) * kOrthInv, aa = v[e];
            if constexpr (TERMS == 1) {
              if (i == j + e) { aij = di; aa = fmaf(di, di, aa); }
              else aa = fmaf(di + dA[j + e], aij, aa);
            }
            v[e] = fmaf(g.c, aa, g.b * aij);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (TERMS == 1) {
            if (i == j + e) { (KIND == kGram ? dA : dB)[i] = v[e]; v[e] = 0.f; }
          }
          half_t a, b;
          split(v[e], a, b);
          h[e] = a; l[e] = b;
        }
        *reinterpret_cast<half4*>(dst + at) = h;
        *reinterpret_cast<half4*>(dst + w.aplane + at) = l;
        if (ti != tj) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dst[(long long)(j + e) * o.Mp + i] = h[e];
            dst[w.aplane + (long long)(j + e) * o.Mp + i] = l[e];
          }
        }
      }
    }
  }
}

// AdamW on the parameters that are no matrices: {offset, count} per workgroup
__global__ __launch_bounds__(256) void muon_rest_kernel(const longlong2* __restrict__ runs, float* __restrict__ p, const float* __restrict__ g,
                                                        float* __restrict__ m, float* __restrict__ v, float keep, float step, float b1, float c1,
                                                        float b2, float c2, float eps, float bc2_sqrt, float grad_scale) {
  const longlong2 r = runs[blockIdx.x];
  for (long long k = threadIdx.x; k < r.y; k += 256) {
    const long long i = r.x + k;
    const float gv = grad_scale * g[i];
    const float mv = b1 * m[i] + c1 * gv, vv = b2 * v[i] + c2 * (gv * gv);
    p[i] = p[i] * keep - step * mv / (sqrtf(vv) / bc2_sqrt + eps);
    m[i] = mv; v[i] = vv;
  }
}

static int up(int v, int q) { return (v + q - 1) / q * q; }
static OrthItem orth_make(int rows, int cols, int tile) {
  OrthItem o;
  memset(&o, 0, sizeof o);
  o.rows = rows; o.cols = cols;
  o.Mp = up(std::min(rows, cols), tile); o.Np = up(std::max(rows, cols), tile);
  o.gain = 1.f;
  return o;
}
// tiles of A or A A (symmetric), and of B X
static long long orth_sym_tiles(const OrthItem& o, int tile) { const long long t = o.Mp / tile; return t * (t + 1) / 2; }
static long long orth_apply_tiles(const OrthItem& o, int tile) { return (long long)(o.Mp / tile) * (o.Np / tile); }

// 128 x 128 tiles move half the bytes per product of 64 x 64 ones, but a launch of them fills the chip only from 256 tiles on
static int orth_tile(int rows, int cols, long long batch) {
  return batch * orth_apply_tiles(orth_make(rows, cols, 128), 128) >= 256 ? 128 : 64;
}

struct OrthCounts { long long flat, pack, sym, apply; };

template <int TERMS, int TILE, typename SRC, typename OUT>
static int orth_run(OrthArgs g, const OrthCounts& n, const int4* const (&lists)[4], const SRC& src, const OUT& out, int steps, const int (&per)[4],
                    hipStream_t s) {
  const dim3 b(256);
  auto with = [&](int k, int buf) { OrthArgs h = g; h.tiles = lists[k]; h.per = per[k]; h.buf = buf; return h; };
  hipLaunchKernelGGL((orth_norm_kernel<SRC>), dim3((unsigned)n.flat), b, 0, s, with(0, 0), src);
  hipLaunchKernelGGL((orth_pack_kernel<SRC>), dim3((unsigned)n.pack), b, 0, s, with(1, 0), src);
  for (int k = 0; k < steps; ++k) {
    hipLaunchKernelGGL((orth_gemm_kernel<TERMS, kGram, TILE, OrthNone>), dim3((unsigned)n.sym), b, 0, s, with(2, k & 1), OrthNone{}, 0);
    hipLaunchKernelGGL((orth_gemm_kernel<TERMS, kPoly, TILE, OrthNone>), dim3((unsigned)n.sym), b, 0, s, with(2, k & 1), OrthNone{}, 0);
    hipLaunchKernelGGL((orth_gemm_kernel<TERMS, kApply, TILE, OUT>), dim3((unsigned)n.apply), b, 0, s, with(3, k & 1), out, k == steps - 1);
  }
  return (int)hipGetLastError();
}

constexpr int kOrthMaxSide = 1 << 20;
constexpr int kOrthMaxSteps = 64;

static bool orth_shape_ok(long long rows, long long cols) {
  // (a matrix of up to 2^31 entries: tile counts and the entries of a plane's row stay in 32 bits, offsets are 64)
  return rows >= 1 && cols >= 1 && rows <= kOrthMaxSide && cols <= kOrthMaxSide && rows * cols <= 0x7fffffffll;
}

}  // namespace pwr

using namespace pwr;

extern "C" size_t pwr_orthogonalize_workspace_bytes(int rows, int cols, long long batch) {
  if (batch <= 0 || !orth_shape_ok(rows, cols)) return 0;
  const OrthItem o = orth_make(rows, cols, orth_tile(rows, cols, batch));
  return (size_t)batch * orth_ws_bytes(rows, cols, o.Mp, o.Np);
}

template <typename T, int TERMS>
static int orthogonalize(const void* x, long long x_batch, long long x_ld, void* out, int rows, int cols, long long batch, int steps, float a, float b,
                         float c, float eps, void* ws, hipStream_t s) {
  const int tile = orth_tile(rows, cols, batch);
  OrthArgs g = {};
  g.one = orth_make(rows, cols, tile);
  g.ws = (char*)ws;
  g.ws_stride = orth_ws_bytes(rows, cols, g.one.Mp, g.one.Np);
  g.a = a; g.b = b; g.c = c; g.eps = eps;
  const long long per[4] = {orth_parts(rows, cols), (long long)(g.one.Mp / 64) * (g.one.Np / 64), orth_sym_tiles(g.one, tile), orth_apply_tiles(g.one, tile)};
  const OrthCounts n = {batch * per[0], batch * per[1], batch * per[2], batch * per[3]};
  if (std::max(std::max(n.flat, n.pack), std::max(n.sym, n.apply)) > 0x7fffffffll) return PWR_EUNSUPPORTED;
  const int4* const lists[4] = {};
  const int iper[4] = {(int)per[0], (int)per[1], (int)per[2], (int)per[3]};
  g.src_stride = x_batch;
  g.dst_stride = (long long)rows * cols;
  const OrthTensor<T> src = {(const T*)x, x_ld};
  const OrthOut<T> dst = {(T*)out, cols};
  return tile == 128 ? orth_run<TERMS, 128>(g, n, lists, src, dst, steps, iper, s) : orth_run<TERMS, 64>(g, n, lists, src, dst, steps, iper, s);
}

extern "C" int pwr_orthogonalize(const void* x, long long x_batch_stride, long long x_row_stride, void* out, int rows, int cols, long long batch,
                                 int dtype, int steps, float a, float b, float c, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch == 0) return 0;
  if (!x || !out || batch < 0 || x_batch_stride < 0 || x_row_stride < 0 || steps < 1 || steps > kOrthMaxSteps || !(eps >= 0.f)) return PWR_EINVAL;
  if (dtype != PWR_F32 && dtype != PWR_BF16) return PWR_EINVAL;
  if (!orth_shape_ok(rows, cols)) return rows < 1 || cols < 1 ? PWR_EINVAL : PWR_EUNSUPPORTED;
  if (!workspace || workspace_bytes < pwr_orthogonalize_workspace_bytes(rows, cols, batch)) return PWR_ENOSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PWR_F32) return orthogonalize<float, 3>(x, x_batch_stride, x_row_stride, out, rows, cols, batch, steps, a, b, c, eps, workspace, s);
  return orthogonalize<bf16_t, 1>(x, x_batch_stride, x_row_stride, out, rows, cols, batch, steps, a, b, c, eps, workspace, s);
}

// ---------------------------------------------------------------------------------------------
// The optimizer step: a PLAN of a parameter list (host bytes, copied to the device once), then one call per step.
// ---------------------------------------------------------------------------------------------
namespace {

constexpr int kRestRun = 4096;           // elements per workgroup of the AdamW part
struct MuonHead {
  unsigned long long magic, bytes, ws_bytes;
  int items, tile;
  long long n[4], rest;                  // workgroups of the norm, pack, symmetric and apply launches; of the rest
  long long at_items, at_list[4], at_rest;
};
constexpr unsigned long long kMuonMagic = 0x31304e4f554d5750ull;

// what the launches of a list cost with a tile: the padded products, in units of one product of a 64 x 64 x 64 block
long long muon_cost(const std::vector<OrthItem>& v, int tile, long long* blocks) {
  long long c = 0;
  *blocks = 0;
  for (const OrthItem& k : v) {
    const OrthItem o = orth_make(k.rows, k.cols, tile);
    const long long m = o.Mp / 64, n = o.Np / 64;
    c += m * m * (2 * n + m);
    *blocks += orth_apply_tiles(o, tile);
  }
  return c;
}

bool muon_layout(const pwr_muon_param* params, int n, MuonHead& h, std::vector<OrthItem>& items, std::vector<longlong2>& rest) {
  std::vector<std::pair<long long, long long>> used;
  std::vector<pwr_muon_param> vec;
  for (int k = 0; k < n; ++k) {
    const pwr_muon_param& q = params[k];
    if (q.offset < 0 || q.rows < 1 || q.cols < 1) return false;
    used.push_back({q.offset, q.offset + (long long)q.rows * q.cols});
    if (std::min(q.rows, q.cols) == 1) { vec.push_back(q); continue; }
    if (!orth_shape_ok(q.rows, q.cols)) return false;
    OrthItem o = orth_make(q.rows, q.cols, 64);
    o.src = o.dst = q.offset;
    items.push_back(o);
  }
  std::sort(used.begin(), used.end());
  for (size_t k = 1; k < used.size(); ++k)
    if (used[k].first < used[k - 1].second) return false;               // (an element that two parameters share would be updated twice)
  for (const pwr_muon_param& q : vec)
    for (long long at = 0, e = (long long)q.rows * q.cols; at < e; at += kRestRun)
      rest.push_back(longlong2{q.offset + at, std::min<long long>(kRestRun, e - at)});
  memset(&h, 0, sizeof h);
  h.magic = kMuonMagic;
  h.items = (int)items.size();
  // (the rule of orth_tile, and no wide tile where its padding costs over a quarter more)
  long long b64, b128;
  const long long c64 = muon_cost(items, 64, &b64), c128 = muon_cost(items, 128, &b128);
  h.tile = b128 >= 256 && 4 * c128 <= 5 * c64 ? 128 : 64;
  long long ws = 0;
  for (OrthItem& o : items) {
    const OrthItem q = orth_make(o.rows, o.cols, h.tile);
    o.Mp = q.Mp; o.Np = q.Np;
    o.gain = sqrtf((float)std::max(o.rows, o.cols));
    o.ws = ws;
    ws += orth_ws_bytes(o.rows, o.cols, o.Mp, o.Np);
    h.n[0] += orth_parts(o.rows, o.cols);
    h.n[1] += (long long)(o.Mp / 64) * (o.Np / 64);
    h.n[2] += orth_sym_tiles(o, h.tile);
    h.n[3] += orth_apply_tiles(o, h.tile);
  }
  h.ws_bytes = ws;
  h.rest = (long long)rest.size();
  long long at = (sizeof(MuonHead) + 255) / 256 * 256;
  auto take = [&](long long bytes) { const long long r = at; at += (bytes + 255) / 256 * 256; return r; };
  h.at_items = take(h.items * (long long)sizeof(OrthItem));
  for (int k = 0; k < 4; ++k) h.at_list[k] = take(h.n[k] * (long long)sizeof(int4));
  h.at_rest = take(h.rest * (long long)sizeof(longlong2));
  h.bytes = at;
  for (int k = 0; k < 4; ++k)
    if (h.n[k] > 0x7fffffffll) return false;
  return h.rest <= 0x7fffffffll;
}

}  // namespace

extern "C" size_t pwr_muon_plan_bytes(const pwr_muon_param* params, int n) {
  if (!params || n < 1) return 0;
  MuonHead h;
  std::vector<OrthItem> items;
  std::vector<longlong2> rest;
  return muon_layout(params, n, h, items, rest) ? h.bytes : 0;
}

extern "C" int pwr_muon_plan(const pwr_muon_param* params, int n, void* host_dst) {
  if (!params || n < 1 || !host_dst) return PWR_EINVAL;
  MuonHead h;
  std::vector<OrthItem> items;
  std::vector<longlong2> rest;
  if (!muon_layout(params, n, h, items, rest)) return PWR_EINVAL;
  char* d = (char*)host_dst;
  memset(d, 0, h.bytes);
  memcpy(d, &h, sizeof h);
  memcpy(d + h.at_items, items.data(), items.size() * sizeof(OrthItem));
  std::vector<int4> list[4];
  for (int k = 0; k < h.items; ++k) {
    const OrthItem& o = items[k];
    for (int t = 0; t < orth_parts(o.rows, o.cols); ++t) list[0].push_back(int4{k, t, 0, 0});
    for (int i = 0; i < o.Mp / 64; ++i)
      for (int j = 0; j < o.Np / 64; ++j) list[1].push_back(int4{k, i, j, 0});
    for (int j = 0; j < o.Mp / h.tile; ++j)
      for (int i = 0; i <= j; ++i) list[2].push_back(int4{k, i, j, 0});
    for (int i = 0; i < o.Mp / h.tile; ++i)
      for (int j = 0; j < o.Np / h.tile; ++j) list[3].push_back(int4{k, i, j, 0});
  }
  for (int k = 0; k < 4; ++k) memcpy(d + h.at_list[k], list[k].data(), list[k].size() * sizeof(int4));
  memcpy(d + h.at_rest, rest.data(), rest.size() * sizeof(longlong2));
  return 0;
}

extern "C" size_t pwr_muon_workspace_bytes(const void* plan_host) {
  const MuonHead* h = (const MuonHead*)plan_host;
  return h && h->magic == kMuonMagic ? h->ws_bytes : 0;
}

extern "C" int pwr_muon_step(const void* plan_host, const void* plan_dev, float* p, const float* g, float* buf, float* v, float lr, float momentum,
                             int nesterov, float weight_decay, float update_rms, int ns_steps, float a, float b, float c, float eps, float beta1,
                             float beta2, float adam_eps, int step, float grad_scale, void* workspace, size_t workspace_bytes, void* stream) {
  const MuonHead* h = (const MuonHead*)plan_host;
  if (!h || h->magic != kMuonMagic || !plan_dev || !p || !g || !buf || (h->rest && !v)) return PWR_EINVAL;
  if (ns_steps < 1 || ns_steps > kOrthMaxSteps || !(eps >= 0.f) || step < 1) return PWR_EINVAL;
  if (h->items && (!workspace || workspace_bytes < h->ws_bytes)) return PWR_ENOSPACE;
  hipStream_t s = (hipStream_t)stream;
  const char* d = (const char*)plan_dev;
  const float keep = 1.f - lr * weight_decay;
  if (h->rest) {
    // (1 - beta and 1 - beta^t in 64 bits: the first steps' 1 - 0.999 would lose 2e-5 of itself)
    const double bc1 = 1.0 - pow((double)beta1, step), bc2 = 1.0 - pow((double)beta2, step);
    hipLaunchKernelGGL(muon_rest_kernel, dim3((unsigned)h->rest), dim3(256), 0, s, (const longlong2*)(d + h->at_rest), p, g, buf, v, keep,
                       (float)(lr / bc1), beta1, (float)(1.0 - (double)beta1), beta2, (float)(1.0 - (double)beta2), adam_eps, (float)sqrt(bc2), grad_scale);
  }
  if (!h->items) return (int)hipGetLastError();
  OrthArgs ga = {};
  ga.items = (const OrthItem*)(d + h->at_items);
  ga.ws = (char*)workspace;
  ga.a = a; ga.b = b; ga.c = c; ga.eps = eps;
  const OrthCounts n = {h->n[0], h->n[1], h->n[2], h->n[3]};
  const int4* lists[4];
  for (int k = 0; k < 4; ++k) lists[k] = (const int4*)(d + h->at_list[k]);
  const int4* const (&ls)[4] = lists;
  const int per[4] = {};
  const OrthMomentum src = {g, buf, momentum, grad_scale, nesterov};
  const OrthUpdate dst = {p, keep, lr * update_rms};
  return h->tile == 128 ? orth_run<3, 128>(ga, n, ls, src, dst, ns_steps, per, s) : orth_run<3, 64>(ga, n, ls, src, dst, ns_steps, per, s);
}
