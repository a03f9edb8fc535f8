// Orthogonalising a matrix by Newton-Schulz products, and the optimizer step built on it (Muon).
//
// X0 = G / (|G|_F + eps); then `steps` times  A = X X^T,  B = b A + c A A,  X <- a X + B X.
// Every singular value s of X goes through s <- a s + b s^3 + c s^5 and the singular vectors stay: with (a, b, c) = (3.4445, -4.7750, 2.0315)
// five steps bring everything above ~1e-3 of the norm into about 0.7 .. 1.2, i.e. X is near the closest orthogonal matrix U V^T.  A matrix with
// more rows than columns is worked on transposed, so A and B are as small as they can be: m x m with m = min(rows, cols), n = max.
//
// Numbers.  Everything between the products is kept as a PAIR of fp16, hi + lo = 22 bits, scaled by 4096 (|X| <= ~1.2, |A| <= ~1.5, |B| <= ~3
// with the coefficients above; others are refused where an entry could reach 16, the end of fp16).  Below 2^-14 = 6e-5 the low half is no normal fp16 any
// more, and an entry is kept to 2^-37 instead of 2^-23 of itself: the result is right in norm, and a row that is 1e-5 of the others right to 1e-4 of
// itself (in fp32 arithmetic: 2e-7).  The matrix cores multiply fp16 pairs exactly and add in fp32.
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
#include <cmath>
#include <type_traits>
#include <vector>

#include "pwr_common.h"
#include "pwr.h"

namespace pwr {

typedef _Float16 half_t;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;

constexpr float kOrthScale = 4096.f;                     // of every stored pair
constexpr float kOrthInv = 1.f / 4096.f;
constexpr int kOrthNarrow = 128;                         // up to this many rows A fits the LDS: its sums go straight into the product A A

// One matrix.  In a table on the device (a parameter list), or made from the launch's arguments (a batch of equal ones).
struct OrthItem {
  long long src, dst;       // offsets of its first element in the source and in the result (in elements)
  long long ws;             // offset of its workspace block (in bytes)
  int rows, cols;           // as the caller has it
  int Mp, Np;               // min / max of the two, up to the tile
  float gain;               // of the update
  int shares, first;        // workgroups along K of a 64 x 64 tile of A; the first of its sums (in a batch: sums per matrix)
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
  const OrthItem* items; const int4* tiles;              // table form (items != null): tiles[t] = {item, ti, tj, share}
  OrthItem one; long long src_stride, dst_stride, ws_stride; int per;     // batch form: t = batch * per + tile
  char* ws;
  int buf;                                               // which X buffer is read
  float a, b, c, eps;
  // a product's tiles from `whole` on are split into `parts` along K: their sums go to slab [tile - whole][part][4 x 4 fragments][256 threads]
  int whole, parts; f32x4* slab;
  // 64 x 64 tiles: a workgroup of A that has only a share of its tile's K, or whose matrix is narrow, leaves its sums at slab + 1024 orth_sums(); those of
  // the first `shared` ones are joined by a launch of their own
  int shared;
};

// the matrix and tile number t of a launch belong to: tile >= 0 is the number within the matrix, else `entry` names it
__device__ __forceinline__ OrthItem orth_item(const OrthArgs& g, int t, int& tile, int4& entry) {
  if (g.items) {
    entry = g.tiles[t];
    tile = -1;
    return g.items[entry.x];
  }
  const int batch = t / g.per;
  tile = t - batch * g.per;
  OrthItem o = g.one;
  o.src += batch * g.src_stride;
  o.dst += batch * g.dst_stride;
  o.ws += batch * g.ws_stride;
  o.first *= batch;
  return o;
}
// Tiles of B X: a die gets every eighth workgroup.  64 x 64 tiles go in bands of eight columns, so that a die has a column of X for all its rows (5 of
// 1031 x 517 fp32 300 -> 265 us, the step of the 42-joint network with 256 features 530 -> 515); 128 x 128 ones row by row: eight columns and eight rows at once on a die (2048 x 8192 2010 us, in bands 2060).
__host__ __device__ __forceinline__ int orth_band(int tile, int nj) { return tile == 64 ? 8 : nj; }
// (ti, tj) of a tile of B X, or of a symmetric product: ti <= tj, in blocks of 4 x 4 tiles, block column J from tile 2 J (4 J + 1) on: workgroups that run
// together on a chip die read few different rows.  T: tiles a side; nj: tiles a row of X, `band` of them at a time.
__device__ __forceinline__ void orth_place(bool symmetric, int tile, const int4& entry, int T, int nj, int band, int& ti, int& tj) {
  if (tile < 0) { ti = entry.y; tj = entry.z; }
  else if (!symmetric) {
    const int b = tile / (band * T), rest = tile - b * band * T, wide = min(band, nj - b * band);
    ti = rest / wide;
    tj = b * band + rest - ti * wide;
  }
  else {
    int J = (int)((sqrtf(4.f + 32.f * tile) - 2.f) * (1.f / 16.f));
    while (2 * J * (4 * J + 1) > tile) --J;
    while (2 * (J + 1) * (4 * J + 5) <= tile) ++J;
    const int wide = min(4, T - 4 * J), rest = tile - 2 * J * (4 * J + 1), I = min(rest / (4 * wide), J), in = rest - I * 4 * wide;
    if (I < J) { ti = 4 * I + in / wide; tj = 4 * J + in % wide; }
    else {
      int c = 0;
      while ((c + 1) * (c + 2) / 2 <= in) ++c;
      tj = 4 * J + c;
      ti = 4 * J + in - c * (c + 1) / 2;
    }
  }
}
// where the sums of share `part` of a 64 x 64 tile of A are (t: the tile's number in a batch)
__device__ __forceinline__ long long orth_sums(const OrthArgs& g, const OrthItem& o, int t, int ti, int tj, int part) {
  return (g.items ? o.first + (long long)(tj * (tj + 1) / 2 + ti) * o.shares : (long long)t * o.shares) + part;
}
// Workgroup b of n, dealt round over the 8 chip dies: the die's share of the numbers 0 .. n - 1 is a run of neighbours.
__device__ __forceinline__ int orth_die_order(int b, int n) {
  const int x = b & 7, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + (b >> 3);
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
  const OrthItem o = orth_item(g, blockIdx.x, t, tile);
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
  const OrthItem o = orth_item(g, blockIdx.x, t, tile);
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

// ---- what the last step does with N neighbouring entries X[i][j .. j + N) of an m x n matrix.  Everything is read before anything is written: behind one
// another's stores the reads would cost a latency each (the last B X of the 42-joint step with 256 features: 92 us, all together 55).
template <typename T> struct OrthOut {
  T* out; long long ld;
  template <int N> __device__ __forceinline__ void put(const OrthItem& o, bool tall, int m, int n, int i, int j, const float (&v)[N]) const {
    if (i >= m) return;
    if (!tall && j + N <= n) {
      T* q = out + o.dst + (long long)i * ld + j;
#pragma unroll
      for (int e = 0; e < N; e += 4)
        *reinterpret_cast<Quad<T>*>(q + e) = Quad<T>{{Elem<T>::from_f(v[e]), Elem<T>::from_f(v[e + 1]), Elem<T>::from_f(v[e + 2]), Elem<T>::from_f(v[e + 3])}};
      return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (j + e < n) out[o.dst + (tall ? (j + e) * ld + i : i * ld + j + e)] = Elem<T>::from_f(v[e]);
  }
};
struct OrthUpdate {
  float* p; float keep, lr;           // keep = 1 - lr weight_decay
  template <int N> __device__ __forceinline__ void put(const OrthItem& o, bool tall, int m, int n, int i, int j, const float (&v)[N]) const {
    if (i >= m) return;
    const float step = lr * o.gain;
    float* base = p + o.dst;
    constexpr int C = N < 8 ? N : 8;                                  // (sixteen together spill)
    if (!tall && j + N <= n) {
      float* q = base + (long long)i * o.cols + j;
#pragma unroll
      for (int h = 0; h < N; h += C) {
        Quad<float> x[C / 4];
#pragma unroll
        for (int k = 0; k < C / 4; ++k) x[k] = *reinterpret_cast<const Quad<float>*>(q + h + 4 * k);
#pragma unroll
        for (int k = 0; k < C / 4; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k].v[e] = x[k].v[e] * keep - step * v[h + 4 * k + e];
          *reinterpret_cast<Quad<float>*>(q + h + 4 * k) = x[k];
        }
      }
      return;
    }
    auto at = [&](int jj) { return tall ? (long long)jj * o.cols + i : (long long)i * o.cols + jj; };
#pragma unroll
    for (int h = 0; h < N; h += C) {
      float x[C];
#pragma unroll
      for (int e = 0; e < C; ++e) x[e] = base[at(min(j + h + e, n - 1))];
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (j + h + e < n) base[at(j + h + e)] = x[e] * keep - step * v[h + e];
    }
  }
};
struct OrthNone {
  template <int N> __device__ __forceinline__ void put(const OrthItem&, bool, int, int, int, int, const float (&)[N]) const {}
};

enum { kGram = 0, kPoly = 1, kApply = 2 };

// N neighbouring entries of one row as pairs
template <int N> struct alignas(N >= 8 ? 16 : 8) Halves { half_t v[N]; };
template <int N> struct OrthPair { Halves<N> h, l; };

// What finished entries need besides their sums: the pairs of A (for B) or X (for the next X) at the same place.
template <int KIND, int N>
__device__ __forceinline__ OrthPair<N> orth_beside(const OrthArgs& g, const OrthItem& o, const OrthWs& w, int i, int j) {
  OrthPair<N> r;
  if constexpr (KIND != kGram) {
    const char* base = g.ws + o.ws;
    const half_t* p = reinterpret_cast<const half_t*>(base + (KIND == kPoly ? w.a() : w.x(g.buf))) + (long long)i * (KIND == kPoly ? o.Mp : o.Np) + j;
    r.h = *reinterpret_cast<const Halves<N>*>(p);
    r.l = *reinterpret_cast<const Halves<N>*>(p + (KIND == kPoly ? w.aplane : w.xplane));
  }
  return r;
}

// Entries (i, j .. j + N) of a finished product, and what becomes of them: A, B or the next X, as pairs (returned too); after the last step the result.
template <int TERMS, int KIND, int N, typename OUT>
__device__ __forceinline__ OrthPair<N> orth_finish(const OrthArgs& g, const OrthItem& o, const OrthWs& w, const OUT& fin, int last, int i, int j,
                                                   const float (&sum)[N], const OrthPair<N>& beside, const float* diag = nullptr) {
  char* base = g.ws + o.ws;
  float v[N];
  OrthPair<N> r;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = sum[e] * (kOrthInv * kOrthInv);
  float* dA = reinterpret_cast<float*>(base + w.diag(o.Mp));
  float* dB = dA + o.Mp;
  if constexpr (KIND == kApply) {
    const float d = TERMS == 1 ? dB[i] : 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xhf = (float)beside.h.v[e] * kOrthInv;
      float x = fmaf(g.a, xhf + (float)beside.l.v[e] * kOrthInv, v[e]);
      if constexpr (TERMS == 1) x = fmaf(d, xhf, x);
      v[e] = x;
    }
    if (last) {
      const bool tall = o.rows > o.cols;
      const int m = tall ? o.cols : o.rows, n = tall ? o.rows : o.cols;
      fin.put(o, tall, m, n, i, j, v);
      return r;
    }
  } else {
    if constexpr (KIND == kPoly) {
      const float* const da = diag ? diag : dA;
      const float di = TERMS == 1 ? da[i] : 0.f;
      float dj[N];
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const f32x4 d = TERMS == 1 ? *reinterpret_cast<const f32x4*>(da + j + e) : f32x4{0.f, 0.f, 0.f, 0.f};
        dj[e] = d.x; dj[e + 1] = d.y; dj[e + 2] = d.z; dj[e + 3] = d.w;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float aij = ((float)beside.h.v[e] + (float)beside.l.v[e]) * kOrthInv, aa = v[e];
        if constexpr (TERMS == 1) {
          const bool same = i == j + e;
          aa = fmaf(same ? di : di + dj[e], same ? di : aij, aa);
          aij = same ? di : aij;
        }
        v[e] = fmaf(g.c, aa, g.b * aij);
      }
    }
    if constexpr (TERMS == 1) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i == j + e) { (KIND == kGram ? dA : dB)[i] = v[e]; v[e] = 0.f; }
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) split(v[e], r.h.v[e], r.l.v[e]);
  half_t* dst = reinterpret_cast<half_t*>(base + (KIND == kApply ? w.x(g.buf ^ 1) : KIND == kGram ? w.a() : w.b()));
  const long long at = (long long)i * (KIND == kApply ? o.Np : o.Mp) + j;
  *reinterpret_cast<Halves<N>*>(dst + at) = r.h;
  *reinterpret_cast<Halves<N>*>(dst + (KIND == kApply ? w.xplane : w.aplane) + at) = r.l;
  return r;
}
// the same entries on the other side of the diagonal
template <int KIND, int N>
__device__ __forceinline__ void orth_mirror(const OrthArgs& g, const OrthItem& o, const OrthWs& w, int i, int j, const OrthPair<N>& r) {
  half_t* dst = reinterpret_cast<half_t*>(g.ws + o.ws + (KIND == kGram ? w.a() : w.b())) + i;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    dst[(long long)(j + e) * o.Mp] = r.h.v[e];
    dst[w.aplane + (long long)(j + e) * o.Mp] = r.l.v[e];
  }
}

// A A of a matrix of one or two 64 x 64 tiles a side: the workgroup (16 waves, a fragment each) adds the shares of all of A into LDS, which is never
// written out, and multiplies from there.
template <int TERMS>
__device__ __forceinline__ void orth_narrow_poly(const OrthArgs& g, const OrthItem& o, const OrthWs& w, int ti, int tj, char* lds) {
  __shared__ __attribute__((aligned(16))) float diag[kOrthNarrow];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  const int Mp = o.Mp, plane = Mp * Mp * 2, flip = Mp == 128 ? 15 : 7, shift = Mp == 128 ? 0 : 1;
  // rows of Mp * 2 bytes, their 16-byte units swizzled by the row
  auto at = [&](int row, int j) { return row * Mp * 2 + (((j >> 3) ^ ((row >> shift) & flip)) << 4) + (j & 7) * 2; };
  const f32x4* s = g.slab + (long long)o.first * 1024 + tid;
  const int gi = ((wave >> 1) & 1) * 32 + (wave >> 3) * 16 + li, gj = (wave & 1) * 32 + 8 * lg + ((wave >> 2) & 1) * 4;     // the entries that A's launch gave this thread
  auto place = [&](const f32x4& a, int i, int j, bool mirror) {
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = a[e] * (kOrthInv * kOrthInv);
      if (TERMS == 1 && i == j + e) { diag[i] = v; v = 0.f; }
      half_t p, q;
      split(v, p, q);
      h[e] = p; l[e] = q;
    }
    *reinterpret_cast<half4*>(lds + at(i, j)) = h;
    *reinterpret_cast<half4*>(lds + plane + at(i, j)) = l;
    if (mirror) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        *reinterpret_cast<half_t*>(lds + at(j + e, i)) = h[e];
        *reinterpret_cast<half_t*>(lds + plane + at(j + e, i)) = l[e];
      }
    }
  };
  const int n = o.shares;
  if (Mp == 64) {
    f32x4 a = s[0];
    for (int u = 1; u < n; ++u) a += s[u * 1024];
    place(a, gi, gj, false);
  } else {
    f32x4 a[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) a[q] = s[q * n * 1024];
    for (int u = 1; u < n; ++u)
#pragma unroll
      for (int q = 0; q < 3; ++q) a[q] += s[(q * n + u) * 1024];
    place(a[0], gi, gj, false);
    place(a[1], gi, 64 + gj, true);
    place(a[2], 64 + gi, 64 + gj, false);
  }
  __syncthreads();
  const int i = ti * 64 + (wave >> 2) * 16, j = tj * 64 + (wave & 3) * 16;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = 8 * lg; k < Mp; k += 32) {
    const half8 qh = *reinterpret_cast<const half8*>(lds + at(i + li, k)), ph = *reinterpret_cast<const half8*>(lds + at(j + li, k));
    if constexpr (TERMS == 3) {
      const half8 ql = *reinterpret_cast<const half8*>(lds + plane + at(i + li, k)), pl = *reinterpret_cast<const half8*>(lds + plane + at(j + li, k));
      acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, acc, 0, 0, 0);
    }
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
  }
  const int jj = j + 4 * lg;
  OrthPair<4> beside;
  beside.h = *reinterpret_cast<const Halves<4>*>(lds + at(i + li, jj));
  beside.l = *reinterpret_cast<const Halves<4>*>(lds + plane + at(i + li, jj));
  const float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  const OrthPair<4> d = orth_finish<TERMS, kPoly, 4, OrthNone>(g, o, w, OrthNone{}, 0, i + li, jj, v, beside, diag);
  if (ti != tj) orth_mirror<kPoly, 4>(g, o, w, i + li, jj, d);
}

// ---- the products: one TILE x TILE tile of the result per workgroup of four waves.
// First MFMA operand P: the entries j, second operand Q: the rows i.  A lane ends up with four neighbouring j of one row i per fragment; row 4 g + e of
// fragment p is entry 4 NF g + 4 p + e, so that its NF fragments are 4 NF neighbours, and the 16 x 4 lanes hold whole cache lines.
// A and A A are symmetric: tiles tj >= ti only, written twice.  In B X the columns of X are needed along K: its rows are staged as they are
// and read transposed by the LDS hardware.
// TILE 128, large matrices: a wave has (TILE / 2)^2; two stages in LDS, the next one in registers on its way; few tiles, or a last round of few, are split
// along K over workgroups.  2048 x 8192 fp32: A 131 us and its join 10, A A 38 + 12, B X 204 = 1010 TFLOP/s of fp16 products.  4096 x 4096 bf16: A 88, A A
// 99, B X 168 = 815 TFLOP/s: the LDS reads of 64 x 64 a wave take as long as its matrix instructions.
// TILE 64, for the few workgroups of smaller ones, where a stage costs its latency.  B X: stages of 64 along K.  A and A A (KG = 4): stages of 128, two on
// their way in registers, their four steps of 32 shared out over four groups of four waves, which add their sums through LDS.  (Measured and not kept:
// fragments straight from memory, no LDS along K, 1.4 to 2 times slower; four waves with the whole tile and a step each, 3 - 8 % slower.)
// (Registers for two 128 x 128 workgroups a CU, or four of B X in 64 x 64: with three the 14-joint step takes 168 us instead of 160, with five it spills.)
template <int TERMS, int KIND, int TILE, int KG, typename OUT>
__global__ __launch_bounds__(256 * KG, KG > 1 ? 1 : TILE == 64 ? 4 : 2) void orth_gemm_kernel(OrthArgs g, OUT fin, int last) {
  constexpr int NT = 256 * KG;
  constexpr int KS = TILE == 128 ? (TERMS == 3 ? 32 : 64) : KG == 4 ? 128 : 64;        // K per stage
  constexpr int STAGES = TILE == 128 ? 2 : 1;
  constexpr int SIDE = TILE / 2, NF = SIDE / 16;                        // of a wave's part of the tile; 16 x 16 fragments a side
  constexpr int PLANES = TERMS == 3 ? 2 : 1;
  constexpr int OPB = TILE * KS * 2;                                    // bytes of one operand plane of a stage
  constexpr int UNITS = OPB / 16 / NT;                                  // 16-byte units per thread and plane
  constexpr int STAGE = 2 * PLANES * OPB;
  constexpr int CK = KS / 8, CT = TILE / 8;                             // 16-byte units of a row along K, and along the tile
  constexpr int SUMS = KG > 1 ? KG * TILE * TILE * 4 : 0;               // the groups' sums
  __shared__ __attribute__((aligned(16))) char lds[STAGES * STAGE > SUMS ? STAGES * STAGE : SUMS];
  int t = blockIdx.x, part = 0;
  const bool split_k = TILE == 128 && KIND != kApply && t >= g.whole;
  if (TILE == 128 && KIND != kApply) {
    // a die's workgroups: the same share of K of all tiles (parts in eighths), else neighbouring tiles
    if (split_k && !(g.parts & 7)) { const int v = t - g.whole; part = v % g.parts; t = g.whole + v / g.parts; }
    else if (split_k) {
      const int n = ((int)gridDim.x - g.whole) / g.parts, v = t - g.whole;
      part = v / n;
      t = g.whole + orth_die_order(v - part * n, n);
    } else t = orth_die_order(t, min(g.whole, (int)gridDim.x));
  }
  constexpr bool SHARED = TILE == 64 && KIND == kGram;
  // (64 x 64 tiles: neighbours on a die from 16 tiles a die on.  5 of 1031 x 517 fp32 265 -> 247 us; 700 x 1000, 66 tiles, would be 198 -> 206)
  if (TILE == 64 && KIND != kApply && !g.items && gridDim.x >= 128 && (KIND == kPoly || g.one.shares == 1)) t = orth_die_order(t, gridDim.x);
  if (SHARED && !g.items) { part = t % g.one.shares; t /= g.one.shares; }
  int tile, ti, tj; int4 entry;
  const OrthItem o = orth_item(g, t, tile, entry);
  if (SHARED && g.items) part = entry.w;
  const OrthWs w(o.Mp, o.Np);
  orth_place(KIND != kApply, tile, entry, o.Mp / TILE, o.Np / TILE, orth_band(TILE, o.Np / TILE), ti, tj);
  const int tid = threadIdx.x, lane = tid & 63, wid = (tid >> 6) & 3, group = tid >> 8;
  if constexpr (TILE == 64 && KIND == kPoly) {
    if (o.Mp <= kOrthNarrow) {
      orth_narrow_poly<TERMS>(g, o, w, ti, tj, lds);
      return;
    }
  }
  const int wp = (wid & 1) * SIDE, wq = (wid >> 1) * SIDE;              // this wave's part of the tile: entries j, rows i
  char* base = g.ws + o.ws;
  const half_t* X = reinterpret_cast<const half_t*>(base + w.x(g.buf));
  const half_t* A = reinterpret_cast<const half_t*>(base + w.a());
  const half_t* B = reinterpret_cast<const half_t*>(base + w.b());
  const half_t* Q = KIND == kGram ? X : KIND == kPoly ? A : B;
  const half_t* P = KIND == kPoly ? A : X;
  const long long qplane = KIND == kGram ? w.xplane : w.aplane, pplane = KIND == kPoly ? w.aplane : w.xplane;
  const int ldq = KIND == kGram ? o.Np : o.Mp, ldp = KIND == kPoly ? o.Mp : o.Np;
  const int K = KIND == kGram ? o.Np : o.Mp;                            // a multiple of 64

  // Staging.  A plane is [row][CK units of 16 bytes along K], the unit swizzled by the row, or (columns of X) [k][CT units], swizzled by k: so that the
  // sixteen rows of a fragment -- neighbours (Q), or four runs of four (P) --, or the four pieces of four rows of a transposing read, meet no bank twice.  Where K ends inside a stage the units beyond are loaded from inside and not used.
  constexpr int SETS = KG == 4 ? 2 : 1;                             // stages on their way in registers
  half8 rq[SETS][PLANES][UNITS], rp[SETS][PLANES][UNITS];
  const bool same = KIND != kApply && ti == tj;                         // both operands are the same rows
  const int pbase = same ? 0 : PLANES * OPB;
  auto ntq = [](int row) { return CK == 4 ? (row >> 2) & 3 : CK == 8 ? (row >> 1) & 7 : row & 15; };
  auto ntp = [](int row) { return CK == 4 ? (row >> 4) & 3 : CK == 8 ? ((row >> 1) & 1) | ((row >> 4) & 3) << 1 : (row & 3) | ((row >> 3) & 3) << 2; };
  auto trf = [](int k) { return TILE == 128 ? (k & 1) << 3 | ((k >> 1) & 1) : ((k >> 1) & 1) << 2; };
  auto load = [&](int k0, int set) {
    const int left = K - k0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int id = u * NT + tid, row = id / CK, c = KS > 64 ? min(id % CK, left / 8 - 1) : id % CK;
      const int kr = KS > 64 ? min(id / CT, left - 1) : id / CT;
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        rq[set][p][u] = *reinterpret_cast<const half8*>(Q + p * qplane + (long long)(ti * TILE + row) * ldq + k0 + c * 8);
        if constexpr (KIND == kApply)
          rp[set][p][u] = *reinterpret_cast<const half8*>(P + p * pplane + (long long)(k0 + kr) * ldp + tj * TILE + (id % CT) * 8);
        else if (!same)
          rp[set][p][u] = *reinterpret_cast<const half8*>(P + p * pplane + (long long)(tj * TILE + row) * ldp + k0 + c * 8);
      }
    }
  };
  auto store = [&](int stage, int set) {
    char* s = lds + stage * STAGE;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int id = u * NT + tid;
      const int row = id / CK, k = id / CT;
      const int aq = row * KS * 2 + (((id % CK) ^ ntq(row)) << 4);
      const int ap = KIND == kApply ? k * TILE * 2 + (((id % CT) ^ trf(k)) << 4) : row * KS * 2 + (((id % CK) ^ ntp(row)) << 4);
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        *reinterpret_cast<half8*>(s + p * OPB + aq) = rq[set][p][u];
        if (!same) *reinterpret_cast<half8*>(s + (PLANES + p) * OPB + ap) = rp[set][p][u];
      }
    }
  };
  const int li = lane & 15, lg = lane >> 4;
  auto frag_q = [&](const char* plane, int f, int kk) {
    const int row = wq + 16 * f + li;
    return *reinterpret_cast<const half8*>(plane + row * KS * 2 + (((kk * 4 + lg) ^ ntq(row)) << 4));
  };
  auto frag_p = [&](const char* plane, int f, int kk) {
    const int row = wp + 4 * NF * (li >> 2) + 4 * f + (li & 3);
    return *reinterpret_cast<const half8*>(plane + row * KS * 2 + (((kk * 4 + lg) ^ (same ? ntq(row) : ntp(row))) << 4));
  };
  auto frag_tr = [&](const char* plane, int f, int kk) {
    typedef __attribute__((address_space(3))) bf16x4* lptr;              // (the read moves 16-bit patterns, whatever they mean)
    const int k = kk * 32 + 8 * lg + (li >> 2), j = wp + 4 * NF * (li & 3) + 4 * f;
    const char* a0 = plane + k * TILE * 2 + (((j >> 3) ^ trf(k)) << 4) + ((j & 4) << 1);
    const half4 lo = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(a0)));
    const half4 hi = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(a0 + 4 * TILE * 2)));
    half8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) { r[e] = lo[e]; r[4 + e] = hi[e]; }
    return r;
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
        fq[p][f] = frag_q(s + p * OPB, f, kk);
        if constexpr (KIND == kApply) fp[p][f] = frag_tr(s + (PLANES + p) * OPB, f, kk);
        else fp[p][f] = frag_p(s + pbase + p * OPB, f, kk);
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

  // a group finishes ROWS fragment rows (16 rows i) of 4 NP neighbours
  constexpr int NP = NF * NF / KG < NF ? NF * NF / KG : NF, ROWS = NF * NF / KG / NP;
  static_assert(NP * ROWS * KG == NF * NF, "every group finishes as many fragments");
  const int q0 = NP < NF ? group * NP / NF : group * ROWS, p0 = NP < NF ? group * NP % NF : 0;
  OrthPair<4 * NP> beside[ROWS];
  int kb = 0, ke = K;
  if (split_k) { const int n = K / KS; kb = n * part / g.parts * KS; ke = n * (part + 1) / g.parts * KS; }
  if (SHARED) { const int n = (K + KS - 1) / KS; kb = n * part / o.shares * KS; ke = min(K, n * (part + 1) / o.shares * KS); }
  const int i0 = ti * TILE + wq + 16 * q0 + li, j0 = tj * TILE + wp + 4 * NF * lg + 4 * p0;
  if constexpr (STAGES == 2) {
    if (kb < ke) { load(kb, 0); store(0, 0); }
    __syncthreads();
    int stage = 0;
    for (int k0 = kb; k0 < ke; k0 += KS) {
      const bool more = k0 + KS < ke;
      if (more) load(k0 + KS, 0);
#pragma unroll
      for (int kk = 0; kk < KS / 32; ++kk) compute(lds + stage * STAGE, kk);
      if (more) store(stage ^ 1, 0);
      __syncthreads();
      stage ^= 1;
    }
  } else {
    load(kb, 0);
    if (SETS == 2 && kb + KS < ke) load(kb + KS, SETS - 1);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) beside[r] = orth_beside<KIND, 4 * NP>(g, o, w, i0 + 16 * r, j0);
    auto turn = [&](int k0, int set) {
      if (k0 > kb) __syncthreads();                                          // (everyone has read the stage before)
      store(0, set);
      __syncthreads();
      if (k0 + SETS * KS < ke) load(k0 + SETS * KS, set);
#pragma unroll
      for (int kk = 0; kk < KS / 32 / KG; ++kk)
        if (k0 + (group * (KS / 32 / KG) + kk) * 32 < ke) compute(lds, group * (KS / 32 / KG) + kk);
    };
    for (int k0 = kb; k0 < ke; k0 += SETS * KS) {
      turn(k0, 0);
      if (SETS == 2 && k0 + KS < ke) turn(k0 + KS, SETS - 1);
    }
  }

  if (split_k) {
    f32x4* s = g.slab + (long long)((t - g.whole) * g.parts + part) * (NF * NF * 256);
#pragma unroll
    for (int p = 0; p < NF; ++p)
#pragma unroll
      for (int q = 0; q < NF; ++q) s[(p * NF + q) * 256 + tid] = acc[p][q];
    return;
  }
  const bool mirror = KIND != kApply && ti != tj;
  // (all loads together: behind one another's stores they would cost a latency each; before the last stages, or beside the parameters of an update, they would
  // cost registers that are needed)
  constexpr bool TOGETHER = STAGES == 2 && !std::is_same<OUT, OrthUpdate>::value;
  if (TOGETHER) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) beside[r] = orth_beside<KIND, 4 * NP>(g, o, w, i0 + 16 * r, j0);
  }
  f32x4* sums = reinterpret_cast<f32x4*>(lds);
  if constexpr (KG > 1) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < NF; ++p)
#pragma unroll
      for (int q = 0; q < NF; ++q) sums[((p * NF + q) * KG + group) * 256 + wid * 64 + lane] = acc[p][q];
    __syncthreads();
  }
  // (the tile's other side: a wave's 64 x 64 block goes through LDS, where the transposing reads make 16 bytes along i of it)
  char* turn = lds + (wid & 3) * 16384;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float v[4 * NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      f32x4 a = acc[k][r];
      if constexpr (KG > 1) {
        const int f = (p0 + k) * NF + q0 + r;
        a = sums[f * KG * 256 + wid * 64 + lane];
#pragma unroll
        for (int u = 1; u < KG; ++u) a += sums[(f * KG + u) * 256 + wid * 64 + lane];
      }
      if constexpr (SHARED) {
        static_assert(NP == 1 && ROWS == 1, "a thread has one fragment");
        if (o.shares > 1 || o.Mp <= kOrthNarrow) {
          g.slab[orth_sums(g, o, t, ti, tj, part) * 1024 + tid] = a;
          return;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * k + e] = a[e];
    }
    const int i = i0 + 16 * r;
    if (STAGES == 2 && !TOGETHER) beside[r] = orth_beside<KIND, 4 * NP>(g, o, w, i, j0);
    const OrthPair<4 * NP> d = orth_finish<TERMS, KIND, 4 * NP, OUT>(g, o, w, fin, last, i, j0, v, beside[r]);
    if (!mirror) continue;
    if constexpr (TILE == 128) {
      // row i of the block: 128 bytes per plane, its 16-byte units swizzled
      const int row = 16 * r + li;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int at = row * 128 + (((2 * lg + k) ^ ((row >> 1) & 7)) << 4);
        *reinterpret_cast<Halves<8>*>(turn + at) = *reinterpret_cast<const Halves<8>*>(d.h.v + 8 * k);
        *reinterpret_cast<Halves<8>*>(turn + 8192 + at) = *reinterpret_cast<const Halves<8>*>(d.l.v + 8 * k);
      }
    } else orth_mirror<KIND, 4 * NP>(g, o, w, i, j0, d);
  }
  if constexpr (TILE == 128 && KIND != kApply) {
    if (mirror) {                                                       // (a wave's own block: its reads follow its writes)
      typedef __attribute__((address_space(3))) bf16x4* lptr;
      half_t* dst = reinterpret_cast<half_t*>(base + (KIND == kGram ? w.a() : w.b()));
#pragma unroll
      for (int plane = 0; plane < 2; ++plane)
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)
#pragma unroll
          for (int ib = 0; ib < 2; ++ib) {
            // lane (lg, li): entry jb 16 + li of the rows ib 32 + 8 lg ... + 7
            const int row = ib * 32 + 8 * lg + (li >> 2), j = jb * 16 + 4 * (li & 3);
            auto at = [&](int r) { return turn + plane * 8192 + r * 128 + (((j >> 3) ^ ((r >> 1) & 7)) << 4) + ((j & 4) << 1); };
            const half4 lo = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)at(row)));
            const half4 hi = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)at(row + 4)));
            half8 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = lo[e]; x[4 + e] = hi[e]; }
            *reinterpret_cast<half8*>(dst + plane * w.aplane + (long long)(tj * TILE + wp + jb * 16 + li) * o.Mp + ti * TILE + wq + ib * 32 + 8 * lg) = x;
          }
    }
  }
}

// the shared 64 x 64 tiles of A: the workgroup of a tile's first share adds all of them
template <int TERMS>
__global__ __launch_bounds__(1024) void orth_join_shared_kernel(OrthArgs g) {
  const int tid = threadIdx.x, lane = tid & 63, wid = (tid >> 6) & 3, group = tid >> 8;
  const int t = g.items ? blockIdx.x : blockIdx.x / g.one.shares;
  int tile, ti, tj; int4 entry;
  const OrthItem o = orth_item(g, t, tile, entry);
  if ((g.items ? entry.w : (int)blockIdx.x % g.one.shares) != 0) return;
  const OrthWs w(o.Mp, o.Np);
  orth_place(true, tile, entry, o.Mp / 64, o.Np / 64, 1, ti, tj);
  const f32x4* s = g.slab + orth_sums(g, o, t, ti, tj, 0) * 1024 + tid;
  f32x4 a = s[0];
  for (int u = 1; u < o.shares; ++u) a += s[u * 1024];
  const int i = ti * 64 + (wid >> 1) * 32 + 16 * (group >> 1) + (lane & 15), j = tj * 64 + (wid & 1) * 32 + 8 * (lane >> 4) + 4 * (group & 1);
  const float v[4] = {a[0], a[1], a[2], a[3]};
  const OrthPair<4> d = orth_finish<TERMS, kGram, 4, OrthNone>(g, o, w, OrthNone{}, 0, i, j, v, orth_beside<kGram, 4>(g, o, w, i, j));
  if (ti != tj) orth_mirror<kGram, 4>(g, o, w, i, j, d);
}

// the split 128 x 128 tiles of A or A A: a workgroup adds the parts of one of a tile's four fragment rows and finishes it
template <int TERMS, int KIND>
__global__ __launch_bounds__(256) void orth_join_kernel(OrthArgs g) {
  const int t = blockIdx.x >> 2, q = blockIdx.x & 3, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int tile, ti, tj; int4 entry;
  const OrthItem o = orth_item(g, g.whole + t, tile, entry);
  const OrthWs w(o.Mp, o.Np);
  orth_place(true, tile, entry, o.Mp / 128, o.Np / 128, 1, ti, tj);
  const int i = ti * 128 + (wid >> 1) * 64 + 16 * q + (lane & 15), j = tj * 128 + (wid & 1) * 64 + 16 * (lane >> 4);
  const OrthPair<16> beside = orth_beside<KIND, 16>(g, o, w, i, j);
  const f32x4* s = g.slab + (long long)t * g.parts * 4096 + q * 256 + tid;
  f32x4 a[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) a[p] = s[p * 1024];
  for (int k = 1; k < g.parts; ++k)
#pragma unroll
    for (int p = 0; p < 4; ++p) a[p] += s[(long long)k * 4096 + p * 1024];
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = a[e / 4][e % 4];
  const OrthPair<16> d = orth_finish<TERMS, KIND, 16, OrthNone>(g, o, w, OrthNone{}, 0, i, j, v, beside);
  if (ti != tj) orth_mirror<KIND, 16>(g, o, w, i, j, d);
}

// ---- small matrices: one workgroup of eight waves does a whole matrix, X in LDS for all steps.  MT x 16 rows (m <= 32 or 64), up to NCAP columns.
// Every product is all four products of the halves, for bf16 tensors too: what is left is latency, not arithmetic, and a sum this short loses less than
// lo lo: 16 x 40 and 30 x 800 have 0.75 of the error without it, 1 x 7 a seventh, in the same time.
//   A: a wave pair per quarter of K, each wave half of the 16 x 16 tiles on and above the diagonal; the quarters are added through LDS.
//   B + a I: two tiles a wave, written over A.      X: a wave takes 16 columns at a time, (B + a I) in registers, and writes them in place.
template <int MT> struct OrthTri;                       // the tiles (p, q), p <= q, of the two waves of a pair
template <> struct OrthTri<4> {
  static constexpr int n[2] = {5, 5}, p[2][5] = {{0, 0, 0, 0, 1}, {1, 1, 2, 2, 3}}, q[2][5] = {{0, 1, 2, 3, 1}, {2, 3, 2, 3, 3}};
};
template <> struct OrthTri<2> {
  static constexpr int n[2] = {2, 1}, p[2][2] = {{0, 0}, {1, 1}}, q[2][2] = {{0, 1}, {1, 1}};
};

template <int MT, int NCAP, typename SRC, typename OUT>
__global__ __launch_bounds__(512) void orth_small_kernel(OrthArgs g, SRC src, OUT fin, int steps) {
  typedef OrthTri<MT> Tri;
  constexpr int MP = 16 * MT, KK = MP / 32, TRI = Tri::n[0] + Tri::n[1];
  constexpr int REGION = 3 * TRI * 1024 > MP * MP * 4 ? 3 * TRI * 1024 : MP * MP * 4;      // A or B, or the quarters' sums
  __shared__ __attribute__((aligned(16))) char lds[MP * NCAP * 4 + REGION];
  __shared__ double red[8];
  int t; int4 tile;
  const OrthItem o = orth_item(g, blockIdx.x, t, tile);
  // (the wave's number as a scalar: branches on it are jumps; as a lane's value the phases of A below spill three registers)
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, lg = lane >> 4;
  const bool tall = o.rows > o.cols;
  const int m = tall ? o.cols : o.rows, n = tall ? o.rows : o.cols;
  const int NP = (n + 63) & ~63;                        // <= NCAP
  const int xplane = MP * NP * 2;                       // bytes
  constexpr int aplane = MP * MP * 2;
  char* X = lds;
  char* R = lds + MP * NCAP * 4;
  // rows are NP * 2 (a multiple of 128) and MP * 2 bytes long, their 16-byte units swizzled by the row
  const bool odd = (NP & 64) != 0;
  auto xat = [&](int row, int unit) { return row * NP * 2 + ((unit ^ (odd ? (row >> 1) & 7 : row & 7)) << 4); };
  auto aat = [&](int row, int unit) { return row * MP * 2 + ((unit ^ ((row >> 1) & (MP / 8 - 1))) << 4); };

  // |G|, then X0: the source is read once, all of a thread's loads under way together: four neighbours of a row at a time, number tid + 512 k
  for (int k = tid * 16; k < 2 * xplane; k += 512 * 16) *reinterpret_cast<uint4*>(X + k) = uint4{0, 0, 0, 0};
  constexpr int PER = MP * NCAP / 2048, RUN = PER < 4 ? PER : 4;
  const int wide = (o.cols + 3) >> 2, quads = o.rows * wide, dr = 512 / wide, dc = 512 % wide, r0 = tid / wide;
  const long long ld = src.stride(o);
  float v[PER][4];
  auto sweep = [&](auto&& use) {                        // (r, c): the row and the first column of the four
    int r = r0, c = tid - r0 * wide;
#pragma unroll
    for (int k0 = 0; k0 < PER; k0 += RUN)
      if (k0 * 512 < quads) {
#pragma unroll
        for (int k = k0; k < k0 + RUN; ++k) {
          use(v[k], r, 4 * c);
          r += dr; c += dc;
          if (c >= wide) { c -= wide; ++r; }
        }
      }
  };
  if (o.cols & 3) {
    sweep([&](float (&q)[4], int r, int c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = src.one(o, min(r, o.rows - 1) * ld + min(c + e, o.cols - 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = r < o.rows && c + e < o.cols ? q[e] : 0.f;
    });
  } else {
    sweep([&](float (&q)[4], int r, int c) {
      src.quad(o, min(r, o.rows - 1) * ld + c, q);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = r < o.rows ? q[e] : 0.f;
    });
  }
  double s = 0.0;
  sweep([&](float (&q)[4], int, int) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s += (double)q[e] * q[e];
  });
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if (lane == 0) red[wid] = s;
  __syncthreads();
  s = ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
  const double inv = 1.0 / (sqrt(s) + (double)g.eps);
  sweep([&](float (&q)[4], int r, int c) {
    if (r >= o.rows) return;
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) { half_t a, b; split((float)((double)q[e] * inv), a, b); h[e] = a; l[e] = b; }
    if (!tall) {                                        // (zeros up to the fourth: NP is a multiple of 64)
      const int at = xat(r, c >> 3) + (c & 7) * 2;
      *reinterpret_cast<half4*>(X + at) = h;
      *reinterpret_cast<half4*>(X + xplane + at) = l;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {                       // (rows beyond m are zero: MP is a multiple of 16)
      const int at = xat(c + e, r >> 3) + (r & 7) * 2;
      *reinterpret_cast<half_t*>(X + at) = h[e];
      *reinterpret_cast<half_t*>(X + xplane + at) = l[e];
    }
  });
  __syncthreads();

  auto mfma4 = [](const half8 (&p)[2], const half8 (&q)[2], f32x4 acc) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[1], q[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[1], q[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[0], q[1], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(p[0], q[0], acc, 0, 0, 0);
  };
  auto put4 = [&](char* at, int plane, const float (&v)[4], half4& h, half4& l) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { half_t a, b; split(v[e], a, b); h[e] = a; l[e] = b; }
    *reinterpret_cast<half4*>(at) = h;
    *reinterpret_cast<half4*>(at + plane) = l;
  };
  // A, in phases between the workgroup's barriers: the waves of a pair have tiles of their own, the barriers are everyone's
  constexpr int MOST = Tri::n[0] > Tri::n[1] ? Tri::n[0] : Tri::n[1];
  f32x4 sums[MOST];
  const int quarter = wid >> 1;
  auto halves = [&](auto&& phase) {
    if (wid & 1) phase(std::integral_constant<int, 1>{});
    else phase(std::integral_constant<int, 0>{});
  };
  // tile k is finished by the wave of quarter k & 3: the other three leave it their sums
  auto slot = [&](int h, int u, int k) { return reinterpret_cast<f32x4*>(R + ((u * TRI + h * Tri::n[0] + k) * 64 + lane) * 16); };
  auto gram_sums = [&](auto half) {
    constexpr int H = decltype(half)::value, NT = Tri::n[H];
#pragma unroll
    for (int k = 0; k < NT; ++k) sums[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int ks = quarter; ks < NP / 32; ks += 4) {
      half8 f[MT][2];
#pragma unroll
      for (int r = Tri::p[H][0]; r < MT; ++r)
#pragma unroll
        for (int p = 0; p < 2; ++p) f[r][p] = *reinterpret_cast<const half8*>(X + p * xplane + xat(16 * r + li, ks * 4 + lg));
#pragma unroll
      for (int k = 0; k < NT; ++k) sums[k] = mfma4(f[Tri::p[H][k]], f[Tri::q[H][k]], sums[k]);
    }
#pragma unroll
    for (int k = 0; k < NT; ++k)
      if ((k & 3) != quarter) *slot(H, (quarter - k - 1) & 3, k) = sums[k];
  };
  auto gram_add = [&](auto half) {
    constexpr int H = decltype(half)::value, NT = Tri::n[H];
#pragma unroll
    for (int k = 0; k < NT; ++k)
      if ((k & 3) == quarter)
#pragma unroll
        for (int u = 0; u < 3; ++u) sums[k] += *slot(H, u, k);
  };
  auto gram_put = [&](auto half) {
    constexpr int H = decltype(half)::value, NT = Tri::n[H];
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      if ((k & 3) != quarter) continue;
      const int i = 16 * Tri::q[H][k] + li, j = 16 * Tri::p[H][k] + 4 * lg;
      float v[4];
      half4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = sums[k][e] * (kOrthInv * kOrthInv);
      put4(R + aat(i, j >> 3) + (j & 7) * 2, aplane, v, h, l);
      if (Tri::p[H][k] != Tri::q[H][k]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = aat(j + e, i >> 3) + (i & 7) * 2;
          *reinterpret_cast<half_t*>(R + at) = h[e];
          *reinterpret_cast<half_t*>(R + aplane + at) = l[e];
        }
      }
    }
  };
  for (int step = 0; step < steps; ++step) {
    halves(gram_sums);
    __syncthreads();
    halves(gram_add);
    __syncthreads();
    halves(gram_put);
    __syncthreads();
    // B + a I
    constexpr int PW = MT == 4 ? 2 : 1;
    const int q = MT == 4 ? wid >> 1 : (wid >> 1) & 1, p0 = MT == 4 ? 2 * (wid & 1) : wid & 1;
    float v[PW][4];
    if (MT == 4 || wid < 4) {
      f32x4 acc[PW];
#pragma unroll
      for (int k = 0; k < PW; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        half8 fq[2], fp[PW][2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          fq[p] = *reinterpret_cast<const half8*>(R + p * aplane + aat(16 * q + li, kk * 4 + lg));
#pragma unroll
          for (int k = 0; k < PW; ++k) fp[k][p] = *reinterpret_cast<const half8*>(R + p * aplane + aat(16 * (p0 + k) + li, kk * 4 + lg));
        }
#pragma unroll
        for (int k = 0; k < PW; ++k) acc[k] = mfma4(fp[k], fq, acc[k]);
      }
#pragma unroll
      for (int k = 0; k < PW; ++k) {
        const int i = 16 * q + li, j = 16 * (p0 + k) + 4 * lg, at = aat(i, j >> 3) + (j & 7) * 2;
        const half4 h = *reinterpret_cast<const half4*>(R + at), l = *reinterpret_cast<const half4*>(R + aplane + at);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[k][e] = fmaf(g.c, acc[k][e] * (kOrthInv * kOrthInv), g.b * (((float)h[e] + (float)l[e]) * kOrthInv)) + (i == j + e ? g.a : 0.f);
      }
    }
    __syncthreads();
    if (MT == 4 || wid < 4) {
#pragma unroll
      for (int k = 0; k < PW; ++k) {
        const int i = 16 * q + li, j = 16 * (p0 + k) + 4 * lg;
        half4 h, l;
        put4(R + aat(i, j >> 3) + (j & 7) * 2, aplane, v[k], h, l);
      }
    }
    __syncthreads();
    // X
    half8 b[KK][MT][2];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int p = 0; p < 2; ++p) b[kk][r][p] = *reinterpret_cast<const half8*>(R + p * aplane + aat(16 * r + li, kk * 4 + lg));
    half8 f[KK][2], next[KK][2];
    auto columns = [&](int jb, half8 (&f)[KK][2]) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          typedef __attribute__((address_space(3))) bf16x4* lptr;
          const int k = kk * 32 + 8 * lg + (li >> 2), j = jb * 16 + 4 * (li & 3);
          const half4 lo = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(X + p * xplane + xat(k, j >> 3) + (j & 7) * 2)));
          const half4 hi = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lptr)(X + p * xplane + xat(k + 4, j >> 3) + (j & 7) * 2)));
#pragma unroll
          for (int e = 0; e < 4; ++e) { f[kk][p][e] = lo[e]; f[kk][p][4 + e] = hi[e]; }
        }
    };
    if (wid < NP / 16) columns(wid, f);
    for (int jb = wid; jb < NP / 16; jb += 8) {
      if (jb + 8 < NP / 16) columns(jb + 8, next);
      f32x4 acc[MT];
#pragma unroll
      for (int r = 0; r < MT; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int r = 0; r < MT; ++r) acc[r] = mfma4(f[kk], b[kk][r], acc[r]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int p = 0; p < 2; ++p) f[kk][p] = next[kk][p];
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        const int i = 16 * r + li, j = jb * 16 + 4 * lg;
        float x[4];
        half4 h, l;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[r][e] * (kOrthInv * kOrthInv);
        if (step < steps - 1) put4(X + xat(i, j >> 3) + (j & 7) * 2, xplane, x, h, l);
        else fin.put(o, tall, m, n, i, j, x);
      }
    }
    __syncthreads();
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
  o.shares = 1;
  return o;
}
// tiles of A or A A (symmetric), and of B X
static long long orth_sym_tiles(const OrthItem& o, int tile) { const long long t = o.Mp / tile; return t * (t + 1) / 2; }
static long long orth_apply_tiles(const OrthItem& o, int tile) { return (long long)(o.Mp / tile) * (o.Np / tile); }

// 128 x 128 tiles move half the bytes per product of 64 x 64 ones, and pad more.  They pay from six tiles a side on, where B X has a tile per CU, by about
// m / 8192 of the time; that is compared with what padding and a last round of B X (512 places) cost.  In 128 / 64: 2048 x 2048 fp32 854 / 1086 us,
// 4000 x 8000 bf16 3495 / 5462, 2 of 1000 x 3000 fp32 630 / 728, 1024 x 4096 487 / 521; 1300 x 6000 (517 tiles) 1021 / 878, 900 x 8000 728 / 652,
// 4 of 640 x 2560 496 / 448, 16 of 400 x 1600 746 / 556, 64 of 128 x 1152 348 / 250.
constexpr int kOrthWideSide = 705, kOrthWideTiles = 256;
static double orth_cost(int rows, int cols, long long batch, int tile) {
  const OrthItem o = orth_make(rows, cols, tile);
  long long t = batch * orth_apply_tiles(o, tile);
  if (tile == 128 && t > 512) t = (t + 511) / 512 * 512;
  const double area = (tile / 64) * (tile / 64);
  return area * ((double)t * o.Mp + (double)batch * orth_sym_tiles(o, tile) * (o.Np + (double)o.Mp));
}
static int orth_tile(int rows, int cols, long long batch) {
  const int m = std::min(rows, cols);
  if (m < kOrthWideSide || batch * orth_apply_tiles(orth_make(rows, cols, 128), 128) < kOrthWideTiles) return 64;
  return orth_cost(rows, cols, batch, 128) * 8192 <= orth_cost(rows, cols, batch, 64) * (8192.0 + m) ? 128 : 64;
}

// X of such a matrix fits the LDS of one CU.  In one workgroup a matrix / by launches: 64 x 128 fp32 21 / 78 us, 64 x 512 46 / 90, 32 x 1024 38 / 92,
// 600 of 64 x 500 bf16 142 / 374, 2000 of 64 x 128 bf16 165 / 470.
static bool orth_is_small(int rows, int cols) {
  const long long m = std::min(rows, cols), n = (std::max(rows, cols) + 63ll) / 64 * 64;
  return m <= 32 ? n <= 1024 : m <= 64 && n <= 512;
}

struct OrthCounts { long long n[5]; int gram_k, poly_k; };       // workgroups of the norm, pack, A A, B X and A launches; K of the symmetric ones

// 64 x 64 tiles of A: a workgroup has no more of K than a CU on average (`mean`), but 512 at least, and the rest of its tile is other workgroups'.  The
// sums of a narrow matrix go into A A as they are; others need a launch that joins them, which has to save ten stages of 128.  fp32, unshared / shared:
// 20 x 8000 342 / 117 us, 13 of 128 x 1152 132 / 116, 200 x 8000 461 / 193, 4 of 300 x 2000 243 / 201.  (In shares of 256 the first is 132; more than 32
// take one workgroup too long to add.  The last workgroup to arrive adding them cost up to 170 us a launch: every one has to write back and drop its L2.)
static int orth_shares(const OrthItem& o, double mean) {
  const int shares = std::max(1, std::min(32, (int)(o.Np / std::max(512.0, mean) + 0.5)));
  return o.Mp <= kOrthNarrow || o.Np - o.Np / shares >= 1280 ? shares : 1;
}

// How the tiles of a symmetric product share out over 512 places (two workgroups of 128 x 128 tiles per CU): a launch, or its last round, that fills at
// most three quarters of them is split along K, into parts of 256 at least.  4096 x 4096, 528 tiles: 16 of them alone cost a round as long as the first.
// (Dealing the stages out evenly instead was slower, 198 against 160 us for 2048 x 8192: workgroups that start at different k share no rows in the L2s.)
struct OrthSplit { int whole, parts; };
static OrthSplit orth_split(long long tiles, int K) {
  const long long rest = tiles % 512;
  long long parts = rest ? std::min<long long>(512 / rest, K / 256) : 1;
  if (parts > 8) parts &= ~7ll;                          // (in eighths: a chip die's workgroups then share a part's rows in its L2)
  if (rest == 0 || rest > 384 || parts < 2) return {(int)tiles, 1};
  return {(int)(tiles - rest), (int)parts};
}
static long long orth_slab_bytes(long long tiles, int gram_k, int poly_k) {
  long long most = 0;
  for (const int K : {gram_k, poly_k}) {
    const OrthSplit s = orth_split(tiles, K);
    most = std::max(most, (tiles - s.whole) * s.parts * 65536);
  }
  return most;
}

template <int TERMS, int TILE, typename SRC, typename OUT>
static int orth_run(const OrthArgs& g, const OrthCounts& n, const int4* const (&lists)[5], const SRC& src, const OUT& out, int steps, const int (&per)[5],
                    hipStream_t s) {
  const dim3 b(256);
  constexpr int KG = TILE == 64 ? 4 : 1;
  auto with = [&](int k, int buf) { OrthArgs h = g; h.tiles = lists[k]; h.per = per[k]; h.buf = buf; h.whole = 0x7fffffff; h.parts = 1; return h; };
  hipLaunchKernelGGL((orth_norm_kernel<SRC>), dim3((unsigned)n.n[0]), b, 0, s, with(0, 0), src);
  hipLaunchKernelGGL((orth_pack_kernel<SRC>), dim3((unsigned)n.n[1]), b, 0, s, with(1, 0), src);
  auto symmetric = [&](auto kind, int K, int buf) {
    constexpr int KIND = decltype(kind)::value;
    constexpr int LIST = KIND == kGram ? 4 : 2;
    OrthArgs h = with(LIST, buf);
    long long blocks = n.n[LIST];
    if constexpr (TILE == 128) {
      const OrthSplit sp = orth_split(n.n[2], K);
      h.whole = sp.whole; h.parts = sp.parts;
      blocks = sp.whole + (n.n[2] - sp.whole) * sp.parts;
    }
    hipLaunchKernelGGL((orth_gemm_kernel<TERMS, KIND, TILE, KG, OrthNone>), dim3((unsigned)blocks), dim3(256 * KG), 0, s, h, OrthNone{}, 0);
    if constexpr (TILE == 64 && KIND == kGram) {
      if (h.shared) hipLaunchKernelGGL((orth_join_shared_kernel<TERMS>), dim3((unsigned)h.shared), dim3(1024), 0, s, h);
    }
    if constexpr (TILE == 128) {
      if (h.whole < n.n[2])
        hipLaunchKernelGGL((orth_join_kernel<TERMS, KIND>), dim3((unsigned)(4 * (n.n[2] - h.whole))), b, 0, s, h);
    }
  };
  for (int k = 0; k < steps; ++k) {
    symmetric(std::integral_constant<int, kGram>{}, n.gram_k, k & 1);
    symmetric(std::integral_constant<int, kPoly>{}, n.poly_k, k & 1);
    hipLaunchKernelGGL((orth_gemm_kernel<TERMS, kApply, TILE, 1, OUT>), dim3((unsigned)n.n[3]), b, 0, s, with(3, k & 1), out, k == steps - 1);
  }
  return (int)hipGetLastError();
}

constexpr int kOrthMaxSide = 1 << 20;
constexpr int kOrthMaxSteps = 64;
constexpr long long kOrthMaxBlocks = 0xffffffffll / 1024;         // a launch has at most 2^32 - 1 threads

// Every entry that is stored as a pair has to stay below 65504 / 4096 = 15.99.  The singular values of X0 fill [0, 1]; those of the next X are
// s |a + b s^2 + c s^4|, and A, B and (in one workgroup) B + a I have s^2, b s^2 + c s^4 and a more than that.  A continuous odd map takes [-s, s] to
// [-m, m], so the largest ones are followed exactly (0.2 % a step are left for the roundings); the last X is not stored.
constexpr double kOrthLargest = 15.9;
static double orth_quadratic(double k, double b, double c, double u) {         // max |k + b t + c t^2| over 0 <= t <= u
  const double m = std::max(fabs(k), fabs(k + u * (b + c * u))), t = -b / (2 * c);                 // (c = 0: no number in between)
  return t > 0.0 && t < u ? std::max(m, fabs(k + t * (b + c * t))) : m;
}
static bool orth_range_ok(int steps, double a, double b, double c) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double s = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double u = s * s;
    if (!(u < kOrthLargest) || !(orth_quadratic(0.0, b, c, u) < kOrthLargest) || !(orth_quadratic(a, b, c, u) < kOrthLargest)) return false;
    auto next = [&](double t) { return sqrt(t) * fabs(a + t * (b + c * t)); };
    double m = next(u);
    // where the map turns: a + 3 b t + 5 c t^2 = 0 (its roots without a difference of near numbers, c = 0 included)
    const double disc = 9 * b * b - 20 * a * c, q = -0.5 * (3 * b + (b < 0.0 ? -1.0 : 1.0) * sqrt(std::max(disc, 0.0)));
    if (disc >= 0.0)
      for (const double t : {q / (5 * c), a / q})
        if (t > 0.0 && t < u) m = std::max(m, next(t));
    s = 1.002 * m;
  }
  return true;
}

static bool orth_shape_ok(long long rows, long long cols) {
  // (a matrix of up to 2^31 entries: tile counts and the entries of a plane's row stay in 32 bits, offsets are 64)
  return rows >= 1 && cols >= 1 && rows <= kOrthMaxSide && cols <= kOrthMaxSide && rows * cols <= 0x7fffffffll;
}

}  // namespace pwr

using namespace pwr;

extern "C" int pwr_orthogonalize_range(int steps, float a, float b, float c) {
  if (steps < 1 || steps > kOrthMaxSteps) return PWR_EINVAL;
  return orth_range_ok(steps, a, b, c) ? 0 : PWR_EUNSUPPORTED;
}

extern "C" size_t pwr_orthogonalize_workspace_bytes(int rows, int cols, long long batch) {
  if (batch <= 0 || !orth_shape_ok(rows, cols)) return 0;
  if (orth_is_small(rows, cols)) return 256;
  const int tile = orth_tile(rows, cols, batch);
  const OrthItem o = orth_make(rows, cols, tile);
  const long long tiles = batch * orth_sym_tiles(o, tile), shares = orth_shares(o, tiles * (double)o.Np / 256);
  const long long sums = tile == 128 ? orth_slab_bytes(tiles, o.Np, o.Mp) : shares > 1 || o.Mp <= kOrthNarrow ? tiles * shares * 16384 : 0;
  return (size_t)(batch * orth_ws_bytes(rows, cols, o.Mp, o.Np) + sums);
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
  const long long sym = orth_sym_tiles(g.one, tile);
  const long long per[5] = {orth_parts(rows, cols), (long long)(g.one.Mp / 64) * (g.one.Np / 64), sym, orth_apply_tiles(g.one, tile), sym};
  const int shares = g.one.shares = tile == 64 ? orth_shares(g.one, batch * sym * (double)g.one.Np / 256) : 1;
  g.one.first = (int)(sym * shares);
  const OrthCounts n = {{batch * per[0], batch * per[1], batch * sym, batch * per[3], batch * sym * shares}, g.one.Np, g.one.Mp};
  for (const long long k : n.n)
    if (k > kOrthMaxBlocks) return PWR_EUNSUPPORTED;
  g.shared = shares > 1 && g.one.Mp > kOrthNarrow ? (int)n.n[4] : 0;
  g.slab = (f32x4*)(g.ws + batch * g.ws_stride);
  const int4* const lists[5] = {};
  const int iper[5] = {(int)per[0], (int)per[1], (int)per[2], (int)per[3], (int)per[4]};
  g.src_stride = x_batch;
  g.dst_stride = (long long)rows * cols;
  const OrthTensor<T> src = {(const T*)x, x_ld};
  const OrthOut<T> dst = {(T*)out, cols};
  if (orth_is_small(rows, cols)) {
    g.per = 1;
    const dim3 grid((unsigned)batch), block(512);
    const int m = std::min(rows, cols), np = up(std::max(rows, cols), 64);
    if (m <= 32 && np <= 256) hipLaunchKernelGGL((orth_small_kernel<2, 256, OrthTensor<T>, OrthOut<T>>), grid, block, 0, s, g, src, dst, steps);
    else if (m <= 32) hipLaunchKernelGGL((orth_small_kernel<2, 1024, OrthTensor<T>, OrthOut<T>>), grid, block, 0, s, g, src, dst, steps);
    else if (np <= 128) hipLaunchKernelGGL((orth_small_kernel<4, 128, OrthTensor<T>, OrthOut<T>>), grid, block, 0, s, g, src, dst, steps);
    else hipLaunchKernelGGL((orth_small_kernel<4, 512, OrthTensor<T>, OrthOut<T>>), grid, block, 0, s, g, src, dst, steps);
    return (int)hipGetLastError();
  }
  return tile == 128 ? orth_run<TERMS, 128>(g, n, lists, src, dst, steps, iper, s) : orth_run<TERMS, 64>(g, n, lists, src, dst, steps, iper, s);
}

extern "C" int pwr_orthogonalize(const void* x, long long x_batch_stride, long long x_row_stride, void* out, int rows, int cols, long long batch,
                                 int dtype, int steps, float a, float b, float c, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch == 0) return 0;
  if (!x || !out || batch < 0 || x_batch_stride < 0 || x_row_stride < 0 || steps < 1 || steps > kOrthMaxSteps || !(eps >= 0.f)) return PWR_EINVAL;
  if (dtype != PWR_F32 && dtype != PWR_BF16) return PWR_EINVAL;
  if (!orth_shape_ok(rows, cols)) return rows < 1 || cols < 1 ? PWR_EINVAL : PWR_EUNSUPPORTED;
  if (!orth_range_ok(steps, a, b, c)) return PWR_EUNSUPPORTED;
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
  unsigned long long magic, bytes, ws_bytes, slab;
  int items, tile, gram_k, poly_k, shared, pad;
  long long n[5], rest;                  // workgroups of the norm, pack, A A, B X and A launches; of the rest
  long long at_items, at_list[5], at_rest;
};
constexpr unsigned long long kMuonMagic = 0x32304e4f554d5750ull;

// A list is worked on in the tile that most of its products want (in units of a 64 x 64 x 64 block), after orth_tile, padding aside.  A step in 128 / 64:
// 4 of 2048 x 2048 2347 / 3673 us, 12 of 1024 x 4096 3241 / 4143, 12 of 1024 x 1024 1106 / 1397, 4 of 768 x 3000 690 / 747; half of the work in one
// 2048 x 2048, the rest in 60 of 256 x 2304, 2053 / 1982; a list of 1000 x 2100, 2500 x 900, 1000 x 1000 and small ones 644 / 620.
int muon_tile(const std::vector<OrthItem>& v) {
  double wide = 0, all = 0;
  long long tiles = 0;
  for (const OrthItem& k : v) {
    const OrthItem o = orth_make(k.rows, k.cols, 64);
    const double m = o.Mp / 64, n = o.Np / 64, c = m * m * (2 * n + m);
    all += c;
    if (std::min(k.rows, k.cols) >= kOrthWideSide) { wide += c; tiles += orth_apply_tiles(orth_make(k.rows, k.cols, 128), 128); }
  }
  return 2 * wide >= all && tiles >= kOrthWideTiles ? 128 : 64;
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
  h.tile = muon_tile(items);
  long long ws = 0;
  double k_sum = 0;
  bool sums = false;
  for (OrthItem& o : items) {
    const OrthItem q = orth_make(o.rows, o.cols, h.tile);
    o.Mp = q.Mp; o.Np = q.Np;
    k_sum += orth_sym_tiles(o, h.tile) * (double)o.Np;
  }
  for (OrthItem& o : items) {
    o.shares = h.tile == 64 ? orth_shares(o, k_sum / 256) : 1;
    o.gain = sqrtf((float)std::max(o.rows, o.cols));
    o.ws = ws;
    ws += orth_ws_bytes(o.rows, o.cols, o.Mp, o.Np);
    h.n[0] += orth_parts(o.rows, o.cols);
    h.n[1] += (long long)(o.Mp / 64) * (o.Np / 64);
    h.n[2] += orth_sym_tiles(o, h.tile);
    h.n[3] += orth_apply_tiles(o, h.tile);
    h.n[4] += orth_sym_tiles(o, h.tile) * o.shares;
    if (o.shares > 1 && o.Mp > kOrthNarrow) h.shared += (int)(orth_sym_tiles(o, h.tile) * o.shares);
    sums = sums || o.shares > 1 || o.Mp <= kOrthNarrow;
    h.gram_k = std::max(h.gram_k, o.Np);
    h.poly_k = std::max(h.poly_k, o.Mp);
  }
  h.slab = ws;
  h.ws_bytes = ws + (h.tile == 128 ? orth_slab_bytes(h.n[2], h.gram_k, h.poly_k) : sums ? h.n[4] * 16384 : 0);
  h.rest = (long long)rest.size();
  long long at = (sizeof(MuonHead) + 255) / 256 * 256;
  auto take = [&](long long bytes) { const long long r = at; at += (bytes + 255) / 256 * 256; return r; };
  h.at_items = take(h.items * (long long)sizeof(OrthItem));
  for (int k = 0; k < 5; ++k) h.at_list[k] = take(h.n[k] * (long long)sizeof(int4));
  h.at_rest = take(h.rest * (long long)sizeof(longlong2));
  h.bytes = at;
  for (int k = 0; k < 5; ++k)
    if (h.n[k] > kOrthMaxBlocks) return false;
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
  // The longest sums first (of A: the longest rows; of A A and B X: the most rows), so that a launch does not end on them; of A the tiles with a
  // launch that joins them are in front.
  std::vector<int> by_k(h.items), by_m(h.items);
  auto joined = [](const OrthItem& o) { return o.shares > 1 && o.Mp > kOrthNarrow; };
  for (int k = 0; k < h.items; ++k) by_k[k] = by_m[k] = k;
  std::stable_sort(by_k.begin(), by_k.end(), [&](int p, int q) {
    const bool jp = joined(items[p]), jq = joined(items[q]);
    return jp != jq ? jp : items[p].Np > items[q].Np;
  });
  std::stable_sort(by_m.begin(), by_m.end(), [&](int p, int q) { return items[p].Mp > items[q].Mp; });
  std::vector<int4> list[5];
  for (int k = 0; k < h.items; ++k) {
    const OrthItem& o = items[k];
    for (int t = 0; t < orth_parts(o.rows, o.cols); ++t) list[0].push_back(int4{k, t, 0, 0});
    for (int i = 0; i < o.Mp / 64; ++i)
      for (int j = 0; j < o.Np / 64; ++j) list[1].push_back(int4{k, i, j, 0});
  }
  // Tiles of equally long sums go to the dies in runs of neighbours (64 x 64 tiles, four a die or more; wide ones: see the kernel), so that a
  // die reads few matrices.  The step of the 42-joint network with 256 features 515 -> 479 us, 224 features 455 -> 424.
  auto deal = [&](std::vector<int4>& v, size_t from) {
    const size_t n = v.size() - from;
    if (h.tile != 64 || n < 32) return;
    const std::vector<int4> in(v.begin() + from, v.end());
    size_t next = 0;
    for (size_t die = 0; die < 8; ++die)
      for (size_t p = from + (die + 8 - from % 8) % 8; p < v.size(); p += 8) v[p] = in[next++];
  };
  size_t from = 0;
  for (size_t q = 0; q < by_m.size(); ++q) {
    const int k = by_m[q];
    const OrthItem& o = items[k];
    for (int j = 0; j < o.Mp / h.tile; ++j)
      for (int i = 0; i <= j; ++i) list[2].push_back(int4{k, i, j, 0});
    if (q + 1 == by_m.size() || items[by_m[q + 1]].Mp != o.Mp) { deal(list[2], from); from = list[2].size(); }
    const int nj = o.Np / h.tile, band = orth_band(h.tile, nj);
    for (int j0 = 0; j0 < nj; j0 += band)
      for (int i = 0; i < o.Mp / h.tile; ++i)
        for (int j = j0; j < std::min(nj, j0 + band); ++j) list[3].push_back(int4{k, i, j, 0});
  }
  from = 0;
  for (size_t q = 0; q < by_k.size(); ++q) {
    const int k = by_k[q];
    OrthItem& o = items[k];
    o.first = (int)list[4].size();
    for (int j = 0; j < o.Mp / h.tile; ++j)
      for (int i = 0; i <= j; ++i)
        for (int u = 0; u < o.shares; ++u) list[4].push_back(int4{k, i, j, u});
    const bool more = q + 1 < by_k.size();
    if (!more || items[by_k[q + 1]].Np != o.Np || joined(items[by_k[q + 1]]) != joined(o)) { deal(list[4], from); from = list[4].size(); }
  }
  memcpy(d + h.at_items, items.data(), items.size() * sizeof(OrthItem));
  for (int k = 0; k < 5; ++k) memcpy(d + h.at_list[k], list[k].data(), list[k].size() * sizeof(int4));
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
  if (h->items && !orth_range_ok(ns_steps, a, b, c)) return PWR_EUNSUPPORTED;
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
  const OrthCounts n = {{h->n[0], h->n[1], h->n[2], h->n[3], h->n[4]}, h->gram_k, h->poly_k};
  ga.shared = h->shared;
  ga.slab = (f32x4*)(ga.ws + h->slab);
  const int4* lists[5];
  for (int k = 0; k < 5; ++k) lists[k] = (const int4*)(d + h->at_list[k]);
  const int4* const (&ls)[5] = lists;
  const int per[5] = {};
  const OrthMomentum src = {g, buf, momentum, grad_scale, nesterov};
  const OrthUpdate dst = {p, keep, lr * update_rms};
  return h->tile == 128 ? orth_run<3, 128>(ga, n, ls, src, dst, ns_steps, per, s) : orth_run<3, 64>(ga, n, ls, src, dst, ns_steps, per, s);
}
