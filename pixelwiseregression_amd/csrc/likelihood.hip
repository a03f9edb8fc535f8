// The log likelihood of one pixel per heat map, the map's entropy and its K most likely pixels, and the gradient of the first two.
//
// A heat map is the categorical distribution the decoder reads its joint from (/root/reference/model.py:83-85): p = softmax_i(s), s_i = w_j z_i
// over the pixels i a mask allows.  With M = max s, c = the number of pixels that reach it, r = sum_{s_i < M} exp(s_i - M) and
// q = sum exp(s_i - M)(s_i - M):
//     log p_i = (s_i - M) - log(c + r),        entropy = log(c + r) - q / (c + r),
// forward, and with the upstream gradients g of log p_t and h of the entropy
//     dL/ds_i = g (1[i = t] - p_i) - h p_i (log p_i + entropy),     dL/dz_i = w_j dL/ds_i,     dL/dw_j = sum dL/ds_i z_i.
// The pixels at the maximum are COUNTED and the others summed apart from them: for a map that is almost one pixel, log(c + r) = log c +
// log1p(r / c) and 1 - p_t = -expm1(log p_t) then keep all 24 bits of a sum whose leading 1 would swallow them.
//
// Bound: memory.  Forward reads s once (the row stays in registers between the maximum and the sums), backward reads it once more and writes the
// gradient.  Sums, maxima and statistics are fp32; bf16 logits are widened on load, the gradient of a bf16 tensor is rounded once on store.
#include <hip/hip_runtime.h>
#include <math.h>

#include "pwr_common.h"
#include "pwr.h"

namespace pwr {

constexpr int kLikeMaxTop = 32;         // of the K most likely pixels
constexpr int kLikeCand = 256;          // candidates the selection sorts (one per thread)
constexpr int kLikeChunk = 16384;       // values of a row one workgroup holds in registers (256 threads x 64)
constexpr int kLikeWaveMax = 512;       // rows up to here: one wave per row (64 lanes x 8)

struct LikeArgs {
  const void* z; long long ldz;         // [rows] of V values, ldz apart
  const float* w; int J;                // row r belongs to joint r % J; w may be null
  const float* mask; int mask_rows;     // mask row of row r: r / mask_rows (J: one per sample; 1: one per row); null: every pixel
  const long long* index;               // may be null
  long long rows; int V, K;
  float* logp; float* entropy; float* stats;      // stats [rows][2] = {M, log(c + r)}
  float* top_logp; long long* top_index;
  // chunked rows
  int chunks, chunk;                    // chunk = values per workgroup
  float* part;                          // [rows][chunks][4] = {M, c, r, q}
  float* cand_s; int* cand_i;           // [rows][chunks][K]
};

// four neighbouring values of T at any element alignment (rows of odd length start anywhere; the hardware takes such an address)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Quad { T v[4]; };

template <typename T>
__device__ __forceinline__ void load4(const T* p, int i, int V, float (&o)[4], float fill) {
  if (i + 3 < V) {
    const Quad<T> q = *reinterpret_cast<const Quad<T>*>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = Elem<T>::to_f(q.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = i + k < V ? Elem<T>::to_f(p[i + k]) : fill;
  }
}

// The statistics of a set of values, and how two sets join.  M = -inf: nothing in the set (c = q = 0, r = 0 or NaN).
struct LikeStat { float M, c, r, q; };
__device__ __forceinline__ LikeStat like_join(const LikeStat& a, const LikeStat& b) {
  const float M = fmaxf(a.M, b.M);
  LikeStat o = {M, 0.f, 0.f, 0.f};
  auto add = [&](const LikeStat& x) {
    if (x.M == M) { o.c += x.c; o.r += x.r; o.q += x.q; }
    else if (x.M == -INFINITY) { o.r += x.r; }                     // (empty: adds 0, or the NaN it saw)
    else {
      const float d = x.M - M, f = __expf(d), t = x.c + x.r;
      o.r += f * t;
      if (f > 0.f) o.q += f * (x.q + d * t);
    }
  };
  add(a); add(b);
  return o;
}
// log of the sum of exp(s - M)
__device__ __forceinline__ float like_log_total(const LikeStat& a) {
  if (a.c == 0.f && a.r == 0.f) return -INFINITY;
  return a.c > 0.f ? (a.c == 1.f ? 0.f : logf(a.c)) + log1pf(a.r / a.c) : a.r * INFINITY;      // (c == 0 with r != 0: a NaN was seen)
}

template <typename T>
__device__ __forceinline__ float like_value(const LikeArgs& a, long long row, long long t, float w) {
  const float s = Elem<T>::to_f(reinterpret_cast<const T*>(a.z)[row * a.ldz + t]) * w;
  return a.mask && a.mask[(row / a.mask_rows) * a.V + t] == 0.f ? -INFINITY : s;
}

// what one thread writes for a finished row
template <typename T>
__device__ __forceinline__ float like_finish(const LikeArgs& a, long long row, const LikeStat& st, float w) {
  const float lt = like_log_total(st);
  const bool none = st.c == 0.f && st.r == 0.f;
  if (a.logp) {
    float lp = 0.f;
    const long long t = a.index ? a.index[row] : -1;
    if (t >= a.V) lp = NAN;                                        // (not a pixel: loud, and nothing is read)
    else if (t >= 0) {
      const float s = like_value<T>(a, row, t, w);
      lp = none || s == -INFINITY ? (lt == lt ? -INFINITY : lt) : (s - st.M) - lt;
    }
    a.logp[row] = lp;
  }
  if (a.entropy) a.entropy[row] = none ? 0.f : lt - st.q / (st.c + st.r);
  if (a.stats) { a.stats[2 * row] = st.M; a.stats[2 * row + 1] = lt; }
  return lt;
}

// (s, i) before (t, j) in the order of the alternatives: the larger value, among equals the lower index
__device__ __forceinline__ bool like_before(float s, int i, float t, int j) { return s > t || (s == t && i < j); }

// The K first of the (s, i) a workgroup of 256 threads holds, in order, to emit(rank, s, i); ranks beyond what is there get (-inf, -1).
// The K-th largest of the threads' own maxima bounds the K-th value from below (K threads hold one each): what reaches it are the candidates,
// rarely more than a few over K, sorted by counting who comes before whom.  More candidates than threads (long ties): K rounds of a
// maximum over what comes after the last one instead.
template <int VPT, typename IndexOf, typename Emit>
__device__ __forceinline__ void like_select(const float (&s)[VPT], IndexOf index_of, int K, char* lds, Emit emit) {
  float* tm = reinterpret_cast<float*>(lds);                       // [256] maxima, then candidates' values
  int* ti = reinterpret_cast<int*>(lds + 1024);                    // [256] candidates' indices
  int* cnt = reinterpret_cast<int*>(lds + 2048);
  float* thr = reinterpret_cast<float*>(lds + 2052);
  const int tid = threadIdx.x;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) m = fmaxf(m, s[k]);
  __syncthreads();
  tm[tid] = m;
  if (tid == 0) *cnt = 0;
  __syncthreads();
  int rank = 0;
  for (int k = 0; k < 256; k += 4) {
    const f32x4 o = *reinterpret_cast<const f32x4*>(tm + k);
#pragma unroll
    for (int e = 0; e < 4; ++e) rank += o[e] > m || (o[e] == m && k + e < tid);
  }
  if (rank == K - 1) *thr = m;
  __syncthreads();
  const float bound = *thr;
  if (m >= bound && m > -INFINITY) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (s[k] >= bound && s[k] > -INFINITY) {
        const int at = atomicAdd(cnt, 1);                          // (the order of arrival is not the order of the result)
        if (at < kLikeCand) { tm[at] = s[k]; ti[at] = index_of(k); }
      }
  }
  __syncthreads();
  const int n = *cnt;
  if (n <= kLikeCand) {
    if (tid < n) {
      const float v = tm[tid];
      const int i = ti[tid];
      int r = 0;
      for (int k = 0; k < n; ++k) r += like_before(tm[k], ti[k], v, i);
      if (r < K) emit(r, v, i);
    } else if (tid < K) emit(tid, -INFINITY, -1);                  // (n < K only when that is all there is)
    return;
  }
  float last_s = INFINITY;
  int last_i = -1;
  for (int r = 0; r < K; ++r) {
    float bs = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int i = index_of(k);
      if (s[k] > -INFINITY && like_before(last_s, last_i, s[k], i) && like_before(s[k], i, bs, bi)) { bs = s[k]; bi = i; }
    }
    for (int o = 32; o; o >>= 1) {
      const float xs = __shfl_xor(bs, o);
      const int xi = __shfl_xor(bi, o);
      if (like_before(xs, xi, bs, bi)) { bs = xs; bi = xi; }
    }
    __syncthreads();
    if ((tid & 63) == 0) { tm[tid >> 6] = bs; ti[tid >> 6] = bi; }
    __syncthreads();
    bs = tm[0]; bi = ti[0];
#pragma unroll
    for (int k = 1; k < 4; ++k)
      if (like_before(tm[k], ti[k], bs, bi)) { bs = tm[k]; bi = ti[k]; }
    if (tid == 0) emit(r, bs, bs > -INFINITY ? bi : -1);
    last_s = bs; last_i = bi;
  }
}

// One workgroup: one chunk of one row (CHUNKED), or a whole row.
template <typename T, int VPT, bool CHUNKED>
__global__ __launch_bounds__(256) void like_fwd_kernel(LikeArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[2064];
  __shared__ float red[16];
  const int tid = threadIdx.x;
  const long long row = CHUNKED ? (long long)blockIdx.x / a.chunks : blockIdx.x;
  const int ch = CHUNKED ? (int)(blockIdx.x - row * a.chunks) : 0;
  const int base = ch * a.chunk, end = CHUNKED ? min(a.V, base + a.chunk) : a.V;
  const float w = a.w ? a.w[row % a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  const float* mk = a.mask ? a.mask + (row / a.mask_rows) * a.V : nullptr;
  float s[VPT];
#pragma unroll
  for (int k = 0; k < VPT / 4; ++k) {
    const int i = base + (k * 256 + tid) * 4;
    float v[4];
    load4(z, i, end, v, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * k + e] = i + e < end ? v[e] * w : -INFINITY;
  }
  if (mk) {
#pragma unroll
    for (int k = 0; k < VPT / 4; ++k) {
      const int i = base + (k * 256 + tid) * 4;
      float v[4];
      load4(mk, i, end, v, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] == 0.f) s[4 * k + e] = -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) m = fmaxf(m, s[k]);
  m = block_max<4>(m, red);
  const float m0 = m == -INFINITY ? 0.f : m;
  float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const float d = s[k] - m0, e = __expf(d);
    const bool at = d == 0.f && m0 == m;
    sum[0] += at ? 1.f : 0.f;
    sum[1] += at ? 0.f : e;
    if (e != 0.f) sum[2] = fmaf(e, d, sum[2]);                     // (0 x -inf is 0 here; NaN passes)
  }
  block_sum<3, 4>(sum, red);
  const LikeStat st = {m, sum[0], sum[1], sum[2]};
  auto index_of = [&](int k) { return base + ((k >> 2) * 256 + tid) * 4 + (k & 3); };
  if constexpr (CHUNKED) {
    if (tid == 0) *reinterpret_cast<f32x4*>(a.part + 4 * (long long)blockIdx.x) = f32x4{st.M, st.c, st.r, st.q};
    if (a.K) {
      float* cs = a.cand_s + (long long)blockIdx.x * a.K;
      int* ci = a.cand_i + (long long)blockIdx.x * a.K;
      like_select<VPT>(s, index_of, a.K, lds, [&](int r, float v, int i) { cs[r] = v; ci[r] = i; });
    }
  } else {
    if (tid == 0) like_finish<T>(a, row, st, w);
    if (a.K) {
      const float lt = like_log_total(st);
      float* ts = a.top_logp + row * a.K;
      long long* ix = a.top_index + row * a.K;
      like_select<VPT>(s, index_of, a.K, lds, [&](int r, float v, int i) { ts[r] = i < 0 ? v : (v - st.M) - lt; ix[r] = i; });
    }
  }
}

// Joins the chunks of a row: one workgroup per row, the candidates of all chunks (at most 256 x VPT) selected again.
template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_join_kernel(LikeArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[2064];
  __shared__ LikeStat part[256];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x;
  const float w = a.w ? a.w[row % a.J] : 1.f;
  LikeStat st = {-INFINITY, 0.f, 0.f, 0.f};
  for (int c = tid; c < a.chunks; c += 256) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + 4 * (row * a.chunks + c));
    st = like_join(st, LikeStat{v.x, v.y, v.z, v.w});
  }
  part[tid] = st;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (tid < o) part[tid] = like_join(part[tid], part[tid + o]);
    __syncthreads();
  }
  st = part[0];
  if (tid == 0) like_finish<T>(a, row, st, w);
  if (a.K) {
    const float lt = like_log_total(st);
    const int n = a.chunks * a.K;
    float s[VPT];
    int ix[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int at = k * 256 + tid;
      s[k] = at < n ? a.cand_s[row * n + at] : -INFINITY;
      ix[k] = at < n ? a.cand_i[row * n + at] : -1;
    }
    float* ts = a.top_logp + row * a.K;
    long long* to = a.top_index + row * a.K;
    auto index_of = [&](int k) { return ix[k]; };
    like_select<VPT>(s, index_of, a.K, lds, [&](int r, float v, int i) { ts[r] = i < 0 ? v : (v - st.M) - lt; to[r] = i; });
  }
}

// Rows of at most 512 values: one wave per row, four rows per workgroup, no barrier.
template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_fwd_wave_kernel(LikeArgs a) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const float w = a.w ? a.w[row % a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  const float* mk = a.mask ? a.mask + (row / a.mask_rows) * a.V : nullptr;
  float s[VPT];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * 64 + lane;
    s[k] = i < a.V && (!mk || mk[i] != 0.f) ? Elem<T>::to_f(z[i]) * w : -INFINITY;
    m = fmaxf(m, s[k]);
  }
  m = wave_max(m);
  const float m0 = m == -INFINITY ? 0.f : m;
  float c = 0.f, r = 0.f, q = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const float d = s[k] - m0, e = __expf(d);
    const bool at = d == 0.f && m0 == m;
    c += at ? 1.f : 0.f;
    r += at ? 0.f : e;
    if (e != 0.f) q = fmaf(e, d, q);
  }
  const LikeStat st = {m, wave_sum(c), wave_sum(r), wave_sum(q)};
  if (lane == 0) like_finish<T>(a, row, st, w);
  if (!a.K) return;
  const float lt = like_log_total(st);
  float last_s = INFINITY;
  int last_i = -1;
  for (int rank = 0; rank < a.K; ++rank) {
    float bs = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int i = k * 64 + lane;
      if (s[k] > -INFINITY && like_before(last_s, last_i, s[k], i) && like_before(s[k], i, bs, bi)) { bs = s[k]; bi = i; }
    }
    for (int o = 32; o; o >>= 1) {
      const float xs = __shfl_xor(bs, o);
      const int xi = __shfl_xor(bi, o);
      if (like_before(xs, xi, bs, bi)) { bs = xs; bi = xi; }
    }
    const bool some = bs > -INFINITY;
    if (lane == 0) { a.top_logp[row * a.K + rank] = some ? (bs - st.M) - lt : bs; a.top_index[row * a.K + rank] = some ? bi : -1; }
    last_s = bs; last_i = bi;
  }
}

struct LikeBwdArgs {
  const void* z; long long ldz; const float* w; int J; const float* mask; int mask_rows; const long long* index;
  const float* stats; const float* entropy; const float* glogp; const float* gentropy;
  void* gz; float* gw_part; long long rows; int V, chunks;
};

// dL/ds of one value; what it has to know about its row
struct LikeRow { float M, lt, H, g, h, zr; long long t; };
__device__ __forceinline__ LikeRow like_row(const LikeBwdArgs& a, long long row, float w) {
  LikeRow o;
  o.M = a.stats[2 * row]; o.lt = a.stats[2 * row + 1];
  o.t = a.index ? a.index[row] : -1;
  o.g = a.glogp && o.t >= 0 ? a.glogp[row] : 0.f;
  o.h = a.gentropy ? a.gentropy[row] : 0.f;
  o.H = a.entropy[row];
  if (o.t >= a.V) o.g = NAN;                                       // (as the log likelihood of such a pixel)
  o.zr = w != 0.f && o.M > -INFINITY ? o.M / w : 0.f;              // the logit at the maximum
  return o;
}
// dL/dw_j of a row is sum ds z.  The ds add up to 0 -- or to -g where the given pixel has no probability --, so the row's largest logit is taken out
// of every z: what is left of the sum does not cancel, also where the logits are 1e38.
__device__ __forceinline__ float like_gw_rest(const LikeRow& o, float st) { return st == -INFINITY && o.g != 0.f && o.M > -INFINITY ? -o.g * o.zr : 0.f; }
__device__ __forceinline__ float like_ds(const LikeRow& o, float s, bool hit) {
  if (s == -INFINITY) return 0.f;                                  // no probability: masked, or the row has no pixel at all
  const float lp = (s - o.M) - o.lt, p = __expf(lp);
  const float e = p != 0.f ? o.h * p * (lp + o.H) : 0.f;
  return o.g * (hit ? -expm1f(lp) : -p) - e;
}

constexpr int kLikeBwdChunk = 4096;     // 256 threads x 16
template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_bwd_kernel(LikeBwdArgs a) {
  __shared__ float red[4];
  const int tid = threadIdx.x;
  const long long row = (long long)blockIdx.x / a.chunks;
  const int base = (int)(blockIdx.x - row * a.chunks) * (256 * VPT);
  const float w = a.w ? a.w[row % a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  T* gz = reinterpret_cast<T*>(a.gz) + row * (long long)a.V;
  const float* mk = a.mask ? a.mask + (row / a.mask_rows) * a.V : nullptr;
  float v[VPT], mv[VPT];
#pragma unroll
  for (int k = 0; k < VPT / 4; ++k) {
    float t[4];
    load4(z, base + (k * 256 + tid) * 4, a.V, t, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[4 * k + e] = t[e]; mv[4 * k + e] = 1.f; }
  }
  if (mk) {
#pragma unroll
    for (int k = 0; k < VPT / 4; ++k) {
      float t[4];
      load4(mk, base + (k * 256 + tid) * 4, a.V, t, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) mv[4 * k + e] = t[e];
    }
  }
  const LikeRow o = like_row(a, row, w);
  float gw = 0.f;
#pragma unroll
  for (int k = 0; k < VPT / 4; ++k) {
    const int i = base + (k * 256 + tid) * 4;
    Quad<T> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = v[4 * k + e];
      const float ds = i + e < a.V ? like_ds(o, mv[4 * k + e] == 0.f ? -INFINITY : x * w, i + e == o.t) : 0.f;
      if (ds != 0.f) gw = fmaf(ds, x - o.zr, gw);
      q.v[e] = Elem<T>::from_f(ds * w);
    }
    if (i + 3 < a.V) *reinterpret_cast<Quad<T>*>(gz + i) = q;
    else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < a.V) gz[i + e] = q.v[e];
    }
  }
  if (a.gw_part) {
    gw = block_sum1(gw, red);
    if (tid == 0) {
      if (base == 0 && o.t >= 0 && o.t < a.V) gw += like_gw_rest(o, mk && mk[o.t] == 0.f ? -INFINITY : Elem<T>::to_f(z[o.t]) * w);
      a.gw_part[blockIdx.x] = gw;
    }
  }
}

template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_bwd_wave_kernel(LikeBwdArgs a) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const float w = a.w ? a.w[row % a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  T* gz = reinterpret_cast<T*>(a.gz) + row * (long long)a.V;
  const float* mk = a.mask ? a.mask + (row / a.mask_rows) * a.V : nullptr;
  const LikeRow o = like_row(a, row, w);
  float gw = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * 64 + lane;
    if (i < a.V) {
      const float x = Elem<T>::to_f(z[i]);
      const float ds = like_ds(o, mk && mk[i] == 0.f ? -INFINITY : x * w, i == o.t);
      if (ds != 0.f) gw = fmaf(ds, x - o.zr, gw);
      gz[i] = Elem<T>::from_f(ds * w);
    }
  }
  if (a.gw_part) {
    gw = wave_sum(gw);
    if (lane == 0) {
      if (o.t >= 0 && o.t < a.V) gw += like_gw_rest(o, mk && mk[o.t] == 0.f ? -INFINITY : Elem<T>::to_f(z[o.t]) * w);
      a.gw_part[row] = gw;
    }
  }
}

// gw[j] = the partial sums of the rows of joint j, in their order
__global__ __launch_bounds__(256) void like_gw_kernel(const float* __restrict__ part, float* __restrict__ gw, long long samples, int J, int chunks) {
  __shared__ float red[4];
  const int j = blockIdx.x;
  float s = 0.f;
  for (long long k = threadIdx.x; k < samples * chunks; k += 256) s += part[((k / chunks) * J + j) * chunks + k % chunks];
  s = block_sum1(s, red);
  if (threadIdx.x == 0) gw[j] = s;
}

}  // namespace pwr

using namespace pwr;

// Values per workgroup of a row that is split: as many as the registers hold -- but a few long rows do not fill 256 CUs that way, so the chunk is
// halved (down to 4096 = one wide load per lane and instruction, 16 values per thread) until the launch has 512 workgroups.
static int like_chunk(long long rows, int V) {
  int c = kLikeChunk;
  while (c > 4096 && rows * ((V + c - 1) / c) < 512) c >>= 1;
  return c;
}
static int like_chunks(long long rows, int V) {
  const int c = like_chunk(rows, V);
  return (V + c - 1) / c;
}

extern "C" size_t pwr_likelihood_workspace_bytes(long long rows, int V, int K) {
  if (rows <= 0 || V <= 0 || K < 0) return 0;
  const int n = like_chunks(rows, V);
  return n == 1 ? 0 : (size_t)rows * n * (16 + 8 * (size_t)K);
}

template <typename T>
static int like_forward(const LikeArgs& a, hipStream_t s) {
  const long long rows = a.rows;
  if (a.V <= kLikeWaveMax) {
    const dim3 g((unsigned)((rows + 3) / 4));
    if (a.V <= 64) hipLaunchKernelGGL((like_fwd_wave_kernel<T, 1>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((like_fwd_wave_kernel<T, 8>), g, dim3(256), 0, s, a);
    return (int)hipGetLastError();
  }
  const dim3 g((unsigned)(rows * a.chunks));
  if (a.chunks == 1) {
    if (a.V <= 4096) hipLaunchKernelGGL((like_fwd_kernel<T, 16, false>), g, dim3(256), 0, s, a);
    else if (a.V <= 8192) hipLaunchKernelGGL((like_fwd_kernel<T, 32, false>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((like_fwd_kernel<T, 64, false>), g, dim3(256), 0, s, a);
    return (int)hipGetLastError();
  }
  if (a.chunk == 4096) hipLaunchKernelGGL((like_fwd_kernel<T, 16, true>), g, dim3(256), 0, s, a);
  else if (a.chunk == 8192) hipLaunchKernelGGL((like_fwd_kernel<T, 32, true>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((like_fwd_kernel<T, 64, true>), g, dim3(256), 0, s, a);
  if (a.chunks * a.K <= 1024) hipLaunchKernelGGL((like_join_kernel<T, 4>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((like_join_kernel<T, 16>), dim3((unsigned)rows), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

extern "C" int pwr_likelihood_fwd(const void* z, long long ldz, const float* w, int J, const float* mask, int mask_rows, const long long* index,
                                  float* logp, float* entropy, float* stats, float* top_logp, long long* top_index, long long rows, int V, int K,
                                  int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return 0;
  if (!z || rows < 0 || V <= 0 || K < 0 || J <= 0 || mask_rows <= 0 || ldz < 0 || (K && (!top_logp || !top_index))) return PWR_EINVAL;
  if (dtype != PWR_F32 && dtype != PWR_BF16) return PWR_EINVAL;
  LikeArgs a = {z, ldz, w, J, mask, mask_rows, index, rows, V, K, logp, entropy, stats, top_logp, top_index, 1, V, nullptr, nullptr, nullptr};
  a.chunk = like_chunk(rows, V);
  a.chunks = like_chunks(rows, V);
  if (K > kLikeMaxTop || (long long)a.chunks * K > 4096 || rows * a.chunks > 0x7fffffffll) return PWR_EUNSUPPORTED;
  if (a.chunks > 1) {
    if (!workspace || workspace_bytes < pwr_likelihood_workspace_bytes(rows, V, K)) return PWR_ENOSPACE;
    a.part = (float*)workspace;
    a.cand_s = a.part + 4 * rows * a.chunks;
    a.cand_i = (int*)(a.cand_s + rows * a.chunks * K);
  }
  return dtype == PWR_F32 ? like_forward<float>(a, (hipStream_t)stream) : like_forward<bf16_t>(a, (hipStream_t)stream);
}

static int like_bwd_chunks(int V) { return V <= kLikeWaveMax ? 1 : (V + kLikeBwdChunk - 1) / kLikeBwdChunk; }

extern "C" size_t pwr_likelihood_bwd_workspace_bytes(long long rows, int V) { return rows <= 0 || V <= 0 ? 0 : (size_t)rows * like_bwd_chunks(V) * 4; }

template <typename T>
static void like_backward(const LikeBwdArgs& a, hipStream_t s) {
  if (a.V <= kLikeWaveMax) {
    const dim3 g((unsigned)((a.rows + 3) / 4));
    if (a.V <= 64) hipLaunchKernelGGL((like_bwd_wave_kernel<T, 1>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((like_bwd_wave_kernel<T, 8>), g, dim3(256), 0, s, a);
  } else hipLaunchKernelGGL((like_bwd_kernel<T, 16>), dim3((unsigned)(a.rows * a.chunks)), dim3(256), 0, s, a);
}

extern "C" int pwr_likelihood_bwd(const void* z, long long ldz, const float* w, int J, const float* mask, int mask_rows, const long long* index,
                                  const float* stats, const float* entropy, const float* glogp, const float* gentropy, void* gz, float* gw,
                                  long long rows, int V, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0 && !gw) return 0;
  if (rows < 0 || V <= 0 || J <= 0 || mask_rows <= 0 || ldz < 0 || (rows && (!z || !stats || !entropy || !gz)) || (gw && (!w || rows % J))) return PWR_EINVAL;
  if (dtype != PWR_F32 && dtype != PWR_BF16) return PWR_EINVAL;
  LikeBwdArgs a = {z, ldz, w, J, mask, mask_rows, index, stats, entropy, glogp, gentropy, gz, nullptr, rows, V, like_bwd_chunks(V)};
  if (rows * a.chunks > 0x7fffffffll) return PWR_EUNSUPPORTED;
  if (gw) {
    if (rows && (!workspace || workspace_bytes < pwr_likelihood_bwd_workspace_bytes(rows, V))) return PWR_ENOSPACE;
    a.gw_part = (float*)workspace;
  }
  hipStream_t s = (hipStream_t)stream;
  if (rows) { if (dtype == PWR_F32) like_backward<float>(a, s); else like_backward<bf16_t>(a, s); }
  if (gw) hipLaunchKernelGGL(like_gw_kernel, dim3(J), dim3(256), 0, s, a.gw_part, gw, rows / J, J, a.chunks);
  return (int)hipGetLastError();
}
