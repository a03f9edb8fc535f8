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
constexpr int kLikeChunk = 16384;       // values of a row one workgroup holds in registers (512 threads x 32)
// Without alternatives a workgroup walks a row of over 4096 values; only a row of several chunks is split over workgroups, where there are fewer
// rows than this.  Walked / split: 512 rows of 50001 fp32 18.6 / 24.0 us, bf16 19.6 / 22.2; 256 rows 13.0 / 15.4 and 15.3 / 13.9.
constexpr int kLikeWalkRows = 512;
constexpr int kLikeWaveMax = 512;       // rows up to here: one wave per row (64 lanes x 8)
constexpr int kLikeMaxRow = 0x7fffffff - kLikeChunk + 1;       // 2^31 - 2^14: the end of a row's last piece is an int too

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

// 16 bytes of T at any element alignment (rows of odd length start anywhere; the hardware takes such an address)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[16 / sizeof(T)]; };

// VPT of a row's n values per thread, 16 bytes at a time, and the mask's: value k belongs to index value_index(k).  No load hides behind a branch (one
// that does is waited for before the next is sent): where the workgroup has room for more than n values, every piece is read at an index that has one,
// n >= N (or N values in front of p), and moved into place by values().
template <typename T, int NT, int VPT>
struct RowPart {
  static constexpr int N = 16 / sizeof(T);
  Piece<T> q[VPT / N];
  Piece<float> mq[VPT / 4];
  __device__ __forceinline__ void load(const T* p, const float* mask, int n) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < VPT / N; ++k) q[k] = *reinterpret_cast<const Piece<T>*>(p + min((k * NT + tid) * N, n - N));
    if (mask) {
#pragma unroll
      for (int k = 0; k < VPT / 4; ++k)
        mq[k] = *reinterpret_cast<const Piece<float>*>(mask + min((k * 4 / N * NT + tid) * N, n - N) + k * 4 % N);
    }
  }
  // v = z, s = w z of the allowed ones, -inf where the mask says so and beyond n
  __device__ __forceinline__ void values(bool mask, int n, float w, float (&v)[VPT], float (&s)[VPT]) const {
    const int tid = threadIdx.x;
    if (n >= NT * VPT) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) { v[k] = Elem<T>::to_f(q[k / N].v[k % N]); s[k] = v[k] * w; }
      if (mask) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) s[k] = mq[k / 4].v[k % 4] == 0.f ? -INFINITY : s[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < VPT / N; ++k) {
        const int d = (k * NT + tid) * N - (n - N);             // how far the piece reaches beyond n
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float x = Elem<T>::to_f(q[k].v[e]), in = mask ? mq[(k * N + e) / 4].v[e % 4] : 1.f;
#pragma unroll
          for (int j = e + 1; j < N; ++j) {
            x = d == j - e ? Elem<T>::to_f(q[k].v[j]) : x;
            in = mask && d == j - e ? mq[(k * N + j) / 4].v[j % 4] : in;
          }
          v[k * N + e] = x;
          s[k * N + e] = e + d < N && in != 0.f ? x * w : -INFINITY;
        }
      }
    }
  }
};
// the index of value k of a RowPart
template <typename T, int NT>
__device__ __forceinline__ int value_index(int k) {
  constexpr int N = 16 / sizeof(T);
  return ((k / N) * NT + (int)threadIdx.x) * N + k % N;
}

// The statistics of a set of values, and how sets join.  M = -inf: nothing in the set (c = q = 0, r = 0 or NaN).
struct LikeStat { float M, c, r, q; };
// x's sums relative to the joint maximum M >= x.M
__device__ __forceinline__ LikeStat like_shift(const LikeStat& x, float M) {
  if (x.M == M) return x;
  if (x.M == -INFINITY) return {M, 0.f, x.r, 0.f};                  // (empty: adds 0, or the NaN it saw)
  const float d = x.M - M, f = __expf(d), t = x.c + x.r;
  return {M, 0.f, f * t, f > 0.f ? f * (x.q + d * t) : 0.f};
}
// log of the sum of exp(s - M)
__device__ __forceinline__ float like_log_total(const LikeStat& a) {
  if (a.c == 0.f) return a.r == 0.f ? -INFINITY : a.r * INFINITY;                // (nothing, or a NaN was seen)
  return a.c == 1.f ? log1pf(a.r) : __logf(a.c + a.r);                            // (from 2 on the sum swallows nothing)
}

// The given pixel t of a row: its s, or NaN for one that is no pixel.  Its index is read at the start of a kernel and s behind the row's own loads, so
// that the two reads in a row cost no time of their own.
struct LikeGiven { bool any; float s; };
template <typename T>
__device__ __forceinline__ LikeGiven like_given(const LikeArgs& a, long long t, const T* z, const float* mask, float w) {
  if (t < 0) return {false, 0.f};
  if (t >= a.V) return {true, NAN};                                // (nothing is read, and the result is loud)
  const float s = Elem<T>::to_f(z[t]) * w;
  return {true, mask && mask[t] == 0.f ? -INFINITY : s};
}

// what one thread writes for a finished row
__device__ __forceinline__ void like_finish(const LikeArgs& a, unsigned row, const LikeStat& st, float lt, const LikeGiven& g) {
  const bool none = st.c == 0.f && st.r == 0.f;
  if (a.logp) {
    float lp = 0.f;
    if (g.any) lp = g.s != g.s ? NAN : none || g.s == -INFINITY ? (lt == lt ? -INFINITY : lt) : (g.s - st.M) - lt;
    a.logp[row] = lp;
  }
  if (a.entropy) a.entropy[row] = none ? 0.f : lt - st.q / (st.c + st.r);
  if (a.stats) { a.stats[2ll * row] = st.M; a.stats[2ll * row + 1] = lt; }
}

// (s, i) before (t, j) in the order of the alternatives: the larger value, among equals the lower index
__device__ __forceinline__ bool like_before(float s, int i, float t, int j) { return s > t || (s == t && i < j); }

// Shared memory of a workgroup of NW waves.
template <int NW> struct LikeShared {
  float group[NW][32];
  float sum[3][NW];
  int count;
  __attribute__((aligned(16))) float cs[kLikeCand];
  __attribute__((aligned(16))) int ci[kLikeCand];
};

// The workgroup's maximum, and a bound that at least K of its values reach: the values fall into G >= K groups (lane mod G, over all waves), each group's
// maximum is a value, so K values reach the least of these maxima -- and by the coupon collector's count about G ln G values do in all.
// One barrier.  m: this thread's maximum.
template <int NW>
__device__ __forceinline__ void like_maximum(float m, int K, LikeShared<NW>& sh, float& M, float& bound) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  m = fmaxf(m, lane_xor<32>(m));
  if (lane < 32) sh.group[wid][lane] = m;
  if (threadIdx.x == 0) sh.count = 0;
  if (K)
    for (int k = threadIdx.x; k < kLikeCand; k += NW * 64) sh.cs[k] = -INFINITY;
  __syncthreads();
  m = sh.group[0][lane & 31];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, sh.group[w][lane & 31]);
  if (K <= 16) m = fmaxf(m, lane_xor<16>(m));
  if (K <= 8) m = fmaxf(m, lane_xor<8>(m));
  if (K <= 4) m = fmaxf(m, lane_xor<4>(m));
  float lo = m, hi = m;
  lo = fminf(lo, lane_xor<16>(lo)); hi = fmaxf(hi, lane_xor<16>(hi));
  lo = fminf(lo, lane_xor<8>(lo)); hi = fmaxf(hi, lane_xor<8>(hi));
  lo = fminf(lo, lane_xor<4>(lo)); hi = fmaxf(hi, lane_xor<4>(hi));
  lo = fminf(lo, lane_xor<2>(lo)); hi = fmaxf(hi, lane_xor<2>(hi));
  lo = fminf(lo, lane_xor<1>(lo)); hi = fmaxf(hi, lane_xor<1>(hi));
  M = hi; bound = lo;
}

// What reaches the bound becomes a candidate (in any order); a barrier has to follow.  own: this thread's maximum.
template <int NW, int VPT, typename IndexOf>
__device__ __forceinline__ void like_push(LikeShared<NW>& sh, const float (&s)[VPT], IndexOf index_of, float own, float bound) {
  if (own < bound || own == -INFINITY) return;
  int n = 0;
#pragma unroll
  for (int k = 0; k < VPT; ++k) n += s[k] >= bound && s[k] > -INFINITY;
  int at = atomicAdd(&sh.count, n);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (s[k] >= bound && s[k] > -INFINITY) {
      if (at < kLikeCand) { sh.cs[at] = s[k]; sh.ci[at] = index_of(k); }
      ++at;
    }
}

// The K first of the workgroup's (s, i) in order, to emit(rank, s, i); ranks beyond what is there get (-inf, -1).  Candidates are placed by counting
// who comes before them; more of them than there is room for (long ties, or a mask that leaves one group empty): K rounds of a maximum over what
// comes after the last one.
template <int NW, int VPT, typename IndexOf, typename Emit>
__device__ __forceinline__ void like_select(const float (&s)[VPT], IndexOf index_of, int K, LikeShared<NW>& sh, Emit emit) {
  const int tid = threadIdx.x, n = sh.count;
  if (n <= kLikeCand) {
    for (int c = tid; c < n; c += NW * 64) {
      const float v = sh.cs[c];
      const int i = sh.ci[c];
      int r = 0;
      for (int k = 0; k < n; k += 4) {                               // (beyond n: -inf, which comes before nobody)
        const f32x4 x = *reinterpret_cast<const f32x4*>(sh.cs + k);
        const int4 j = *reinterpret_cast<const int4*>(sh.ci + k);
        r += like_before(x.x, j.x, v, i) + like_before(x.y, j.y, v, i) + like_before(x.z, j.z, v, i) + like_before(x.w, j.w, v, i);
      }
      if (r < K) emit(r, v, i);
    }
    for (int r = n + tid; r < K; r += NW * 64) emit(r, -INFINITY, -1);       // (n < K only when that is all there is)
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
    if ((tid & 63) == 0) { sh.cs[tid >> 6] = bs; sh.ci[tid >> 6] = bi; }
    __syncthreads();
    bs = sh.cs[0]; bi = sh.ci[0];
#pragma unroll
    for (int k = 1; k < NW; ++k)
      if (like_before(sh.cs[k], sh.ci[k], bs, bi)) { bs = sh.cs[k]; bi = sh.ci[k]; }
    if (tid == 0) emit(r, bs, bs > -INFINITY ? bi : -1);
    last_s = bs; last_i = bi;
  }
}

// One workgroup: one chunk of one row (CHUNKED), or a whole row.  Two barriers: maximum and bound, then sums and candidates.
template <typename T, int NT, int VPT, bool CHUNKED, bool TOP>
__device__ __forceinline__ void like_fwd_block(const LikeArgs& a, LikeShared<NT / 64>& sh, unsigned row, int base, int n) {
  constexpr int NW = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  const float* mrow = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const long long t = !CHUNKED && a.index ? a.index[row] : -1;
  RowPart<T, NT, VPT> part;
  part.load(z + base, mrow ? mrow + base : nullptr, n);
  const LikeGiven given = like_given<T>(a, t, z, mrow, w);
  float s[VPT], v[VPT];
  part.values(mrow != nullptr, n, w, v, s);
  float own = -INFINITY, m, bound;
#pragma unroll
  for (int k = 0; k < VPT; ++k) own = fmaxf(own, s[k]);
  like_maximum<NW>(own, a.K, sh, m, bound);
  const float m0 = m == -INFINITY ? 0.f : m;
  float c = 0.f, r = 0.f, q = 0.f;
  if (__any(own == m0)) {
    // the wave that has the maximum (or a few): its values at the maximum are counted, the others summed
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const float d = s[k] - m0, e = __expf(d);
      const bool at = d == 0.f && m0 == m;
      c += at ? 1.f : 0.f;
      r += at ? 0.f : e;
      q = fmaf(e, fmaxf(d, -1e30f), q);
    }
  } else {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const float d = s[k] - m0, e = __expf(d);
      r += e;
      q = fmaf(e, fmaxf(d, -1e30f), q);                            // (0 x -inf is 0 here; a NaN has passed through e)
    }
  }
  c = wave_sum(c); r = wave_sum(r); q = wave_sum(q);
  if (lane == 0) { sh.sum[0][wid] = c; sh.sum[1][wid] = r; sh.sum[2][wid] = q; }
  auto index_of = [&](int k) { return base + value_index<T, NT>(k); };
  if constexpr (TOP) like_push<NW, VPT>(sh, s, index_of, own, bound);
  __syncthreads();
  c = r = q = 0.f;
#pragma unroll
  for (int k = 0; k < NW; ++k) { c += sh.sum[0][k]; r += sh.sum[1][k]; q += sh.sum[2][k]; }
  const LikeStat st = {m, c, r, q};
  if constexpr (CHUNKED) {
    if (tid == 0) *reinterpret_cast<f32x4*>(a.part + 4 * (long long)blockIdx.x) = f32x4{st.M, st.c, st.r, st.q};
    if constexpr (TOP) {
      float* cs = a.cand_s + (long long)blockIdx.x * a.K;
      int* ci = a.cand_i + (long long)blockIdx.x * a.K;
      like_select<NW, VPT>(s, index_of, a.K, sh, [&](int rk, float v, int i) { cs[rk] = v; ci[rk] = i; });
    }
  } else {
    const float lt = like_log_total(st);
    if (tid == NT - 1) like_finish(a, row, st, lt, given);         // (not a thread that has an alternative to place)
    if constexpr (TOP) {
      float* ts = a.top_logp + (long long)row * a.K;
      long long* ix = a.top_index + (long long)row * a.K;
      like_select<NW, VPT>(s, index_of, a.K, sh, [&](int rk, float v, int i) { ts[rk] = i < 0 ? v : (v - st.M) - lt; ix[rk] = i; });
    }
  }
}

// (Straight-line code runs once per workgroup and the instruction cache starts cold: rows of up to 4096 values take one 16-byte piece a thread, long ones 32
// values.  128 x 42 maps of 128 x 128, fp32: 512 threads x 32 values 74 us = 4.8 TB/s, 1024 x 16 82 us, 256 x 64 79 us.  Alternatives are a form of
// their own: compiled in and unused they took 50 us of the same launch, in registers and copies.)
template <typename T, int NT, int VPT, bool CHUNKED, bool TOP>
__global__ __launch_bounds__(NT) void like_fwd_kernel(LikeArgs a) {
  __shared__ LikeShared<NT / 64> sh;
  constexpr int N = 16 / sizeof(T);
  if constexpr (CHUNKED) {
    const unsigned row = blockIdx.x / (unsigned)a.chunks;          // (below 2^31: 64-bit divisions would cost more than the loads)
    const int base = (int)(blockIdx.x - row * (unsigned)a.chunks) * a.chunk, n = min(a.V - base, a.chunk);
    if (VPT > N && n <= NT * N) like_fwd_block<T, NT, N, true, TOP>(a, sh, row, base, n);       // (a row's short end)
    else like_fwd_block<T, NT, VPT, true, TOP>(a, sh, row, base, n);
  } else like_fwd_block<T, NT, VPT, false, TOP>(a, sh, blockIdx.x, 0, a.V);
}

// Long rows, enough of them to fill the chip, without alternatives: one workgroup walks its row in parts of NT x VPT values, the next part's loads under
// way while it works on one.  The sums are kept relative to the largest value so far, per thread; one barrier per part.  A part's sixteen values are added up
// by themselves and the parts by compensated additions: the length of the row costs no bits, a new maximum three roundings of what is there.  4096 rows of 50001 bf16: 256 threads
// x 16 values 102 us = 4.0 TB/s (50000, rows that start aligned: 88 us = 4.7), 256 x 32 112, 512 x 16 128, 1024 x 16 189, a workgroup per chunk and a
// join 161; 5376 rows of 16384 fp32: 64 us = 5.5 TB/s against 74 in one piece.
template <typename T, int NT, int VPT>
__global__ __launch_bounds__(NT) void like_walk_kernel(LikeArgs a) {
  constexpr int NW = NT / 64, N = 16 / sizeof(T), PART = NT * VPT;
  __shared__ float top[2][NW], sum[3][NW];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const unsigned row = blockIdx.x;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  const float* mrow = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const long long t = a.index ? a.index[row] : -1;
  RowPart<T, NT, VPT> part;
  part.load(z, mrow, a.V);
  const LikeGiven given = like_given<T>(a, t, z, mrow, w);
  float M = -INFINITY, c = 0.f, r = 0.f, q = 0.f, dr = 0.f, dq = 0.f;     // (what the last additions to r and q lost)
  for (int base = 0, turn = 0; base < a.V; base += PART, turn ^= 1) {
    const int n = a.V - base;
    float s[VPT], v[VPT];
    part.values(mrow != nullptr, n, w, v, s);
    if (base + PART < a.V) part.load(z + base + PART, mrow ? mrow + base + PART : nullptr, n - PART);
    float own = -INFINITY;
#pragma unroll
    for (int k = 0; k < VPT; ++k) own = fmaxf(own, s[k]);
    const float mw = wave_max(own);
    if (lane == 0) top[turn][wid] = mw;
    __syncthreads();                                               // (the other buffer is read by nobody any more)
    float m = M;
#pragma unroll
    for (int k = 0; k < NW; ++k) m = fmaxf(m, top[turn][k]);
    if (m > M) {
      const LikeStat x = like_shift(LikeStat{M, c, r - dr, q - dq}, m);
      c = x.c; r = x.r; q = x.q; M = m;
      dr = dq = 0.f;
    }
    float pr = 0.f, pq = 0.f;                                      // of this part
    const float m0 = M == -INFINITY ? 0.f : M;
    if (__any(own == m0 && M > -INFINITY)) {                        // a wave that has values at the maximum counts them
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const float d = s[k] - m0, x = __expf(d);
        const bool at = d == 0.f;
        c += at ? 1.f : 0.f;
        pr += at ? 0.f : x;
        pq = fmaf(x, fmaxf(d, -1e30f), pq);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VPT / N; ++k) {
        if (k * NT * N >= n) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = s[k * N + e] - m0, x = __expf(d);
          pr += x;
          pq = fmaf(x, fmaxf(d, -1e30f), pq);
        }
      }
    }
    const float yr = pr - dr, yq = pq - dq, nr = r + yr, nq = q + yq;
    dr = (nr - r) - yr; dq = (nq - q) - yq;
    r = nr; q = nq;
  }
  r -= dr; q -= dq;
  c = wave_sum(c); r = wave_sum(r); q = wave_sum(q);
  if (lane == 0) { sum[0][wid] = c; sum[1][wid] = r; sum[2][wid] = q; }
  __syncthreads();
  if (tid != NT - 1) return;
  c = r = q = 0.f;
#pragma unroll
  for (int k = 0; k < NW; ++k) { c += sum[0][k]; r += sum[1][k]; q += sum[2][k]; }
  const LikeStat st = {M, c, r, q};
  like_finish(a, row, st, like_log_total(st), given);
}

// Joins the chunks of a row: one workgroup per row.  Every wave joins the statistics for itself; the candidates of all chunks (at most 256 x VPT)
// are selected again.
template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_join_kernel(LikeArgs a) {
  __shared__ LikeShared<4> sh;
  const unsigned row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const int n = a.chunks * a.K;
  const float* mrow = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const LikeGiven given = like_given<T>(a, a.index ? a.index[row] : -1, reinterpret_cast<const T*>(a.z) + row * a.ldz, mrow, w);
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part) + (long long)row * a.chunks;
  float s[VPT];
  int ix[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int at = min(k * 256 + tid, n - 1);
    s[k] = n ? a.cand_s[(long long)row * n + at] : -INFINITY;
    ix[k] = n ? a.cand_i[(long long)row * n + at] : -1;
    if (k * 256 + tid >= n) s[k] = -INFINITY;
  }
  float M = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) M = fmaxf(M, part[c].x);
  M = wave_max(M);
  double tc = 0.0, tr = 0.0, tq = 0.0;                              // (a row may have 2^17 pieces, 2048 a lane)
  for (int c = lane; c < a.chunks; c += 64) {
    const f32x4 v = part[c];
    const LikeStat x = like_shift(LikeStat{v.x, v.y, v.z, v.w}, M);
    tc += x.c; tr += x.r; tq += x.q;
  }
  const LikeStat st = {M, wave_sum((float)tc), wave_sum((float)tr), wave_sum((float)tq)};
  const float lt = like_log_total(st);
  if (tid == 255) like_finish(a, row, st, lt, given);
  if (!a.K) return;
  float own = -INFINITY, m, bound;
#pragma unroll
  for (int k = 0; k < VPT; ++k) own = fmaxf(own, s[k]);
  like_maximum<4>(own, a.K, sh, m, bound);
  like_push<4, VPT>(sh, s, [&](int k) { return ix[k]; }, own, bound);
  __syncthreads();
  float* ts = a.top_logp + (long long)row * a.K;
  long long* to = a.top_index + (long long)row * a.K;
  auto index_of = [&](int k) { return ix[k]; };
  like_select<4, VPT>(s, index_of, a.K, sh, [&](int rk, float v, int i) { ts[rk] = i < 0 ? v : (v - st.M) - lt; to[rk] = i; });
}

// Rows of at most 512 values: one wave per row, four rows per workgroup, no barrier.
template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_fwd_wave_kernel(LikeArgs a) {
  const int lane = threadIdx.x & 63;
  const unsigned row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  const float* mk = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const long long t = a.index ? a.index[row] : -1;
  float s[VPT];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * 64 + lane, c = min(i, a.V - 1);
    const float v = Elem<T>::to_f(z[c]) * w, in = mk ? mk[c] : 1.f;
    s[k] = i < a.V && in != 0.f ? v : -INFINITY;
    m = fmaxf(m, s[k]);
  }
  const LikeGiven given = like_given<T>(a, t, z, mk, w);
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
  const float lt = like_log_total(st);
  if (lane == 0) like_finish(a, row, st, lt, given);
  if (!a.K) return;
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
    if (lane == 0) { a.top_logp[(long long)row * a.K + rank] = some ? (bs - st.M) - lt : bs; a.top_index[(long long)row * a.K + rank] = some ? bi : -1; }
    last_s = bs; last_i = bi;
  }
}

struct LikeBwdArgs {
  const void* z; long long ldz; const float* w; int J; const float* mask; int mask_rows; const long long* index;
  const float* stats; const float* entropy; const float* glogp; const float* gentropy;
  void* gz; float* gw_part; long long rows; int V, chunks;
};

// What dL/ds of a value has to know about its row.
// dL/dw_j of a row is sum ds z.  The ds add up to 0 -- or to -g where the given pixel has no probability --, so the row's largest logit zr is taken out of
// every z: what is left of the sum does not cancel, also where the logits are 1e38.
struct LikeRow { float M, lt, H, g, h, zr; long long t; };
__device__ __forceinline__ LikeRow like_row(const LikeBwdArgs& a, unsigned row, float w) {
  LikeRow o;
  o.M = a.stats[2ll * row]; o.lt = a.stats[2ll * row + 1];
  o.t = a.index ? a.index[row] : -1;
  o.g = a.glogp && o.t >= 0 ? a.glogp[row] : 0.f;
  o.h = a.gentropy ? a.gentropy[row] : 0.f;
  o.H = a.entropy[row];
  if (o.t >= a.V) o.g = NAN;                                       // (as the log likelihood of such a pixel)
  o.zr = w != 0.f && o.M > -INFINITY ? o.M / w : 0.f;              // the logit at the maximum
  return o;
}
__device__ __forceinline__ float like_ds(const LikeRow& o, float s) {
  const float lp = (s - o.M) - o.lt, p = __expf(lp);
  const float ds = -p * (o.g + o.h * (fmaxf(lp, -1e30f) + o.H));
  return s == -INFINITY ? 0.f : ds;                                // no probability: masked, or the row has no pixel at all
}
// ... of the given pixel
__device__ __forceinline__ float like_ds_given(const LikeRow& o, float s) {
  const float lp = (s - o.M) - o.lt, p = __expf(lp);
  return s == -INFINITY ? 0.f : -o.g * expm1f(lp) - p * o.h * (fmaxf(lp, -1e30f) + o.H);
}

// The gradient, 4096 values of a row per workgroup.  The rows are taken from the last to the first -- the forward pass went the other way, and what it read
// last is still in the memory-side cache -- and the gradient is stored past the caches, which keep z instead.  Forward and backward of 4096 rows of 50001
// bf16: 323 us, with both 255 (reading z twice and writing once at copy rate: 249); 5376 rows of 16384 fp32: 205 and 179.
constexpr int kLikeBwdChunk = 4096;     // 256 threads x 16
template <typename T>
__global__ __launch_bounds__(256) void like_bwd_kernel(LikeBwdArgs a) {
  constexpr int VPT = kLikeBwdChunk / 256, N = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned Bits;
  __shared__ float red[4];
  const int tid = threadIdx.x;
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const unsigned row = block / (unsigned)a.chunks;
  // (a last chunk of less than one piece reads what lies before it too, and writes its own)
  const int chunk = (int)(block - row * (unsigned)a.chunks), first = chunk * kLikeBwdChunk;
  const int n = min(a.V - first, kLikeBwdChunk), base = n < N ? a.V - N : first, own = first - base, len = n < N ? N : n;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  T* gz = reinterpret_cast<T*>(a.gz) + row * (long long)a.V + base;
  const float* mk = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const LikeRow o = like_row(a, row, w);
  float v[VPT], s[VPT];
  RowPart<T, 256, VPT> part;
  part.load(z + base, mk ? mk + base : nullptr, len);
  part.values(mk != nullptr, len, w, v, s);
  const int t = o.t >= first && o.t < first + n ? (int)(o.t - base) : -1;
  float gw = 0.f, st = 0.f, vt = 0.f;
  bool mine = false;
#pragma unroll
  for (int k = 0; k < VPT; k += N) {
    const int i = value_index<T, 256>(k);
    Piece<T> q;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float ds = like_ds(o, s[k + e]);
      q.v[e] = Elem<T>::from_f(ds * w);
      if (i + e == t) { mine = true; st = s[k + e]; vt = v[k + e]; ds = 0.f; }
      if (ds != 0.f && i + e >= own) gw = fmaf(ds, v[k + e] - o.zr, gw);
    }
    if (i >= own && i + N <= len) __builtin_nontemporal_store(__builtin_bit_cast(Bits, q), reinterpret_cast<Bits*>(gz + i));
    else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e >= own && i + e < len) gz[i + e] = q.v[e];
    }
  }
  if (mine) {                                                      // (after its neighbours: the same thread's stores stay in order)
    const float ds = like_ds_given(o, st);
    gz[t] = Elem<T>::from_f(ds * w);
    if (ds != 0.f) gw = fmaf(ds, vt - o.zr, gw);
    if (o.g != 0.f && st == -INFINITY && o.M > -INFINITY) gw -= o.g * o.zr;
  }
  if (a.gw_part) {
    gw = block_sum1(gw, red);
    if (tid == 0) a.gw_part[block] = gw;
  }
}

template <typename T, int VPT>
__global__ __launch_bounds__(256) void like_bwd_wave_kernel(LikeBwdArgs a) {
  const int lane = threadIdx.x & 63;
  const unsigned row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const float w = a.w ? a.w[row % (unsigned)a.J] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
  T* gz = reinterpret_cast<T*>(a.gz) + row * (long long)a.V;
  const float* mk = a.mask ? a.mask + (long long)(row / (unsigned)a.mask_rows) * a.V : nullptr;
  const LikeRow o = like_row(a, row, w);
  float gw = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * 64 + lane, c = min(i, a.V - 1);
    const float x = Elem<T>::to_f(z[c]), s = mk && mk[c] == 0.f ? -INFINITY : x * w;
    float ds = like_ds(o, s);
    if (i == o.t) {
      ds = like_ds_given(o, s);
      if (o.g != 0.f && s == -INFINITY && o.M > -INFINITY) gw -= o.g * o.zr;
    }
    if (i < a.V) {
      if (ds != 0.f) gw = fmaf(ds, x - o.zr, gw);
      gz[i] = Elem<T>::from_f(ds * w);
    }
  }
  if (a.gw_part) {
    gw = wave_sum(gw);
    if (lane == 0) a.gw_part[row] = gw;
  }
}

// gw[j] = the partial sums of the rows of joint j, in their order.  In 64 bits: a thread adds every 256th of them, thousands where the rows are many.
__global__ __launch_bounds__(256) void like_gw_kernel(const float* __restrict__ part, float* __restrict__ gw, long long samples, int J, int chunks) {
  __shared__ double red[4];
  const int j = blockIdx.x;
  double s = 0.0;
  for (long long k = threadIdx.x; k < samples * chunks; k += 256) s += part[((k / chunks) * J + j) * chunks + k % chunks];
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) gw[j] = (float)((red[0] + red[1]) + (red[2] + red[3]));
}

}  // namespace pwr

using namespace pwr;

// Values per workgroup of a row that is split: as many as the registers of 512 threads hold -- but a few long rows do not fill 256 CUs that way, so
// the chunk is halved (down to 4096) until the launch has 256 workgroups, as long as a row's alternatives still fit the join.
constexpr int kLikeJoin = 4096;         // candidates of all chunks of a row
static int like_chunk(long long rows, int V, int K) {
  int c = kLikeChunk;
  while (V > c && c > 4096 && rows * ((V + c - 1) / c) < 256 && (V + c / 2 - 1) / (c / 2) * (long long)K <= kLikeJoin) c >>= 1;
  return c;
}
static int like_chunks(long long rows, int V, int K) {
  const int c = like_chunk(rows, V, K);
  return (int)((V + (long long)c - 1) / c);
}
// a launch has at most 2^32 - 1 threads
static bool like_fits(long long blocks, int threads) { return blocks <= 0xffffffffll / threads; }
// what the kernels count in 32 bits (and no product of the checks below leaves 64)
static bool like_countable(long long rows, int V) { return rows <= 0xffffffffll && V <= kLikeMaxRow; }

// rows that one workgroup each walks
static bool like_walks(long long rows, int V, int K) { return !K && V > 4096 && (rows >= kLikeWalkRows || like_chunks(rows, V, K) == 1); }

extern "C" size_t pwr_likelihood_workspace_bytes(long long rows, int V, int K) {
  if (rows <= 0 || V <= 0 || K < 0 || !like_countable(rows, V) || like_walks(rows, V, K)) return 0;
  const int n = like_chunks(rows, V, K);
  return n == 1 ? 0 : (size_t)rows * n * (16 + 8 * (size_t)K);
}

template <typename T, bool TOP>
static int like_forward(const LikeArgs& a, hipStream_t s) {
  const long long rows = a.rows;
  if (a.V <= kLikeWaveMax) {
    if (!like_fits((rows + 3) / 4, 256)) return PWR_EUNSUPPORTED;
    const dim3 g((unsigned)((rows + 3) / 4));
    if (a.V <= 64) hipLaunchKernelGGL((like_fwd_wave_kernel<T, 1>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((like_fwd_wave_kernel<T, 8>), g, dim3(256), 0, s, a);
    return (int)hipGetLastError();
  }
  constexpr int N = 16 / sizeof(T);
  if constexpr (!TOP) {
    if (like_walks(rows, a.V, 0)) {
      if (!like_fits(rows, 256)) return PWR_EUNSUPPORTED;
      hipLaunchKernelGGL((like_walk_kernel<T, 256, 16>), dim3((unsigned)rows), dim3(256), 0, s, a);
      return (int)hipGetLastError();
    }
  }
  if (!like_fits(rows * a.chunks, a.V <= 256 * N ? 256 : 1024)) return PWR_EUNSUPPORTED;
  const dim3 g((unsigned)(rows * a.chunks));
  if (a.chunks == 1) {
    if (a.V <= 256 * N) hipLaunchKernelGGL((like_fwd_kernel<T, 256, N, false, TOP>), g, dim3(256), 0, s, a);
    else if (a.V <= 1024 * N) hipLaunchKernelGGL((like_fwd_kernel<T, 1024, N, false, TOP>), g, dim3(1024), 0, s, a);
    else if constexpr (TOP) hipLaunchKernelGGL((like_fwd_kernel<T, 512, 32, false, true>), g, dim3(512), 0, s, a);
    return (int)hipGetLastError();
  }
  if (a.chunk <= 1024 * N) hipLaunchKernelGGL((like_fwd_kernel<T, 1024, N, true, TOP>), g, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((like_fwd_kernel<T, 512, 32, true, TOP>), g, dim3(512), 0, s, a);
  const int n = a.chunks * a.K;
  if (n <= 256) hipLaunchKernelGGL((like_join_kernel<T, 1>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else if (n <= 1024) hipLaunchKernelGGL((like_join_kernel<T, 4>), dim3((unsigned)rows), dim3(256), 0, s, a);
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
  if (K > kLikeMaxTop || !like_countable(rows, V)) return PWR_EUNSUPPORTED;
  const bool walks = like_walks(rows, V, K);
  a.chunk = walks ? V : like_chunk(rows, V, K);
  a.chunks = walks ? 1 : like_chunks(rows, V, K);
  if ((long long)a.chunks * K > kLikeJoin || rows * a.chunks > 0x7fffffffll) return PWR_EUNSUPPORTED;
  if (a.chunks > 1) {
    if (!workspace || workspace_bytes < pwr_likelihood_workspace_bytes(rows, V, K)) return PWR_ENOSPACE;
    a.part = (float*)workspace;
    a.cand_s = a.part + 4 * rows * a.chunks;
    a.cand_i = (int*)(a.cand_s + rows * a.chunks * K);
  }
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PWR_F32) return K ? like_forward<float, true>(a, s) : like_forward<float, false>(a, s);
  return K ? like_forward<bf16_t, true>(a, s) : like_forward<bf16_t, false>(a, s);
}

static int like_bwd_chunks(int V) { return V <= kLikeWaveMax ? 1 : (V + kLikeBwdChunk - 1) / kLikeBwdChunk; }

extern "C" size_t pwr_likelihood_bwd_workspace_bytes(long long rows, int V) {
  return rows <= 0 || V <= 0 || !like_countable(rows, V) ? 0 : (size_t)rows * like_bwd_chunks(V) * 4;
}

template <typename T>
static void like_backward(const LikeBwdArgs& a, hipStream_t s) {
  if (a.V <= kLikeWaveMax) {
    const dim3 g((unsigned)((a.rows + 3) / 4));
    if (a.V <= 64) hipLaunchKernelGGL((like_bwd_wave_kernel<T, 1>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((like_bwd_wave_kernel<T, 8>), g, dim3(256), 0, s, a);
  } else hipLaunchKernelGGL((like_bwd_kernel<T>), dim3((unsigned)(a.rows * a.chunks)), dim3(256), 0, s, a);
}

extern "C" int pwr_likelihood_bwd(const void* z, long long ldz, const float* w, int J, const float* mask, int mask_rows, const long long* index,
                                  const float* stats, const float* entropy, const float* glogp, const float* gentropy, void* gz, float* gw,
                                  long long rows, int V, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0 && !gw) return 0;
  if (rows < 0 || V <= 0 || J <= 0 || mask_rows <= 0 || ldz < 0 || (rows && (!z || !stats || !entropy || !gz)) || (gw && (!w || rows % J))) return PWR_EINVAL;
  if (dtype != PWR_F32 && dtype != PWR_BF16) return PWR_EINVAL;
  if (!like_countable(rows, V)) return PWR_EUNSUPPORTED;
  LikeBwdArgs a = {z, ldz, w, J, mask, mask_rows, index, stats, entropy, glogp, gentropy, gz, nullptr, rows, V, like_bwd_chunks(V)};
  if (!like_fits(V <= kLikeWaveMax ? (rows + 3) / 4 : rows * a.chunks, 256) || (gw && !like_fits(J, 256))) return PWR_EUNSUPPORTED;
  if (gw) {
    if (rows && (!workspace || workspace_bytes < pwr_likelihood_bwd_workspace_bytes(rows, V))) return PWR_ENOSPACE;
    a.gw_part = (float*)workspace;
  }
  hipStream_t s = (hipStream_t)stream;
  if (rows) { if (dtype == PWR_F32) like_backward<float>(a, s); else like_backward<bf16_t>(a, s); }
  if (gw) hipLaunchKernelGGL(like_gw_kernel, dim3(J), dim3(256), 0, s, a.gw_part, gw, rows / J, J, a.chunks);
  return (int)hipGetLastError();
}
