// The next token under temperature, top-k, top-p and min-p, from one given uniform number a row.
//
//   order: logits falling, equal ones by index;   w_i = exp((x_i - max) * inv_temp)
//   top-k: the first k of the order;  top-p: of those, every one before which the sum of w is <= top_p * their total
//   min-p: w_i >= min_p;  W = sum of the kept w;  token = the lowest index whose running sum (by index) passes u * W
//   log-prob = ln(w / W); a greedy row takes the first of the order and its log-prob over all tokens
//
// A token next to a border (of the nucleus, or of u) must not depend on how a sum was rounded, so weights and sums are 64-bit floats.
//
// One thread-block cluster = one row; its blocks hold the row in their shared memory, so that the logits are read from memory once,
// and exchange what they find through distributed shared memory.
//   (1) Load; every thread leaves the largest of its logits (its peak). The k-th largest peak bounds the k-th largest logit from below, and
//       closely while k is small against the number of threads.
//   (2) A usual row: everything down to that bound (k = top_k, or 256 for a nucleus) goes to a list in the first block while the exact
//       total is summed; the sums say whether the nucleus is in the list, and the first block sorts it and finishes alone.
//   (3) A longer nucleus: a histogram of the depth below the maximum in steps of 1/64 nat. The edges of the bins bound the sums before and
//       behind each bin, which leaves a bin or two in which the border can lie. What comes before is kept and only summed, what is in them is
//       listed, and the first block finds the last value that is kept and how many tokens with that value are.
//   (4) Where even those bins are too full (thousands of equal logits, a long top-k), the range is cut again, until one value is left.
// Then the blocks sum their kept weights by index, and the one in whose share u * W falls looks for the token.
//
// Measured (one B200, 151936 logits, device time): 1 row top-k 19 us, 64 rows of nuclei 94 us, of min-p 44 us, 256 rows of all kinds 170 us. Reading the logits
// would take 0.1, 6 and 24 us: the time goes to a row's chain of steps (18 us for a usual row, 42 for a nucleus of tens of thousands), of which
// 33 rows run at a time (two blocks on an SM, and whole clusters of eight in a GPC); inside them to issue slots, shared-memory atomics and the exchanges. (Read again
// from the second-level cache instead, with clusters of four and twice the rows at a time, the same cases took 21, 99 and 178 us where this took 19, 99 and 181.)
#include <cmath>

#include <cooperative_groups.h>

#include "common.cuh"

namespace ab2 {
namespace cg = cooperative_groups;

constexpr int SF_THREADS = 512, SF_WARPS = SF_THREADS / 32;
constexpr int SF_BINS = 2048;          // four for each thread
constexpr int SF_CAP = 2048;           // entries of the list
constexpr int SF_SEG = 256;            // logits of a piece of a block's share that has a sum of its own
constexpr int SF_SEGS = 200;           // at most
constexpr float SF_FAR = 52.f;         // nats below the maximum from where tokens are left out of a total: 2^19 of them sum to less than 2^-56 of it
constexpr int SF_LOADS = 10;           // 16-byte loads of a thread on their way: a share of 20480 logits at once
constexpr int SF_GUESS = 256;          // tokens of a nucleus that is tried without a histogram of the row
constexpr int SF_MAX_CLUSTER = 8;
constexpr float SF_PER_NAT = 64.f;
constexpr double SF_NONE = 0x1p-1015;  // weights above it count: the smallest is e^-700.0005, above 2^-1010; 2^19 tokens without weight sum to less than 2^-1023

struct SampleArgs {
  const float* logits;
  long long ld;
  const float *u, *inv_temp, *top_p, *min_p;
  const int *top_k, *greedy;           // greedy may be null
  int* out_tok;
  float* out_logp;
  int V, share;                        // share: logits of one block, a multiple of 4
  int aligned;                         // rows start on 16 bytes
  int index_shift;                     // index >> index_shift numbers at most SF_BINS buckets
  double tab[32];                      // 2^(j/32)
};

struct SampleShared {
  unsigned long long list[SF_CAP];
  unsigned int hist[SF_BINS];
  float peak[SF_THREADS];              // the largest logit of each thread's
  uint2 hist16[SF_BINS / 4];           // the same in 16 bits, for the other blocks (a share is below 65536)
  double tab[32];                      // 2^(j/32): the entries of a half warp fall on banks of their own
  double seg_sum[SF_SEGS];
  int seg_tie[SF_SEGS];
  // what the blocks of the cluster tell one another; two sets in turn, since a fast block may write the next before a slow one has read
  double pub_sum[2][SF_MAX_CLUSTER], pub_sum2[2][SF_MAX_CLUSTER];
  float pub_hi[2][SF_MAX_CLUSTER], pub_lo[2][SF_MAX_CLUSTER], pub_hi2[2][SF_MAX_CLUSTER], pub_lo2[2][SF_MAX_CLUSTER];
  int pub_int[2][SF_MAX_CLUSTER];
  double red[SF_WARPS], red2[SF_WARPS];
  float fred[4][SF_WARPS];
  int ired[SF_WARPS];
  float thr;
  int ties, list_n, cut[4];
  unsigned int arg[6];                 // of the row: inv_temp, top_p, min_p, u, top_k, greedy
};

// exp(d) for d <= 0 in 64 bits: exp(d) = 2^k * 2^(j/32) * exp(r), |r| <= ln 2 / 64, the last by its Taylor polynomial (table-driven
// exponentials after P. T. P. Tang, 1989; relative error below 2e-12). From -(700 + 2^-11) down a token has no weight: what is returned there is below 2^-1042 (its
// high word is cleared; clearing the low one too cost 8 %), in sums nothing, and below SF_NONE however many there are.
__device__ __forceinline__ double weight(double d, const double* tab) {
  const double big = 6755399441055744.0;                       // 1.5 * 2^52: adding it rounds to a whole number
  const double t = fma(d, 46.166241308446828, big);            // 32 / ln 2
  const int k = __double2loint(t);
  const double r = fma(t - big, -0.021660849392498290, d);     // ln 2 / 32
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double w = p * tab[k & 31];
  // (the high word of a negative number rises as it falls, 2^-11 at a time here; minus infinity and NaN are above them all)
  const bool gone = (unsigned int)__double2hiint(d) > 0xc085e000u;
  return __hiloint2double(gone ? 0 : __double2hiint(w) + ((k >> 5) << 20), __double2loint(w));
}
// Order-preserving map of floats to unsigned; the two zeros are one value.
__device__ __forceinline__ unsigned int key_of(float x) {
  const unsigned int b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int warp_sum_i(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sorts list[0 .. n2), n2 a power of two, falling.
__device__ __forceinline__ void sort_falling(unsigned long long* list, int n2) {
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n2 / 2; i += SF_THREADS) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const unsigned long long x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
      }
      __syncthreads();
    }
}
__device__ __forceinline__ int pow2_above(int n) {
  int p = 2;
  while (p < n) p <<= 1;
  return p;
}

// Sorts list[0 .. n) falling, n <= SF_CAP, given each entry's bucket (rising as the keys fall) and end[b] = entries of the buckets before b on
// entry: an entry goes behind what its bucket holds already, and then to its rank among the few of its bucket. Keys are all different.
// With VALUES the order of equal values (the keys' high halves) is left open, and a bucket of one value is left alone.
template <bool VALUES = false, typename F>
__device__ __forceinline__ void sort_buckets(unsigned long long* list, int n, unsigned int* end, F bucket) {
  unsigned long long e[SF_CAP / SF_THREADS];
  int at[SF_CAP / SF_THREADS];
#pragma unroll
  for (int j = 0; j < SF_CAP / SF_THREADS; ++j) {
    const int i = threadIdx.x + j * SF_THREADS;
    if (i < n) {
      e[j] = list[i];
      at[j] = atomicAdd(&end[bucket(e[j])], 1u);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < SF_CAP / SF_THREADS; ++j)
    if ((int)threadIdx.x + j * SF_THREADS < n) list[at[j]] = e[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < SF_CAP / SF_THREADS; ++j)
    if ((int)threadIdx.x + j * SF_THREADS < n) {
      const int b = bucket(e[j]), last = (int)(end[b] & 0xffffu);
      const int from = b > 0 ? (int)(end[b - 1] & 0xffffu) : 0;
      if constexpr (VALUES) {
        // a mark in the bucket's high half: it holds two values
        if ((list[from] ^ e[j]) >> 32) atomicOr(&end[b], 0x10000u);
      } else {
        int r = from;
        for (int i = from; i < last; ++i) r += list[i] > e[j];
        at[j] = r;
      }
    }
  __syncthreads();
  if constexpr (VALUES) {
#pragma unroll
    for (int j = 0; j < SF_CAP / SF_THREADS; ++j)
      if ((int)threadIdx.x + j * SF_THREADS < n) {
        const int b = bucket(e[j]), last = (int)(end[b] & 0xffffu);
        if (end[b] >> 16) {
          int r = b > 0 ? (int)(end[b - 1] & 0xffffu) : 0;
          const int from = r;
          for (int i = from; i < last; ++i) r += list[i] > e[j];
          at[j] = r;
        }
      }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < SF_CAP / SF_THREADS; ++j)
    if ((int)threadIdx.x + j * SF_THREADS < n) list[at[j]] = e[j];
  __syncthreads();
}

// Sum over the block of each thread's value before this thread (exclusive, in thread order), and the total.
// Where only the first `warps` warps have any, theirs are enough.
__device__ __forceinline__ double block_scan(double v, double* red, double* total, int warps = SF_WARPS) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  // every warp sums the warps' totals: lane w takes warp w's
  double p = lane < warps ? red[lane] : 0.0;
#pragma unroll
  for (int o = 1; o < SF_WARPS; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, p, o);
    if (lane >= o) p += t;
  }
  const double all = __shfl_sync(0xffffffffu, p, SF_WARPS - 1), before = warp ? __shfl_sync(0xffffffffu, p, warp - 1) : 0.0;
  *total = all;
  return before + (s - v);
}
__device__ __forceinline__ float block_scan_f(float v, float* red, float* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  float p = lane < SF_WARPS ? red[lane] : 0.f;
#pragma unroll
  for (int o = 1; o < SF_WARPS; o <<= 1) {
    const float t = __shfl_up_sync(0xffffffffu, p, o);
    if (lane >= o) p += t;
  }
  const float all = __shfl_sync(0xffffffffu, p, SF_WARPS - 1), before = warp ? __shfl_sync(0xffffffffu, p, warp - 1) : 0.f;
  *total = all;
  return before + (s - v);
}
__device__ __forceinline__ int block_scan_i(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  int p = lane < SF_WARPS ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < SF_WARPS; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, p, o);
    if (lane >= o) p += t;
  }
  const int all = __shfl_sync(0xffffffffu, p, SF_WARPS - 1), before = warp ? __shfl_sync(0xffffffffu, p, warp - 1) : 0;
  *total = all;
  return before + s - v;
}

// The range of values that is being cut into bins: x in [lo, hi], bin = (hi - x) * scale, the last bin open below.
struct Range {
  float hi, lo;
  double scale;
  bool first;                          // the whole row, 64 bins a nat: single precision is enough
};
__device__ __forceinline__ int bin_of(const Range& r, float x) {
  if (r.first) return (int)fminf((r.hi - x) * (float)r.scale, (float)(SF_BINS - 1));
  return (int)fmin(((double)r.hi - (double)x) * r.scale, (double)(SF_BINS - 1));
}

__global__ void __launch_bounds__(SF_THREADS, 2) sample_filtered_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dsm[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(dsm);
  float* xs = reinterpret_cast<float*>(dsm + (sizeof(SampleShared) + 15) / 16 * 16);
  cg::cluster_group cl = cg::this_cluster();
  const int nb = cl.num_blocks(), me = cl.block_rank();
  const int row = blockIdx.x / nb, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const int begin = min(me * a.share, a.V), n = min(a.share, a.V - begin);       // this block's logits
  int buf = 0;                                                                   // set of the published values in use
  // the row's arguments are read once, beside the logits, and the first block's are everyone's: all blocks take the same path
  unsigned int arg = 0u;
  if (me == 0 && tid < 6) {
    const void* p = tid == 0 ? (const void*)a.inv_temp : tid == 1 ? a.top_p : tid == 2 ? a.min_p : tid == 3 ? a.u : tid == 4 ? (const void*)a.top_k : a.greedy;
    if (p) arg = reinterpret_cast<const unsigned int*>(p)[row];
  }
  // ---- the row into shared memory, its maximum
  float mx = -INFINITY;
  {
    const float* src = a.logits + (size_t)row * a.ld + begin;
    auto clean = [](float x) { return fmaxf(x, -INFINITY); };               // NaN has no weight
    if (a.aligned) {
      const int n4 = n >> 2;
      for (int i0 = tid; i0 < n4; i0 += SF_LOADS * SF_THREADS) {
        float4 v[SF_LOADS];                                                 // all on their way before the first is used
#pragma unroll
        for (int j = 0; j < SF_LOADS; ++j)
          v[j] = i0 + j * SF_THREADS < n4 ? __ldcs(reinterpret_cast<const float4*>(src) + i0 + j * SF_THREADS) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
        for (int j = 0; j < SF_LOADS; ++j) {
          v[j].x = clean(v[j].x); v[j].y = clean(v[j].y); v[j].z = clean(v[j].z); v[j].w = clean(v[j].w);
          if (i0 + j * SF_THREADS < n4) reinterpret_cast<float4*>(xs)[i0 + j * SF_THREADS] = v[j];
          mx = fmaxf(mx, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
        }
      }
      for (int i = 4 * n4 + tid; i < n; i += SF_THREADS) { const float v = clean(src[i]); xs[i] = v; mx = fmaxf(mx, v); }
    } else {
      for (int i = tid; i < n; i += SF_THREADS) { const float v = clean(src[i]); xs[i] = v; mx = fmaxf(mx, v); }
    }
    for (int i = max(n, 0) + tid; i < a.share; i += SF_THREADS) xs[i] = -INFINITY;
  }
  for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
  if (tid < 32) sh.tab[tid] = a.tab[tid];
  if (tid == 0) sh.list_n = 0;
  if (me == 0 && tid < 6) sh.arg[tid] = arg;
  sh.peak[tid] = mx;
  cl.sync();
  if (me != 0 && tid < 6) sh.arg[tid] = cl.map_shared_rank(sh.arg, 0)[tid];
  float peaks[SF_MAX_CLUSTER], xmax = -INFINITY;                                 // every block looks at all threads' largest
#pragma unroll
  for (int i = 0; i < SF_MAX_CLUSTER; ++i) {
    peaks[i] = i < nb ? cl.map_shared_rank(sh.peak, i)[tid] : -INFINITY;
    xmax = fmaxf(xmax, peaks[i]);
  }
  xmax = warp_max(xmax);
  if (lane == 0) sh.fred[0][warp] = xmax;
  __syncthreads();
  xmax = warp_max(sh.fred[0][lane % SF_WARPS]);
  if (xmax == -INFINITY) {                                                       // nothing has any weight
    if (me == 0 && tid == 0) { a.out_tok[row] = -1; a.out_logp[row] = -INFINITY; }
    cl.sync();                                                                   // the others may still be reading this block's peaks
    return;
  }
  if (xmax == INFINITY) {                                                        // only infinite logits have weight, all the same
    for (int i = tid; i < a.share; i += SF_THREADS) xs[i] = xs[i] == INFINITY ? 0.f : -INFINITY;
#pragma unroll
    for (int i = 0; i < SF_MAX_CLUSTER; ++i) peaks[i] = peaks[i] == INFINITY ? 0.f : -INFINITY;
    xmax = 0.f;
  }
  __syncthreads();
  const float it_in = __uint_as_float(sh.arg[0]), tpf = __uint_as_float(sh.arg[1]), mpf = __uint_as_float(sh.arg[2]);
  const bool greedy = sh.arg[5] != 0u;
  int K = (int)sh.arg[4];
  const float itf = it_in >= 0.f ? fminf(it_in, 1e30f) : 0.f;
  const double it = (double)itf, top = (double)xmax;
  const double top_it = top * it;
  // the same for every use of a logit: (x - max) * inv_temp in one rounding
  auto w_of = [&](float x) { return x == xmax ? 1.0 : weight(fma((double)x, it, -top_it), sh.tab); };
  const double top_p = (double)fmaxf(tpf, 0.f), min_p = (double)fminf(mpf, 1.f);
  const bool by_mass = !greedy && tpf < 1.f;
  if (greedy || K <= 0 || K >= a.V) K = 0;
  const bool by_min = !greedy && min_p > 0.0;

  // publishes one sum for each block; after the next cluster barrier pub_sum[buf] has them all
  auto publish_sum = [&](double v) {
    v = warp_sum_d(v);
    __syncthreads();
    if (lane == 0) sh.red[warp] = v;
    __syncthreads();
    if (tid < nb) {
      double s = 0.0;
#pragma unroll
      for (int w = 0; w < SF_WARPS; ++w) s += sh.red[w];
      cl.map_shared_rank(&sh, tid)->pub_sum[buf][me] = s;
    }
  };
  auto all_sum = [&]() {
    double s = 0.0;
    for (int i = 0; i < nb; ++i) s += sh.pub_sum[buf][i];
    return s;
  };

  if (greedy) {
    double s = 0.0;
    int first = 0x7fffffff;
#pragma unroll 2
    for (int i = tid; i < a.share / 4; i += SF_THREADS) {
      const float4 v = reinterpret_cast<const float4*>(xs)[i];
      const float x[4] = {v.x, v.y, v.z, v.w};
      double w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
        if (x[j] == xmax) { first = min(first, begin + 4 * i + j); w[j] = 1.0; }
      }
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.ired[warp] = first;
    publish_sum(s);                                                              // its barriers cover ired too
    if (tid < nb) {
      int f = sh.ired[0];
#pragma unroll
      for (int w = 1; w < SF_WARPS; ++w) f = min(f, sh.ired[w]);
      cl.map_shared_rank(&sh, tid)->pub_int[buf][me] = f;
    }
    cl.sync();
    if (me == 0 && tid == 0) {
      int f = 0x7fffffff;
      for (int i = 0; i < nb; ++i) f = min(f, sh.pub_int[buf][i]);
      a.out_tok[row] = f;
      a.out_logp[row] = (float)-log(all_sum());
    }
    return;
  }

  float thr = -INFINITY;                // kept: x > thr, and the first `ties` (by index) of those equal to it
  int ties = 0;
  double total = 0.0;                   // what top_p is a share of
  // The list holds, in order (a long one by value only), everything that can be kept: what of it is, and the token.
  auto finish = [&](int cnt) {
    const int k = K > 0 ? min(K, cnt) : cnt;
    if (cnt <= SF_THREADS) {
      // one thread for each: its place in the sum by index is found by going through them all
      double* ws = reinterpret_cast<double*>(sh.hist);
      const unsigned long long e = tid < cnt ? sh.list[tid] : 0ull;
      const double w = tid < k ? w_of(float_of((unsigned int)(e >> 32))) : 0.0;
      double sum;
      const double run = block_scan(w, sh.red, &sum, (cnt + 31) >> 5);
      const bool kept = w > SF_NONE && (!by_mass || run <= top_p * (K > 0 ? sum : total)) && w >= min_p;
      const int m = max(1, __syncthreads_count(kept));                            // its barrier also ends the use of hist
      const int index = (int)(0xffffffffu - (unsigned int)e);
      if (tid < m) ws[tid] = w;
      if (tid == 0) { sh.cut[0] = 0x7fffffff; sh.cut[1] = -1; }
      if (tid == m - 1) sh.red2[0] = run + w;
      __syncthreads();
      const double all = sh.red2[0], goal = fmax((double)__uint_as_float(sh.arg[3]) * all, SF_NONE);
      if (tid < m) {
        double q[4] = {0.0, 0.0, 0.0, 0.0};
        for (int j = 0; j < m; j += 4) {
#pragma unroll
          for (int h = 0; h < 4; ++h)
            if (j + h < m && (int)(0xffffffffu - (unsigned int)sh.list[j + h]) <= index) q[h] += ws[j + h];
        }
        if ((q[0] + q[1]) + (q[2] + q[3]) > goal) atomicMin(&sh.cut[0], index);
        atomicMax(&sh.cut[1], index);
      }
      __syncthreads();
      const int tok = sh.cut[0] != 0x7fffffff ? sh.cut[0] : sh.cut[1];
      if (tid < m && index == tok) {
        a.out_tok[row] = tok;
        a.out_logp[row] = (float)log(w / all);
      }
      return;
    }
    double w[4], mine = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * tid + j;
      w[j] = i < k ? w_of(float_of((unsigned int)(sh.list[i] >> 32))) : 0.0;
      mine += w[j];
    }
    double sum;
    double run = block_scan(mine, sh.red, &sum);
    const double all = K > 0 ? sum : total;
    int kept = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * tid + j;
      if (i < k && w[j] > SF_NONE && (!by_mass || run <= top_p * all) && w[j] >= min_p) ++kept;
      run += w[j];
    }
    int m;
    block_scan_i(kept, sh.ired, &m);
    if (m == 0) m = 1;
    // a long list is in order by value only: of the entries equal to the last kept one, those with the lowest indices go first
    const unsigned int edge = (unsigned int)(sh.list[m - 1] >> 32);
    if (m < cnt && (unsigned int)(sh.list[m] >> 32) == edge) {
      int above = 0, same = 0;
      for (int i = tid; i < cnt; i += SF_THREADS) {
        const unsigned int v = (unsigned int)(sh.list[i] >> 32);
        above += v > edge;
        same += v == edge;
      }
      int from, size;
      block_scan_i(above, sh.ired, &from);
      block_scan_i(same, sh.ired, &size);
      unsigned long long e[SF_CAP / SF_THREADS];
      int at[SF_CAP / SF_THREADS];
#pragma unroll
      for (int j = 0; j < SF_CAP / SF_THREADS; ++j) {
        const int i = tid + j * SF_THREADS;
        at[j] = -1;
        if (i >= from && i < from + size) {
          e[j] = sh.list[i];
          at[j] = from;
          for (int q = from; q < from + size; ++q) at[j] += sh.list[q] > e[j];
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < SF_CAP / SF_THREADS; ++j)
        if (at[j] >= 0) sh.list[at[j]] = e[j];
    }
    __syncthreads();
    // the kept ones by index: the key's low half, the index's complement, to the front
    for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
    __syncthreads();
    auto bucket = [&](unsigned long long e) { return (int)((0xffffffffu - (unsigned int)(e >> 32)) >> a.index_shift); };
    for (int i = tid; i < m; i += SF_THREADS) {
      const unsigned long long e = (sh.list[i] << 32) | (sh.list[i] >> 32);
      sh.list[i] = e;
      atomicAdd(&sh.hist[bucket(e)], 1u);
    }
    __syncthreads();
    const uint4 c = reinterpret_cast<const uint4*>(sh.hist)[tid];
    int all_i;
    const unsigned int at = block_scan_i((int)(c.x + c.y + c.z + c.w), sh.ired, &all_i);
    reinterpret_cast<uint4*>(sh.hist)[tid] = make_uint4(at, at + c.x, at + c.x + c.y, at + c.x + c.y + c.z);
    __syncthreads();
    sort_buckets(sh.list, m, sh.hist, bucket);
    mine = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * tid + j;
      w[j] = i < m ? w_of(float_of((unsigned int)sh.list[i])) : 0.0;
      mine += w[j];
    }
    run = block_scan(mine, sh.red, &sum);
    const double goal = fmax((double)__uint_as_float(sh.arg[3]) * sum, SF_NONE);
    int hit = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      run += w[j];
      if (4 * tid + j < m && run > goal) hit = min(hit, 4 * tid + j);
    }
    hit = __reduce_min_sync(0xffffffffu, hit);
    __syncthreads();
    if (lane == 0) sh.ired[warp] = hit;
    __syncthreads();
    if (tid == 0) {
      for (int w2 = 1; w2 < SF_WARPS; ++w2) hit = min(hit, sh.ired[w2]);
      if (hit >= m) hit = m - 1;
      const unsigned long long v = sh.list[hit];
      a.out_tok[row] = (int)(0xffffffffu - (unsigned int)(v >> 32));
      a.out_logp[row] = (float)log(w_of(float_of((unsigned int)v)) / sum);
    }
  };

  const int n4 = a.share / 4, segs = (a.share + SF_SEG - 1) / SF_SEG;
  const float4* xs4 = reinterpret_cast<const float4*>(xs);
  bool decided = !(K > 0 || by_mass || by_min);         // thr and ties are known
  bool summed = false;                                   // s_own has this block's weights before t_sure
  double s_own = 0.0;
  float t_sure = -INFINITY;                              // a depth: what is before is kept, whatever thr is
  const float scale = itf * SF_PER_NAT, top_t = xmax * scale;
  // how far a logit is below the largest, in bins of 1/64 nat: one rounding, so it falls as the logit rises; off by 1e-3 bins at most
  // as long as `plain` holds (within 300 nats of zero: any sane row), else the general way below takes the row
  auto depth = [&](float x) { return fmaf(x, -scale, top_t); };
  const bool plain = itf >= 1e-6f && fabsf(top_t) < 300.f * SF_PER_NAT;
  bool have_total = false;
  // ---- a list guessed from the peaks: the k-th largest of the threads' largest logits bounds the k-th largest logit, so its bin and those
  // before hold k tokens at least and usually few more; for top-p it is a guess (SF_GUESS tokens), which the sums confirm or not
  if (plain && !decided && K <= nb * (SF_THREADS / 4)) {
    const int want = K > 0 ? K : SF_GUESS;
    float t_list = INFINITY;
    bool from_min = false;                               // what is not listed is dropped by min-p
    bool guess = true;
    if (K > 0 || by_mass) {
#pragma unroll
      for (int i = 0; i < SF_MAX_CLUSTER; ++i) {
        const float t = depth(peaks[i]);
        if (t < (float)(SF_BINS - 1)) atomicAdd(&sh.hist[__float2uint_rz(t)], 1u);
      }
      if (tid == 0) sh.cut[0] = SF_BINS;
      __syncthreads();
      const uint4 c = reinterpret_cast<const uint4*>(sh.hist)[tid];
      int all_i;
      int at = block_scan_i((int)(c.x + c.y + c.z + c.w), sh.ired, &all_i);
      const unsigned int cc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (at < want && at + (int)cc[j] >= want) sh.cut[0] = 4 * tid + j;
        at += (int)cc[j];
      }
      if (by_mass && K == 0) {
        // the peaks' own weights, those in front against all: a share below top_p already says that the nucleus is longer
        float e = fast_exp2(tid * (-4.f * 1.4426950408889634f / SF_PER_NAT)), m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { m += (float)cc[j] * e; e *= 0.98449643700540842f; }
        float m_all;
        const float m_before = block_scan_f(m, sh.fred[1], &m_all);
        if (sh.cut[0] < SF_BINS && sh.cut[0] >> 2 == tid) sh.fred[3][0] = m_before + m;
        __syncthreads();
        guess = sh.cut[0] >= SF_BINS || sh.fred[3][0] > (float)top_p * m_all;
      }
      reinterpret_cast<uint4*>(sh.hist)[tid] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      if (sh.cut[0] < SF_BINS) t_list = (float)(sh.cut[0] + 1);                   // the last bin is not counted above
    }
    if (by_min && !(K > 0 && by_mass)) {
      const float t = (float)(-log(min_p)) * SF_PER_NAT * 1.0001f + 1.f;          // ln(1 / min_p), and what rounding does to it
      if (t <= t_list) { t_list = t; from_min = guess = true; }
    }
    if (guess) {
      const bool to_end = t_list == INFINITY, sums = by_mass && K == 0;
      double s = 0.0, s_head = 0.0;                        // (a list that does not go to the end is no deeper than the bins, 32 nats)
      int listed = 0;                                      // lane 31: entries of this warp
#pragma unroll 2
      for (int i0 = 0; i0 < n4; i0 += SF_THREADS) {
        const int i = i0 + tid;
        const float4 v = i < n4 ? xs4[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const float x[4] = {v.x, v.y, v.z, v.w};
        float t[4];
        bool some = to_end, near = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t[j] = depth(x[j]);
          some |= t[j] < t_list;
          near |= t[j] < SF_FAR * SF_PER_NAT;
        }
        if (sums && near) {
          double w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
          s += (w[0] + w[1]) + (w[2] + w[3]);
          if (some) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s_head += to_end || t[j] < t_list ? w[j] : 0.0;
          }
        }
        if (__any_sync(0xffffffffu, some)) {
          int mine = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) mine += (to_end || t[j] < t_list) && x[j] > -INFINITY;
          int at = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int q = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += q;
          }
          int base = 0;
          if (lane == 31 && at) base = atomicAdd(&sh.list_n, at);
          listed += at;
          at += __shfl_sync(0xffffffffu, base, 31) - mine;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((to_end || t[j] < t_list) && x[j] > -INFINITY) {
              if (at < SF_CAP) sh.list[at] = ((unsigned long long)key_of(x[j]) << 32) | (0xffffffffu - (unsigned int)(begin + 4 * i + j));
              ++at;
            }
        }
      }
      if (lane == 31) sh.seg_tie[warp] = listed;
      __syncthreads();
      if (me != 0) {                                                                // the first block's list takes them all
        SampleShared* head = cl.map_shared_rank(&sh, 0);
        const int k = sh.list_n;
        if (tid == 0 && k) sh.ired[0] = atomicAdd(&head->list_n, k);
        __syncthreads();
        const int at = sh.ired[0];
        for (int i = tid; i < k && at + i < SF_CAP; i += SF_THREADS) head->list[at + i] = sh.list[i];
      }
      if (sums) {
        s = warp_sum_d(s);
        s_head = warp_sum_d(s_head);
        if (lane == 0) { sh.red[warp] = s; sh.red2[warp] = s_head; }
      }
      __syncthreads();
      if (tid < nb) {
        double q = 0.0, q2 = 0.0;
        int k = 0;
#pragma unroll
        for (int w = 0; w < SF_WARPS; ++w) {
          if (sums) { q += sh.red[w]; q2 += sh.red2[w]; }
          k += sh.seg_tie[w];
        }
        SampleShared* o = cl.map_shared_rank(&sh, tid);
        o->pub_sum[buf][me] = q;
        o->pub_sum2[buf][me] = q2;
        o->pub_int[buf][me] = k;
      }
      cl.sync();
      double in_list = 0.0;
      int cnt = 0;
      for (int i = 0; i < nb; ++i) { in_list += sh.pub_sum2[buf][i]; cnt += sh.pub_int[buf][i]; }
      if (sums) total = all_sum();
      have_total = sums;
      buf ^= 1;
      if (cnt <= SF_CAP && (!sums || to_end || from_min || in_list > top_p * total)) {
        if (me != 0) return;
        const float fine = to_end ? 1.f : (float)(SF_BINS - 1) / t_list;
        auto bucket = [&](unsigned long long q) { return (int)fmaxf(fminf(depth(float_of((unsigned int)(q >> 32))) * fine, (float)(SF_BINS - 1)), 0.f); };
        for (int i = tid; i < cnt; i += SF_THREADS) atomicAdd(&sh.hist[bucket(sh.list[i])], 1u);
        __syncthreads();
        const uint4 q = reinterpret_cast<const uint4*>(sh.hist)[tid];
        int all_i;
        const unsigned int at = block_scan_i((int)(q.x + q.y + q.z + q.w), sh.ired, &all_i);
        reinterpret_cast<uint4*>(sh.hist)[tid] = make_uint4(at, at + q.x, at + q.x + q.y, at + q.x + q.y + q.z);
        __syncthreads();
        if (cnt <= SF_THREADS) sort_buckets(sh.list, cnt, sh.hist, bucket);
        else sort_buckets<true>(sh.list, cnt, sh.hist, bucket);
        finish(cnt);
        return;
      }
    }
    if (tid == 0) sh.list_n = 0;
    decided = K == 0 && !by_mass;                        // min-p alone: every token is looked at anyway
    __syncthreads();
  }
  // ---- one histogram of the whole row, one look at what the border needs
  if (plain && !decided) {
    {
      // logits without weight fall into the last bin, which is open below. The shared-memory atomics bound this loop; the exact sums that
      // top-p needs fit between them.
      const bool sums = by_mass && K == 0 && !have_total;
      double q = 0.0;
#pragma unroll 2
      for (int i = tid; i < n4; i += SF_THREADS) {
        const float4 v = xs4[i];
        const float x[4] = {v.x, v.y, v.z, v.w};
        float t[4];
        bool near = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t[j] = depth(x[j]);
          near |= t[j] < SF_FAR * SF_PER_NAT;
          atomicAdd(&sh.hist[__float2uint_rz(fminf(t[j], (float)(SF_BINS - 1)))], 1u);
        }
        if (sums && near) {
          double w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
          q += (w[0] + w[1]) + (w[2] + w[3]);
        }
      }
      if (sums) publish_sum(q);
    }
    __syncthreads();
    {
      const uint4 v = reinterpret_cast<const uint4*>(sh.hist)[tid];
      sh.hist16[tid] = make_uint2(v.x | v.y << 16, v.z | v.w << 16);
    }
    cl.sync();
    if (by_mass && K == 0 && !have_total) { total = all_sum(); buf ^= 1; }
    unsigned int c[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
    for (int i = 0; i < nb; ++i) {
      const uint2 v = cl.map_shared_rank(sh.hist16, i)[tid];
      c[0] += v.x & 0xffffu; c[1] += v.x >> 16; c[2] += v.y & 0xffffu; c[3] += v.y >> 16;
    }
    int c_total;
    const int c_before = block_scan_i((int)(c[0] + c[1] + c[2] + c[3]), sh.ired, &c_total);
    do {
      if (tid == 0) { sh.cut[0] = SF_BINS; sh.cut[1] = SF_BINS; sh.cut[2] = c_total; sh.cut[3] = 0; }
      __syncthreads();
      if (K > 0) {
        int at = c_before;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (at < K && at + (int)c[j] >= K) { sh.cut[0] = 0; sh.cut[1] = 4 * tid + j; sh.cut[2] = at + (int)c[j]; sh.cut[3] = 0; }
          at += (int)c[j];
        }
      } else if (by_mass) {
        const float f = 0.98449643700540842f, slack = 4e-5f;                      // exp(-1 / 64)
        const float w0 = fast_exp2(tid * (-4.f * 1.4426950408889634f / SF_PER_NAT));
        float part[4], m = 0.f, e = w0;                                           // the bins' masses from below
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[j] = 4 * tid + j < SF_BINS - 1 ? (float)c[j] * e * f : 0.f;
          m += part[j];
          e *= f;
        }
        float m_all;
        float m_cum = block_scan_f(m, sh.fred[0], &m_all);
        if (tid == SF_THREADS - 1) sh.fred[1][0] = (float)c[3] * e / f;           // the open last bin, from above
        __syncthreads();
        const float last_hi = sh.fred[1][0];
        const float want = (float)(top_p * total), rest = (float)(total - top_p * total);
        int at = c_before, b1 = SF_BINS, b2 = SF_BINS, c1 = 0, c2 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m_cum += part[j];
          const bool end = 4 * tid + j == SF_BINS - 1;
          // a bin's weights lie between those of its edges, but for the last one: from those, bounds on what is before and behind a
          // bin's end. Single precision, and the rounding of x to its bin, stay well within `slack`.
          const float behind = fmaxf(m_all - m_cum, 0.f), fuzz = slack * m_all;                  // the difference of two sums is off by a part of them
          const bool maybe = m_cum / f * (1.f + slack) > want && (behind - fuzz) * (1.f - slack) < rest;
          const bool sure = m_cum * (1.f - slack) > want || ((behind + fuzz) / f + last_hi) * (1.f + slack) < rest;
          if (c[j] && (maybe || end) && b1 == SF_BINS) { b1 = 4 * tid + j; c1 = at; }
          at += (int)c[j];
          if (c[j] && (sure || end) && b2 == SF_BINS) { b2 = 4 * tid + j; c2 = at; }
        }
        if (b1 < SF_BINS) atomicMin(&sh.cut[0], b1);
        if (b2 < SF_BINS) atomicMin(&sh.cut[1], b2);
        __syncthreads();
        if (b1 < SF_BINS && sh.cut[0] == b1) sh.cut[3] = c1;
        if (b2 < SF_BINS && sh.cut[1] == b2) sh.cut[2] = c2;
      }
      __syncthreads();
      int b1 = sh.cut[0], b2 = sh.cut[1], before = sh.cut[3];
      const int upto = sh.cut[2];
      if (b2 >= SF_BINS) b2 = SF_BINS - 1;
      if (b1 > b2) b1 = before = 0;
      const bool whole = upto <= SF_CAP, part = !whole && K == 0 && upto - before <= SF_CAP;
      if (!whole && !part) break;
      const bool to_end = b2 == SF_BINS - 1;
      const float t_list = (float)(b2 + 1);
      t_sure = part && b1 > 0 ? (float)b1 : -INFINITY;                            // (the largest logit may be a rounding before zero)
      const float t_from = whole ? 0.f : (float)b1;
      SampleShared* head = cl.map_shared_rank(&sh, 0);
      double s = 0.0;
#pragma unroll 2
      for (int i0 = 0; i0 < n4; i0 += SF_THREADS) {
        {
          const int i = i0 + tid;
          const float4 v = i < n4 ? xs4[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          const float x[4] = {v.x, v.y, v.z, v.w};
          float t[4];
          bool some = false, sure = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            t[j] = depth(x[j]);
            some |= (to_end || t[j] < t_list) && !(t[j] < t_sure);
            sure |= t[j] < t_sure;
          }
          if (sure) {
            double w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = t[j] < t_sure ? w[j] : 0.0;
            s += (w[0] + w[1]) + (w[2] + w[3]);
          }
          if (__any_sync(0xffffffffu, some)) {
            int mine = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) mine += (to_end || t[j] < t_list) && !(t[j] < t_sure) && x[j] > -INFINITY;
            int at = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int q = __shfl_up_sync(0xffffffffu, at, o);
              if (lane >= o) at += q;
            }
            int base = 0;
            if (lane == 31 && at) base = atomicAdd(&sh.list_n, at);
            at += __shfl_sync(0xffffffffu, base, 31) - mine;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((to_end || t[j] < t_list) && !(t[j] < t_sure) && x[j] > -INFINITY) {
                if (at < SF_CAP) sh.list[at] = ((unsigned long long)key_of(x[j]) << 32) | (0xffffffffu - (unsigned int)(begin + 4 * i + j));
                ++at;
              }
          }
        }
      }
      __syncthreads();
      if (me != 0) {                                                   // the first block's list takes them all
        const int k = sh.list_n;
        if (tid == 0 && k) sh.ired[0] = atomicAdd(&head->list_n, k);
        __syncthreads();
        const int at = sh.ired[0];
        for (int i = tid; i < k && at + i < SF_CAP; i += SF_THREADS) head->list[at + i] = sh.list[i];
      }
      publish_sum(s);
      cl.sync();
      const double s_above = all_sum();
      s_own = sh.pub_sum[buf][me];
      buf ^= 1;
      if (whole && me != 0) return;
      const int cnt = me == 0 ? min(sh.list_n, SF_CAP) : 0;
      if (me == 0) {
        // order: by bins of the list's own range, finely enough that most hold one value. Of equal values the lowest index comes first only
        // where the list is all there is; for the last kept value and its number the order among them does not matter.
        const float fine = (float)(SF_BINS - 1) / (t_list - t_from);
        auto bucket = [&](unsigned long long q) {
          return (int)fmaxf(fminf((depth(float_of((unsigned int)(q >> 32))) - t_from) * fine, (float)(SF_BINS - 1)), 0.f);
        };
        for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
        __syncthreads();
        for (int i = tid; i < cnt; i += SF_THREADS) atomicAdd(&sh.hist[bucket(sh.list[i])], 1u);
        __syncthreads();
        const uint4 q = reinterpret_cast<const uint4*>(sh.hist)[tid];
        int all_i;
        const unsigned int at = block_scan_i((int)(q.x + q.y + q.z + q.w), sh.ired, &all_i);
        reinterpret_cast<uint4*>(sh.hist)[tid] = make_uint4(at, at + q.x, at + q.x + q.y, at + q.x + q.y + q.z);
        __syncthreads();
        if (whole && cnt <= SF_THREADS) sort_buckets(sh.list, cnt, sh.hist, bucket);
        else sort_buckets<true>(sh.list, cnt, sh.hist, bucket);
      }
      if (whole) {
        finish(cnt);
        return;
      }
      if (me == 0) {
        double w[4], mine = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * tid + j;
          w[j] = i < cnt ? w_of(float_of((unsigned int)(sh.list[i] >> 32))) : 0.0;
          mine += w[j];
        }
        double sum;
        double run = s_above + block_scan(mine, sh.red, &sum);
        int kept = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * tid + j < cnt && run <= top_p * total) ++kept;
          run += w[j];
        }
        int m;
        block_scan_i(kept, sh.ired, &m);
        const unsigned int last = m > 0 ? (unsigned int)(sh.list[m - 1] >> 32) : 0u;
        int same = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * tid + j < m && (unsigned int)(sh.list[4 * tid + j] >> 32) == last) ++same;
        int eq;
        block_scan_i(same, sh.ired, &eq);
        __syncthreads();
        if (tid < nb) {
          SampleShared* o = cl.map_shared_rank(&sh, tid);
          // nothing of the list kept (the border at its very start): what is above it, up to the lowest value that is
          o->thr = m > 0 ? float_of(last) : INFINITY;
          o->ties = eq;
        }
      }
      cl.sync();
      thr = sh.thr;
      ties = sh.ties;
      decided = true;
      summed = !by_min;                                                           // min-p may take some of those away
    } while (false);
    if (!decided) {
      cl.sync();                                                                  // every block has read the histograms
      for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
      if (tid == 0) sh.list_n = 0;
      __syncthreads();
    }
  }

  // ---- where that did not do (a top-k beyond the list, or thousands of tokens in the undecided bins): by count first, then by mass
  for (int stage = 0; stage < 2 && !decided; ++stage) {
    const bool counting = stage == 0 && K > 0;
    const bool mass = stage == 1 && by_mass;
    const bool min_only = stage == 1 && !by_mass && by_min && K == 0;
    if (!counting && !mass && !min_only) continue;
    // top-p behind a top-k that was too long for the list: its total is that of the kept ones
    const bool limited = stage == 1 && K > 0;
    Range r{xmax, -INFINITY, (double)(itf * SF_PER_NAT), true};
    double s_above = 0.0;               // exact mass and number of what is certainly kept
    int c_above = 0;
    for (int round = 0;; ++round) {
      // ---- histogram of this range
      double s = 0.0;
      const bool sum_now = mass && round == 0;
      for (int i = tid; i < n; i += SF_THREADS) {
        const float x = xs[i];
        if (x == -INFINITY) continue;
        if (limited && x <= thr) continue;                                        // of those equal to thr `ties` are there: added below
        if (sum_now) s += w_of(x);
        if (x <= r.hi && x >= r.lo) atomicAdd(&sh.hist[bin_of(r, x)], 1u);
      }
      if (sum_now) publish_sum(s);
      cl.sync();
      if (sum_now) {
        total = all_sum();
        if (limited) total += ties * w_of(thr);
        buf ^= 1;
      }
      // ---- counts of the cluster, and where the border can be
      unsigned int c[4] = {0u, 0u, 0u, 0u};
      for (int i = 0; i < nb; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(cl.map_shared_rank(sh.hist, i))[tid];
        c[0] += v.x; c[1] += v.y; c[2] += v.z; c[3] += v.w;
      }
      if (limited && thr <= r.hi && thr >= r.lo && (bin_of(r, thr) >> 2) == tid) c[bin_of(r, thr) & 3] += ties;
      const int own = (int)(c[0] + c[1] + c[2] + c[3]);
      int c_total;
      const int c_before = block_scan_i(own, sh.ired, &c_total);
      if (tid == 0) { sh.cut[0] = SF_BINS; sh.cut[1] = SF_BINS; sh.cut[2] = c_total; sh.cut[3] = 0; }
      __syncthreads();
      if (counting) {
        if (round == 0 && c_total < K) { K = 0; break; }                          // fewer than k tokens have any weight
        int at = c_above + c_before;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (at < K && at + (int)c[j] >= K) { sh.cut[0] = sh.cut[1] = 4 * tid + j; sh.cut[2] = c_before + (at - c_above - c_before) + (int)c[j]; sh.cut[3] = at - c_above; }
          at += (int)c[j];
        }
      } else if (mass) {
        // weights of bin b lie in w0 * f^b * [f, 1], f the ratio of neighbouring edges, but for the open last bin
        const double f = exp(-it / r.scale), w0 = exp(((double)r.hi - top) * it) * exp(-it / r.scale * 4.0 * tid);
        double lo[4], m = 0.0, e = w0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = (4 * tid + j < SF_BINS - 1) ? c[j] * e * f : 0.0;
          m += lo[j];
          e *= f;
        }
        double m_all;
        double m_cum = block_scan(m, sh.red, &m_all);
        if (tid == SF_THREADS - 1) sh.red2[0] = c[3] * (e / f);                   // upper bound of the last bin
        __syncthreads();
        const double last_hi = sh.red2[0], slack = 2e-5;
        const double want = top_p * total - s_above;                              // mass up to the border, of this range
        const double rest = total - top_p * total;                               // mass behind it
        // mass behind the last bin of the range (later rounds): total - s_above - what the range holds; only bounded by the head then
        int at = c_before, b1 = SF_BINS, b2 = SF_BINS, c1 = 0, c2 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m_cum += lo[j];
          const double head_hi = m_cum / f * (1.0 + slack), head_lo = m_cum * (1.0 - slack);
          const double tail_hi = ((m_all - m_cum) / f + last_hi) * (1.0 + slack), tail_lo = (m_all - m_cum) * (1.0 - slack);
          const bool end = 4 * tid + j == SF_BINS - 1;
          const bool maybe = c[j] && (end || (head_hi > want && (!r.first || tail_lo < rest)));
          const bool sure = c[j] && (head_lo > want || (r.first && tail_hi < rest));
          if (maybe && b1 == SF_BINS) { b1 = 4 * tid + j; c1 = at; }
          at += (int)c[j];
          if (sure && b2 == SF_BINS) { b2 = 4 * tid + j; c2 = at; }
        }
        if (b1 < SF_BINS) atomicMin(&sh.cut[0], b1);
        if (b2 < SF_BINS) atomicMin(&sh.cut[1], b2);
        __syncthreads();
        if (b1 < SF_BINS && sh.cut[0] == b1) sh.cut[3] = c1;
        if (b2 < SF_BINS && sh.cut[1] == b2) sh.cut[2] = c2;
      } else {
        // min-p: ln(1 / min_p) below the maximum, a bin further for what rounding does to the edges
        const double t = -log(min(min_p, 1.0)) * (double)SF_PER_NAT + 1.0;
        const int b2 = t < (double)(SF_BINS - 1) ? (int)t : SF_BINS - 1;
        if (tid == b2 >> 2) {
          int at = c_before;
          for (int j = 0; j <= (b2 & 3); ++j) at += (int)c[j];
          sh.cut[0] = 0; sh.cut[1] = b2; sh.cut[2] = at; sh.cut[3] = 0;
        }
      }
      __syncthreads();
      int b1 = sh.cut[0], b2 = sh.cut[1], before = sh.cut[3];
      const int upto = sh.cut[2];
      if (b2 >= SF_BINS) b2 = SF_BINS - 1;
      if (b1 > b2) b1 = before = 0;
      const bool whole = r.first && upto <= SF_CAP && !limited;
      const int undecided = upto - before;
      if (min_only && !whole) break;                                              // every token is looked at anyway
      const bool listed = whole || undecided <= SF_CAP;
      // ---- second look: the list, or the mass and range of what is decided
      s = 0.0;
      double s_one = 0.0;
      float hi1 = -INFINITY, lo1 = INFINITY, hi2 = -INFINITY, lo2 = INFINITY;
      SampleShared* head = cl.map_shared_rank(&sh, 0);
      for (int i0 = 0; i0 < n; i0 += SF_THREADS) {
        const int i = i0 + tid;
        const float x = i < n ? xs[i] : -INFINITY;
        bool take = false;
        if (x != -INFINITY && !(limited && x <= thr) && x >= r.lo) {
          const int b = x > r.hi ? -1 : bin_of(r, x);
          if (whole) {
            take = b <= b2;
          } else {
            if (b < b1) s += mass && b >= 0 ? w_of(x) : 0.0;                      // those above the range were summed before
            else if (b <= b2) {
              if (listed) take = true;
              else if (b == b1) { s_one += mass ? w_of(x) : 0.0; hi1 = fmaxf(hi1, x); lo1 = fminf(lo1, x); }
              else { hi2 = fmaxf(hi2, x); lo2 = fminf(lo2, x); }
            }
          }
        }
        const unsigned int who = __ballot_sync(0xffffffffu, take);
        if (who) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&sh.list_n, __popc(who));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
          if (take && at < SF_CAP) sh.list[at] = ((unsigned long long)key_of(x) << 32) | (0xffffffffu - (unsigned int)(begin + i));
        }
      }
      __syncthreads();
      if (listed && me != 0) {                                                    // the first block's list takes them all
        const int k = sh.list_n;
        if (tid == 0 && k) sh.ired[0] = atomicAdd(&head->list_n, k);
        __syncthreads();
        const int at = sh.ired[0];
        for (int i = tid; i < k && at + i < SF_CAP; i += SF_THREADS) head->list[at + i] = sh.list[i];
      }
      // the first block fills its own list through the same counter, from its own shared memory: no copy
      if (!whole) {
        if (mass) publish_sum(s);
        if (!listed) {
          // the border bin and those behind it apart: whichever holds the border, fewer tokens remain
          const double one = warp_sum_d(s_one);
          const float h1 = warp_max(hi1), l1 = warp_min(lo1), h2 = warp_max(hi2), l2 = warp_min(lo2);
          if (lane == 0) { sh.red2[warp] = one; sh.fred[0][warp] = h1; sh.fred[1][warp] = l1; sh.fred[2][warp] = h2; sh.fred[3][warp] = l2; }
          __syncthreads();
          if (tid < nb) {
            double o = 0.0;
            float p1 = -INFINITY, q1 = INFINITY, p2 = -INFINITY, q2 = INFINITY;
            for (int w = 0; w < SF_WARPS; ++w) {
              o += sh.red2[w];
              p1 = fmaxf(p1, sh.fred[0][w]); q1 = fminf(q1, sh.fred[1][w]);
              p2 = fmaxf(p2, sh.fred[2][w]); q2 = fminf(q2, sh.fred[3][w]);
            }
            SampleShared* t = cl.map_shared_rank(&sh, tid);
            t->pub_sum2[buf][me] = o;
            t->pub_hi[buf][me] = p1; t->pub_lo[buf][me] = q1; t->pub_hi2[buf][me] = p2; t->pub_lo2[buf][me] = q2;
          }
        }
      }
      cl.sync();
      if (whole) {
        if (me != 0) return;
        const int cnt = min(sh.list_n, SF_CAP), n2 = pow2_above(cnt);
        for (int i = cnt + tid; i < n2; i += SF_THREADS) sh.list[i] = 0ull;
        __syncthreads();
        sort_falling(sh.list, n2);
        finish(cnt);
        return;
      }
      if (mass) s_above += all_sum();
      c_above += before;
      if (listed) {
        // ---- the undecided ones are in the first block's list: it finds the last value that is kept, and how many have it
        if (me == 0) {
          const int cnt = min(sh.list_n, SF_CAP), n2 = pow2_above(cnt);
          const int extra = limited && thr >= r.lo && thr <= r.hi && bin_of(r, thr) >= b1 && bin_of(r, thr) <= b2 ? ties : 0;
          for (int i = cnt + tid; i < n2; i += SF_THREADS) sh.list[i] = 0ull;
          __syncthreads();
          sort_falling(sh.list, n2);
          double w[4], mine = 0.0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * tid + j;
            w[j] = mass && i < cnt ? w_of(float_of((unsigned int)(sh.list[i] >> 32))) : 0.0;
            mine += w[j];
          }
          double sum;
          double run = s_above + block_scan(mine, sh.red, &sum);
          int kept = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * tid + j;
            if (i < cnt && (counting ? c_above + i < K : run <= top_p * total)) ++kept;
            run += w[j];
          }
          int m;
          block_scan_i(kept, sh.ired, &m);
          __syncthreads();
          // all of the list kept, and tokens equal to the top-k's last value behind it: some of those
          const bool into = m == cnt && extra > 0;
          const unsigned int last = m > 0 ? (unsigned int)(sh.list[m - 1] >> 32) : 0u;
          int same = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * tid + j;
            if (i < m && (unsigned int)(sh.list[i] >> 32) == last) ++same;
          }
          int eq;
          block_scan_i(same, sh.ired, &eq);
          if (tid < nb) {
            float t = m > 0 ? float_of(last) : r.hi;
            if (into) {
              const double w1 = w_of(thr), have = s_above + sum;
              const double q = floor((top_p * total - have) / w1) + 1.0;
              eq = q < 1.0 ? 0 : q > (double)ties ? ties : (int)q;
              t = thr;
            }
            SampleShared* o = cl.map_shared_rank(&sh, tid);
            o->thr = t;
            o->ties = eq;
          }
        }
        cl.sync();
        thr = sh.thr;
        ties = sh.ties;
        break;
      }
      // ---- too many: the bin of the border, or what is behind it
      float p1 = -INFINITY, q1 = INFINITY, p2 = -INFINITY, q2 = INFINITY;
      double one = 0.0;
      for (int i = 0; i < nb; ++i) {
        one += sh.pub_sum2[buf][i];
        p1 = fmaxf(p1, sh.pub_hi[buf][i]); q1 = fminf(q1, sh.pub_lo[buf][i]);
        p2 = fmaxf(p2, sh.pub_hi2[buf][i]); q2 = fminf(q2, sh.pub_lo2[buf][i]);
      }
      if (limited && thr >= r.lo && thr <= r.hi) {                                // the top-k's last value is not in the sums above
        const int b = bin_of(r, thr);
        if (b == b1) { one += ties * w_of(thr); p1 = fmaxf(p1, thr); q1 = fminf(q1, thr); }
        else if (b > b1 && b <= b2) { p2 = fmaxf(p2, thr); q2 = fminf(q2, thr); }
      }
      buf ^= 1;
      if (counting || s_above + one > top_p * total || !(p2 >= q2)) {
        r = Range{p1, q1, 0.0, false};
      } else {
        // what is in the border bin is kept after all; how many those are is only needed for a top-k, which is not cut here
        s_above += one;
        r = Range{p2, q2, 0.0, false};
      }
      if (round >= 400) {                                                         // not reached by finite arguments: ends the loop whatever they are
        thr = r.hi;
        ties = a.V;
        break;
      }
      if (r.hi == r.lo) {                                                         // equal logits all through
        double q;
        if (counting) q = (double)(K - c_above);
        else q = fmin(floor((top_p * total - s_above) / w_of(r.hi)) + 1.0, limited && r.hi == thr ? (double)ties : 1e9);
        thr = r.hi;
        ties = (int)fmax(q, 0.0);
        break;
      }
      r.scale = fmax((double)(SF_BINS - 1) / ((double)r.hi - (double)r.lo), it * (double)SF_PER_NAT);
      for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
      if (tid == 0) sh.list_n = 0;
      __syncthreads();
    }
    // the histogram and the list are free again: every block has passed a barrier since it last read them
    cl.sync();
    for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = 0u;
    if (tid == 0) sh.list_n = 0;
    __syncthreads();
  }

  // ---- kept weights by index: sums of the blocks, and in the block that has the token sums of pieces of its share
  {
    double s = 0.0;
    int eq = 0;
#pragma unroll 2
    for (int i = tid; i < n4; i += SF_THREADS) {
      const float4 v = xs4[i];
      const float x[4] = {v.x, v.y, v.z, v.w};
      bool in[4], any = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool sure = depth(x[j]) < t_sure;
        in[j] = summed ? x[j] > thr && !sure : x[j] > thr || sure;                // those before t_sure are in the sum already
        any |= in[j];
        eq += x[j] == thr && x[j] != -INFINITY;
      }
      if (any) {
        double w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
          if (!in[j] || w[j] < min_p) w[j] = 0.0;
        }
        s += (w[0] + w[1]) + (w[2] + w[3]);
      }
    }
    s = warp_sum_d(s);
    eq = warp_sum_i(eq);
    __syncthreads();
    if (lane == 0) { sh.red[warp] = s; sh.ired[warp] = eq; }
    __syncthreads();
    if (tid < nb) {
      s = summed ? s_own : 0.0;
      eq = 0;
#pragma unroll
      for (int w = 0; w < SF_WARPS; ++w) { s += sh.red[w]; eq += sh.ired[w]; }
      SampleShared* t = cl.map_shared_rank(&sh, tid);
      t->pub_sum[buf][me] = s;
      t->pub_int[buf][me] = eq;
    }
  }
  double w_tie = thr == -INFINITY || thr == INFINITY ? 0.0 : w_of(thr);
  if (w_tie < min_p) w_tie = 0.0;
  cl.sync();
  double sum = 0.0, my_begin = 0.0, my_sum = 0.0;
  int ties_left = ties, my_ties = 0, last = 0;
  for (int i = 0; i < nb; ++i) {
    const int t = min(sh.pub_int[buf][i], ties_left);
    const double s = sh.pub_sum[buf][i] + t * w_tie;
    if (i == me) { my_begin = sum; my_sum = s; my_ties = ties_left; }
    if (s > SF_NONE) last = i;
    sum += s;
    ties_left -= t;
  }
  const double goal = fmax((double)__uint_as_float(sh.arg[3]) * sum, SF_NONE);      // (above nothing: u may be 0)
  // the first block whose end passes the goal (the last one with any weight, should rounding leave none)
  const bool mine = my_sum > SF_NONE && my_begin <= goal && (my_begin + my_sum > goal || me == last);
  if (!mine) return;
  for (int g = warp; g < segs; g += SF_WARPS) {
    double s = 0.0;
    int eq = 0;
#pragma unroll
    for (int h = 0; h < SF_SEG / 128; ++h) {
      const int i = g * (SF_SEG / 4) + h * 32 + lane;
      const float4 v = i < n4 ? xs4[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      const float x[4] = {v.x, v.y, v.z, v.w};
      double w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = weight(fma((double)x[j], it, -top_it), sh.tab);
        if (!(x[j] > thr || depth(x[j]) < t_sure) || w[j] < min_p) w[j] = 0.0;
        eq += x[j] == thr && x[j] != -INFINITY;
      }
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    s = warp_sum_d(s);
    eq = warp_sum_i(eq);
    if (lane == 0) { sh.seg_sum[g] = s; sh.seg_tie[g] = eq; }
  }
  __syncthreads();
  if (warp != 0) return;
  // the piece: 32 at a time, lane by lane
  double run = my_begin, sg_run = 0.0;
  int left = my_ties, sg = -1, sg_left = 0;
  for (int g0 = 0; g0 < segs; g0 += 32) {
    const int g = g0 + lane, eq = g < segs ? sh.seg_tie[g] : 0;
    int before = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += t;
    }
    const int here = max(0, min(eq, left - (before - eq)));
    const double own = (g < segs ? sh.seg_sum[g] : 0.0) + here * w_tie;
    double s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    const unsigned int some = __ballot_sync(0xffffffffu, own > SF_NONE), hit = __ballot_sync(0xffffffffu, own > SF_NONE && run + s > goal);
    if (some) {
      const int from = hit ? __ffs(hit) - 1 : 31 - __clz(some);
      sg = g0 + from;
      sg_run = run + __shfl_sync(0xffffffffu, s - own, from);
      sg_left = max(0, left - __shfl_sync(0xffffffffu, before - eq, from));
    }
    if (hit) break;
    run += __shfl_sync(0xffffffffu, s, 31);
    left = max(0, left - __shfl_sync(0xffffffffu, before, 31));
  }
  int tok = -1;
  double w_tok = 0.0;
  run = sg_run;
  left = sg_left;
  for (int i0 = sg * SF_SEG; i0 < min(a.share, (sg + 1) * SF_SEG); i0 += 32) {
    const int i = i0 + lane;
    const float x = i < a.share ? xs[i] : -INFINITY;
    const unsigned int eq = __ballot_sync(0xffffffffu, x == thr && x != -INFINITY);
    const int rank = __popc(eq & ((1u << lane) - 1u));
    double w = 0.0;
    if (x > thr || depth(x) < t_sure) { w = w_of(x); if (w < min_p) w = 0.0; }
    else if ((eq >> lane & 1u) && rank < left) w = w_tie;
    double s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    const unsigned int some = __ballot_sync(0xffffffffu, w > SF_NONE), hit = __ballot_sync(0xffffffffu, w > SF_NONE && run + s > goal);
    if (some) {
      const int from = hit ? __ffs(hit) - 1 : 31 - __clz(some);
      tok = begin + i0 + from;
      w_tok = __shfl_sync(0xffffffffu, w, from);
    }
    if (hit) break;
    run += __shfl_sync(0xffffffffu, s, 31);
    left -= min(left, __popc(eq));
  }
  if (lane == 0) {
    a.out_tok[row] = tok;
    a.out_logp[row] = (float)log(w_tok / sum);
  }
}

}  // namespace ab2

extern "C" {
using namespace ab2;

// logits [B, V] fp32, rows `ld` elements apart; u, inv_temp (> 0), top_p, min_p fp32 [B]; top_k, greedy int32 [B] (greedy may be null).
// top_k <= 0, top_p >= 1, min_p <= 0 switch a filter off. A row in which nothing has weight gives token -1 and log-prob -inf.
int ab2_sample_filtered(const void* logits, long long ld, int B, int V, const void* u, const void* inv_temp, const int* top_k, const void* top_p,
                        const void* min_p, const int* greedy, int* out_tok, float* out_logp, void* stream) {
  if (B <= 0) return 0;
  if (V <= 0 || ld < V) return 10;
  int nb = 1;
  while (nb < SF_MAX_CLUSTER && (V + nb - 1) / nb > 20480) nb *= 2;              // two blocks an SM as long as a share is below 80 KB
  SampleArgs a;
  a.share = ((V + nb - 1) / nb + 3) / 4 * 4;
  const int head = (int)((sizeof(SampleShared) + 15) / 16 * 16), smem = head + a.share * 4;
  if (smem > 227 * 1024 || a.share > SF_SEG * SF_SEGS) return 11;
  if ((long long)B * nb > 0x7fffffffLL) return 10;
  a.logits = (const float*)logits; a.ld = ld; a.u = (const float*)u; a.inv_temp = (const float*)inv_temp; a.top_p = (const float*)top_p;
  a.min_p = (const float*)min_p; a.top_k = top_k; a.greedy = greedy; a.out_tok = out_tok; a.out_logp = out_logp; a.V = V;
  a.aligned = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
  a.index_shift = 0;
  while ((V - 1) >> a.index_shift >= SF_BINS) ++a.index_shift;
  for (int j = 0; j < 32; ++j) a.tab[j] = exp2(j / 32.0);
  static ab2host::DevState st;
  if (ab2host::prepare_launch(sample_filtered_kernel, 227 * 1024, st, nullptr)) return 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B * nb);
  cfg.blockDim = dim3(SF_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = nb; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (ab2host::pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, sample_filtered_kernel, a) == cudaSuccess ? 0 : 1;
}
}
