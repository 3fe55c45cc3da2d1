// Paged key/value cache held in 8 bits, and the page copies of either cache.
//
// Layout: codes e4m3 [pages, Hkv, page_size, D], so that the block of one page and head is one contiguous run; scales fp32
// [pages, Hkv], powers of two, one for each such block. value = code * scale. A power of two divides and multiplies exactly:
// quantising rounds once, and a block whose scale has to grow (a larger row arrives) is re-coded without a second rounding
// except where a code falls below e4m3's normal range. e4m3 is a floating format, so a scale that is not a power of two would
// not make its relative steps any finer.
#include <mutex>

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

extern "C" int ab2_num_sms();

namespace ab2 {

constexpr long long KV8_WIDEST = 0x7fffffffLL - 63;   // tokens of a table: the end of the last page or tile still is an int
constexpr int KV8_E_MIN = -100, KV8_E_MAX = 120;       // exponents a scale may have; both its value and its inverse are normal

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e with amax <= 448 * 2^e, 448 = 1.75 * 2^8 the largest e4m3 value. amax is finite and >= 0.
__device__ __forceinline__ int scale_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - ((bits & 0x7fffff) > 0x600000 ? 7 : 8);
  return min(max(e, KV8_E_MIN), KV8_E_MAX);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;                       // infinities saturate and NaN stays NaN: neither sets a scale
}
// Sizes of bf16 numbers order as their bits do without the sign: two at a time in one word.
__device__ __forceinline__ uint32_t size2(uint32_t a, uint32_t w) {
  uint32_t r;
  asm("max.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(w & 0x7fff7fffu));
  return r;
}
__device__ __forceinline__ uint32_t size8(uint32_t a, const uint4& v) { return size2(size2(size2(size2(a, v.x), v.y), v.z), v.w); }
// The same without infinities and NaN, for the rare rows that hold any.
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = w & 0x7fff0000u;
  return (lo < 0x7f80u ? lo : 0u) | (hi < 0x7f800000u ? hi : 0u);
}
__device__ __forceinline__ float larger_half(uint32_t a) { return __uint_as_float(max(a << 16, a & 0xffff0000u)); }
constexpr uint32_t BF16_INF = 0x7f800000u;

__device__ __forceinline__ uint32_t code4(uint32_t lo, uint32_t hi, float inv) {
  const float2 a = unpack_bf16(lo), b = unpack_bf16(hi);
  const uint32_t c0 = __nv_cvt_float2_to_fp8x2(make_float2(a.x * inv, a.y * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t c1 = __nv_cvt_float2_to_fp8x2(make_float2(b.x * inv, b.y * inv), __NV_SATFINITE, __NV_E4M3);
  return c0 | (c1 << 16);
}
__device__ __forceinline__ uint32_t recode4(uint32_t c, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * i)), __NV_E4M3));
    const float2 f = __half22float2(h);
    r |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3) << (16 * i);
  }
  return r;
}
// Multiplies the codes of one block (16 bytes at a time) by `ratio`, all slots but [lo, hi).
template <int D>
__device__ __forceinline__ void recode_block(unsigned char* block, int page_size, int lo, int hi, float ratio, int tid, int nthr) {
  for (int i = tid; i < page_size * (D / 16); i += nthr) {
    const int slot = i / (D / 16);
    if (slot >= lo && slot < hi) continue;
    uint4 v = reinterpret_cast<uint4*>(block)[i];
    v.x = recode4(v.x, ratio); v.y = recode4(v.y, ratio); v.z = recode4(v.z, ratio); v.w = recode4(v.w, ratio);
    reinterpret_cast<uint4*>(block)[i] = v;
  }
}

struct Kv8Args {
  const __nv_bfloat16* x[2];     // keys, values: [rows, Hkv, D], heads dense, rows `stride` elements apart
  unsigned char* codes[2];
  float* scales[2];
  long long stride[2];
};

// ------------------------------------------------------------------ append, one token for each row of the batch
// One warp = (row, head, keys or values). The whole call is a few hundred KB at most and bound by latency (64 rows of 8 heads of 128: 2.1 us): one load of the
// row, one of the scale, one store of each; a warp re-codes its block (8 KB at 64 x 128) only when the scale grows.
template <int D>
__global__ void __launch_bounds__(128)
kv8_append_row_kernel(const __grid_constant__ Kv8Args a, const int* __restrict__ table, const int* __restrict__ lens, int B, int Hkv, int page_size, int width,
                      int num_pages, int* __restrict__ err) {
  pdl_wait();
  pdl_trigger();
  const int w = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = w / (2 * Hkv), r = w - b * 2 * Hkv, kv = r & 1, h = r >> 1;
  if (b >= B) return;
  const int pos = lens[b] - 1;
  if (pos < 0) return;
  const int j = pos / page_size, slot = pos - j * page_size;
  const int page = j < width ? table[(size_t)b * width + j] : -1;
  if (page < 0 || page >= num_pages) {
    if (lane == 0) set_error(err, ERR_BOUNDS);
    return;
  }
  const size_t blk = (size_t)page * Hkv + h;
  float* scale = kv ? a.scales[1] : a.scales[0];
  const float old = slot ? scale[blk] : 0.f;
  const __nv_bfloat16* x = kv ? a.x[1] + (size_t)b * a.stride[1] + h * D : a.x[0] + (size_t)b * a.stride[0] + h * D;
  uint32_t v[D / 64];
  float m = 0.f;
  if constexpr (D == 128) {
    const uint2 t = reinterpret_cast<const uint2*>(x)[lane];
    v[0] = t.x; v[1] = t.y;
  } else {
    v[0] = reinterpret_cast<const uint32_t*>(x)[lane];
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const float2 f = unpack_bf16(v[i]);
    m = fmaxf(m, fmaxf(finite_abs(f.x), finite_abs(f.y)));
  }
  m = warp_max(m);
  const float s = fmaxf(old, pow2i(scale_exponent(m)));
  unsigned char* block = (kv ? a.codes[1] : a.codes[0]) + blk * page_size * D;
  if (old > 0.f && s > old) recode_block<D>(block, page_size, slot, slot + 1, old / s, lane, 32);
  const float inv = 1.f / s;
  unsigned char* dst = block + (size_t)slot * D;
  if constexpr (D == 128) {
    reinterpret_cast<uint32_t*>(dst)[lane] = code4(v[0], v[1], inv);
  } else {
    const float2 f = unpack_bf16(v[0]);
    reinterpret_cast<__nv_fp8x2_storage_t*>(dst)[lane] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
  }
  if (lane == 0 && s != old) scale[blk] = s;
}

// ------------------------------------------------------------------ append, packed rows of several sequences
// Sequence b brings rows cu[b] .. cu[b+1], its last ones: it is lens[b] long with them. One block = (page that gets rows, head,
// keys or values): its rows (16 KB at 64 x 128) are read once into registers, their maximum decides the scale, and the codes go out
// in one contiguous run. Bound by issue slots (62 % used) and the chain sequence, page, rows: 16384 rows of 8 heads of 128 take 16.2 us, 4.9 TB/s
// of 79 MB. Which page a block has: the pages of sequence b are numbered from cu[b] / page_size + 2 b on, which
// leaves room for the floor(n / page_size) + 2 that n rows can touch, so no scan over the batch is needed.
template <int D, int NV>          // NV: 16-byte pieces of a thread = page_size * D / 8 / 128
__global__ void __launch_bounds__(128, NV <= 8 ? 8 : 4)
kv8_append_page_kernel(const __grid_constant__ Kv8Args a, const int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ cu, int B, int rows,
                       int Hkv, int page_size, int width, int num_pages, int* __restrict__ err) {
  __shared__ float red[4];
  __shared__ int found[4];             // of this block's sequence: first row, first row of the next, length
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, item = blockIdx.x, h = blockIdx.y >> 1, kv = blockIdx.y & 1;
  int b = -1;
  for (int i0 = 0; i0 < B; i0 += 128) {                // numbers grow with b: the last one that does not pass this block's
    const int i = i0 + tid, k = min(i, B - 1);
    const int c = cu[k], next = cu[k + 1], len = lens[k];
    const int n = __syncthreads_count(i < B && c / page_size + 2 * i <= item);
    if (n && tid == n - 1) { found[0] = c; found[1] = next; found[2] = len; }
    b += n;
    if (n < 128) break;
  }
  __syncthreads();
  if (b < 0) return;
  const int c0 = found[0], n = found[1] - c0, end = found[2], start = end - n;
  if (n <= 0) return;
  const int j = start / page_size + item - (c0 / page_size + 2 * b);
  const int lo = max(start, j * page_size), hi = min(end, (j + 1) * page_size);
  if (start >= 0 && lo >= hi) return;
  const bool fits = start >= 0 && j < width && c0 >= 0 && c0 + n <= rows;
  // the rows do not need the page's number: they are on their way while it is looked up
  const int page = fits ? table[(size_t)b * width + j] : -1;
  const int slot = lo - j * page_size, cnt = fits ? hi - lo : 0;
  const long long stride = kv ? a.stride[1] : a.stride[0];
  const __nv_bfloat16* x = (kv ? a.x[1] : a.x[0]) + (fits ? (size_t)(c0 + lo - start) * stride + h * D : 0);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = tid + i * 128, row = p / (D / 8), piece = p % (D / 8);
    v[i] = row < cnt ? *reinterpret_cast<const uint4*>(x + row * stride + piece * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (page < 0 || page >= num_pages) {
    if (tid == 0) set_error(err, ERR_BOUNDS);
    return;
  }
  const size_t blk = (size_t)page * Hkv + h;
  float* scale = kv ? a.scales[1] : a.scales[0];
  const float old = slot ? scale[blk] : 0.f;
  uint32_t most = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) most = size8(most, v[i]);
  float m = larger_half(most);
  if (__float_as_uint(m) >= BF16_INF) {
    most = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      most = size2(size2(size2(size2(most, finite2(v[i].x)), finite2(v[i].y)), finite2(v[i].z)), finite2(v[i].w));
    m = larger_half(most);
  }
  m = warp_max(m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float s = fmaxf(old, pow2i(scale_exponent(m)));
  unsigned char* block = (kv ? a.codes[1] : a.codes[0]) + blk * page_size * D;
  if (old > 0.f && s > old) recode_block<D>(block, page_size, slot, slot + cnt, old / s, tid, 128);
  const float inv = 1.f / s;
  uint2* dst = reinterpret_cast<uint2*>(block + (size_t)slot * D);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = tid + i * 128;
    if (p / (D / 8) < cnt) dst[p] = make_uint2(code4(v[i].x, v[i].y, inv), code4(v[i].z, v[i].w, inv));
  }
  if (tid == 0 && s != old) scale[blk] = s;
}

// ------------------------------------------------------------------ attention of single tokens
// o = softmax(scale * q K^T) V over the first lens[b] tokens, G query heads for each key/value head. Bound by the codes' bytes: 256 x 2000..4001
// tokens, 28 / 4 heads of 128, 140 us, 5.7 TB/s; 64 x 750..1500, 32 / 8 heads, 35 us, 4.0 TB/s, of which 8 us pass until the first tiles are here.
//
// Split: every (sequence, head) item is cut into units of U chunks of 64 tokens, U from the whole batch's tokens, whatever the lengths are.
// Block i takes units i, i + grid, ...: about one each, so that taking them from a counter instead (SMs do not get equal shares of the
// memory's rate) gained 1 % on the largest case and cost a launch that clears it in every captured call. A second kernel joins the
// units of items that were split (the last block of an item joining it cost 1.4 us a unit for the fence, which waits for its copies too).
// Warp w of a block takes tokens 16 w .. 16 w + 15 of each chunk and fetches them itself, with 16-byte asynchronous copies into a ring
// of its own in shared memory, so there is no barrier in the loop and the bytes in flight are not bounded by registers.
//   S^T[16 tokens, 8 heads] = K Q^T: the sum over dims may be taken in any order, so 16 contiguous bytes of a row serve a thread as
//     four steps of k = 16 (the queries are laid out to match);
//   O^T[D dims, 8 heads] += V^T P^T: rows (dims) may stand in any order too, so a thread's 16 contiguous dims of four tokens are
//     paired by byte permutes; P^T comes from S^T by an 8 x 8 transpose between registers.
// The 16-byte pieces of a 128-byte line stand where their number is xor-ed with the line's, so that both patterns of reads are free of
// bank conflicts. e4m3 converts to fp16 exactly; q is divided by a power of two for its head (exact), and both sums are fp32.
// P is rounded to fp16 (half a step 2^-11) and multiplies codes, so it holds the page's value scale: probability times scale, what the token can add to
// the result, as 2^(x + log2 scale - d). The largest of it seen lies between 2^8 and 2^15 (m and d only move when a token leaves that range), so that all
// down to 2^-22 of the largest keep all bits, whatever the scales are and in whatever order the pages come. The sum of the probabilities
// alone has a reference of its own, m: a token may have all the weight and add next to nothing, or the other way round. d is counted from m, so
// that it stays within a few hundred and is not rounded where scores are large.
constexpr int KV8_CHUNK = 64, KV8_MOST_ROWS = 8192;
constexpr int KV8_LEAST = 4;        // chunks of the smallest unit: what a split saves of so short an item, the join costs
constexpr float KV8_LOW = -300.f;   // below every d: a scale is 2^-100 or more

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Two e4m3 codes (low / high half of a word) as two fp16.
__device__ __forceinline__ uint32_t half2_lo(uint32_t c) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(r) : "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t half2_hi(uint32_t c) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p));
  return v;
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// log2 of a scale; a power of two gives a whole number.
__device__ __forceinline__ float log2_scale(float s) {
  const int bits = __float_as_int(s);
  const float e = (float)((bits >> 23) - 127);
  if (s > 0.f) return bits & 0x7fffff ? e + __log2f(__int_as_float((bits & 0x7fffff) | 0x3f800000)) : e;
  return s == 0.f ? -INFINITY : NAN;
}
// a * 2^d, d whole, in two steps: 2^d alone may be out of range where the product is not.
__device__ __forceinline__ float times_pow2(float a, float d) {
  const int k = (int)fminf(fmaxf(d, -250.f), 250.f), h = k >> 1;
  return a * pow2i(h) * pow2i(k - h);
}

struct Kv8Decode {
  const __nv_bfloat16* q;
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens;
  __nv_bfloat16* out;
  float* part_o;                // [slots][HP][D]: units of items that are split, divided by 2^(m + d)
  float4* part_ml;              // [slots][HP]: m, the sum of probabilities divided by 2^m, d
  int2* meta;                   // [B] units of an item of the sequence, and its first slot
  int* err;
  int B, Hq, Hkv, G, groups, page_size, page_bits, width, num_pages;
  float scale_log2;             // softmax scale * log2(e)
  long long q_stride;
};

// Where piece `c` (16 bytes) of row `r` stands in a 16-row tile.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if constexpr (D == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ ((r & 6))) << 4);            // two rows in a line; line r / 2, xor 2 * (line % 4)
}

template <int D, int NT>
struct Kv8Cfg {
  static constexpr int BLOCKS = NT == 1 ? 4 : 2;           // resident on an SM
  static constexpr int STAGES = NT == 1 ? 3 : 4;           // of each warp's ring: 4 KB at D = 128
  static constexpr int TILE = 16 * D;                      // bytes of one operand
  static constexpr int RING = (STAGES * 2 * TILE > 8 * NT * (D + 4) * 4 ? STAGES * 2 * TILE : (8 * NT * (D + 4) * 4 + 127) / 128 * 128);
};

template <int D, int NT>        // NT: tiles of 8 query heads
__global__ void __launch_bounds__(128, Kv8Cfg<D, NT>::BLOCKS)
kv8_decode_kernel(const __grid_constant__ Kv8Decode a) {
  using Cfg = Kv8Cfg<D, NT>;
  constexpr int HP = 8 * NT;
  constexpr int KS = D / 16;            // steps of S; also D / 16 row tiles of O
  constexpr int S = Cfg::STAGES;
  extern __shared__ __align__(128) unsigned char dsm[];       // four rings; where a unit ends, each holds its warp's result [HP][D + 4]
  float* mm = reinterpret_cast<float*>(dsm + 4 * Cfg::RING);  // [4][HP]
  float* ml = mm + 4 * HP;                                    // [4][HP]
  float* md = ml + 4 * HP;                                    // [4][HP]
  int* units = reinterpret_cast<int*>(md + 4 * HP);           // [B + 1] units of one head before sequence b
  int* slots = units + a.B + 1;                               // [B + 1] those of split items only
  __shared__ int wsum[2][4];
  __shared__ float s_scale[4][S][2];                          // scales of the tiles in the rings
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  const int Hv = a.Hkv * a.groups;
  const uint32_t ring = smem_u32(dsm) + warp * Cfg::RING;
  const uint32_t in_off = tile_at<D>(lane / (D / 16), lane % (D / 16)), k_off = tile_at<D>(gq, (D / 64) * tq);
  const uint32_t v_off = D == 128 ? tile_at<D>(2 * tq, gq) : tile_at<D>(2 * tq, gq >> 1) + 8 * (gq & 1);
  const int room = a.width * a.page_size;
  auto length = [&](int b) { return min(max(a.lens[b], 0), room); };
  // ---- chunks of the batch, and with them the size of a unit: every block counts them all (a few loads a thread)
  int sum = 0;
  for (int i = tid; i < a.B; i += 128) {
    if (blockIdx.x == 0 && a.lens[i] > room) set_error(a.err, ERR_BOUNDS);
    const int n = (length(i) + KV8_CHUNK - 1) / KV8_CHUNK;
    units[i] = n;
    sum += n;
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (lane == 0) wsum[0][warp] = sum;
  __syncthreads();
  const int chunks = (wsum[0][0] + wsum[0][1] + wsum[0][2] + wsum[0][3]) * Hv;
  // A unit's chunks: an equal share of the wave. Where the items alone fill half of the wave or more, twice that: a unit costs about 4 us
  // beside its chunks (queries, first copies, join), and fewer of them cost less than the uneven end does (64 x 1k: 35 us against 39; 12 items of
  // 32k: 24 us with single shares, 25 with double ones; shares halved or the last quarter cut finer: 2 to 20 % slower in every case).
  const unsigned share = (unsigned)chunks * (2 * Hv * a.B >= (int)gridDim.x ? 2u : 1u);
  const int U = max(KV8_LEAST, (int)((share + gridDim.x - 1) / gridDim.x));
  {
    int carry_u = 0, carry_s = 0;
    for (int i0 = 0; i0 < a.B; i0 += 128) {
      const int i = i0 + tid;
      const int np = i < a.B ? (units[i] + U - 1) / U : 0, sp = np > 1 ? np : 0;
      int u = np, s = sp;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, u, o), y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) { u += x; s += y; }
      }
      __syncthreads();
      if (lane == 31) { wsum[0][warp] = u; wsum[1][warp] = s; }
      __syncthreads();
      int bu = carry_u, bs = carry_s;
      for (int w = 0; w < 4; ++w) {
        if (w < warp) { bu += wsum[0][w]; bs += wsum[1][w]; }
        carry_u += wsum[0][w]; carry_s += wsum[1][w];
      }
      if (i < a.B) { units[i] = bu + u - np; slots[i] = bs + s - sp; }
    }
    if (tid == 0) { units[a.B] = carry_u; slots[a.B] = carry_s; }
    __syncthreads();
  }
  const int total = units[a.B] * Hv;                            // units
  for (int i = blockIdx.x * 128 + tid; i < a.B; i += gridDim.x * 128) a.meta[i] = make_int2(units[i + 1] - units[i], slots[i] * Hv);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)            // rows without tokens
    if (units[b] == units[b + 1])
      for (int i = tid; i < a.Hq * D / 8; i += 128) reinterpret_cast<uint4*>(a.out + (size_t)b * a.Hq * D)[i] = make_uint4(0u, 0u, 0u, 0u);

  struct Unit { int b, np, hv, part, len, c0, c1; };
  auto unit_of = [&](int unit) {
    int lo = 0, hi = a.B;                                       // last b with Hv * units[b] <= unit and units of its own
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (units[mid] * Hv <= unit) lo = mid; else hi = mid;
    }
    Unit u;
    u.b = lo;
    u.np = units[lo + 1] - units[lo];
    const int rest = unit - units[lo] * Hv;
    u.hv = rest / u.np;
    u.part = rest - u.hv * u.np;
    u.len = length(lo);
    const int nc = (u.len + KV8_CHUNK - 1) / KV8_CHUNK, per = (nc + u.np - 1) / u.np;
    u.c0 = u.part * per;
    u.c1 = min(nc, u.c0 + per);
    return u;
  };
  // What the next unit is and its pages (lane i: of this warp's tile i) are looked up while this one runs: its first copies then
  // start at once.
  Unit u = {};
  int pg_first = 0;
  auto tiles_of = [&](const Unit& x) { return min(x.c1 - x.c0, max(0, (x.len - x.c0 * KV8_CHUNK - warp * 16 + KV8_CHUNK - 1) / KV8_CHUNK)); };
  auto page_of = [&](const Unit& x, int i, int n) {
    int p = 0;
    if (i < n) {
      p = a.table[(size_t)x.b * a.width + (((x.c0 + i) * KV8_CHUNK + warp * 16) >> a.page_bits)];
      if ((unsigned)p >= (unsigned)a.num_pages) { set_error(a.err, ERR_BOUNDS); p = 0; }
    }
    return p;
  };
  if ((int)blockIdx.x < total) {
    u = unit_of(blockIdx.x);
    pg_first = page_of(u, lane, tiles_of(u));
  }
  for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
    const int b = u.b, np = u.np, hv = u.hv, part = u.part, len = u.len;
    const int h = hv / a.groups, g0 = (hv - h * a.groups) * 16, ng = min(a.G - g0, HP);
    // ---- this warp's tiles: tokens 64 c + 16 warp of the unit's chunks
    const int t_first = u.c0 * KV8_CHUNK + warp * 16, n_tiles = tiles_of(u);
    const Unit now = u;
    int pg = 0, pg_next = pg_first;                             // pages of 32 tiles, and of the next 32
    uint32_t st_in = ring, st_out = ring;                       // stages that the next tile goes to and comes from
    int sc_in = 0, sc_out = 0;
    auto fetch = [&](int i) {                                   // tile i into its stage; an empty group where there is none
      if (i < n_tiles) {
        if ((i & 31) == 0) {
          pg = pg_next;
          pg_next = n_tiles > i + 32 ? page_of(now, i + 32 + lane, n_tiles) : 0;
        }
        const size_t blk = (size_t)__shfl_sync(0xffffffffu, pg, i & 31) * a.Hkv + h;
        const size_t at = ((blk << a.page_bits) + ((t_first + i * KV8_CHUNK) & (a.page_size - 1))) * D + lane * 16;
        if (lane < 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&s_scale[warp][sc_in][lane])), "l"((lane ? a.vs : a.ks) + blk) : "memory");
        const unsigned char *ksrc = a.kc + at, *vsrc = a.vc + at;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {                      // 512 bytes of each, contiguous
          // D = 128: 4 rows on, which flips bit 2 of a line's xor; D = 64: 8 rows, 4 lines on, which leaves it
          const uint32_t d = st_in + (D == 128 ? in_off ^ ((j & 1) << 6) : in_off) + j * 512;
          copy16_async(d, ksrc + j * 512);
          copy16_async(d + Cfg::TILE, vsrc + j * 512);
        }
        st_in = st_in == ring + (S - 1) * 2 * Cfg::TILE ? ring : st_in + 2 * Cfg::TILE;
        sc_in = sc_in == S - 1 ? 0 : sc_in + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i);
    if (unit + (int)gridDim.x < total) {
      u = unit_of(unit + gridDim.x);
      pg_first = page_of(u, lane, tiles_of(u));
    }

    // ---- queries as the B operand: head gq of the tile, dims in the order of the keys' bytes
    uint32_t qf[NT][KS][2];
    float qs[NT][2];                                          // score factor of heads 2 tq, 2 tq + 1
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int hd = t * 8 + gq;
      uint32_t raw[KS][2];
      float m = 0.f;
      const __nv_bfloat16* qp = a.q + (size_t)b * a.q_stride + (size_t)(h * a.G + g0 + hd) * D;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint2 w = hd < ng ? *reinterpret_cast<const uint2*>(qp + (D == 128 ? tq * 32 : tq * 16) + s * 4) : make_uint2(0u, 0u);
        raw[s][0] = w.x; raw[s][1] = w.y;
        const float2 x = unpack_bf16(w.x), y = unpack_bf16(w.y);
        m = fmaxf(m, fmaxf(fmaxf(finite_abs(x.x), finite_abs(x.y)), fmaxf(finite_abs(y.x), finite_abs(y.y))));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int e = scale_exponent(m);                        // m <= 448 * 2^e: fp16 holds q / 2^e with steps below 2^-24
      const float inv = pow2i(-e);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float2 x = unpack_bf16(raw[s][0]), y = unpack_bf16(raw[s][1]);
        qf[t][s][0] = pack_f16(x.x * inv, x.y * inv);
        qf[t][s][1] = pack_f16(y.x * inv, y.y * inv);
      }
      const float f = pow2i(e) * a.scale_log2;
      qs[t][0] = __shfl_sync(0xffffffffu, f, 8 * tq);         // lane 4 * (2 tq) holds head 2 tq
      qs[t][1] = __shfl_sync(0xffffffffu, f, 8 * tq + 4);
    }

    float o[NT][KS][4], m_run[NT][2], l_run[NT][2], d_run[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < KS; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      m_run[t][0] = m_run[t][1] = -3e38f;                       // below every finite score, and a difference of two such is no NaN
      l_run[t][0] = l_run[t][1] = 0.f;
      d_run[t][0] = d_run[t][1] = KV8_LOW;
    }

    float v_last = -1.f, lv = 0.f;                              // value scale of the page, and its log2
    auto work = [&](int i) {
      const float kscale = s_scale[warp][sc_out][0], vscale = s_scale[warp][sc_out][1];
      sc_out = sc_out == S - 1 ? 0 : sc_out + 1;
      const int left = len - (t_first + i * KV8_CHUNK);         // tokens of the tile that exist (16 or more: all)
      const uint32_t kt = st_out, vt = st_out + Cfg::TILE;
      st_out = st_out == ring + (S - 1) * 2 * Cfg::TILE ? ring : st_out + 2 * Cfg::TILE;
      uint32_t k[2][D / 16], v[4][D / 32];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) *reinterpret_cast<uint4*>(&k[r][4 * c]) = lds16(kt + (k_off ^ (c << 4)) + r * 8 * D);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 128) *reinterpret_cast<uint4*>(&v[r][0]) = lds16(vt + (v_off ^ ((r & 1) << 4)) + (r & 1) * 128 + (r >> 1) * 1024);
        else *reinterpret_cast<uint2*>(&v[r][0]) = lds8(vt + (v_off ^ ((r & 1) << 6)) + (r >> 1) * 512);
      }
      float s[NT][4], s2[NT][4];                                // two sums of half the dims each: chains half as long
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = s2[t][e] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint32_t a0 = half2_lo(k[0][j]), a2 = half2_hi(k[0][j]), a1 = half2_lo(k[1][j]), a3 = half2_hi(k[1][j]);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16_16816(j & 1 ? s2[t] : s[t], a0, a1, a2, a3, qf[t][j][0], qf[t][j][1]);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] += s2[t][e];
      if (left < 16) {                                          // what stands behind the last token may be anything
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (2 * tq + (r >> 1) * 8 + (r & 1) >= left)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) v[r][c] = 0u;
      }
      if (vscale != v_last) {                                   // another page
        v_last = vscale;
        lv = log2_scale(vscale);
      }
      // x = score - m; both of a head's tokens. The product is rounded as the maximum's was: with one rounding for both steps, large
      // scores (2^24 and more) would be off by the rounding of the maximum's product, whole powers of two.
      float x[NT][4], f[NT][2];
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[t][e & 1] = qs[t][e & 1] * kscale;
          x[t][e] = __fmul_rn(s[t][e], f[t][e & 1]) - m_run[t][e & 1];
        }
        if (left < 16) {
          if (gq >= left) x[t][0] = x[t][1] = -INFINITY;
          if (gq + 8 >= left) x[t][2] = x[t][3] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) grow |= fmaxf(x[t][e], x[t][e + 2]) > fminf(15.f, 15.f - (lv - d_run[t][e]));
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // from the products: the old maximum may be so far off that the difference has lost its low bits. Every lane takes
            // part in the exchange; which heads move is the same for the eight lanes of a head only.
            const bool in0 = gq < left, in1 = gq + 8 < left;
            float top = fmaxf(in0 ? __fmul_rn(s[t][e], f[t][e]) : -INFINITY, in1 ? __fmul_rn(s[t][e + 2], f[t][e]) : -INFINITY);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float m = fmaxf(m_run[t][e], top - 9.f);                              // the largest probability becomes 2^9, which fp16 holds exactly
            const float d_old = d_run[t][e] - (m - m_run[t][e]);                        // the same unit of the sums, counted from the new m
            const float d = fmaxf(fmaxf(d_old, ceilf(top - m + lv) - 9.f), KV8_LOW);    // and the largest share of the result 2^8 to 2^9
            if (m > m_run[t][e]) {
              l_run[t][e] *= fast_exp2(m_run[t][e] - m);
              m_run[t][e] = m;
              x[t][e] = in0 ? __fmul_rn(s[t][e], f[t][e]) - m : -INFINITY;
              x[t][e + 2] = in1 ? __fmul_rn(s[t][e + 2], f[t][e]) - m : -INFINITY;
            }
            d_run[t][e] = d;
            if (d > d_old) {
              const float al = fast_exp2(d_old - d);
#pragma unroll
              for (int i2 = 0; i2 < KS; ++i2) { o[t][i2][e] *= al; o[t][i2][e + 2] *= al; }
            }
          }
      }
      uint32_t p0[NT], p1[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float e0 = fast_exp2(x[t][0]), e1 = fast_exp2(x[t][1]), e2 = fast_exp2(x[t][2]), e3 = fast_exp2(x[t][3]);
        l_run[t][0] += e0 + e2;
        l_run[t][1] += e1 + e3;
        const float c0 = lv - d_run[t][0], c1 = lv - d_run[t][1];
        p0[t] = transpose8x8(pack_f16(fast_exp2(x[t][0] + c0), fast_exp2(x[t][1] + c1)));
        p1[t] = transpose8x8(pack_f16(fast_exp2(x[t][2] + c0), fast_exp2(x[t][3] + c1)));
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) {                            // dims gq * D/8 + 2 j and + 2 j + 1
        const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
        const uint32_t w0 = __byte_perm(v[0][j >> 1], v[1][j >> 1], sel), w1 = __byte_perm(v[2][j >> 1], v[3][j >> 1], sel);
        const uint32_t a0 = half2_lo(w0), a1 = half2_hi(w0), a2 = half2_lo(w1), a3 = half2_hi(w1);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16_16816(o[t][j], a0, a1, a2, a3, p0[t], p1[t]);
      }
    };
    for (int i = 0; i < n_tiles; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
      __syncwarp();                                             // every lane's copies are here, and tile i - 1 has been read
      fetch(i + S - 1);
      work(i);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float* mo = reinterpret_cast<float*>(dsm + warp * Cfg::RING);

    // ---- join the four warps; O^T fragments: element 0/1 = dim gq * D/8 + 2 j of heads 2 tq, 2 tq + 1; 2/3 = the next dim
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[t][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int hd = t * 8 + 2 * tq + e;
        if (gq == 0) {
          mm[warp * HP + hd] = m_run[t][e];
          ml[warp * HP + hd] = l;
          md[warp * HP + hd] = d_run[t][e];
        }
#pragma unroll
        for (int j = 0; j < KS; ++j)
          *reinterpret_cast<float2*>(&mo[hd * (D + 4) + gq * (D / 8) + 2 * j]) = make_float2(o[t][j][e], o[t][j][e + 2]);
      }
    }
    __syncthreads();
    const int slot = slots[b] * Hv + hv * np + part;
    for (int i = tid; i < ng * D; i += 128) {
      const int g = i / D, d = i - g * D;
      float mx = mm[g];
#pragma unroll
      for (int w = 1; w < 4; ++w) mx = fmaxf(mx, mm[w * HP + g]);
      float dx = mm[g] - mx + md[g];                            // the warps' units, counted from the largest m
#pragma unroll
      for (int w = 1; w < 4; ++w) dx = fmaxf(dx, mm[w * HP + g] - mx + md[w * HP + g]);
      dx = ceilf(dx);                                           // (whole, for times_pow2)
      float l = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float below = mm[w * HP + g] - mx;
        l += ml[w * HP + g] * fast_exp2(below);
        acc += reinterpret_cast<const float*>(dsm + w * Cfg::RING)[g * (D + 4) + d] * fast_exp2(below + md[w * HP + g] - dx);
      }
      if (np == 1) {
        a.out[((size_t)b * a.Hq + h * a.G + g0 + g) * D + d] = __float2bfloat16(times_pow2(acc / l, dx));
      } else {
        a.part_o[((size_t)slot * HP + g) * D + d] = acc;
        if (d == 0) a.part_ml[(size_t)slot * HP + g] = make_float4(mx, l, dx, 0.f);
      }
    }
    __syncthreads();                                            // the rings are free for the next unit
  }
}

// Joins the units of split items. Block (b, y) takes the heads y, y + gridDim.y, ... of sequence b: four warps share an item's units, lane i
// weighs unit i, all lanes read its row together, eight rows on their way at a time.
template <int D, int NT>
__global__ void __launch_bounds__(128) kv8_join_kernel(const __grid_constant__ Kv8Decode a) {
  constexpr int HP = 8 * NT, PER = D / 32;
  __shared__ float so[4][D], sm[4], sl[4], sd[4];
  pdl_wait();
  pdl_trigger();
  const int2 meta = a.meta[blockIdx.x];
  const int b = blockIdx.x, np = meta.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (np <= 1) return;
  for (int hq = blockIdx.y; hq < a.Hq; hq += gridDim.y) {
    const int h = hq / a.G, gh = hq - h * a.G, grp = gh / 16, g = gh - grp * 16;
    const size_t first = (size_t)(meta.y + (h * a.groups + grp) * np);
    float mx = -INFINITY, l = 0.f, dx = -INFINITY, acc[PER];   // acc: divided by 2^(mx + dx)
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
    for (int i0 = warp; i0 < np; i0 += 128) {                   // units i0, i0 + 4, ...: 32 of them
      const int i = i0 + 4 * lane, n = min(32, (np - i0 + 3) / 4);
      const float4 p = i < np ? a.part_ml[(first + i) * HP + g] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      const float m = fmaxf(mx, warp_max(p.x));
      l = l * fast_exp2(mx - m) + p.y * fast_exp2(p.x - m);
      const float d_old = mx - m + dx, d_own = p.x - m + p.z, d = fmaxf(d_old, warp_max(d_own));
      const float f0 = fast_exp2(d_old - d), f = fast_exp2(d_own - d);
      mx = m;
      dx = d;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] *= f0;
      for (int j0 = 0; j0 < n; j0 += 8) {
        float x[8][PER];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float* q = a.part_o + ((first + i0 + 4 * min(j0 + j, n - 1)) * HP + g) * D + lane * PER;
          if constexpr (D == 128) *reinterpret_cast<float4*>(x[j]) = *reinterpret_cast<const float4*>(q);
          else *reinterpret_cast<float2*>(x[j]) = *reinterpret_cast<const float2*>(q);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = __shfl_sync(0xffffffffu, f, j0 + j);  // lanes behind the last unit hold zero
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += x[j][e] * w;
        }
      }
    }
    l = warp_sum(l);
#pragma unroll
    for (int e = 0; e < PER; ++e) so[warp][lane * PER + e] = acc[e];
    if (lane == 0) { sm[warp] = mx; sl[warp] = l; sd[warp] = dx; }
    __syncthreads();
    mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    l = 0.f;
    dx = -INFINITY;
    float f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      l += sl[w] * fast_exp2(sm[w] - mx);
      f[w] = sm[w] - mx + sd[w];
      dx = fmaxf(dx, f[w]);
    }
    dx = ceilf(dx);
#pragma unroll
    for (int w = 0; w < 4; ++w) f[w] = fast_exp2(f[w] - dx);
    for (int d = threadIdx.x; d < D; d += 128)
      a.out[((size_t)b * a.Hq + hq) * D + d] = __float2bfloat16(times_pow2((so[0][d] * f[0] + so[1][d] * f[1] + so[2][d] * f[2] + so[3][d] * f[3]) / l, dx));
    __syncthreads();
  }
}

// Host threads that share a stream share its workspace: one call's two launches must not have another's between them.
static std::mutex g_kv8_pair;

template <int D, int NT>
static int launch_kv8_decode(const Kv8Decode& a, int grid, cudaStream_t s) {
  constexpr int HP = 8 * NT, RING = 4 * Kv8Cfg<D, NT>::RING + 12 * HP * 4;
  const int smem = RING + 2 * (a.B + 1) * 4;
  auto kern = kv8_decode_kernel<D, NT>;
  static ab2host::DevState st;
  if (ab2host::prepare_launch(kern, RING + 2 * (KV8_MOST_ROWS + 1) * 4, st, nullptr)) return 2;
  std::lock_guard<std::mutex> lk(g_kv8_pair);
  launch_pdl(kern, dim3(grid), dim3(128), (size_t)smem, s, a);
  if (((long long)a.width * a.page_size + KV8_CHUNK - 1) / KV8_CHUNK > KV8_LEAST) {              // some item may have been split
    int y = 4736 / a.B;
    y = y < 1 ? 1 : y > a.Hq ? a.Hq : y;
    launch_pdl(kv8_join_kernel<D, NT>, dim3(a.B, y), dim3(128), 0, s, a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

// ------------------------------------------------------------------ page copies
// Copies pages src -> dst of up to four buffers in one launch: all planes (layers, keys and values, scales) of all pairs. A page of
// a plane is `rows` runs of bytes, `row_stride` apart, of which the first tokens * token_bytes of each are copied (all of them where
// tokens < 0). The pairs travel as kernel arguments, so a call needs no transfer. Bound by memory: 16 KB a block, 64 bytes a thread in flight
// (32 KB and 128 bytes cost 15 % where the runs do not fill the blocks, and gain nothing on whole pages). 90 pages of 28 layers, 16 bits, 330 MB read
// and 330 MB written: 101 us, 6.5 TB/s; 15 tails of 40 tokens of 36 layers in 8 bits: 10 us.
constexpr int COPY_PAIRS = 256, COPY_BUFFERS = 4, COPY_PER = 4, COPY_BYTES = 256 * 16 * COPY_PER;
struct CopyBuffer {
  unsigned char* base;
  long long plane_stride, page_stride, row_stride;
  int planes, rows, row_bytes, token_bytes, first_block, per, unit;     // per: blocks of one plane; unit: bytes of one access (16, 4 or 1)
};
struct CopyArgs {
  CopyBuffer buf[COPY_BUFFERS];
  int src[COPY_PAIRS], dst[COPY_PAIRS], tokens[COPY_PAIRS];
  int n_buf;
};
template <typename T>
__device__ __forceinline__ void copy_run(const unsigned char* s, unsigned char* d, int run, long long row_stride, int first, int last) {
  constexpr int U = sizeof(T), PER = COPY_PER;
  // the row of access i without an integer division for each: counted from the block's first row, where a quotient in single precision is
  // off by one at most
  const int len = run / U, row0 = first / run, base = row0 * len;
  const float inv = 1.f / (float)len;
  for (int i0 = first / U + threadIdx.x; i0 < last / U; i0 += PER * 256) {
    T v[PER];
    long long off[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = i0 + j * 256;
      if (i < last / U) {
        int q = (int)((float)(i - base) * inv), rest = i - base - q * len;
        if (rest < 0) { --q; rest += len; }
        if (rest >= len) { ++q; rest -= len; }
        off[j] = (row0 + q) * row_stride + (long long)rest * U;
        v[j] = *reinterpret_cast<const T*>(s + off[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (i0 + j * 256 < last / U) *reinterpret_cast<T*>(d + off[j]) = v[j];
  }
}
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  const int pair = blockIdx.y;
  int n = 0;
#pragma unroll
  for (int i = 1; i < COPY_BUFFERS; ++i)
    if (i < a.n_buf && (int)blockIdx.x >= a.buf[i].first_block) n = i;
  const CopyBuffer& c = a.buf[n];
  const int k = blockIdx.x - c.first_block, plane = k / c.per, part = k - plane * c.per;
  if (plane >= c.planes) return;
  const int tok = a.tokens[pair];
  const int run = tok < 0 || c.token_bytes == 0 ? c.row_bytes : tok * c.token_bytes;
  const int first = part * COPY_BYTES, last = min(first + COPY_BYTES, run * c.rows);
  if (first >= last) return;
  const unsigned char* s = c.base + plane * c.plane_stride + a.src[pair] * c.page_stride;
  unsigned char* d = c.base + plane * c.plane_stride + a.dst[pair] * c.page_stride;
  if (c.unit == 16) copy_run<uint4>(s, d, run, c.row_stride, first, last);
  else if (c.unit == 4) copy_run<uint32_t>(s, d, run, c.row_stride, first, last);
  else copy_run<unsigned char>(s, d, run, c.row_stride, first, last);
}

}  // namespace ab2

extern "C" {
using namespace ab2;

// k, v: [rows, Hkv, D] bf16 (rows k_stride / v_stride elements apart, multiples of 8); kc, vc [num_pages, Hkv, page_size, D]; ks, vs
// [num_pages, Hkv]; table [B, width]; lens [B] with the new rows. cu == null: row b is the last token of sequence b (none where
// lens[b] is 0); else sequence b brings rows cu[b] .. cu[b+1]. A page out of range or a table too narrow sets the error word and is skipped.
int ab2_kv8_append(const void* k, const void* v, void* kc, void* vc, void* ks, void* vs, const int* table, const int* lens, const int* cu,
                   int B, int rows, int Hkv, int D, int page_size, int width, int num_pages, long long k_stride, long long v_stride, void* stream) {
  if (B <= 0 || rows <= 0) return 0;
  if (!cu && rows < B) return 10;
  if (D != 64 && D != 128) return 11;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return 12;
  if (Hkv <= 0 || Hkv > 4096 || (k_stride & 7) || (v_stride & 7) || width <= 0 || num_pages <= 0) return 10;
  if ((long long)width * page_size >= KV8_WIDEST) return 13;
  int* err = ab2host::error_flag();
  Kv8Args a;
  a.x[0] = (const __nv_bfloat16*)k; a.x[1] = (const __nv_bfloat16*)v;
  a.codes[0] = (unsigned char*)kc; a.codes[1] = (unsigned char*)vc;
  a.scales[0] = (float*)ks; a.scales[1] = (float*)vs;
  a.stride[0] = k_stride; a.stride[1] = v_stride;
  cudaStream_t s = (cudaStream_t)stream;
  if (!cu) {
    const long long warps = (long long)B * Hkv * 2;
    if (warps > 0x7fffffffLL) return 10;
    const dim3 grid((unsigned)((warps + 3) / 4));
    if (D == 128) launch_pdl(kv8_append_row_kernel<128>, grid, dim3(128), 0, s, a, table, lens, B, Hkv, page_size, width, num_pages, err);
    else launch_pdl(kv8_append_row_kernel<64>, grid, dim3(128), 0, s, a, table, lens, B, Hkv, page_size, width, num_pages, err);
    return cudaGetLastError() == cudaSuccess ? 0 : 1;
  }
  if (rows / page_size + 2LL * B > 0x7fffffffLL || Hkv * 2 > 65535) return 10;
  const dim3 grid(rows / page_size + 2 * B, Hkv * 2);
#define AB2_APPEND(DD, NN) launch_pdl(kv8_append_page_kernel<DD, NN>, grid, dim3(128), 0, s, a, table, lens, cu, B, rows, Hkv, page_size, width, num_pages, err)
  switch (page_size * D / 1024) {
    case 1: AB2_APPEND(64, 1); break;
    case 2: if (D == 64) AB2_APPEND(64, 2); else AB2_APPEND(128, 2); break;
    case 4: if (D == 64) AB2_APPEND(64, 4); else AB2_APPEND(128, 4); break;
    case 8: if (D == 64) AB2_APPEND(64, 8); else AB2_APPEND(128, 8); break;
    case 16: AB2_APPEND(128, 16); break;
    default: return 12;
  }
#undef AB2_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

// Blocks that ab2_kv8_decode launches, and with them the bytes of its workspace.
static int kv8_grid(int B, int Hq, int Hkv, int width, int page_size, int sms) {
  const int G = Hq / Hkv, groups = (G + 15) / 16;
  const long long most = (long long)B * Hkv * groups * (((long long)width * page_size + KV8_CHUNK - 1) / KV8_CHUNK);
  const long long wave = (long long)sms * (G <= 8 ? Kv8Cfg<128, 1>::BLOCKS : Kv8Cfg<128, 2>::BLOCKS);
  return (int)(most < wave ? most : wave);
}
// Bytes of the workspace. A split item has at least two units, and a unit is a block's share or more, so no more than 2 * blocks units belong to split items.
long long ab2_kv8_decode_workspace(int B, int Hq, int Hkv, int D, int page_size, int width) {
  if (B <= 0 || Hkv <= 0 || Hq % Hkv) return 0;
  const int G = Hq / Hkv, HP = G <= 8 ? 8 : 16;
  const long long slots = 2LL * kv8_grid(B, Hq, Hkv, width, page_size, ab2_num_sms());
  return slots * HP * (D + 4) * 4 + (long long)B * 8;
}

// q [B, Hq, D] bf16 (rows q_stride elements apart, heads dense), out [B, Hq, D] dense; cache and table as above; lens [B]. Calls that
// may run at the same time must not share the workspace.
int ab2_kv8_decode(const void* q, const void* kc, const void* vc, const void* ks, const void* vs, const int* table, const int* lens, void* out,
                   void* workspace, int B, int Hq, int Hkv, int D, int page_size, int width, int num_pages, float scale, long long q_stride,
                   void* stream) {
  if (B <= 0) return 0;
  if (D != 64 && D != 128) return 11;
  if (page_size < 16 || (page_size & (page_size - 1))) return 12;
  if (Hkv <= 0 || Hq % Hkv || (q_stride & 7) || width <= 0 || num_pages <= 0 || B > KV8_MOST_ROWS) return 10;
  const int G = Hq / Hkv, groups = (G + 15) / 16;
  // chunks of the whole batch are counted in 32 bits
  if ((long long)width * page_size >= KV8_WIDEST || (long long)B * Hkv * groups * (((long long)width * page_size + 63) / 64) > 0x7fffffffLL - 65536) return 13;
  Kv8Decode a;
  const int grid = kv8_grid(B, Hq, Hkv, width, page_size, ab2_num_sms());
  a.q = (const __nv_bfloat16*)q; a.kc = (const unsigned char*)kc; a.vc = (const unsigned char*)vc;
  a.ks = (const float*)ks; a.vs = (const float*)vs; a.table = table; a.lens = lens; a.out = (__nv_bfloat16*)out;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = G; a.groups = groups;
  a.page_size = page_size; a.page_bits = __builtin_ctz(page_size); a.width = width; a.num_pages = num_pages;
  a.scale_log2 = scale * 1.4426950408889634f; a.q_stride = q_stride; a.err = ab2host::error_flag();
  const int HP = G <= 8 ? 8 : 16;
  a.part_o = (float*)workspace;
  a.part_ml = (float4*)(a.part_o + 2LL * grid * HP * D);
  a.meta = (int2*)(a.part_ml + 2LL * grid * HP);
  cudaStream_t s = (cudaStream_t)stream;
  if (D == 128) return G <= 8 ? launch_kv8_decode<128, 1>(a, grid, s) : launch_kv8_decode<128, 2>(a, grid, s);
  return G <= 8 ? launch_kv8_decode<64, 1>(a, grid, s) : launch_kv8_decode<64, 2>(a, grid, s);
}

// n_buf buffers, each ten values in `desc`: address, plane, page and row strides in bytes, planes, rows, bytes of a row, bytes of a token in a
// row, pages, 0. pairs: n sources, n destinations, n numbers of tokens (host memory; < 0: whole page). No page may be both source and destination, or
// destination twice: the caller has checked it.
int ab2_copy_pages(const long long* desc, int n_buf, const int* pairs, int n, void* stream) {
  if (n <= 0 || n_buf <= 0) return 0;
  if (n_buf > COPY_BUFFERS) return 10;
  CopyArgs a;
  a.n_buf = n_buf;
  long long blocks = 0;
  int longest = 0;                                     // tokens of the longest copy; -1: whole pages
  for (int i = 0; i < n; ++i) {
    const int t = pairs[2 * n + i];
    if (t < 0) { longest = -1; break; }
    longest = t > longest ? t : longest;
  }
  for (int i = 0; i < n_buf; ++i) {
    const long long* d = desc + 10 * i;
    CopyBuffer& c = a.buf[i];
    if (d[6] * d[5] > 0x7fffffffLL - COPY_BYTES || d[6] <= 0 || d[5] <= 0 || d[4] <= 0) return 10;
    c.base = (unsigned char*)d[0];
    c.plane_stride = d[1]; c.page_stride = d[2]; c.row_stride = d[3];
    c.planes = (int)d[4]; c.rows = (int)d[5]; c.row_bytes = (int)d[6]; c.token_bytes = (int)d[7];
    c.first_block = (int)blocks;
    if (c.rows == 1 && c.token_bytes == 0 && c.row_bytes <= COPY_BYTES / 8) {       // a few bytes in each plane (scales): planes as rows
      c.rows = c.planes;
      c.planes = 1;
      c.row_stride = c.plane_stride;
      if ((long long)c.rows * c.row_bytes > 0x7fffffffLL - COPY_BYTES) return 10;
    }
    const long long most = c.token_bytes && longest >= 0 ? (long long)longest * c.token_bytes : c.row_bytes;
    c.per = (int)((most * c.rows + COPY_BYTES - 1) / COPY_BYTES);
    if (c.per < 1) c.per = 1;
    const long long all = d[0] | d[1] | d[2] | d[3] | d[6] | d[7];
    c.unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    blocks += (long long)c.per * c.planes;
    if (blocks > 0x7fffffffLL) return 10;
  }
  for (int at = 0; at < n; at += COPY_PAIRS) {
    const int m = n - at < COPY_PAIRS ? n - at : COPY_PAIRS;
    for (int i = 0; i < m; ++i) {
      a.src[i] = pairs[at + i]; a.dst[i] = pairs[n + at + i]; a.tokens[i] = pairs[2 * n + at + i];
    }
    launch_pdl(copy_pages_kernel, dim3((unsigned)blocks, m), dim3(256), 0, (cudaStream_t)stream, a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}
}
