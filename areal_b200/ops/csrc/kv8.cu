// Paged key/value cache held in 8 bits, and the page copies of either cache.
//
// Layout: codes e4m3 [pages, Hkv, page_size, D], so that the block of one page and head is one contiguous run; scales fp32
// [pages, Hkv], powers of two, one for each such block. value = code * scale. A power of two divides and multiplies exactly:
// quantising rounds once, and a block whose scale has to grow (a larger row arrives) is re-coded without a second rounding
// except where a code falls below e4m3's normal range. e4m3 is a floating format, so a scale that is not a power of two would
// not make its relative steps any finer.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

extern "C" int ab2_num_sms();

namespace ab2 {

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
__device__ __forceinline__ float amax8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16(w[i]);
    a = fmaxf(a, fmaxf(finite_abs(f.x), finite_abs(f.y)));
  }
  return a;
}
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
// One warp = (row, head, keys or values). The whole call is a few hundred KB at most and bound by latency: one load of the
// row, one of the scale, one store of each; a warp re-codes its block (8 KB at 64 x 128) only when the scale grows.
template <int D>
__global__ void __launch_bounds__(128)
kv8_append_row_kernel(Kv8Args a, const int* __restrict__ table, const int* __restrict__ lens, int B, int Hkv, int page_size, int width,
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
// in one contiguous run. Which page a block has: the pages of sequence b are numbered from cu[b] / page_size + 2 b on, which
// leaves room for the floor(n / page_size) + 2 that n rows can touch, so no scan over the batch is needed.
template <int D, int NV>          // NV: 16-byte pieces of a thread = page_size * D / 8 / 128
__global__ void __launch_bounds__(128)
kv8_append_page_kernel(Kv8Args a, const int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ cu, int B, int rows,
                       int Hkv, int page_size, int width, int num_pages, int* __restrict__ err) {
  __shared__ float red[4];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, item = blockIdx.x, h = blockIdx.y >> 1, kv = blockIdx.y & 1;
  int b = -1;
  for (int i0 = 0; i0 < B; i0 += 128) {                // numbers grow with b: how many do not pass this block's
    const int i = i0 + tid;
    const int n = __syncthreads_count(i < B && cu[min(i, B - 1)] / page_size + 2 * i <= item);
    b += n;
    if (n < 128) break;
  }
  if (b < 0) return;
  const int c0 = cu[b], n = cu[b + 1] - c0, end = lens[b], start = end - n;
  if (n <= 0) return;
  const int j = start / page_size + item - (c0 / page_size + 2 * b);
  const int lo = max(start, j * page_size), hi = min(end, (j + 1) * page_size);
  if (start >= 0 && lo >= hi) return;
  const int page = start >= 0 && j < width && c0 >= 0 && c0 + n <= rows ? table[(size_t)b * width + j] : -1;
  if (page < 0 || page >= num_pages) {
    if (tid == 0) set_error(err, ERR_BOUNDS);
    return;
  }
  const size_t blk = (size_t)page * Hkv + h;
  const int slot = lo - j * page_size, cnt = hi - lo;
  float* scale = kv ? a.scales[1] : a.scales[0];
  const float old = slot ? scale[blk] : 0.f;
  const long long stride = kv ? a.stride[1] : a.stride[0];
  const __nv_bfloat16* x = (kv ? a.x[1] : a.x[0]) + (size_t)(c0 + lo - start) * stride + h * D;
  uint4 v[NV];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = tid + i * 128, row = p / (D / 8), piece = p % (D / 8);
    v[i] = row < cnt ? *reinterpret_cast<const uint4*>(x + row * stride + piece * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, amax8(v[i]));
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
// o = softmax(scale * q K^T) V over the first lens[b] tokens, G query heads for each key/value head. Bound by the codes' bytes.
//
// Split: the tokens of all (sequence, head) items are cut into chunks of 64 and the chunks, in order, dealt evenly to the blocks of
// one resident wave, whatever the lengths are; a block that ends inside an item leaves (m, l, o) for the join kernel.
// Warp w of a block takes tokens 16 w .. 16 w + 15 of each chunk. Its codes go from global memory straight into the registers
// that the matrix instruction wants, one tile ahead, so there is no shared-memory round trip and no barrier in the loop:
//   S^T[16 tokens, 8 heads] = K Q^T: the sum over dims may be taken in any order, so a thread's 16 contiguous bytes of a row serve as
//     four steps of k = 16 (the queries are laid out to match);
//   O^T[D dims, 8 heads] += V^T P^T: rows (dims) may stand in any order too, so a thread's 16 contiguous dims of four tokens are
//     paired by byte permutes; P^T comes from S^T by an 8 x 8 transpose between registers.
// e4m3 converts to fp16 exactly; q is divided by a power of two for its head (exact), P is rounded to fp16 (11 bits, half a step
// 2^-12) around a running maximum that is only moved when a score passes it by 2^6, and both sums are fp32.
constexpr int KV8_CHUNK = 64;

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
__device__ __forceinline__ uint4 ldg_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

struct Kv8Decode {
  const __nv_bfloat16* q;
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens;
  __nv_bfloat16* out;
  float *part_o, *part_ml;      // [2 * grid][HP][D], [2 * grid][HP][2]
  int* meta;                    // [items]: how the item is split, for the join kernel
  int* err;
  int B, Hq, Hkv, G, groups, page_size, width, num_pages;
  float scale_log2;             // softmax scale * log2(e)
  long long q_stride;
};

// Codes of one 16-token tile in a thread's registers.
template <int D>
struct Kv8Tile {
  uint32_t k[2][D / 16];        // tokens gq and gq + 8: D / 64 pieces of 16 bytes at dims 64 c + 16 tq
  uint32_t v[4][D / 32];        // tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9: D / 8 bytes at dim gq * D / 8
};

template <int D, int NT>        // NT: tiles of 8 query heads
__global__ void __launch_bounds__(128, NT == 1 ? 3 : 2)
kv8_decode_kernel(Kv8Decode a) {
  constexpr int HP = 8 * NT;
  constexpr int KS = D / 16;            // steps of S; also D / 16 row tiles of O
  extern __shared__ __align__(16) unsigned char dsm[];
  float* mo = reinterpret_cast<float*>(dsm);                  // [4][HP][D + 4]
  float* mm = mo + 4 * HP * (D + 4);                          // [4][HP]
  float* ml = mm + 4 * HP;                                    // [4][HP]
  int* prefix = reinterpret_cast<int*>(ml + 4 * HP);          // [B + 1] chunks before sequence b
  __shared__ int wsum[4];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  const int Hv = a.Hkv * a.groups;
  const int room = a.width * a.page_size;
  auto length = [&](int b) { return min(max(a.lens[b], 0), room); };
  // ---- chunks of the sequences before each, the whole batch in every block (a few loads a thread)
  {
    int carry = 0;
    for (int i0 = 0; i0 < a.B; i0 += 128) {
      const int i = i0 + tid;
      if (i < a.B && blockIdx.x == 0 && a.lens[i] > room) set_error(a.err, ERR_BOUNDS);
      const int n = i < a.B ? (length(i) + KV8_CHUNK - 1) / KV8_CHUNK : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (lane == 31) wsum[warp] = s;
      __syncthreads();
      int before = carry;
      for (int w = 0; w < warp; ++w) before += wsum[w];
      if (i < a.B) prefix[i] = before + s - n;
      carry += wsum[0] + wsum[1] + wsum[2] + wsum[3];
      __syncthreads();
    }
    if (tid == 0) prefix[a.B] = carry;
    __syncthreads();
  }
  const long long total = (long long)prefix[a.B] * Hv;
  const long long grid = min((long long)gridDim.x, total);      // blocks with a share: none of them is empty
  if (blockIdx.x >= grid) return;
  long long pos = total * blockIdx.x / grid;
  const long long stop = total * (blockIdx.x + 1) / grid;
  bool first_segment = true;

  while (pos < stop) {
    // ---- which item, which of its chunks
    int lo = 0, hi = a.B;                                     // last b with Hv * prefix[b] <= pos and chunks of its own
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)prefix[mid] * Hv <= pos) lo = mid; else hi = mid;
    }
    const int b = lo, nc = prefix[b + 1] - prefix[b];
    const long long base = (long long)prefix[b] * Hv;
    const int hv = (int)((pos - base) / nc);
    const long long item0 = base + (long long)hv * nc;
    const int c0 = (int)(pos - item0), c1 = (int)min((long long)nc, stop - item0);
    const int h = hv / a.groups, g0 = (hv - h * a.groups) * 16, ng = min(a.G - g0, HP);
    const int len = length(b);
    const int* pt = a.table + (size_t)b * a.width;

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
        const uint2 w = hd < ng ? *reinterpret_cast<const uint2*>(qp + (s >> 2) * 64 + tq * 16 + (s & 3) * 4) : make_uint2(0u, 0u);
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

    float o[NT][KS][4], m_run[NT][2], l_run[NT][2], v_ref = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < KS; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      m_run[t][0] = m_run[t][1] = -1e30f;
      l_run[t][0] = l_run[t][1] = 0.f;
    }

    // ---- this warp's tiles: tokens 64 c + 16 warp of chunks c0 .. c1
    const int t_first = c0 * KV8_CHUNK + warp * 16;
    const int n_tiles = min(c1 - c0, max(0, (len - t_first + KV8_CHUNK - 1) / KV8_CHUNK));
    int pg = 0, pg_next = 0;                                   // lane i: page of tile 32 k + i
    float ksc = 0.f, vsc = 0.f;
    auto page_of = [&](int i) {
      int p = 0;
      if (i < n_tiles) {
        p = pt[(t_first + i * KV8_CHUNK) / a.page_size];
        if (p < 0 || p >= a.num_pages) { set_error(a.err, ERR_BOUNDS); p = 0; }
      }
      return p;
    };
    auto load = [&](int i, Kv8Tile<D>& x) {
      const int p = __shfl_sync(0xffffffffu, pg, i & 31);
      const int t = (t_first + i * KV8_CHUNK) % a.page_size;
      const size_t at = (((size_t)p * a.Hkv + h) * a.page_size + t) * D;
      const unsigned char* kp = a.kc + at + gq * D + tq * 16;
      const unsigned char* vp = a.vc + at + 2 * tq * D + gq * (D / 8);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          *reinterpret_cast<uint4*>(&x.k[r][4 * c]) = ldg_stream16(kp + r * 8 * D + c * 64);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned char* p4 = vp + ((r >> 1) * 8 + (r & 1)) * D;
        if constexpr (D == 128) *reinterpret_cast<uint4*>(&x.v[r][0]) = ldg_stream16(p4);
        else *reinterpret_cast<uint2*>(&x.v[r][0]) = ldg_stream8(p4);
      }
    };
    auto work = [&](int i, Kv8Tile<D>& x) {
      const float kscale = __shfl_sync(0xffffffffu, ksc, i & 31), vscale = __shfl_sync(0xffffffffu, vsc, i & 31);
      const int left = len - (t_first + i * KV8_CHUNK);         // tokens of the tile that exist (16 or more: all)
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint32_t a0 = half2_lo(x.k[0][j]), a2 = half2_hi(x.k[0][j]), a1 = half2_lo(x.k[1][j]), a3 = half2_hi(x.k[1][j]);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16_16816(s[t], a0, a1, a2, a3, qf[t][j][0], qf[t][j][1]);
      }
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f0 = qs[t][0] * kscale, f1 = qs[t][1] * kscale;
        s[t][0] = gq < left ? s[t][0] * f0 : -INFINITY;
        s[t][1] = gq < left ? s[t][1] * f1 : -INFINITY;
        s[t][2] = gq + 8 < left ? s[t][2] * f0 : -INFINITY;
        s[t][3] = gq + 8 < left ? s[t][3] * f1 : -INFINITY;
        grow |= fmaxf(s[t][0], s[t][2]) > m_run[t][0] + 6.f || fmaxf(s[t][1], s[t][3]) > m_run[t][1] + 6.f;
      }
      if (left < 16) {                                          // what stands behind the last token may be anything
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (2 * tq + (r >> 1) * 8 + (r & 1) >= left)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) x.v[r][c] = 0u;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = fmaxf(s[t][e], s[t][e + 2]);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            m = fmaxf(m, m_run[t][e]);
            const float al = fast_exp2(m_run[t][e] - m);
            m_run[t][e] = m;
            l_run[t][e] *= al;
#pragma unroll
            for (int i2 = 0; i2 < KS; ++i2) { o[t][i2][e] *= al; o[t][i2][e + 2] *= al; }
          }
      }
      if (vscale > v_ref) {                                     // values of this page have a larger scale than those before
        const float r = v_ref / vscale;
        v_ref = vscale;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i2 = 0; i2 < KS; ++i2) { o[t][i2][0] *= r; o[t][i2][1] *= r; o[t][i2][2] *= r; o[t][i2][3] *= r; }
      }
      const float pv = v_ref > 0.f ? vscale / v_ref * 512.f : 0.f;                  // p <= 2^6: 2^15 at most, and fp16 goes down to 2^-24
      uint32_t p0[NT], p1[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float e0 = fast_exp2(s[t][0] - m_run[t][0]), e1 = fast_exp2(s[t][1] - m_run[t][1]);
        const float e2 = fast_exp2(s[t][2] - m_run[t][0]), e3 = fast_exp2(s[t][3] - m_run[t][1]);
        l_run[t][0] += e0 + e2;
        l_run[t][1] += e1 + e3;
        p0[t] = transpose8x8(pack_f16(e0 * pv, e1 * pv));
        p1[t] = transpose8x8(pack_f16(e2 * pv, e3 * pv));
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) {                            // dims gq * D/8 + 2 j and + 2 j + 1
        const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
        const uint32_t w0 = __byte_perm(x.v[0][j >> 1], x.v[1][j >> 1], sel), w1 = __byte_perm(x.v[2][j >> 1], x.v[3][j >> 1], sel);
        const uint32_t a0 = half2_lo(w0), a1 = half2_hi(w0), a2 = half2_lo(w1), a3 = half2_hi(w1);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16_16816(o[t][j], a0, a1, a2, a3, p0[t], p1[t]);
      }
    };
    auto scales_of = [&]() {
      ksc = a.ks[(size_t)pg * a.Hkv + h];
      vsc = a.vs[(size_t)pg * a.Hkv + h];
    };
    if (n_tiles > 0) {
      pg = page_of(lane);
      scales_of();
      pg_next = page_of(32 + lane);
      Kv8Tile<D> x, y;
      load(0, x);
      for (int i = 0; i < n_tiles; i += 2) {                    // blocks of 32 tiles start at an even tile
        if (i + 1 < n_tiles) load(i + 1, y);
        work(i, x);
        const float ks1 = ksc, vs1 = vsc;
        if (i + 2 < n_tiles) {
          if (((i + 2) & 31) == 0) {
            pg = pg_next;
            scales_of();
            pg_next = page_of(i + 34 + lane);
          }
          load(i + 2, x);
        }
        if (i + 1 < n_tiles) {
          const float ks2 = ksc, vs2 = vsc;
          ksc = ks1; vsc = vs1;
          work(i + 1, y);
          ksc = ks2; vsc = vs2;
        }
      }
    }

    // ---- join the four warps; O^T fragments: element 0/1 = dim gq * D/8 + 2 j of heads 2 tq, 2 tq + 1; 2/3 = the next dim
    const float unit = v_ref * (1.f / 512.f);
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
        }
#pragma unroll
        for (int j = 0; j < KS; ++j)
          *reinterpret_cast<float2*>(&mo[(warp * HP + hd) * (D + 4) + gq * (D / 8) + 2 * j]) = make_float2(o[t][j][e] * unit, o[t][j][e + 2] * unit);
      }
    }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == nc;
    const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
    for (int i = tid; i < ng * D; i += 128) {
      const int g = i / D, d = i - g * D;
      float mx = mm[g];
#pragma unroll
      for (int w = 1; w < 4; ++w) mx = fmaxf(mx, mm[w * HP + g]);
      float l = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = fast_exp2(mm[w * HP + g] - mx);
        l += ml[w * HP + g] * f;
        acc += mo[(w * HP + g) * (D + 4) + d] * f;
      }
      if (whole) {
        a.out[((size_t)b * a.Hq + h * a.G + g0 + g) * D + d] = __float2bfloat16(acc / l);
      } else {
        a.part_o[((size_t)slot * HP + g) * D + d] = acc;
        if (d == 0) {
          a.part_ml[((size_t)slot * HP + g) * 2] = mx;
          a.part_ml[((size_t)slot * HP + g) * 2 + 1] = l;
        }
      }
    }
    if (c0 == 0 && tid == 0) {
      // blocks that hold the item: this one to the one with its last chunk, c * grid / total rounded up as the shares are
      int last = (int)(((item0 + nc) * grid - 1) / total);
      a.meta[b * Hv + hv] = whole ? 0 : (slot << 10) | (last - (int)blockIdx.x);
    }
    __syncthreads();                                            // the buffers are free for the next segment
    pos = item0 + c1;
    first_segment = false;
  }
}

// Joins the partial results of items that were split over blocks: the first in slot `slot`, the others in the first slot of the
// blocks behind. A row without tokens gets zeros.
template <int D, int NT>
__global__ void __launch_bounds__(D) kv8_join_kernel(Kv8Decode a) {
  constexpr int HP = 8 * NT;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq, d = threadIdx.x;
  const int h = hq / a.G, gh = hq - h * a.G, grp = gh / 16, g = gh - grp * 16;
  __nv_bfloat16* out = a.out + (size_t)blockIdx.x * D + d;
  if (a.lens[b] <= 0) {
    *out = __float2bfloat16(0.f);
    return;
  }
  const int meta = a.meta[b * a.Hkv * a.groups + h * a.groups + grp];
  if (meta == 0) return;
  const int slot = meta >> 10, more = meta & 1023, next = (slot >> 1) + 1;
  auto row = [&](int i) { return (size_t)(i == 0 ? slot : 2 * (next + i - 1)) * HP + g; };
  float mx = -INFINITY;
  for (int i = 0; i <= more; ++i) mx = fmaxf(mx, a.part_ml[row(i) * 2]);
  float l = 0.f, acc = 0.f;
#pragma unroll 8
  for (int i = 0; i <= more; ++i) {
    const float f = fast_exp2(a.part_ml[row(i) * 2] - mx);
    l += a.part_ml[row(i) * 2 + 1] * f;
    acc += a.part_o[row(i) * D + d] * f;
  }
  *out = __float2bfloat16(acc / l);
}

template <int D, int NT>
static int launch_kv8_decode(const Kv8Decode& a, int grid, cudaStream_t s) {
  constexpr int HP = 8 * NT;
  const int smem = (4 * HP * (D + 4) + 8 * HP + a.B + 1) * 4;
  auto kern = kv8_decode_kernel<D, NT>;
  static ab2host::DevState st;
  if (ab2host::prepare_launch(kern, (4 * HP * (D + 4) + 8 * HP + 8192 + 1) * 4, st, nullptr)) return 2;
  launch_pdl(kern, dim3(grid), dim3(128), (size_t)smem, s, a);
  launch_pdl(kv8_join_kernel<D, NT>, dim3(a.B * a.Hq), dim3(D), 0, s, a);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

// ------------------------------------------------------------------ page copies
// Copies pages src -> dst of up to four buffers in one launch: all planes (layers, keys and values, scales) of all pairs. A page of
// a plane is `rows` runs of bytes, `row_stride` apart, of which the first tokens * token_bytes of each are copied (all of them where
// tokens < 0). The pairs travel as kernel arguments, so a call needs no transfer. Bound by memory: 16 KB a block, 64 bytes a thread in flight.
constexpr int COPY_PAIRS = 256, COPY_BUFFERS = 4, COPY_BYTES = 16384;
struct CopyBuffer {
  unsigned char* base;
  long long plane_stride, page_stride, row_stride;
  int planes, rows, row_bytes, token_bytes, first_block, unit;     // unit: bytes of one access (16, 4 or 1)
};
struct CopyArgs {
  CopyBuffer buf[COPY_BUFFERS];
  int src[COPY_PAIRS], dst[COPY_PAIRS], tokens[COPY_PAIRS];
  int n_buf;
};
template <typename T>
__device__ __forceinline__ void copy_run(const unsigned char* s, unsigned char* d, int run, long long row_stride, int first, int last) {
  constexpr int U = sizeof(T), PER = 4;
  for (int i0 = first / U + threadIdx.x; i0 < last / U; i0 += PER * 256) {
    T v[PER];
    long long off[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = i0 + j * 256;
      if (i < last / U) {
        const int row = i / (run / U);
        off[j] = row * row_stride + (long long)(i - row * (run / U)) * U;
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
  const int per = (int)(((long long)c.rows * c.row_bytes + COPY_BYTES - 1) / COPY_BYTES);      // blocks of one plane
  const int k = blockIdx.x - c.first_block, plane = k / per, part = k - plane * per;
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
  const long long wave = (long long)sms * (G <= 8 ? 3 : 2);
  return (int)(most < wave ? most : wave);
}
long long ab2_kv8_decode_workspace(int B, int Hq, int Hkv, int D, int page_size, int width) {
  if (B <= 0 || Hkv <= 0 || Hq % Hkv) return 0;
  const int G = Hq / Hkv, groups = (G + 15) / 16, HP = G <= 8 ? 8 : 16;
  const long long slots = 2LL * kv8_grid(B, Hq, Hkv, width, page_size, ab2_num_sms());
  return slots * HP * (D + 2) * 4 + (long long)B * Hkv * groups * 4;
}

// q [B, Hq, D] bf16 (rows q_stride elements apart, heads dense), out [B, Hq, D] dense; cache and table as above; lens [B].
int ab2_kv8_decode(const void* q, const void* kc, const void* vc, const void* ks, const void* vs, const int* table, const int* lens, void* out,
                   void* workspace, int B, int Hq, int Hkv, int D, int page_size, int width, int num_pages, float scale, long long q_stride, void* stream) {
  if (B <= 0) return 0;
  if (D != 64 && D != 128) return 11;
  if (page_size <= 0 || page_size % 16) return 12;
  if (Hkv <= 0 || Hq % Hkv || (q_stride & 7) || width <= 0 || num_pages <= 0 || B > 8192 || (long long)width * page_size > 0x7fffffffLL - 64) return 10;
  Kv8Decode a;
  const int grid = kv8_grid(B, Hq, Hkv, width, page_size, ab2_num_sms());
  if (grid > 1023) return 13;
  a.q = (const __nv_bfloat16*)q; a.kc = (const unsigned char*)kc; a.vc = (const unsigned char*)vc;
  a.ks = (const float*)ks; a.vs = (const float*)vs; a.table = table; a.lens = lens; a.out = (__nv_bfloat16*)out;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.groups = (a.G + 15) / 16;
  a.page_size = page_size; a.width = width; a.num_pages = num_pages;
  a.scale_log2 = scale * 1.4426950408889634f; a.q_stride = q_stride; a.err = ab2host::error_flag();
  const int HP = a.G <= 8 ? 8 : 16;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + 2LL * grid * HP * D;
  a.meta = (int*)(a.part_ml + 2LL * grid * HP * 2);
  cudaStream_t s = (cudaStream_t)stream;
  if (D == 128) return a.G <= 8 ? launch_kv8_decode<128, 1>(a, grid, s) : launch_kv8_decode<128, 2>(a, grid, s);
  return a.G <= 8 ? launch_kv8_decode<64, 1>(a, grid, s) : launch_kv8_decode<64, 2>(a, grid, s);
}

// n_buf buffers, each ten values in `desc`: address, plane, page and row strides in bytes, planes, rows, bytes of a row, bytes of a token in a
// row, pages, 0. pairs: src, dst, tokens of n pairs (host memory), tokens < 0 = whole page. No page may be both source and destination, or
// destination twice: the caller has checked it.
int ab2_copy_pages(const long long* desc, int n_buf, const int* pairs, int n, void* stream) {
  if (n <= 0 || n_buf <= 0) return 0;
  if (n_buf > COPY_BUFFERS) return 10;
  CopyArgs a;
  a.n_buf = n_buf;
  long long blocks = 0;
  for (int i = 0; i < n_buf; ++i) {
    const long long* d = desc + 10 * i;
    CopyBuffer& c = a.buf[i];
    if (d[6] * d[5] > 0x7fffffffLL - COPY_BYTES || d[6] <= 0 || d[5] <= 0 || d[4] <= 0) return 10;
    c.base = (unsigned char*)d[0];
    c.plane_stride = d[1]; c.page_stride = d[2]; c.row_stride = d[3];
    c.planes = (int)d[4]; c.rows = (int)d[5]; c.row_bytes = (int)d[6]; c.token_bytes = (int)d[7];
    c.first_block = (int)blocks;
    const long long all = d[0] | d[1] | d[2] | d[3] | d[6] | d[7];
    c.unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    blocks += (d[6] * d[5] + COPY_BYTES - 1) / COPY_BYTES * d[4];
    if (blocks > 0x7fffffffLL) return 10;
  }
  for (int at = 0; at < n; at += COPY_PAIRS) {
    const int m = n - at < COPY_PAIRS ? n - at : COPY_PAIRS;
    for (int i = 0; i < m; ++i) {
      a.src[i] = pairs[3 * (at + i)]; a.dst[i] = pairs[3 * (at + i) + 1]; a.tokens[i] = pairs[3 * (at + i) + 2];
    }
    launch_pdl(copy_pages_kernel, dim3((unsigned)blocks, m), dim3(256), 0, (cudaStream_t)stream, a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}
}
