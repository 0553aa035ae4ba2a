// Writing rows to the 4-bit key/value cache and reading them back.
//
// Both are bound by memory and, for two-byte types, nearly as much by instructions, so a thread stays with one
// eight-channel chunk of a head (its column) and walks down packed rows: what depends on the column is
// computed once. A block finds its rows' places in the cache once (sequence, length, page: a chain
// of three loads), behind the first loads of the rows. A warp's accesses are whole lines on the float side, and a
// group's largest magnitude is a butterfly over G / 8 neighbouring lanes. 8 heads of 128 channels, bfloat16: 16384
// tokens are written in 24 us (3.5 TB/s, 145 instructions for eight channels), 65536 read in 59 us (5.8 TB/s).
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "kv_cache.cuh"
#include "attn_int4.cuh"
#include "kv_host.cuh"
#include "w4a8.h"

namespace {

using namespace w4a8;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kMostRows = 32;    // packed rows of a block
constexpr int kCuCached = 1024;  // row offsets a block keeps in shared memory

struct RowParams {
  KvView view;
  FastDiv by_cols, by_head;  // columns of a block and of a head
  int cols;                  // columns of a row: keys' heads, then values'
  int tile_rows;             // packed rows of a block
};

// The column of a thread: keys (0) or values (1), head, eight-channel chunk of the head; and its first row.
struct Column {
  unsigned which, head, c, row;
  bool some;
};
__device__ __forceinline__ Column column_of(const RowParams& p) {
  Column k;
  unsigned col, hd;
  p.by_cols.divmod(threadIdx.x, &k.row, &col);
  col += blockIdx.y * p.by_cols.d;
  k.some = threadIdx.x < kThreads / p.by_cols.d * p.by_cols.d && col < unsigned(p.cols);
  p.by_head.divmod(col, &hd, &k.c);
  k.which = hd >= unsigned(p.view.heads);
  k.head = hd - k.which * unsigned(p.view.heads);
  return k;
}

// Sequence of packed row `row`: the last b with cu[b] <= row.
__device__ __forceinline__ int seq_of_row(const KvView& v, const int* cu, int row) {
  int lo = 0, hi = v.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Where the rows of a block lie: byte offset of the codes of head 0 (-1: nowhere) and offset of the scales.
struct Places {
  long long codes[kMostRows], scales[kMostRows];
  int cu[kCuCached];
};

__device__ __forceinline__ void find_places(const KvView& v, Places& s, int row0, int rows) {
  const int* cu = v.cu_q;
  if (cu && v.batch < kCuCached) {  // one latency in place of a search's chain of them
    for (int i = threadIdx.x; i <= v.batch; i += kThreads) s.cu[i] = v.cu_q[i];
    cu = s.cu;
    __syncthreads();
  }
  if (int(threadIdx.x) < rows) {
    const int row = row0 + threadIdx.x;
    const int b = cu ? seq_of_row(v, cu, row) : row / (v.rows / v.batch);
    const KvSeq seq = kv_seq(v, b);
    const int t = seq.len - seq.n + (row - seq.row0);
    long long codes = -1, scales = 0;
    // Outside: a row of no sequence, or one before the sequence's first token.
    if (row >= seq.row0 && row < seq.row0 + seq.n && t >= 0) {
      const int p = kv_page_of(v, t), id = kv_page_id(v, b, p), at = t - p * v.page_size;
      if (id >= 0) {
        codes = id * v.c_page + at * v.c_tok;
        scales = id * v.s_page + at * v.s_tok;
      }
    }
    s.codes[threadIdx.x] = codes;
    s.scales[threadIdx.x] = scales;
  }
  __syncthreads();
}

// Rows are read once, and those of two-byte types take no place in L1 (16384 tokens written and read back: 42.9 us, 44.4 if
// they do). A thread has 32 bytes of a float32 row, in two loads of one sector that the second is to find there (5
// prompts: 12.5 us, 13.1 without).
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 w;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
               : "l"(__cvta_generic_to_global(p))
               : "memory");
  return w;
}

template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) {
        const uint4* from = reinterpret_cast<const uint4*>(p) + i;
        w[i] = sizeof(T) == 2 ? load_once(from) : *from;
      }
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T*>(w)[i]); }
  // Bits of the largest magnitude as a float: magnitudes compare like integers, NaN above infinity.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(get(i)) & 0x7fffffffu);
      return t;
    } else {
      uint32_t t = 0;
      const uint32_t q[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) t = __vmaxu2(t, q[i] & 0x7fff7fffu);
      const uint16_t m = uint16_t(max(t & 0xffffu, t >> 16));
      T e;
      memcpy(&e, &m, 2);
      return __float_as_uint(to_f32<T>(e)) & 0x7fffffffu;
    }
  }
};

// The integer nearest to x / s, ties to even, for s > 0 with at most 8 significant bits:
// the rounded quotient is off by at most one, and (q + 1/2) s is exact in 32 bits.
__device__ __noinline__ int nearest_code(float x, float s, int lo) {
  const float t = __fdiv_rn(x, s);
  int q = __float2int_rn(fminf(fmaxf(t, -16.0f), 16.0f));
  const float up = __fmul_rn(float(q) + 0.5f, s), down = __fmul_rn(float(q) - 0.5f, s);
  if (x > up || (x == up && (q & 1))) ++q;
  else if (x < down || (x == down && (q & 1))) --q;
  return max(lo, min(7, q));
}

// The smallest bfloat16 not below a / 7, for a finite a >= 0: from a bfloat16 that is at most two
// steps below it up to the first whose sevenfold (exact in 32 bits) reaches a.
__device__ __forceinline__ float group_scale(float a) {
  uint32_t u = __float_as_uint(a * 0.142857f) & 0xffff0000u;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (__uint_as_float(u) * 7.0f < a) u += 0x10000u;
  return __uint_as_float(u);
}

// Eight codes x / s (nearest, ties to even) as a word, for a positive s.
// x times the approximate reciprocal is off by less than 2^-19 where |x / s| < 8. With x of at most 11 bits a
// quotient that is no tie is 2^-13 away from one, so rounding to multiples of 2^-18 first (in the product's own
// rounding, 48 added; taken off with the constant that rounds to integers) makes ties exact again. With 24 bits the few quotients that near to a tie are decided
// by the exact form.
template <typename T, bool kClamp>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float s, int lo) {
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
  bool near = s < 1e-30f || s > 1e30f;
  constexpr float kShift = sizeof(T) == 2 ? 48.0f : 0.0f;
  constexpr float kMagic = 12582912.0f;  // 1.5 2^23: the sum's last bits are the nearest integer
  const uint64_t inv2 = pair2(inv, inv), shift = pair2(kShift, kShift), magic = pair2(kMagic - kShift, kMagic - kShift);
  uint32_t r[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    uint64_t t = fma2(pair2(x[e], x[e + 1]), inv2, shift);
    float a, b;
    if constexpr (kClamp) {
      unpair2(t, a, b);
      t = pair2(fminf(fmaxf(a, kShift + float(lo)), kShift + 7.0f), fminf(fmaxf(b, kShift + float(lo)), kShift + 7.0f));
    }
    const uint64_t y = add2(t, magic);
    unpair2(y, a, b);
    r[e] = __float_as_uint(a), r[e + 1] = __float_as_uint(b);
    if constexpr (sizeof(T) == 4) {
      float c, d;
      unpair2(t, c, d);
      near |= fmaxf(fabsf(c - (a - kMagic)), fabsf(d - (b - kMagic))) > 0.49999f;
    }
  }
  if (near) {
    uint32_t w = 0;
    for (int e = 0; e < 8; ++e) w |= (uint32_t(nearest_code(x[e], s, lo)) & 15u) << (4 * e);
    return w;
  }
  // r is the bits of kMagic plus the code. Digits code + 8 of base 16, added up modulo 2^32 with kMagic's share taken
  // off at the end; then the sign bits are turned.
  uint32_t w = r[7];
#pragma unroll
  for (int e = 6; e >= 0; --e) w = w * 16u + r[e];
  return (w + 0x88888888u - 0x4b400000u * 0x11111111u) ^ 0x88888888u;
}

struct WriteParams : RowParams {
  const void* x[2];
  long long x_row[2], x_head[2];  // strides, elements
  const float* step[2];           // learned steps [heads][D / G], or null
  int vec[2];                     // 16-byte loads allowed
};

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 4) kv_write_int4_kernel(const __grid_constant__ WriteParams p) {
  __shared__ Places places;
  pdl_trigger();
  const KvView& v = p.view;
  const int row0 = int(blockIdx.x) * p.tile_rows, rows = min(p.tile_rows, v.rows - row0);
  const Column k = column_of(p);
  const int down = int(kThreads / p.by_cols.d);        // rows that the block's threads take side by side
  constexpr unsigned kLanes = G / 8;                   // lanes of a group; they stay together
  const unsigned groups = unsigned(v.head_dim) / G, gi = k.c / kLanes;
  const bool vec = p.vec[k.which];
  const T* from = static_cast<const T*>(p.x[k.which]) + (row0 + int(k.row)) * p.x_row[k.which] +
                  k.head * p.x_head[k.which] + k.c * 8;
  uint8_t* codes = (k.which ? v.v_codes : v.k_codes) + k.head * v.c_head + k.c * 4;
  __nv_bfloat16* scales = v.scales + k.head * v.s_head + k.which * groups + gi;
  const float* step = p.step[k.which];
  pdl_wait();
  float learned = 0.0f;
  if (step && k.some) learned = __bfloat162float(__float2bfloat16_rn(step[k.head * groups + gi]));
  bool found = false;
  for (int base = 0; base < rows; base += down * kUnroll) {
    Raw8<T> raw[kUnroll] = {};
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (k.some && base + u * down + int(k.row) < rows) raw[u].load(from + (base + u * down) * p.x_row[k.which], vec);
    }
    if (!found) find_places(v, places, row0, rows);  // behind the first loads
    found = true;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {  // by whole warps up to the stores: shuffles with a mask cost more
      if (base + u * down >= rows) break;  // for all
      const int r = base + u * down + int(k.row);
      const long long at = k.some && r < rows ? places.codes[r] : -1;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = raw[u].get(e);
      uint32_t top = raw[u].top();  // bits of the largest magnitude, NaN above infinity
#pragma unroll
      for (unsigned d = kLanes / 2; d; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float kNan = __uint_as_float(0x7fc00000u);
      uint32_t w = 0;
      float s;
      if (step) {
        s = top > 0x7f800000u || !(learned > 0.0f && learned <= 3.4e38f) ? kNan : learned;
        if (s > 0.0f) w = codes_of<T, true>(x, s, -8);
      } else {
        s = top >= 0x7f800000u ? kNan : group_scale(__uint_as_float(top));
        if (s > 0.0f) w = codes_of<T, false>(x, s, -7);
      }
      if (at >= 0) {
        *reinterpret_cast<uint32_t*>(codes + at) = w;
        if (k.c % kLanes == 0) scales[places.scales[r]] = __float2bfloat16_rn(s);
      }
    }
  }
}

struct ReadParams : RowParams {
  void* out[2];  // [rows][heads][D], contiguous
};

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) kv_read_int4_kernel(const __grid_constant__ ReadParams p) {
  __shared__ Places places;
  pdl_trigger();
  const KvView& v = p.view;
  const int row0 = int(blockIdx.x) * p.tile_rows, rows = min(p.tile_rows, v.rows - row0);
  const Column k = column_of(p);
  const int down = int(kThreads / p.by_cols.d);
  constexpr unsigned kLanes = G / 8;
  const unsigned groups = unsigned(v.head_dim) / G;
  const uint8_t* codes = (k.which ? v.v_codes : v.k_codes) + k.head * v.c_head + k.c * 4;
  const __nv_bfloat16* scales = v.scales + k.head * v.s_head + k.which * groups + k.c / kLanes;
  const long long out_row = (long long)v.heads * v.head_dim;
  T* out = static_cast<T*>(p.out[k.which]) + row0 * out_row + k.head * v.head_dim + k.c * 8;
  pdl_wait();
  find_places(v, places, row0, rows);
  if (!k.some) return;
  for (int base = int(k.row); base < rows; base += down * kUnroll) {
    uint32_t w[kUnroll];
    uint16_t s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = base + u * down;
      w[u] = s[u] = 0;
      if (r < rows) {
        const long long at = places.codes[r];
        if (at >= 0) {
          w[u] = *reinterpret_cast<const uint32_t*>(codes + at);
          s[u] = *reinterpret_cast<const uint16_t*>(scales + places.scales[r]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = base + u * down;
      if (r >= rows) break;
      // Pairs (e, e + 4) of codes as bfloat16, exact.
      uint32_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = sub_136(and_xor(w[u] >> (4 * e), 0x000f000fu, 0x43084308u));
      T* to = out + r * out_row;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // The product is rounded once, as it should be.
        const uint32_t s2 = s[u] | uint32_t(s[u]) << 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&c[e]),
                                           *reinterpret_cast<const __nv_bfloat162*>(&s2));
          c[e] = *reinterpret_cast<const uint32_t*>(&y);
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410),
                                                   __byte_perm(c[0], c[1], 0x7632), __byte_perm(c[2], c[3], 0x7632));
      } else {
        const float f = __uint_as_float(uint32_t(s[u]) << 16);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = bf16_lo(c[e]) * f, x[e + 4] = bf16_hi(c[e]) * f;
        if constexpr (sizeof(T) == 4) {
          reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
          reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
          *reinterpret_cast<uint4*>(to) =
              make_uint4(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
        }
      }
    }
  }
}

// A block has columns side by side and rows below each other for its threads. Its rows are shared out so that
// all blocks run at once, four an SM, if that takes at most eight times kUnroll loads of a thread (5 prompts of 1237
// rows of 12 heads of 96, float32, written and read: 15.3 -> 13.0 us; 16384 tokens of 8 heads of 128, bfloat16: 47 ->
// 45); beyond that four times kUnroll are best (65536 tokens read, by read-only loads then: 60.7 us, 62.2 with eight).
template <typename P>
int launch_rows(void (*kern)(P), P p, cudaStream_t st) {
  const KvView& v = p.view;
  const unsigned per_head = unsigned(v.head_dim) / 8;
  const long long cols = 2ll * v.heads * per_head;
  // Columns side by side: of the multiples of 16 (a group's lanes) the one that leaves the fewest threads idle.
  unsigned wide = 16;
  double best = 0.0;
  for (unsigned w = kThreads; w >= 16; w -= 16) {
    const double used = double(kThreads / w * w) / kThreads * double(cols) / double((cols + w - 1) / w * w);
    if (used > best + 1e-9) best = used, wide = w;
  }
  const unsigned col_tiles = unsigned((cols + wide - 1) / wide);
  if (col_tiles > 65535) return W4A8_ERR_UNSUPPORTED;
  p.by_head = fast_div(per_head);
  p.by_cols = fast_div(wide);
  p.cols = int(cols);
  const long long at_once = 4ll * device_sms(), spread = ((long long)v.rows * col_tiles + at_once - 1) / at_once;
  const long long full = std::min<long long>(4ll * kUnroll * (kThreads / wide), kMostRows);
  p.tile_rows = int(spread <= std::min<long long>(2 * full, kMostRows) ? spread : full);
  const unsigned grid = unsigned((v.rows + (long long)p.tile_rows - 1) / p.tile_rows);
  if (launch_kernel(kern, dim3(grid, col_tiles), dim3(kThreads), 0, st, p) != cudaSuccess) return W4A8_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? W4A8_OK : W4A8_ERR_LAUNCH;
}

}  // namespace

extern "C" int w4a8_kv_write_int4(const w4a8_kv_cache* cache, const void* k, int64_t k_row, int64_t k_head,
                                  const void* v, int64_t v_row, int64_t v_head, int dtype, const float* k_step,
                                  const float* v_step, void* stream) {
  WriteParams p;
  const int rc = kv_view(cache, &p.view);
  if (rc != W4A8_OK) return rc;
  if (dtype < W4A8_F32 || dtype > W4A8_BF16) return W4A8_ERR_ARG;
  if (cache->rows == 0 || cache->batch == 0) return W4A8_OK;
  if (!k || !v) return W4A8_ERR_ARG;
  const int size = dtype == W4A8_F32 ? 4 : 2;
  const void* x[2] = {k, v};
  const int64_t strides[2][2] = {{k_row, k_head}, {v_row, v_head}};
  for (int i = 0; i < 2; ++i) {
    if (reinterpret_cast<uintptr_t>(x[i]) % size) return W4A8_ERR_ALIGN;
    p.x[i] = x[i];
    p.x_row[i] = strides[i][0];
    p.x_head[i] = strides[i][1];
    p.vec[i] = reinterpret_cast<uintptr_t>(x[i]) % 16 == 0 && strides[i][0] * size % 16 == 0 &&
               strides[i][1] * size % 16 == 0;
  }
  p.step[0] = k_step;
  p.step[1] = v_step;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // By type and group: 32 / 64 = 0, 64 / 64 = 1, 128 / 64 = 2.
  static void (*const kern[3][3])(WriteParams) = {
      {kv_write_int4_kernel<float, 32>, kv_write_int4_kernel<float, 64>, kv_write_int4_kernel<float, 128>},
      {kv_write_int4_kernel<__half, 32>, kv_write_int4_kernel<__half, 64>, kv_write_int4_kernel<__half, 128>},
      {kv_write_int4_kernel<__nv_bfloat16, 32>, kv_write_int4_kernel<__nv_bfloat16, 64>,
       kv_write_int4_kernel<__nv_bfloat16, 128>}};
  return launch_rows(kern[dtype][p.view.group / 64], p, st);
}

extern "C" int w4a8_kv_read_int4(const w4a8_kv_cache* cache, void* k, void* v, int dtype, void* stream) {
  ReadParams p;
  const int rc = kv_view(cache, &p.view);
  if (rc != W4A8_OK) return rc;
  if (dtype < W4A8_F32 || dtype > W4A8_BF16) return W4A8_ERR_ARG;
  if (cache->rows == 0) return W4A8_OK;
  if (!k || !v || cache->batch == 0) return W4A8_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return W4A8_ERR_ALIGN;
  p.out[0] = k;
  p.out[1] = v;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // By type and group: 32 / 64 = 0, 64 / 64 = 1, 128 / 64 = 2.
  static void (*const kern[3][3])(ReadParams) = {
      {kv_read_int4_kernel<float, 32>, kv_read_int4_kernel<float, 64>, kv_read_int4_kernel<float, 128>},
      {kv_read_int4_kernel<__half, 32>, kv_read_int4_kernel<__half, 64>, kv_read_int4_kernel<__half, 128>},
      {kv_read_int4_kernel<__nv_bfloat16, 32>, kv_read_int4_kernel<__nv_bfloat16, 64>,
       kv_read_int4_kernel<__nv_bfloat16, 128>}};
  return launch_rows(kern[dtype][p.view.group / 64], p, st);
}
