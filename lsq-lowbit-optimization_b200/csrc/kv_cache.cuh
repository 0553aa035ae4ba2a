// The 4-bit key/value cache as the kernels see it: pages of packed int4 codes
// with one bfloat16 scale per token, head and group of channels.
//
//   codes  [pages][heads][page_size][D / 2]    two arrays, keys and values, with the same strides
//   scales [pages][heads][page_size][2][D / G] 0: keys, 1: values
//
// Token t of sequence b lies in row t % page_size of page block_table[b][t / page_size].
// Every index that comes from device memory (block table, lengths, row offsets) is checked
// here before it is used: a bad one reads as zeros, is not written to, and sets
// kErrCacheIndex in the device error word.
//
// All of it is read by ordinary loads: a block may be resident while the kernel ahead, which writes the cache, the rows or
// the tables, still runs (launch.cuh), and the read-only path promises data that nobody writes in a kernel's life.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.cuh"

namespace w4a8 {

constexpr unsigned kErrCacheIndex = 1u << 8;

// floor(t / d) = (umulhi(t, mul) + t) >> shift for 0 <= t < 2^31, with shift = ceil(log2 d) and
// mul = floor(2^32 (2^shift - d) / d) + 1; the sum does not carry.
struct FastDiv {
  unsigned mul, shift, d;
  __device__ __forceinline__ unsigned div(unsigned t) const { return (__umulhi(t, mul) + t) >> shift; }
  __device__ __forceinline__ void divmod(unsigned t, unsigned* q, unsigned* r) const {
    *q = div(t);
    *r = t - *q * d;
  }
};

struct KvView {
  uint8_t* k_codes;
  uint8_t* v_codes;
  __nv_bfloat16* scales;
  long long c_page, c_head, c_tok;  // strides of codes, bytes
  long long s_page, s_head, s_tok;  // strides of scales, elements
  int pages, page_size, heads, head_dim, group;
  FastDiv by_page;  // token / page_size
  const int* table;
  long long table_ld;
  int table_cols;
  int batch;
  const int* seq_lens;
  const int* cu_q;  // null: rows / batch rows a sequence
  int rows;
  unsigned* err;
};

__device__ __forceinline__ void kv_error(const KvView& v) { atomicOr(v.err, kErrCacheIndex); }

__device__ __forceinline__ int kv_page_of(const KvView& v, int t) { return int(v.by_page.div(unsigned(t))); }

// Most tokens of a sequence that the block table can name; the host has seen to at most 2^30.
__device__ __forceinline__ int kv_capacity(const KvView& v) { return v.table_cols * v.page_size; }

struct KvSeq {
  int row0;  // first packed row
  int n;     // packed rows
  int len;   // tokens, the packed rows' own included
};

__device__ __forceinline__ KvSeq kv_seq(const KvView& v, int b) {
  KvSeq s;
  bool bad = false;
  if (v.cu_q) {
    s.row0 = v.cu_q[b];
    const int end = v.cu_q[b + 1];
    if (s.row0 < 0 || end < s.row0 || end > v.rows) {
      bad = true;
      s.row0 = 0;
      s.n = 0;
    } else {
      s.n = end - s.row0;
    }
  } else {
    s.n = v.rows / v.batch;
    s.row0 = b * s.n;
  }
  s.len = v.seq_lens[b];
  const int cap = kv_capacity(v);
  if (s.len < 0 || s.len > cap) {
    bad = true;
    s.len = s.len < 0 ? 0 : cap;
  }
  if (bad) kv_error(v);
  return s;
}

// Page of token t (0 <= t < capacity) of sequence b, or -1 where the table names none.
__device__ __forceinline__ int kv_page_id(const KvView& v, int b, int p) {
  const int id = v.table[(long long)b * v.table_ld + p];
  if (unsigned(id) >= unsigned(v.pages)) {
    kv_error(v);
    return -1;
  }
  return id;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

}  // namespace w4a8
