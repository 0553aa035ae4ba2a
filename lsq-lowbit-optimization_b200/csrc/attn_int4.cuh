// Attention over the 4-bit key/value cache, for few query rows a key head (decode, drafts).
//
// One warp takes 32 tokens at a time and keeps everything of a tile in registers: scores
// S^T = K q^T (tokens x query rows), weights, and O^T += V^T P^T (channels x query rows), so
// that the codes are the left operands of mma.m16n8k16 and are unpacked where they are used,
// each once for all 8 NT query rows. The rows of a key head are its query heads of all the
// sequence's query tokens. Warps of a block take tiles in turn and are joined at the end; blocks
// split the tokens of a sequence, and a second kernel joins those (kv_attn_join_kernel).
//
// Why mma.sync and not tcgen05: a decode step has 8 or 16 query rows for each key head, which
// fills 1/16 of a 128-row tensor-core tile, and unpacked operands would have to pass through
// shared memory at four times the size of the codes. In registers they never leave the warp.
//
// No unit is full: about 700 instructions for 32 tokens of a head, a quarter of them the shifts and logic that unpack, fill
// 57 to 60% of the issue slots, 50% of the ALU's, 29% of the tensor cores', 39% of the memory's. A scheduler has 3.5
// warps, which is what 128 registers a lane allow, and 1.2 of them can issue: their dependent instructions and the start
// of a block bound it. One sequence of 131072 tokens, 32 query heads on 8 of 128 channels, bfloat16:
// 47 us, 3.0 TB/s. 64 sequences of up to 8192 tokens, 64 heads on 8: 109 us, 2.8 TB/s.
//
// Codes. A 32-bit word of a row is eight channels; word & 0x000f000f is the pair (0, 4),
// >> 8 the pair (2, 6). With the sign bit flipped a nibble is n = c + 8 >= 0.
//  * Keys: as float16 bits, n is the subnormal n 2^-24 and n << 4 is 16 n 2^-24, exact and
//    without any conversion. The query is scaled to a largest magnitude near 2^14 by a power of
//    two, its pairs (1, 5) and (3, 7) are divided by 16, and the accumulators start at
//    -8 2^-24 sum(q): sums of a group come out signed. They are multiplied by the key's scale in
//    32 bits. (The tensor cores cut products off 25 bits below the largest of a step, and count a subnormal as 2^-14
//    there: what a channel adds to a score is off by up to 2^-15 of the largest |q| times the key's scale.)
//    For float32 queries 8 is subtracted from n first, and the query is two terms with sums of their own: the scaled
//    query rounded to multiples of 8, whose sums are integers below 2^24 and so exact in spite of that, and what is
//    left. Off by 3e-7 for scores of standard deviation 4, 1e-6 to 2e-6 with two float16 roundings in one sum.
//  * Values: as bfloat16 bits, 0x4300 | n is 128 + n, and 136 is subtracted (exact). Here the
//    sums run over thousands of tokens and would cancel 136 sum(p) to its last bits.
// Weights times the value's scale are bfloat16 terms, whose range is that of the scales: two, which keep 15 bits, and
// for float32 queries three (24 bits), with a product each. The two come from two terms of the weight by three bfloat16
// multiply-adds, since what the first product leaves is exact in bfloat16. With one term a call took 44 us in place of
// 47 (131072 tokens) and 97 in place of 108 (64 sequences), but its rounding adds as much to the error as that of a
// bfloat16 output: 2.3e-3 against 1.7e-3 from the formula in 64 bits.
#pragma once

#include "kv_cache.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace w4a8 {

constexpr int kAttnWarps = 4;
constexpr int kTile = 32;  // tokens of a warp's tile

struct AttnParams {
  CUtensorMap k_map, v_map;  // codes as [pages][heads][page_size][D / 2] bytes, boxes of box_rows rows
  int box_rows;              // 0: the pages do not allow boxes, rows are copied one by one
  KvView view;
  const void* q;
  long long q_row, q_head;  // strides, elements
  int q_vec;                // 16-byte loads of q allowed
  void* out;                // [rows][q_heads][D]
  float* lse;               // [rows][q_heads] or null
  int q_heads, ratio;       // ratio = q_heads / heads
  FastDiv by_ratio, by_splits, by_row_tiles, by_heads;
  float scale_log2;         // |scale| * log2(e)
  float sign;               // of scale
  int causal, window;
  int max_q;                // sequences with more rows are refused
  int row_tiles;            // tiles of 8 NT query rows of a key head
  int splits, chunk;        // blocks a sequence, tokens a block
  float* part_o;            // [rows * q_heads][splits][D]
  float2* part_ml;          // [rows * q_heads][splits]: what scores are taken relative to (log2), sum of weights
  int* handover;            // many rows: for each block, whether its rows are left to kv_attn_redo_kernel
};

// Token and head of query row r of a key head, by division with by_ratio.
struct QueryRow {
  int token, head;
};
__device__ __forceinline__ QueryRow query_row(const AttnParams& p, int r) {
  unsigned t, h;
  p.by_ratio.divmod(unsigned(r), &t, &h);
  return {int(t), int(h)};
}

// Sequence, key head, row tile and split of a block: splits fastest.
struct BlockWork {
  int b, head, row_tile, split;
};
__device__ __forceinline__ BlockWork block_work(const AttnParams& p, unsigned i) {
  unsigned split, row_tile, head;
  p.by_splits.divmod(i, &i, &split);
  p.by_row_tiles.divmod(i, &i, &row_tile);
  p.by_heads.divmod(i, &i, &head);
  return {int(i), int(head), int(row_tile), int(split)};
}

// Tokens that the query rows [r0, r1) of a key head see: [begin, end), begin rounded down to a whole tile
// of `tile` tokens. Row r is query token r / ratio.
__device__ __forceinline__ void attn_range(const AttnParams& p, const KvSeq& s, int r0, int r1, int tile, int* begin,
                                           int* end) {
  const int first = s.len - s.n + query_row(p, r0).token, last = s.len - s.n + query_row(p, r1 - 1).token;
  *end = p.causal ? min(s.len, last + 1) : s.len;
  *begin = p.window > 0 ? max(0, max(0, first) - p.window + 1) / tile * tile : 0;  // first may be -2^31
  if (last < 0) *end = 0;  // rows without a position
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void cp_async_ca(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes),
               "r"(take ? kBytes : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// One box of rows of a page: coordinates byte 0, row of the page, head, page.
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head,
                                              int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(row), "r"(head), "r"(page)
      : "memory");
}
template <int kWords, int kAlign>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&r)[kWords]) {
  if constexpr (kWords % 4 == 0 && kAlign % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
                   : "r"(addr + 4 * i)
                   : "memory");
  } else if constexpr (kWords % 2 == 0 && kAlign % 8 == 0) {
#pragma unroll
    for (int i = 0; i < kWords; i += 2)
      asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[i]), "=r"(r[i + 1]) : "r"(addr + 4 * i) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[i]) : "r"(addr + 4 * i) : "memory");
  }
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint16_t x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void sts_u16(uint32_t addr, uint16_t x) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(x) : "memory");
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t neg_bf16x2(uint32_t a) {
  uint32_t d;
  asm("neg.bf16x2 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (w & mask) ^ flip in one logic instruction.
__device__ __forceinline__ uint32_t and_xor(uint32_t w, uint32_t mask, uint32_t flip) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(w), "r"(mask), "r"(flip));
  return d;
}
__device__ __forceinline__ uint32_t sub_136(uint32_t pair) {
  __nv_bfloat162 x = *reinterpret_cast<__nv_bfloat162*>(&pair);
  x = __hsub2(x, __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
  return *reinterpret_cast<uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t sub_half2(uint32_t x, uint32_t y) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}

template <typename T>
__device__ __forceinline__ void store4(T* dst, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(a, b, c, d);
  else if constexpr (std::is_same<T, __half>::value)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f16(a, b), pack_f16(c, d));
  else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}

// Two float32 at once.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair2(uint64_t d, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Rows [from, to) of the given query heads become zeros, lse -inf; by all threads of a block.
template <typename T>
__device__ void attn_clear_rows(const AttnParams& p, int from, int to, int head0, int heads) {
  const int d = p.view.head_dim;
  const long long n = (long long)max(0, to - from) * heads * d;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) {
    const long long rh = i / d, row = from + rh / heads, at = row * p.q_heads + head0 + rh % heads;
    static_cast<T*>(p.out)[at * d + i % d] = from_f32<T>(0.0f);
    if (i % d == 0 && p.lse) p.lse[at] = __uint_as_float(0xff800000u);
  }
}

// Rows before the first and behind the last sequence, which nobody computes: slices of them by the first
// kClearBlocks blocks.
constexpr int kClearBlocks = 8;

template <typename T>
__device__ void attn_clear_outside(const AttnParams& p, int slice, int slices) {
  const KvView& v = p.view;
  const int first = min(max(v.cu_q[0], 0), v.rows), last = min(max(v.cu_q[v.batch], first), v.rows);
  const int n = first + v.rows - last, from = int((long long)n * slice / slices),
            to = int((long long)n * (slice + 1) / slices);
  attn_clear_rows<T>(p, from, min(to, first), 0, p.q_heads);
  attn_clear_rows<T>(p, max(from, first) - first + last, to - first + last, 0, p.q_heads);
}

// Shared memory of one stage of one warp. Rows of codes are read eight at a time, 16 bytes
// each (ldmatrix): with 2, 4 or 8 pieces a row the piece's place is swizzled as the TMA does it (by
// address bits: the arrays are aligned to eight rows), with 3 the rows fall on different banks by themselves.
template <int D, int G>
struct AttnTile {
  static constexpr int kPieces = D / 32;
  static constexpr int kPitch = kPieces * 16;
  static constexpr int kGroups = D / G;
  static constexpr int kScaleBytes = 4 * kGroups;  // keys' and values' scales of a token
  static constexpr int kScalePiece = kScaleBytes % 16 == 0 ? 16 : kScaleBytes % 8 == 0 ? 8 : 4;
  static constexpr int kCodes = kTile * kPitch;
  static constexpr int kScales = kTile * kScaleBytes;
  static constexpr int kStages = 3;
  static constexpr int kRing = kAttnWarps * kStages;  // stages of a block
  static constexpr int kScalesAt = kRing * 2 * kCodes;
  static constexpr int kBytes = kScalesAt + kRing * kScales;
  static __device__ __forceinline__ int place(int row, int piece) {
    int p = piece;
    if constexpr (kPieces == 2) p ^= (row >> 2) & 1;
    if constexpr (kPieces == 4) p ^= (row >> 1) & 3;
    if constexpr (kPieces == 8) p ^= row & 7;
    return row * kPitch + p * 16;
  }
};

// Values' scales of the token pairs 8 k + 2 t4, + 1 (k = 0 .. 3) for one group, as bfloat16 pairs. Two groups share a word of a
// token where their number is even; where it is odd, words hold a key's and a value's.
template <typename Tile>
struct PairScales {
  static constexpr int kGroups = Tile::kGroups;
  uint32_t w[4][2];
  __device__ __forceinline__ void load(uint32_t scales, int t4, int grp) {
    const int e = kGroups + grp;  // its place among a token's scales
    if (grp && e % 2) return;     // the word of the group before
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t r[1];
        lds_words<1, 4>(scales + (8 * k + 2 * t4 + i) * Tile::kScaleBytes + e / 2 * 4, r);
        w[k][i] = r[0];
      }
  }
  __device__ __forceinline__ uint32_t get(int k, int grp) const {
    return __byte_perm(w[k][0], w[k][1], (kGroups + grp) % 2 ? 0x7632 : 0x5410);
  }
};

// Dynamic shared memory of a block: the warps' stages, later their results.
template <int D, int G, int NT>
constexpr int attn_smem_bytes() {
  const int stages = AttnTile<D, G>::kBytes, join = kAttnWarps * 8 * NT * (D + 4) * 4;
  return stages > join ? stages : join;
}

// Blocks an SM is to hold: what the registers of a lane allow (sums, the query, scores), and the stages.
// 131072 tokens, 128 channels, bfloat16, with one term of a weight: 43 us with 4, 52 with 3, 50 with 5.
constexpr int attn_blocks_sm(int d, int nt, bool f32) {
  return nt == 1 && d <= 128 && !f32 ? 4 : nt == 1 && d <= 128 ? 3 : 2;
}

// Query rows [r0, r1), at most 8 NT, of a key head over the tokens [begin, end), by a block. splits > 1: partial results of
// piece `split`. box_rows: 0, or p.box_rows with barriers that were initialised.
template <typename T, int D, int G, int NT>
__device__ __forceinline__ void attn_rows(const AttnParams& p, const KvSeq& seq, int b, int head, int r0, int r1, int begin,
                                          int end, int split, int splits, int box_rows, uint8_t* smem, uint64_t* full_bar,
                                          int* abort_flag) {
  using Tile = AttnTile<D, G>;
  constexpr int QT = sizeof(T) == 4 ? 2 : 1;                     // float16 terms of a query
  constexpr int PT = sizeof(T) == 4 ? 3 : 2;                     // bfloat16 terms of a weight
  constexpr bool kSigned = QT > 1;  // keys' codes are made signed first
  constexpr bool kPairs = PT == 2;  // weights take up the values' scales in pairs of tokens
  constexpr int kSegs = D / 32, kSegsGroup = G / 32, kGroups = Tile::kGroups, kStages = Tile::kStages;
  const KvView& v = p.view;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;

  const int ring = warp * kStages;
  const uint32_t my_codes = smem_u32(smem) + ring * 2 * Tile::kCodes;
  const uint32_t my_scales = smem_u32(smem) + Tile::kScalesAt + ring * Tile::kScales;
  const int tiles = end > begin ? (end - begin + kTile - 1) / kTile : 0;
  const int my_tiles = tiles > warp ? (tiles - warp + kAttnWarps - 1) / kAttnWarps : 0;

  // Copies of tile j of this warp. Lane l stands for token l: it knows the token's page, asked for
  // one tile earlier, and copies its scales. Codes come as boxes of box_rows tokens of one page, each by the lane
  // of its first token; where pages are not whole boxes, row by row.
  const long long c_head = head * v.c_head, s_head = head * v.s_head;
  const int* table = v.table + (long long)b * v.table_ld;
  int ahead = 0;  // page of token l of the tile that load_tile copies next
  auto ask_page = [&](int j) {
    const int t = begin + (warp + j * kAttnWarps) * kTile + lane;
    ahead = t < end ? table[kv_page_of(v, t)] : 0;
  };
  auto load_tile = [&](int j) {
    if (j < my_tiles) {
      const int t = begin + (warp + j * kAttnWarps) * kTile + lane, st = j % kStages;
      const uint32_t codes = my_codes + st * 2 * Tile::kCodes, scales = my_scales + st * Tile::kScales;
      const int id = ahead, at = t - kv_page_of(v, t) * v.page_size;
      bool have = t < end;
      if (have && unsigned(id) >= unsigned(v.pages)) {
        have = false;
        kv_error(v);
      }
      ask_page(j + 1);
      // Tokens without a page keep old codes; their scales are zeros.
      const uint8_t* src = reinterpret_cast<const uint8_t*>(
          v.scales + (have ? id * v.s_page + s_head + at * v.s_tok : 0));
#pragma unroll
      for (int k = 0; k < Tile::kScaleBytes; k += Tile::kScalePiece) {
        const uint32_t dst = scales + lane * Tile::kScaleBytes + k;
        if constexpr (Tile::kScalePiece == 16) cp_async_16(dst, src + k, have);
        else cp_async_ca<Tile::kScalePiece>(dst, src + k, have);
      }
      if (box_rows) {
        const bool copies = have && lane % box_rows == 0;
        const unsigned boxes = __popc(__ballot_sync(0xffffffffu, copies));
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[ring + st], boxes * 2u * unsigned(box_rows) * Tile::kPitch);
        __syncwarp();
        if (copies) {
          const uint32_t bar = smem_u32(&full_bar[ring + st]), dst = codes + lane * Tile::kPitch;
          tma_load_rows(dst, &p.k_map, bar, at, head, id);
          tma_load_rows(dst + Tile::kCodes, &p.v_map, bar, at, head, id);
        }
      } else {
        const long long c_off = have ? id * v.c_page + c_head + at * v.c_tok : -1;
#pragma unroll
        for (int k = 0; k < Tile::kPieces; ++k) {
          const int piece = k * 32 + lane, row = piece / Tile::kPieces, col = piece % Tile::kPieces;
          const long long off = __shfl_sync(0xffffffffu, c_off, row);
          const long long from = off < 0 ? 0 : off + col * 16;
          const uint32_t dst = codes + Tile::place(row, col);
          cp_async_16(dst, v.k_codes + from, off >= 0);
          cp_async_16(dst + Tile::kCodes, v.v_codes + from, off >= 0);
        }
      }
    }
    cp_async_commit();
  };
  ask_page(0);
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) load_tile(j);

  // The query as right operands: rows g of n-tile nt, channels 32 seg + 8 t4 + 0 .. 7.
  uint32_t qf[QT][NT][kSegs][4];
  float q_mul[NT][2];                // scores' factor for query rows 2 t4, 2 t4 + 1
  float s_init[NT][kGroups][2];      // -8 2^-24 sum(q) of a group
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + nt * 8 + g;
    float x[kSegs][8];
    float top = 0.0f;
    if (r < r1) {
      const QueryRow qr = query_row(p, r);
      const T* src = static_cast<const T*>(p.q) + (seq.row0 + qr.token) * p.q_row +
                     (head * p.ratio + qr.head) * p.q_head + t4 * 8;
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        if (sizeof(T) == 2 && p.q_vec) {
          const uint4 w = *reinterpret_cast<const uint4*>(src + s * 32);
          const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[s][k] = to_f32<T>(e[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[s][k] = to_f32<T>(src[s * 32 + k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[s][k]));
      }
    } else {
#pragma unroll
      for (int s = 0; s < kSegs; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k) x[s][k] = 0.0f;
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^up brings the largest magnitude into [2^13, 2^14); zero and infinite rows stay as they are.
    int up = 0;
    if (top > 0.0f && top < __uint_as_float(0x7f800000u)) {
      int e;
      frexpf(top, &e);
      up = max(-126, min(126, 14 - e));
    }
    const float mul = __int_as_float((127 + up) << 23) * p.sign;
    float sum[kGroups];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) sum[k] = 0.0f;
#pragma unroll
    for (int s = 0; s < kSegs; ++s) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[s][k] *= mul;  // the scale's sign included
#pragma unroll
      for (int term = 0; term < QT; ++term) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // Pairs (k, k + 4); odd ones meet codes that stand 16 times too large.
          const float f = k & 1 ? 0.0625f : 1.0f;
          float first = x[s][k], second = x[s][k + 4];
          if (kSigned && term == 0) {  // to multiples of 8, by 1.5 2^26 added and taken off
            first = __fadd_rn(__fadd_rn(first, 100663296.0f), -100663296.0f);
            second = __fadd_rn(__fadd_rn(second, 100663296.0f), -100663296.0f);
          }
          const uint32_t h = pack_f16(first * f, second * f);
          qf[term][nt][s][k] = h;
          const __half2 h2 = *reinterpret_cast<const __half2*>(&h);
          const float lo = __low2float(h2), hi = __high2float(h2);
          const float back = k & 1 ? 16.0f : 1.0f;
          sum[s / kSegsGroup] += (lo + hi) * back;
          x[s][k] -= lo * back;
          x[s][k + 4] -= hi * back;
        }
      }
    }
    const float factor = p.scale_log2 * 16777216.0f;
    const float unscale = __int_as_float((127 - up) << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      q_mul[nt][h] = fmaxf(__shfl_sync(0xffffffffu, unscale, (2 * t4 + h) * 4) * factor, 1.2e-38f);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s_init[nt][k][h] =
            kSigned ? 0.0f : __shfl_sync(0xffffffffu, sum[k], (2 * t4 + h) * 4) * (-8.0f / 16777216.0f);
    }
  }

  float o[kSegs * 2][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int k = 0; k < kSegs * 2; ++k)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][nt][e] = 0.0f;
  const float kNegInf = __uint_as_float(0xff800000u);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = kNegInf, l[nt][0] = l[nt][1] = 0.0f;

  const int first_pos = seq.len - seq.n;
  // Tokens from whole_from to whole_to are seen by every row of the tile.
  const int top_pos = first_pos + query_row(p, r0).token;
  const int whole_to = top_pos < 0 ? 0 : p.causal ? min(end, top_pos + 1) : end;
  const int whole_from = p.window > 0 ? max(0, first_pos + query_row(p, r1 - 1).token) - p.window + 1 : 0;

  for (int j = 0; j < my_tiles; ++j) {
    load_tile(j + kStages - 1);
    cp_async_wait<kStages - 1>();
    const int st = j % kStages;
    if (box_rows &&
        !__all_sync(0xffffffffu, mbar_wait(&full_bar[ring + st], (j / kStages) & 1, abort_flag))) {
      // A copy did not arrive: leave without any in flight.
      if (lane == 0) atomicOr(v.err, kErrTimeoutProducer);
      for (int k = j; k < min(my_tiles, j + kStages); ++k)
        for (int tries = 0; tries < 100000 && !mbar_try_wait(&full_bar[ring + k % kStages], (k / kStages) & 1); ++tries) {
        }
      break;
    }
    __syncwarp();
    const uint32_t codes = my_codes + st * 2 * Tile::kCodes;
    const int t0 = begin + (warp + j * kAttnWarps) * kTile;

    // Scales of tokens g, g + 8, g + 16, g + 24: keys' groups, then values' (not for pairs).
    const uint32_t scales = my_scales + st * Tile::kScales;
    uint32_t sc[4][kPairs ? (kGroups + 1) / 2 : kGroups];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      lds_words<kPairs ? (kGroups + 1) / 2 : kGroups, Tile::kScaleBytes>(scales + (g + 8 * k) * Tile::kScaleBytes, sc[k]);
    auto scale_of = [&](int k, int e) { return e & 1 ? bf16_hi(sc[k][e >> 1]) : bf16_lo(sc[k][e >> 1]); };

    float s[2][NT][4];  // [16-token half][n-tile]: tokens g, g + 8 x query rows 2 t4, 2 t4 + 1
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[h][nt][e] = 0.0f;
#pragma unroll
    for (int grp = 0; grp < kGroups; ++grp) {
      float acc[QT][2][NT][4];
#pragma unroll
      for (int seg = grp * kSegsGroup; seg < (grp + 1) * kSegsGroup; ++seg) {
        uint32_t w[4];
        ldmatrix_x4(codes + Tile::place(lane, seg), w);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = w[2 * h], w1 = w[2 * h + 1], y0 = w0 >> 8, y1 = w1 >> 8;
          uint32_t a0 = and_xor(w0, 0x000f000fu, 0x00080008u), a1 = and_xor(w1, 0x000f000fu, 0x00080008u);
          uint32_t a2 = and_xor(w0, 0x00f000f0u, 0x00800080u), a3 = and_xor(w1, 0x00f000f0u, 0x00800080u);
          uint32_t b0 = and_xor(y0, 0x000f000fu, 0x00080008u), b1 = and_xor(y1, 0x000f000fu, 0x00080008u);
          uint32_t b2 = and_xor(y0, 0x00f000f0u, 0x00800080u), b3 = and_xor(y1, 0x00f000f0u, 0x00800080u);
          if constexpr (kSigned) {
            a0 = sub_half2(a0, 0x00080008u), a1 = sub_half2(a1, 0x00080008u), b0 = sub_half2(b0, 0x00080008u);
            b1 = sub_half2(b1, 0x00080008u), a2 = sub_half2(a2, 0x00800080u), a3 = sub_half2(a3, 0x00800080u);
            b2 = sub_half2(b2, 0x00800080u), b3 = sub_half2(b3, 0x00800080u);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int term = 0; term < QT; ++term) {
              float(&c)[4] = acc[term][h][nt];
              if (seg == grp * kSegsGroup)
                mma_f16(c, a0, a1, a2, a3, qf[term][nt][seg][0], qf[term][nt][seg][1], s_init[nt][grp][0],
                        s_init[nt][grp][1], s_init[nt][grp][0], s_init[nt][grp][1]);
              else
                mma_f16(c, a0, a1, a2, a3, qf[term][nt][seg][0], qf[term][nt][seg][1], c[0], c[1], c[2], c[3]);
              mma_f16(c, b0, b1, b2, b3, qf[term][nt][seg][2], qf[term][nt][seg][3], c[0], c[1], c[2], c[3]);
            }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sum = QT > 1 ? acc[0][h][nt][e] + acc[QT - 1][h][nt][e] : acc[0][h][nt][e];
            s[h][nt][e] = fmaf(scale_of(2 * h + (e >> 1), grp), sum, s[h][nt][e]);
          }
    }
    if (t0 < whole_from || t0 + kTile > whole_to) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + 16 * h + 8 * (e >> 1) + g;
            const int pos = first_pos + query_row(p, r0 + nt * 8 + 2 * t4 + (e & 1)).token;
            const bool hidden = t >= end || (p.causal && t > pos) || (p.window > 0 && t <= pos - p.window) || pos < 0;
            if (hidden) s[h][nt][e] = kNegInf;
          }
      // A hidden value's weight is 0, and its scale may be NaN or infinite: take those groups out of the products, and
      // give NaN to the rows that do see such a value.
      auto v_scale_at = [&](int k, int grp) {
        return scales + (g + 8 * k) * Tile::kScaleBytes + 2 * (kGroups + grp);
      };
      auto v_scale = [&](int k, int grp) {
        if constexpr (kPairs) return bf16_lo(lds_u16(v_scale_at(k, grp)));
        else return scale_of(k, kGroups + grp);
      };
      bool nan = false;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int grp = 0; grp < kGroups; ++grp) nan |= !(fabsf(v_scale(k, grp)) <= 3.4e38f);
      if (__any_sync(0xffffffffu, nan)) {
#pragma unroll
        for (int grp = 0; grp < kGroups; ++grp) {
          bool hit[NT][2] = {};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (fabsf(v_scale(k, grp)) <= 3.4e38f) continue;
            if constexpr (!kPairs) sc[k][(kGroups + grp) >> 1] &= (kGroups + grp) & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r = 0; r < 2; ++r) hit[nt][r] |= s[k >> 1][nt][2 * (k & 1) + r] != kNegInf;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const unsigned lanes = __ballot_sync(0xffffffffu, hit[nt][r]);
              if (lanes & (0x11111111u << t4)) {
#pragma unroll
                for (int k = 2 * grp * kSegsGroup; k < 2 * (grp + 1) * kSegsGroup; ++k)
                  o[k][nt][r] = o[k][nt][r + 2] = __uint_as_float(0x7fc00000u);
              }
            }
        }
        if constexpr (kPairs) {  // four lanes have the same token
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int grp = 0; grp < kGroups; ++grp)
              if (t4 == 0 && !(fabsf(v_scale(k, grp)) <= 3.4e38f)) sts_u16(v_scale_at(k, grp), 0);
          __syncwarp();
        }
      }
    }

    // Weights 2^(s q_mul - m), q_mul > 0. m is raised only when some score passes it, and then to 8 above that score: most
    // tiles need no exchange between lanes and no rescaling, and weights are at most 1, so that their sums with values
    // near the largest number do not overflow before the mean of those does. The product is rounded
    // before m is taken off, as it was for m: of the largest score a fused one would leave what its rounding cut off.
    float top[NT][2];
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) s[h][nt][e + 2 * k] = __fmul_rn(s[h][nt][e + 2 * k], q_mul[nt][e]);
        top[nt][e] = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
        raise |= top[nt][e] > m[nt][e];
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = top[nt][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = x > m[nt][e] ? x + 8.0f : m[nt][e];
          const float c = x == kNegInf ? 1.0f : exp2_approx(m[nt][e] - x);
          m[nt][e] = x;
          l[nt][e] *= c;
#pragma unroll
          for (int k = 0; k < kSegs * 2; ++k) o[k][nt][e] *= c, o[k][nt][e + 2] *= c;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ref = m[nt][e] == kNegInf ? 0.0f : m[nt][e];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float w = exp2_approx(__fsub_rn(s[h][nt][e + 2 * k], ref));
            s[h][nt][e + 2 * k] = w;
            l[nt][e] += w;
          }
      }

    // O^T += V^T (P scale)^T. Half h holds tokens 16 h .. 16 h + 15 as its 16 products.
    uint32_t wt[2][2][NT][2];  // pairs: terms of the weights as right operands, [term][half][n-tile][tokens 0-7, 8-15]
    if constexpr (kPairs) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x = s[h][nt][2 * k], y = s[h][nt][2 * k + 1];
            const uint32_t w = pack_bf16(x, y);
            wt[0][h][nt][k] = movmatrix(w);
            wt[1][h][nt][k] = movmatrix(pack_bf16(x - bf16_lo(w), y - bf16_hi(w)));
          }
    }
    PairScales<Tile> pair_scales;
#pragma unroll
    for (int grp = 0; grp < kGroups; ++grp) {
      uint32_t pb[PT][2][NT][2];  // [term][half][n-tile][tokens 0-7, 8-15]
      if constexpr (kPairs) {
        pair_scales.load(scales, t4, grp);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t vs = pair_scales.get(2 * h + k, grp);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t x = mul_bf16x2(wt[0][h][nt][k], vs), left = fma_bf16x2(wt[0][h][nt][k], vs, neg_bf16x2(x));
              pb[0][h][nt][k] = x;
              pb[1][h][nt][k] = fma_bf16x2(wt[1][h][nt][k], vs, left);
            }
          }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float vs = scale_of(2 * h + k, kGroups + grp);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float x = s[h][nt][2 * k] * vs, y = s[h][nt][2 * k + 1] * vs;
              float rx = x, ry = y;
#pragma unroll
              for (int term = 0; term < PT; ++term) {
                const uint32_t w = pack_bf16(rx, ry);
                pb[term][h][nt][k] = movmatrix(w);
                rx -= bf16_lo(w), ry -= bf16_hi(w);
              }
            }
          }
      }
#pragma unroll
      for (int seg = grp * kSegsGroup; seg < (grp + 1) * kSegsGroup; ++seg) {
        uint32_t w[4];
        ldmatrix_x4_trans(codes + Tile::kCodes + Tile::place(lane, seg), w);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            const uint32_t w0 = w[2 * h], w1 = w[2 * h + 1];
            const uint32_t x0 = pair ? w0 >> 8 : w0, x1 = pair ? w1 >> 8 : w1;
            const uint32_t y0 = w0 >> (pair ? 12 : 4);
            const uint32_t y1 = w1 >> (pair ? 12 : 4);
            const uint32_t a0 = sub_136(and_xor(x0, 0x000f000fu, 0x43084308u));
            const uint32_t a1 = sub_136(and_xor(y0, 0x000f000fu, 0x43084308u));
            const uint32_t a2 = sub_136(and_xor(x1, 0x000f000fu, 0x43084308u));
            const uint32_t a3 = sub_136(and_xor(y1, 0x000f000fu, 0x43084308u));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int term = 0; term < PT; ++term)
                mma_bf16(o[2 * seg + pair][nt], a0, a1, a2, a3, pb[term][h][nt][0], pb[term][h][nt][1]);
          }
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
  }

  // Join the warps: each lane's sums over its tokens, then the warps' results in shared memory.
  cp_async_wait<0>();
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(smem);                    // [warp][row][D + 2]
  constexpr int kRow = D + 2;
  float* s_m = s_o + kAttnWarps * 8 * NT * kRow;                  // [warp][row]
  float* s_l = s_m + kAttnWarps * 8 * NT;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      const int row = warp * 8 * NT + nt * 8 + 2 * t4 + e;
      if (g == 0) {
        s_m[row] = m[nt][e];
        s_l[row] = x;
      }
#pragma unroll
      for (int k = 0; k < kSegs * 2; ++k) {
        // Channels 32 seg + 4 g + 2 pair, + 1.
        float2* dst = reinterpret_cast<float2*>(s_o + row * kRow + (k >> 1) * 32 + 4 * g + 2 * (k & 1));
        *dst = make_float2(o[k][nt][e], o[k][nt][e + 2]);
      }
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < (r1 - r0) * (D / 4); idx += kAttnWarps * 32) {
    const int row = idx / (D / 4), d = idx % (D / 4) * 4;
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w * 8 * NT + row]);
    const float ref = top == kNegInf ? 0.0f : top;
    float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float c = exp2_approx(s_m[w * 8 * NT + row] - ref);
      sum = fmaf(s_l[w * 8 * NT + row], c, sum);
      const float* src = s_o + (w * 8 * NT + row) * kRow + d;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = fmaf(src[k], c, x[k]);
    }
    const int r = r0 + row;
    const QueryRow qr = query_row(p, r);
    const long long at = (long long)(seq.row0 + qr.token) * p.q_heads + head * p.ratio + qr.head;
    if (splits > 1) {
      float4* dst = reinterpret_cast<float4*>(p.part_o + (at * splits + split) * D + d);
      *dst = make_float4(x[0], x[1], x[2], x[3]);
      if (d == 0) p.part_ml[at * splits + split] = make_float2(top, sum);
    } else {
      const float inv = sum == 0.0f ? 0.0f : __frcp_rn(sum);
      store4(static_cast<T*>(p.out) + at * D + d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      if (d == 0 && p.lse) p.lse[at] = sum == 0.0f ? kNegInf : (top + log2f(sum)) * 0.69314718055994531f;
    }
  }
}

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32, attn_blocks_sm(D, NT, sizeof(T) == 4))
    kv_attn_int4_kernel(const __grid_constant__ AttnParams p) {
  using Tile = AttnTile<D, G>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full_bar[Tile::kRing];
  __shared__ int abort_flag;
  pdl_trigger();
  const KvView& v = p.view;
  if (p.box_rows) {
    if (threadIdx.x < Tile::kRing) mbar_init(&full_bar[threadIdx.x], 1);
    if (threadIdx.x == 0) {
      abort_flag = 0;
      tma_prefetch_desc(&p.k_map);
      tma_prefetch_desc(&p.v_map);
    }
    fence_mbarrier_init();
    __syncthreads();
  }
  const BlockWork work = block_work(p, blockIdx.x);
  const int split = work.split, row_tile = work.row_tile, head = work.head, b = work.b;
  pdl_wait();
  if (v.cu_q && blockIdx.x < kClearBlocks)
    attn_clear_outside<T>(p, int(blockIdx.x), min(int(gridDim.x), kClearBlocks));
  const KvSeq seq = kv_seq(v, b);
  if (seq.n > p.max_q) {
    kv_error(v);
    if (row_tile == 0 && split == 0)
      attn_clear_rows<T>(p, seq.row0, seq.row0 + seq.n, head * p.ratio, p.ratio);
    return;
  }
  const int rows = seq.n * p.ratio, r0 = row_tile * 8 * NT;
  if (r0 >= rows) return;
  const int r1 = min(rows, r0 + 8 * NT);
  int begin, end;
  attn_range(p, seq, r0, r1, kTile, &begin, &end);
  begin += split * p.chunk;
  if (begin >= end && split) return;  // the join counts the splits that have tokens
  if (split + 1 < p.splits) end = min(end, begin + p.chunk);  // the last one takes what is left
  attn_rows<T, D, G, NT>(p, seq, b, head, r0, r1, begin, end, split, p.splits, p.box_rows, smem, full_bar, &abort_flag);
}

// Joins the splits of a sequence, each read once. kLanes = kJoinLanes: a block a query row, D / 4 threads times kLanes
// that take the splits in turn, where there are few rows of many splits. kLanes = 1: a block for kJoinLanes
// rows, where there are many rows (one block each took 14 us for 4096 rows of two splits, against 4).
constexpr int kJoinLanes = 8;

template <typename T, int D, int kLanes>
__global__ void __launch_bounds__(kJoinLanes * D / 4) kv_attn_join_kernel(const __grid_constant__ AttnParams p,
                                                                          int tile_rows, int tile_tokens) {
  pdl_trigger();
  const KvView& v = p.view;
  const BlockWork work = block_work(p, blockIdx.x * unsigned(p.splits));
  const int d = threadIdx.x % (D / 4), y = threadIdx.x / (D / 4), lane = kLanes > 1 ? y : 0;
  pdl_wait();
  const KvSeq seq = kv_seq(v, work.b);
  const int rows = seq.n * p.ratio, r0 = work.row_tile * tile_rows;
  const int r = r0 + int(kLanes > 1 ? blockIdx.y : blockIdx.y * kJoinLanes + y);
  if (r >= min(rows, r0 + tile_rows) || seq.n > p.max_q) return;
  int begin, end;
  attn_range(p, seq, r0, min(rows, r0 + tile_rows), tile_tokens, &begin, &end);
  const int splits = max(1, min(p.splits, (end - begin + p.chunk - 1) / p.chunk));
  const QueryRow qr = query_row(p, r);
  const long long at = (long long)(seq.row0 + qr.token) * p.q_heads + work.head * p.ratio + qr.head;
  const float kNegInf = __uint_as_float(0xff800000u);
  const float2* ml = p.part_ml + at * p.splits;
  float top = kNegInf;
  if constexpr (kLanes > 1) {
    for (int s = threadIdx.x & 31; s < splits; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  } else {
#pragma unroll 4
    for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s].x);
  }
  const float ref = top == kNegInf ? 0.0f : top;
  const float4* o = reinterpret_cast<const float4*>(p.part_o + at * p.splits * D) + d;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
#pragma unroll 8
  for (int s = lane; s < splits; s += kLanes) {
    const float2 w = ml[s];
    const float4 z = o[s * (D / 4)];
    const float c = exp2_approx(w.x - ref);
    sum = fmaf(w.y, c, sum);
    x.x = fmaf(z.x, c, x.x), x.y = fmaf(z.y, c, x.y), x.z = fmaf(z.z, c, x.z), x.w = fmaf(z.w, c, x.w);
  }
  if constexpr (kLanes > 1) {
    __shared__ float4 s_x[kLanes][D / 4];
    __shared__ float s_sum[kLanes];
    s_x[lane][d] = x;
    if (d == 0) s_sum[lane] = sum;
    __syncthreads();
    if (lane) return;
#pragma unroll
    for (int k = 1; k < kLanes; ++k) {
      const float4 z = s_x[k][d];
      x.x += z.x, x.y += z.y, x.z += z.z, x.w += z.w;
      sum += s_sum[k];
    }
  }
  const float inv = sum == 0.0f ? 0.0f : __frcp_rn(sum);
  store4(static_cast<T*>(p.out) + at * D + d * 4, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  if (d == 0 && p.lse) p.lse[at] = sum == 0.0f ? kNegInf : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace w4a8
