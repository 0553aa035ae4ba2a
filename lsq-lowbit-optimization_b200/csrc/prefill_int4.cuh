// Attention over the 4-bit key/value cache for many query rows a key head (prompts and their chunks), on
// the tensor cores of sm_100a.
//
// A block takes 256 query rows of one key head, two tiles of 128, and walks over its tokens 128 at a time:
//   S = Q K^T (tcgen05, operands in shared memory, sums in TMEM), P = 2^(S - m), O += P V (P in TMEM).
// Roles: two groups of four warps, one a tile and a thread a row, turn scores into weights; four warps
// unpack the next keys and four the next values; one issues the products. While one tile's weights are
// made the other's products run. A 128-token tile of codes is read once for 256 rows, and unpacked operands
// live in shared memory only.
//
// Bound by the chain of each tile: scores, weights, their hand-over, products; 4.7 k cycles for 128 tokens of 256
// rows of 128 channels, in which the exponentials alone take 2 k and the products 1.5 k. 8192 tokens, causal, 32
// query heads on 8 of 128 channels, bfloat16: 650 us, 846 TFLOP/s in short runs (half of the rate of a plain bfloat16
// matrix product), 680 us once the power limit lowers the clock.
//
// All operands are float16. code * scale has at most 11 significant bits, so keys and values are exact
// there for scales from 2^-17 to 2^12. Where the largest scale of a block's first tile is not within [2^-9, 2^8] they are
// held divided by a power of two, one for the block's keys and one for its values. A block that meets a scale outside
// of the range all the same (of a token that its rows see or not), or scores near 2^20, says so, and
// kv_attn_redo_kernel takes its rows again with the arithmetic of few rows. Otherwise large values, hidden ones even,
// would set the unit that small ones are lost in. A query is brought to a largest magnitude near 2^14 by a power of two.
//
// Weights are rounded to 11 bits, and to multiples of 2^-31 of the row's largest: that is what a long tail of small
// weights beside one large is off by. Two float16 terms would need twice the products and registers that a row does
// not have; error of float16 outputs 2.7e-4, of their own rounding 2.0e-4.
//
// TMEM (512 columns): S of tile 0 and 1 at 0 and 128, their weights over them; O at 256 and 384.
//
// Order of channels. A word of codes is unpacked as the pairs (0, 4), (1, 5), (2, 6), (3, 7) of
// its eight channels and stored like that; the query is stored in the same order, which a
// sum over channels does not see, and output channels are put back in registers.
#pragma once

#include "attn_int4.cuh"

namespace w4a8 {

constexpr int kPreTile = 128;                // tokens of a tile, and rows of a query tile
constexpr int kPreRows = 2 * kPreTile;       // query rows of a block
constexpr int kPreThreads = 20 * 32;         // 2 x 4 softmax warps, 2 x 4 unpacking warps, 1 issuing warp, 3 idle
constexpr int kPreIssuer = 16;               // its warp
constexpr int kPreStages = 2;                // tiles of keys, and of values, in shared memory
constexpr int kPrePanel = kPreTile * 128;    // 128 rows of 64 channels, swizzled 128-byte rows

template <int D>
struct PreSmem {
  static constexpr int kPanels = (D + 63) / 64;
  static constexpr int kTileBytes = kPanels * kPrePanel;
  static constexpr int kQ = 0;
  static constexpr int kK = 2 * kTileBytes;
  static constexpr int kV = kK + kPreStages * kTileBytes;
  static constexpr int kCodes = kV + kPreStages * kTileBytes;  // packed rows on their way: [stage][keys, values]
  static constexpr int kCodeBytes = kPreTile * D / 2;
  static constexpr int kBytes = kCodes + kPreStages * 2 * kCodeBytes;
};
template <int D>
constexpr int prefill_smem_bytes() {
  // The base is rounded up to 1024; more than half of an SM's, since a block takes all of its TMEM.
  return (PreSmem<D>::kBytes > 118 * 1024 ? PreSmem<D>::kBytes : 118 * 1024) + 1024;
}

// Weights are 2^(score - m). m is set so that the largest is 2^kPreHigh, and raised when one would pass 2^kPreRaise: float16
// goes up to 2^16, and what is small keeps bits down to 2^-24, which is 2^-31 of the largest or less.
constexpr float kPreHigh = 7.0f, kPreRaise = 15.0f, kPreLow = 0x1p-15f;
// A fused multiply-add of a score keeps what the rounding of m cut off: up to 2^-4 for m below 2^20, beyond which rows are
// handed over.
constexpr float kPreMost = 0x1p20f;

// Bits [from, to) of 32, either of them anywhere.
__device__ __forceinline__ uint32_t bits_between(int from, int to) {
  const uint32_t below = to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u;
  return from >= 32 ? 0u : from <= 0 ? below : below & ~((1u << from) - 1u);
}

constexpr bool prefill_ok(int head_dim, bool f32) { return head_dim <= 128 && !f32; }

// Byte offset of channel chunk c (eight channels) of row r in a tile.
__device__ __forceinline__ int pre_place(int r, int c) {
  return (c >> 3) * kPrePanel + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Whether this lane of a converged warp is the elected one.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 r;\n\telect.sync r|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(e));
  return e != 0;
}
// kind::f16: float32 sums of float16 products; A along K; B along K or along N.
__host__ __device__ constexpr uint32_t make_idesc_f16(bool b_along_n, uint32_t m, uint32_t n) {
  return (1u << 4) | (uint32_t(b_along_n) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// Registers a thread from here on: of the block's share, which setmaxnreg moves between warp groups.
template <int kRegs>
__device__ __forceinline__ void regs_less() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&r)[16]) {
  tmem_ld16(taddr, reinterpret_cast<uint32_t(&)[16]>(r));
}
// Waits for this thread's TMEM loads; the values are taken through it, so that no use of them moves ahead.
__device__ __forceinline__ void tmem_ld_wait32(float (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]),
                 "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]),
                 "+f"(r[30]), "+f"(r[31]));
}
__device__ __forceinline__ void tmem_ld_wait16(float (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of codes as signed float16, from bits 0-3 of each half and from bits 4-7.
__device__ __forceinline__ __half2 code_pair(uint32_t w) {
  const uint32_t x = and_xor(w, 0x000f000fu, 0x64086408u);  // 1024 + code + 8
  return __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6408)));
}
__device__ __forceinline__ __half2 code_pair_high(uint32_t w) {
  const uint32_t x = and_xor(w, 0x00f000f0u, 0x64806480u);  // 1024 + 16 (code + 8); / 16 - 72
  return __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x2c00)),
                 __half2half2(__ushort_as_half(0xd480)));
}
// Eight codes times their scale, in the stored order.
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 s) {
  const uint32_t y = w >> 8;
  const __half2 r[4] = {__hmul2(code_pair(w), s), __hmul2(code_pair_high(w), s), __hmul2(code_pair(y), s),
                        __hmul2(code_pair_high(y), s)};
  return *reinterpret_cast<const uint4*>(r);
}
// The power of two that keys or values are held divided by, from the bits of the largest scale of a block's first tile.
__device__ __forceinline__ float pre_unit(uint32_t top) {
  const float f = __uint_as_float(top);
  return f == 0.0f || (f >= 0x1p-9f && f <= 0x1p8f) ? 1.0f : __uint_as_float(max(top & 0x7f800000u, 0x00800000u));
}

// All threads of one of the two groups of unpacking warps.
__device__ __forceinline__ void pre_group_sync(int which) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + which) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) return pack_f16(lo, hi);
  else return pack_bf16(lo, hi);
}

// Bounded wait without a call: a function's fixed registers and setmaxnreg do not go together.
__device__ __forceinline__ bool pre_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  unsigned long long t0 = 0;
  for (uint32_t spins = 1; !mbar_try_wait(bar, parity); ++spins) {
    if (spins & 63) continue;
    if (*abort_flag) return false;
    const unsigned long long t = global_timer_ns();
    if (!t0) t0 = t;
    if (t - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

// The same for warps that are ahead of the others: the hardware suspends them for up to 2 us at a time, and they
// take no issue slots meanwhile.
__device__ __forceinline__ bool pre_wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const unsigned long long t0 = global_timer_ns();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
        : "memory");
    if (done) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      return false;
    }
  }
}

struct PreBars {
  uint64_t q_full, k_full[kPreStages], k_empty[kPreStages], v_full[kPreStages], v_empty[kPreStages];
  uint64_t s_full[2], p_full[2], o_done[2], said;
};

template <typename T, int D, int G>
__global__ void __launch_bounds__(kPreThreads, 1) kv_prefill_int4_kernel(const __grid_constant__ AttnParams p) {
  using Smem = PreSmem<D>;
  constexpr int kGroups = D / G, kChunks = D / 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PreBars bars;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;
  // Values that are NaN: the groups that have some, by stage and unpacking warp, and their tokens.
  __shared__ uint32_t nan_any[kPreStages][4], nan_tokens[kPreStages][kGroups][4];
  __shared__ float row_mul[kPreRows];
  __shared__ uint32_t first_top[2][4];  // largest scale of the first tile, of each unpacking warp
  __shared__ float units[2];            // of keys and values
  __shared__ int handover;
  pdl_trigger();
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = smem_u32(smem);
  const KvView& v = p.view;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float kNegInf = __uint_as_float(0xff800000u);

  if (warp == kPreIssuer) {
    if (lane == 0) {
      abort_flag = 0;
      handover = 0;
      mbar_init(&bars.q_full, 8);
      for (int i = 0; i < kPreStages; ++i) {
        mbar_init(&bars.k_full[i], 4);
        mbar_init(&bars.v_full[i], 4);
        mbar_init(&bars.k_empty[i], 1);
        mbar_init(&bars.v_empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars.s_full[i], 1);
        mbar_init(&bars.p_full[i], 4);
        mbar_init(&bars.o_done[i], 1);
      }
      mbar_init(&bars.said, 2);
      fence_mbarrier_init();
    }
  }

  const BlockWork block = block_work(p, blockIdx.x);
  const int split = block.split, head = block.head, b = block.b;
  const int row_tile = p.row_tiles - 1 - block.row_tile;  // later rows see more tokens: they go first
  pdl_wait();
  if (v.cu_q && blockIdx.x < kClearBlocks)
    attn_clear_outside<T>(p, int(blockIdx.x), min(int(gridDim.x), kClearBlocks));
  const KvSeq seq = kv_seq(v, b);
  const int rows = seq.n * p.ratio, r0 = row_tile * kPreRows;
  bool work = r0 < rows;
  if (seq.n > p.max_q) {
    if (threadIdx.x == 0) kv_error(v);
    if (row_tile == 0 && split == 0) attn_clear_rows<T>(p, seq.row0, seq.row0 + seq.n, head * p.ratio, p.ratio);
    work = false;
  }
  const int r1 = min(rows, r0 + kPreRows);
  int begin = 0, end = 0;
  if (work) {
    attn_range(p, seq, r0, r1, kPreTile, &begin, &end);
    begin += split * p.chunk;
    if (begin >= end && split) work = false;
    if (split + 1 < p.splits) end = min(end, begin + p.chunk);
  }
  const int first_pos = seq.len - seq.n;
  // Tiles of 128 tokens of each query tile: the first one's rows may see fewer.
  int tiles[2] = {0, 0};
  if (work && end > begin) {
    tiles[1] = (end - begin + kPreTile - 1) / kPreTile;
    const int last0 = first_pos + query_row(p, min(r1, r0 + kPreTile) - 1).token;
    const int end0 = p.causal ? min(end, last0 + 1) : end;
    tiles[0] = end0 > begin ? (end0 - begin + kPreTile - 1) / kPreTile : 0;
    if (r0 + kPreTile >= r1) tiles[1] = 0;  // no rows there
  }
  const int all_tiles = max(tiles[0], tiles[1]);
  // After pdl_wait: a block that held TMEM while it waits could keep the kernel ahead from getting its own.
  if (warp == kPreIssuer) {
    __syncwarp();
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  // Of the 640 x 96 registers that the block was launched with, each role takes what it needs:
  // 256 x 128 + 256 x 80 + 128 x 64 = 61440.
  if (!work) {
  } else if (warp >= 8 && warp < kPreIssuer) {
    regs_less<80>();
    // ---- unpacking: a thread a token, four warps keys and four values ------------------------
    // A thread copies its own rows of codes ahead of itself (cp.async) and reads them back from shared memory.
    const int r = threadIdx.x & 127, which = (warp - 8) >> 2, slice = warp & 3;
    const uint8_t* codes = (which ? v.v_codes : v.k_codes) + head * v.c_head;
    const __nv_bfloat16* scales = v.scales + head * v.s_head + which * kGroups;
    uint64_t *full = which ? bars.v_full : bars.k_full, *empty = which ? bars.v_empty : bars.k_empty;
    uint8_t* buffers = smem + (which ? Smem::kV : Smem::kK);
    const uint32_t my_codes = sbase + Smem::kCodes + which * Smem::kCodeBytes;
    __nv_bfloat16 cur_s[kGroups], nxt_s[kGroups];
    auto page_of = [&](int j) {
      const int t = begin + j * kPreTile + r;
      return j < all_tiles && t < end ? kv_page_id(v, b, kv_page_of(v, t)) : -1;
    };
    auto fetch = [&](int j, int id) {
      const uint32_t dst = my_codes + (j % kPreStages) * 2 * Smem::kCodeBytes;
      const int t = begin + j * kPreTile + r, at = id < 0 ? 0 : t - kv_page_of(v, t) * v.page_size;
      const uint8_t* from = id < 0 ? codes : codes + id * v.c_page + at * v.c_tok;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) cp_async_16(dst + AttnTile<D, G>::place(r, k), from + k * 16, id >= 0);
      cp_async_commit();
      const __nv_bfloat16* s_from = scales + (id < 0 ? 0 : id * v.s_page + at * v.s_tok);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) nxt_s[k] = id < 0 ? __ushort_as_bfloat16(0) : s_from[k];
    };
    fetch(0, page_of(0));
    int id = page_of(1);
    float inv;  // of the unit
    {
      uint32_t top = 0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const float f = fabsf(__bfloat162float(nxt_s[g]));
        if (f <= 3.4e38f) top = max(top, __float_as_uint(f));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) first_top[which][slice] = top;
      pre_group_sync(which);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, first_top[which][i]);
      const float unit = pre_unit(top);
      inv = __frcp_rn(unit);
      if (r == 0) {
        units[which] = unit;
        mbar_arrive(&bars.said);
      }
    }
    for (int j = 0; j < all_tiles; ++j) {
#pragma unroll
      for (int k = 0; k < kGroups; ++k) cur_s[k] = nxt_s[k];
      fetch(j + 1, id);  // a tile ahead, and its page two
      id = page_of(j + 2);
      const int st = j % kPreStages;
      uint32_t any = 0;
      bool unfit = false;
      cp_async_wait<1>();
      if (!__all_sync(0xffffffffu, pre_wait_idle(&empty[st], ((j / kPreStages) & 1) ^ 1, &abort_flag))) break;
      uint8_t* dst = buffers + st * Smem::kTileBytes;
      const uint32_t src = my_codes + st * 2 * Smem::kCodeBytes;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const float scale = __bfloat162float(cur_s[g]);
        float f = scale * inv;
        unfit |= scale != 0.0f && fabsf(scale) <= 3.4e38f && !(fabsf(f) >= 0x1p-17f && fabsf(f) <= 0x1p12f);
        if (which) {
          // NaN values (and infinite ones) become zeros here; the rows that see them get NaN at the end.
          const bool bad = !(fabsf(f) <= 3.4e38f);
          const unsigned nan = __ballot_sync(0xffffffffu, bad);
          any |= uint32_t(nan != 0) << g;
          if (lane == 0) nan_tokens[st][g][slice] = nan;
          if (bad) f = 0.0f;
        }
        const __half2 s = __float2half2_rn(f);
#pragma unroll 1
        for (int k = g * (G / 32); k < (g + 1) * (G / 32); ++k) {
          uint32_t w[4];
          lds_words<4, 16>(src + AttnTile<D, G>::place(r, k), w);
#pragma unroll
          for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(dst + pre_place(r, k * 4 + q)) = unpack8(w[q], s);
        }
      }
      if (which && lane == 0) nan_any[st][slice] = any;
      if (unfit) handover = 1;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[st]);
    }
    cp_async_wait<0>();
  } else if (warp >= kPreIssuer) {
    regs_less<64>();
    if (warp == kPreIssuer) {
      // ---- issuing the products: waits by the whole warp, products by its elected lane. It takes the query
      // tiles in turn, which keeps them apart: one's products run while the other's weights are made ------
      constexpr uint32_t kIdescQk = make_idesc_f16(false, kPreTile, kPreTile);
      constexpr uint32_t kIdescPv = make_idesc_f16(true, kPreTile, D);
      const uint64_t rows_desc = make_smem_desc(0, 16, 1024, kLayoutSw128);
      const uint64_t value_desc = make_smem_desc(0, kPrePanel, 1024, kLayoutSw128);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, pre_wait(bar, parity, &abort_flag));
      };
      const bool leader = elect_one();
      auto scores = [&](int s, int j) {
        if (!leader) return;
        const uint64_t q = rows_desc + ((sbase + Smem::kQ + s * Smem::kTileBytes) >> 4);
        const uint64_t k = rows_desc + ((sbase + Smem::kK + (j % kPreStages) * Smem::kTileBytes) >> 4);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint32_t off = ((c >> 2) * kPrePanel + (c & 3) * 32) >> 4;
          mma_f16_ss(tmem + s * 128, q + off, k + off, kIdescQk, c != 0);
        }
        mma_commit(&bars.s_full[s]);
      };
      bool ok = all_tiles == 0 || (wait(&bars.q_full, 0) && wait(&bars.k_full[0], 0));
      if (ok && all_tiles) {
        tc_fence_after();
        for (int s = 0; s < 2; ++s)
          if (tiles[s]) scores(s, 0);
        if (leader) mma_commit(&bars.k_empty[0]);
      }
#pragma unroll 1
      for (int j = 0; ok && j < all_tiles; ++j) {
        const int st = j % kPreStages, next = (j + 1) % kPreStages;
        const uint64_t val = value_desc + ((sbase + Smem::kV + st * Smem::kTileBytes) >> 4);
        ok = wait(&bars.v_full[st], (j / kPreStages) & 1) &&
             (j + 1 == all_tiles || wait(&bars.k_full[next], ((j + 1) / kPreStages) & 1));
#pragma unroll 1
        for (int s = 0; ok && s < 2; ++s) {
          if (j >= tiles[s]) continue;
          ok = wait(&bars.p_full[s], j & 1);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int c = 0; c < kPreTile / 16; ++c)
              mma_f16_ts(tmem + 256 + s * 128, tmem + s * 128 + c * 8, val + c * (2048 >> 4), kIdescPv,
                         j != 0 || c != 0);
            // The next scores overwrite the weights that these products read: products run in the order of issue.
            if (j + 1 < tiles[s]) scores(s, j + 1);
            mma_commit(&bars.o_done[s]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) {
          mma_commit(&bars.v_empty[st]);
          if (j + 1 < all_tiles) mma_commit(&bars.k_empty[next]);
        }
        __syncwarp();
      }
      if (!ok) {  // let what was issued end before TMEM is given back
        if (lane == 0) atomicOr(v.err, kErrTimeoutMma);
        for (const unsigned long long t = global_timer_ns(); global_timer_ns() - t < 100000;) {
        }
      }
    }
  } else {
    regs_more<128>();
    // ---- a thread a query row: the query's tile, weights, the output ----------------------
    const int s = warp >> 2, rl = threadIdx.x & 127, r = r0 + s * kPreTile + rl;
    const bool mine = r < r1;
    const QueryRow qr = query_row(p, mine ? r : 0);
    const int token = qr.token, qh = head * p.ratio + qr.head;
    float mul;  // what a score is multiplied by, without its keys' unit
    {
      // A warp brings its 32 rows, kLanes lanes a row and eight channels a lane; the next four loads are in
      // flight while four are converted. (A loop: straight-line code runs once here, at the instruction cache's pace.)
      constexpr int kLanes = D == 64 ? 8 : 16, kStep = 32 / kLanes, kBatch = 4;
      const int c = lane % kLanes, rw = (warp & 3) * 32 + lane / kLanes;
      uint8_t* dst = smem + Smem::kQ + s * Smem::kTileBytes;
      uint4 w[kBatch], nxt[kBatch];
      auto load = [&](int k0, uint4(&to)[kBatch]) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int rt = rw + (k0 + k) * kStep, rr = r0 + s * kPreTile + rt;
          to[k] = make_uint4(0, 0, 0, 0);
          if (rr >= r1 || c >= kChunks || k0 >= kLanes) continue;
          const QueryRow at = query_row(p, rr);
          const T* src = static_cast<const T*>(p.q) + (seq.row0 + at.token) * p.q_row +
                         (head * p.ratio + at.head) * p.q_head + c * 8;
          if (p.q_vec) {
            to[k] = *reinterpret_cast<const uint4*>(src);
          } else {
            T* e = reinterpret_cast<T*>(&to[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = src[i];
          }
        }
      };
      load(0, nxt);
#pragma unroll 1
      for (int k0 = 0; k0 < kLanes; k0 += kBatch) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) w[k] = nxt[k];
        load(k0 + kBatch, nxt);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const T* e = reinterpret_cast<const T*>(&w[k]);
          // The query's factor is the scale's sign, for bfloat16 times the power of two that brings the row's
          // largest magnitude near 2^14; the scores' factor takes it back.
          float up = p.sign, back = p.scale_log2;
          if constexpr (!std::is_same<T, __half>::value) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_f32<T>(e[i])));
#pragma unroll
            for (int i = kLanes / 2; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
            if (top > 0.0f && top < __uint_as_float(0x7f800000u)) {
              // frexp's exponent for normal numbers; smaller ones are taken up by 2^126.
              const int x = max(-126, min(126, 140 - int(__float_as_uint(top) >> 23)));
              up *= __int_as_float((127 + x) << 23);
              back = fmaxf(back * __int_as_float((127 - x) << 23), 1.2e-38f);
            }
          }
          const int rt = rw + (k0 + k) * kStep;
          if (c == 0) row_mul[s * kPreTile + rt] = back;
          uint4 o;  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
          o.x = pack_f16(to_f32<T>(e[0]) * up, to_f32<T>(e[4]) * up);
          o.y = pack_f16(to_f32<T>(e[1]) * up, to_f32<T>(e[5]) * up);
          o.z = pack_f16(to_f32<T>(e[2]) * up, to_f32<T>(e[6]) * up);
          o.w = pack_f16(to_f32<T>(e[3]) * up, to_f32<T>(e[7]) * up);
          if (c < kChunks) *reinterpret_cast<uint4*>(dst + pre_place(rt, c)) = o;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.q_full);
      mul = row_mul[s * kPreTile + rl];  // written by this warp
    }
    const int pos = first_pos + token;
    const int lo = p.window > 0 ? max(0, max(0, pos) - p.window + 1) : 0;
    const int hi = pos < 0 || !mine ? 0 : p.causal ? min(end, pos + 1) : end;
    const uint32_t quad = uint32_t(warp & 3) << 21, s_addr = tmem + s * 128 + quad, o_addr = tmem + 256 + s * 128 + quad;
    float m = kNegInf, l = 0.0f;
    uint32_t nan_groups = 0;
    bool ok = __all_sync(0xffffffffu, pre_wait(&bars.said, 0, &abort_flag));
    const float m32 = fmaxf(mul * units[0], 1.2e-38f);  // a score's factor; positive, for the hidden scores' -inf
    const uint64_t mul2 = pair2(m32, m32);
    for (int j = 0; ok && j < tiles[s]; ++j) {
      // What the unpacking warps say about the tile (NaN values) is read before the weights are
      // handed over: until the products with them are done it is not written over.
      const int st = j % kPreStages;
      if (!__all_sync(0xffffffffu, pre_wait(&bars.s_full[s], j & 1, &abort_flag) &&
                                       pre_wait(&bars.v_full[st], (j / kPreStages) & 1, &abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int t0 = begin + j * kPreTile;
      const int from = max(lo - t0, 0), to = min(hi - t0, kPreTile);  // columns that this row sees
      const bool partial = __any_sync(0xffffffffu, from > 0 || to < kPreTile);
      if (nan_any[st][0] | nan_any[st][1] | nan_any[st][2] | nan_any[st][3]) {
        for (int g = 0; g < kGroups; ++g)
          for (int k = from; k < to; ++k)
            if (nan_tokens[st][g][k >> 5] >> (k & 31) & 1) nan_groups |= 1u << g;
      }
      // Weights for the reference m of the tiles before, and the largest score on the way. Only when that
      // passes m by more than kPreRaise (or at the first tile) m is raised, the output rescaled and the row done again, so
      // most tiles take one pass. They are held in registers until then, since
      // they go where the scores are. The next 32 columns are loaded while these are worked on.
      // Nothing to go by at the first tile: the largest of 32 columns that the rows of the warp see. This and the masks
      // as bits make the first and last tiles of a row cheaper: 6 chunks of 700 tokens in a window of 1024, 16 heads on 4
      // of 64, 96 and 128 channels 77, 86 and 92 us without, 67, 74 and 81 with; 8192 tokens 591, 649 and 653 without, 592,
      // 628 and 644 with.
      if (j == 0) {
        const int c = min(max(__shfl_sync(0xffffffffu, from, 31), 0), kPreTile - 1) / 32;
        float y[32];
        tmem_ld32(s_addr + c * 32, y);
        tmem_ld_wait32(y);
        const uint32_t seen = bits_between(from - c * 32, to - c * 32);
#pragma unroll
        for (int k = 0; k < 32; ++k) m = fmaxf(m, seen >> k & 1 ? y[k] : kNegInf);
        m = m * m32 - kPreHigh;
        if (m != kNegInf && fabsf(m) > kPreMost) handover = 1;
      }
      uint32_t w[kPreTile / 2];
      float sum;
      bool again = false;
      do {
        const float ref = m == kNegInf ? 0.0f : m;
        const uint64_t sub = pair2(-ref, -ref);
        uint64_t acc0 = 0, acc1 = 0;
        float top = kNegInf, x[2][32];
        tmem_ld32(s_addr, x[0]);
#pragma unroll
        for (int c = 0; c < kPreTile / 32; ++c) {
          float(&y)[32] = x[c & 1];
          tmem_ld_wait32(y);
          if (c + 1 < kPreTile / 32) tmem_ld32(s_addr + (c + 1) * 32, x[(c + 1) & 1]);
          if (partial) {
            const uint32_t seen = bits_between(from - c * 32, to - c * 32);
#pragma unroll
            for (int k = 0; k < 32; ++k) y[k] = seen >> k & 1 ? y[k] : kNegInf;
          }
          float t[2] = {kNegInf, kNegInf};
#pragma unroll
          for (int k = 0; k < 32; k += 2) t[k / 2 & 1] = fmaxf(t[k / 2 & 1], fmaxf(y[k], y[k + 1]));
          top = fmaxf(top, fmaxf(t[0], t[1]) * m32);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float a, d;
            unpair2(fma2(pair2(y[k], y[k + 1]), mul2, sub), a, d);
            a = exp2_approx(a), d = exp2_approx(d);
            if (k & 2) acc1 = add2(acc1, pair2(a, d));
            else acc0 = add2(acc0, pair2(a, d));
            w[c * 16 + k / 2] = pack_f16(a, d);
          }
        }
        float a, d;
        unpair2(add2(acc0, acc1), a, d);
        sum = a + d;
        again = !again && __any_sync(0xffffffffu, top > m + kPreRaise);
        if (again) {
          const float next = fmaxf(m, top - kPreHigh);
          if (next != kNegInf && fabsf(next) > kPreMost) handover = 1;
          const float c = next == kNegInf ? 1.0f : exp2_approx(m - next);
          m = next;
          l *= c;
          if (j) {
            ok = __all_sync(0xffffffffu, pre_wait(&bars.o_done[s], (j - 1) & 1, &abort_flag));
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; ok && k < D / 16; ++k) {
              float y[16];
              tmem_ld16f(o_addr + k * 16, y);
              tmem_ld_wait16(y);
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] *= c;
              tmem_st16(o_addr + k * 16, reinterpret_cast<const uint32_t(&)[16]>(y));
            }
          }
        }
      } while (again);
      if (!ok) break;
#pragma unroll
      for (int k = 0; k < kPreTile / 2; k += 16)
        tmem_st16(s_addr + k, *reinterpret_cast<const uint32_t(*)[16]>(w + k));
      l += sum;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[s]);
    }
    if (ok && tiles[s])
      ok = __all_sync(0xffffffffu, pre_wait(&bars.o_done[s], (tiles[s] - 1) & 1, &abort_flag));
    if (!ok && lane == 0) atomicOr(v.err, kErrTimeoutEpilogue);
    tc_fence_after();
    const long long at = (long long)(seq.row0 + token) * p.q_heads + qh;
    // Partial results are for weights of at most 1: with larger ones the sums of values near the largest number overflow.
    const float inv = units[1] * (p.splits > 1 ? kPreLow : l == 0.0f ? 0.0f : __frcp_rn(l));
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      float x[32];
      if (tiles[s]) {
        tmem_ld32(o_addr + k * 32, x);
        tmem_ld_wait32(x);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0.0f;
      }
      const bool nan = nan_groups >> (k * 32 / G) & 1;
      if (!mine) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float y[8];  // columns 2 e, 2 e + 1 hold channels e, e + 4
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[c * 8 + 2 * e], y[e + 4] = x[c * 8 + 2 * e + 1];
        if (nan) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(0x7fc00000u);
        }
        if (p.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(p.part_o + (at * p.splits + split) * D + k * 32 + c * 8);
          dst[0] = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
          dst[1] = make_float4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
        } else {
          uint4 o;
          o.x = pack_pair<T>(y[0] * inv, y[1] * inv), o.y = pack_pair<T>(y[2] * inv, y[3] * inv);
          o.z = pack_pair<T>(y[4] * inv, y[5] * inv), o.w = pack_pair<T>(y[6] * inv, y[7] * inv);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * D + k * 32 + c * 8) = o;
        }
      }
    }
    if (mine) {
      if (p.splits > 1) p.part_ml[at * p.splits + split] = make_float2(m + kPreRaise, l * kPreLow);
      else if (p.lse) p.lse[at] = l == 0.0f ? kNegInf : (m + log2f(l)) * 0.69314718055994531f;
    }
    tc_fence_before();
  }
  __syncthreads();
  if (threadIdx.x == 0) p.handover[blockIdx.x] = handover;
  if (warp == kPreIssuer) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

// The rows of blocks whose scales are too far apart for float16, by the arithmetic of few rows: kRedoParts blocks for each of the
// prompt kernel's tiles of rows, which all leave at once where no piece of the tile was handed over.
constexpr int kRedoParts = 4;

template <typename T, int D, int G>
__global__ void __launch_bounds__(kAttnWarps * 32, attn_blocks_sm(D, 2, false))
    kv_attn_redo_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kRows = 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_trigger();
  const unsigned tile = blockIdx.x / kRedoParts, part = blockIdx.x % kRedoParts;
  pdl_wait();
  int redo = 0;
  for (int s = 0; s < p.splits; ++s) redo |= p.handover[(long long)tile * p.splits + s];
  if (!redo) return;
  const BlockWork work = block_work(p, tile * unsigned(p.splits));
  const int row_tile = p.row_tiles - 1 - work.row_tile;  // as the prompt kernel counts them
  const KvSeq seq = kv_seq(p.view, work.b);
  const int rows = min(seq.n * p.ratio, (row_tile + 1) * kPreRows);
  for (int r0 = row_tile * kPreRows + int(part) * kRows; r0 < rows; r0 += kRedoParts * kRows) {
    const int r1 = min(rows, r0 + kRows);
    int begin, end;
    attn_range(p, seq, r0, r1, kTile, &begin, &end);
    attn_rows<T, D, G, kRows / 8>(p, seq, work.b, work.head, r0, r1, begin, end, 0, 1, 0, smem, nullptr, nullptr);
    __syncthreads();  // the results have left the shared memory that the next rows' stages take
  }
}

}  // namespace w4a8
