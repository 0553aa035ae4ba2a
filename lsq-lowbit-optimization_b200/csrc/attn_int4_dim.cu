// The attention kernels of one head size (W4A8_HEAD_DIM); one object file each.
#include "attn_int4.cuh"
#include "attn_int4_host.cuh"
#include "prefill_int4.cuh"

namespace w4a8 {
namespace {

constexpr int D = W4A8_HEAD_DIM;

template <typename T>
int join(const AttnParams& p, int tile_rows, int tile_tokens, cudaStream_t st) {
  const unsigned tiles = unsigned(p.view.batch) * p.view.heads * p.row_tiles;
  const dim3 block(kJoinLanes * D / 4);
  const cudaError_t e =
      (long long)tiles * tile_rows >= 1024
          ? launch_kernel(kv_attn_join_kernel<T, D, 1>, dim3(tiles, (tile_rows + kJoinLanes - 1) / kJoinLanes), block, 0,
                          st, p, tile_rows, tile_tokens)
          : launch_kernel(kv_attn_join_kernel<T, D, kJoinLanes>, dim3(tiles, tile_rows), block, 0, st, p, tile_rows,
                          tile_tokens);
  return e == cudaSuccess ? W4A8_OK : W4A8_ERR_LAUNCH;
}

template <typename Kernel>
int allow_smem(Kernel kern, int bytes, PerDevice<int>& ready) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return W4A8_ERR_LAUNCH;
  if (ready.get(dev)) return W4A8_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return W4A8_ERR_LAUNCH;
  ready.set(dev, 1);
  return W4A8_OK;
}

template <typename T, int G>
int run_prefill(const AttnParams& p, unsigned grid, cudaStream_t st) {
  constexpr int smem = prefill_smem_bytes<D>();
  static PerDevice<int> ready;
  if (allow_smem(kv_prefill_int4_kernel<T, D, G>, smem, ready) != W4A8_OK) return W4A8_ERR_LAUNCH;
  return launch_kernel(kv_prefill_int4_kernel<T, D, G>, dim3(grid), dim3(kPreThreads), smem, st, p) == cudaSuccess
             ? W4A8_OK
             : W4A8_ERR_LAUNCH;
}

// The rows that the blocks of run_prefill handed over; behind the join.
template <typename T, int G>
int run_redo(const AttnParams& p, cudaStream_t st) {
  constexpr int smem = attn_smem_bytes<D, G, 2>();
  static PerDevice<int> ready;
  if (allow_smem(kv_attn_redo_kernel<T, D, G>, smem, ready) != W4A8_OK) return W4A8_ERR_LAUNCH;
  const unsigned grid = unsigned(p.view.batch) * p.view.heads * p.row_tiles * kRedoParts;
  return launch_kernel(kv_attn_redo_kernel<T, D, G>, dim3(grid), dim3(kAttnWarps * 32), smem, st, p) == cudaSuccess
             ? W4A8_OK
             : W4A8_ERR_LAUNCH;
}

constexpr int kRedo = -1;  // in place of NT

template <typename T, int G, int NT>
int run(const AttnParams& p, unsigned grid, cudaStream_t st) {
  if constexpr (NT == 0) {
    return run_prefill<T, G>(p, grid, st);
  } else if constexpr (NT == kRedo) {
    return run_redo<T, G>(p, st);
  } else {
    constexpr int smem = attn_smem_bytes<D, G, NT>();
    static PerDevice<int> ready;
    if (allow_smem(kv_attn_int4_kernel<T, D, G, NT>, smem, ready) != W4A8_OK) return W4A8_ERR_LAUNCH;
    return launch_kernel(kv_attn_int4_kernel<T, D, G, NT>, dim3(grid), dim3(kAttnWarps * 32), smem, st, p) ==
                   cudaSuccess
               ? W4A8_OK
               : W4A8_ERR_LAUNCH;
  }
}

// NT: tiles of eight query rows of a warp, 0 for the kernel of many rows, or kRedo.
template <typename T, int NT>
int by_group(const AttnParams& p, unsigned grid, cudaStream_t st) {
  switch (p.view.group) {
    case 32: return run<T, 32, NT>(p, grid, st);
    case 64:
      if constexpr (D % 64 == 0) return run<T, 64, NT>(p, grid, st);
      break;
    case 128:
      if constexpr (D % 128 == 0) return run<T, 128, NT>(p, grid, st);
      break;
  }
  return W4A8_ERR_UNSUPPORTED;
}

template <typename T>
int by_tiles(const AttnParams& p, int n_tiles, unsigned grid, cudaStream_t st) {
  if constexpr (prefill_ok(D, sizeof(T) == 4)) {
    if (n_tiles == 0) return by_group<T, 0>(p, grid, st);
    if (n_tiles == kRedo) return by_group<T, kRedo>(p, grid, st);
  }
  if constexpr (attn_wide_ok(D, sizeof(T) == 4)) {
    if (n_tiles == 2) return by_group<T, 2>(p, grid, st);
  }
  return by_group<T, 1>(p, grid, st);
}

}  // namespace

#define W4A8_CAT2(a, b) a##b
#define W4A8_CAT(a, b) W4A8_CAT2(a, b)
int W4A8_CAT(launch_attn_int4_d, W4A8_HEAD_DIM)(const AttnParams& p, int dtype, int n_tiles, unsigned grid,
                                                cudaStream_t st) {
  auto rows = [&](int tiles) {
    return dtype == W4A8_F32   ? by_tiles<float>(p, tiles, grid, st)
           : dtype == W4A8_F16 ? by_tiles<__half>(p, tiles, grid, st)
                               : by_tiles<__nv_bfloat16>(p, tiles, grid, st);
  };
  const int rc = rows(n_tiles);
  if (rc != W4A8_OK) return rc;
  if (p.splits > 1) {
    const int tile_rows = n_tiles ? 8 * n_tiles : kPreRows, tile_tokens = n_tiles ? kTile : kPreTile;
    const int joined = dtype == W4A8_F32   ? join<float>(p, tile_rows, tile_tokens, st)
                       : dtype == W4A8_F16 ? join<__half>(p, tile_rows, tile_tokens, st)
                                           : join<__nv_bfloat16>(p, tile_rows, tile_tokens, st);
    if (joined != W4A8_OK) return joined;
  }
  if (n_tiles == 0) {
    const int redone = rows(kRedo);
    if (redone != W4A8_OK) return redone;
  }
  return cudaGetLastError() == cudaSuccess ? W4A8_OK : W4A8_ERR_LAUNCH;
}

}  // namespace w4a8
