// Products of every expert's rows with its weight matrix (expert_matmul) and of the rows with the results' gradient
// (expert_matmul_gradient).  The rows lie sorted by expert; how many an expert has is known on the device only, so the
// grid is sized for the most tiles that any split of the rows into experts has, and a workgroup finds its tile's expert in
// indptr.
#include "expert.h"

namespace {

using namespace bpl;

constexpr uint32_t kThreads = 256;

// The rows of expert e, whatever indptr says within the array; e == experts: the rows behind the last.
__device__ __forceinline__ uint2 rows_of(const uint32_t *__restrict__ indptr, uint32_t e, uint32_t experts, uint32_t rows) {
  uint32_t from = e == 0 ? 0u : indptr[e], to = e < experts ? indptr[e + 1] : rows;
  from = from < rows ? from : rows;
  to = to < rows ? to : rows;
  return make_uint2(from, to > from ? to : from);
}

struct Tile {
  uint32_t expert, first, end;  // the rows of the tile: [first, end); expert kNoTile: there is none
};
constexpr uint32_t kNoTile = 0xffffffffu;

// Tile `index` of `height` rows, counted over the experts in their order and the rows behind the last: all threads of
// the workgroup scan the experts' numbers of tiles.
__device__ __forceinline__ Tile find_tile(const uint32_t *__restrict__ indptr, uint32_t experts, uint32_t rows,
                                          uint32_t height, uint32_t index) {
  constexpr uint32_t kPer = (kMostExperts + 1 + kThreads - 1) / kThreads, kWaves = kThreads / kWave;
  __shared__ uint32_t wave_total[kWaves];
  __shared__ Tile found;
  const uint32_t per = (experts + 1 + kThreads - 1) / kThreads;
  if (threadIdx.x == 0) found.expert = kNoTile;
  uint2 range[kPer];
  uint32_t tiles = 0;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    const uint32_t e = threadIdx.x * per + j;
    range[j] = j < per && e <= experts ? rows_of(indptr, e, experts, rows) : make_uint2(0, 0);
    tiles += (range[j].y - range[j].x + height - 1) / height;
  }
  const uint32_t upto = wave_inclusive_scan_u32(tiles);
  if (threadIdx.x % kWave == kWave - 1) wave_total[threadIdx.x / kWave] = upto;
  __syncthreads();
  uint32_t before = upto - tiles;
  for (uint32_t w = 0; w < threadIdx.x / kWave; ++w) before += wave_total[w];
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    const uint32_t n = (range[j].y - range[j].x + height - 1) / height;
    if (index >= before && index - before < n) {
      const uint32_t first = range[j].x + (index - before) * height;
      found.expert = threadIdx.x * per + j;
      found.first = first;
      found.end = range[j].y - first < height ? range[j].y : first + height;
    }
    before += n;
  }
  __syncthreads();
  return found;
}

uint64_t most_tiles(uint32_t rows, uint32_t experts, uint32_t height) {
  // every expert (and the rows behind the last) has at most one tile that is not full
  const uint64_t partly = static_cast<uint64_t>(experts) + 1;
  return static_cast<uint64_t>(rows) / height + (partly < rows ? partly : rows);
}

// out = rows @ weight[expert], tiles of 64 x 64, 16 of the inner dimension at a time in LDS, 4 x 4 results to a thread.
constexpr uint32_t kTile = 64, kStep = 16;

template <typename T, bool OUT_MAJOR>
__global__ __launch_bounds__(kThreads) void product_kernel(const T *__restrict__ rows, const T *__restrict__ weight,
                                                           const uint32_t *__restrict__ indptr, T *__restrict__ out,
                                                           uint32_t n_rows, uint32_t experts, uint32_t inner, uint32_t cols) {
  __shared__ float a[kStep][kTile + 1], b[kStep][kTile + 1];
  const Tile tile = find_tile(indptr, experts, n_rows, kTile, blockIdx.y);
  if (tile.expert == kNoTile) return;
  const uint32_t col0 = blockIdx.x * kTile, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float sum[4][4] = {};
  if (tile.expert < experts) {
    const T *const w = weight + static_cast<size_t>(tile.expert) * inner * cols;
    for (uint32_t k0 = 0; k0 < inner; k0 += kStep) {
      for (uint32_t i = threadIdx.x; i < kTile * kStep; i += kThreads) {
        const uint32_t r = i / kStep, kk = i % kStep;
        a[kk][r] = tile.first + r < tile.end && k0 + kk < inner
                       ? static_cast<float>(rows[static_cast<size_t>(tile.first + r) * inner + k0 + kk]) : 0.f;
        const uint32_t c = OUT_MAJOR ? i / kStep : i % kTile, kb = OUT_MAJOR ? i % kStep : i / kTile;
        b[kb][c] = col0 + c < cols && k0 + kb < inner
                       ? static_cast<float>(w[OUT_MAJOR ? static_cast<size_t>(col0 + c) * inner + k0 + kb
                                                        : static_cast<size_t>(k0 + kb) * cols + col0 + c]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (uint32_t kk = 0; kk < kStep; ++kk)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) sum[i][j] = fmaf(a[kk][ty * 4 + i], b[kk][tx + 16 * j], sum[i][j]);
      __syncthreads();
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t r = tile.first + ty * 4 + i, c = col0 + tx + 16 * j;
      if (r < tile.end && c < cols) out[static_cast<size_t>(r) * cols + c] = static_cast<T>(sum[i][j]);
    }
}

// d_weight[expert] = left_e^T @ right_e over the expert's rows; (left, right) = (rows, ct), or (ct, rows) where the weight is
// stored out-major.
template <typename T>
__global__ __launch_bounds__(kThreads) void gradient_kernel(const T *__restrict__ left, const T *__restrict__ right,
                                                            const uint32_t *__restrict__ indptr, T *__restrict__ d_weight,
                                                            uint32_t n_rows, uint32_t experts, uint32_t n_left, uint32_t n_right) {
  __shared__ float a[kStep][kTile + 1], b[kStep][kTile + 1];
  const uint32_t expert = blockIdx.z, p0 = blockIdx.y * kTile, q0 = blockIdx.x * kTile;
  const uint2 range = rows_of(indptr, expert, experts, n_rows);
  const uint32_t ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float sum[4][4] = {};
  for (uint32_t r0 = range.x; r0 < range.y; r0 += kStep) {
    for (uint32_t i = threadIdx.x; i < kTile * kStep; i += kThreads) {
      const uint32_t r = i / kTile, c = i % kTile;
      const bool inside = r0 + r < range.y;
      a[r][c] = inside && p0 + c < n_left ? static_cast<float>(left[static_cast<size_t>(r0 + r) * n_left + p0 + c]) : 0.f;
      b[r][c] = inside && q0 + c < n_right ? static_cast<float>(right[static_cast<size_t>(r0 + r) * n_right + q0 + c]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t kk = 0; kk < kStep; ++kk)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) sum[i][j] = fmaf(a[kk][ty * 4 + i], b[kk][tx + 16 * j], sum[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t p = p0 + ty * 4 + i, q = q0 + tx + 16 * j;
      if (p < n_left && q < n_right)
        d_weight[(static_cast<size_t>(expert) * n_left + p) * n_right + q] = static_cast<T>(sum[i][j]);
    }
}

template <typename T>
void matmul(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.rows == 0 || d.out == 0) return;
  const uint64_t tiles = most_tiles(d.rows, d.experts, kTile);
  const auto launch = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, dim3(div_up(d.out, kTile), static_cast<unsigned>(tiles)), dim3(kThreads), 0, stream,
                       static_cast<const T *>(buffers[0]), static_cast<const T *>(buffers[1]),
                       static_cast<const uint32_t *>(buffers[2]), static_cast<T *>(buffers[3]), d.rows, d.experts, d.width,
                       d.out);
  };
  if (d.flags & BPL_EXPERT_OUT_MAJOR)
    launch(product_kernel<T, true>);
  else
    launch(product_kernel<T, false>);
  check_launch(target);
}

template <typename T>
void matmul_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.width == 0 || d.out == 0) return;
  const bool out_major = (d.flags & BPL_EXPERT_OUT_MAJOR) != 0;
  const uint32_t n_left = out_major ? d.out : d.width, n_right = out_major ? d.width : d.out;
  hipLaunchKernelGGL(gradient_kernel<T>, dim3(div_up(n_right, kTile), div_up(n_left, kTile), d.experts), dim3(kThreads), 0,
                     stream, static_cast<const T *>(buffers[out_major ? 1 : 0]),
                     static_cast<const T *>(buffers[out_major ? 0 : 1]), static_cast<const uint32_t *>(buffers[2]),
                     static_cast<T *>(buffers[3]), d.rows, d.experts, n_left, n_right);
  check_launch(target);
}

}  // namespace

extern "C" {

BPL_EXPERT_DEFINE(expert_matmul, matmul)
BPL_EXPERT_DEFINE(expert_matmul_gradient, matmul_gradient)

}  // extern "C"
