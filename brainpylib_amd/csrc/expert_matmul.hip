// Products of every expert's rows with its weight matrix (expert_matmul) and of the rows with the results' gradient
// (expert_matmul_gradient).  The rows lie sorted by expert; how many an expert has is known on the device only, so the
// grid is sized for the most tiles that any split of the rows into experts has, and a workgroup finds its tile's expert in
// indptr.
#include <type_traits>

#include "expert.h"

namespace {

using namespace bpl;

// A value that all lanes of a wave have, as the scalar that it is.
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
}

template <typename T>
__device__ __forceinline__ const T *uniform(const T *p) {
  const auto v = reinterpret_cast<uintptr_t>(p);
  const uint32_t low = uniform(static_cast<uint32_t>(v)), high = uniform(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const T *>(static_cast<uintptr_t>(high) << 32 | low);
}

// The rows of expert e, whatever indptr says within the array; e == experts: the rows behind the last.
__device__ __forceinline__ uint2 rows_of(const uint32_t *__restrict__ indptr, uint32_t e, uint32_t experts, uint32_t rows) {
  uint32_t from = e == 0 ? 0u : indptr[e], to = e < experts ? indptr[e + 1] : rows;
  from = from < rows ? from : rows;
  to = to < rows ? to : rows;
  return make_uint2(from, to > from ? to : from);
}

// The experts' rows and where their tiles of `height` rows begin, counted over the experts in their order: in LDS, built
// by all threads of the workgroup (one barrier, and one for the caller to see it).
struct Tile {
  uint32_t expert, first, end;  // the rows of the tile: [first, end)
};
struct TileTable {
  uint32_t start[kMostExperts];
  uint32_t wave_total[16];

  // the number of tiles
  template <uint32_t THREADS>
  __device__ __forceinline__ uint32_t build(const uint32_t *__restrict__ indptr, uint32_t experts, uint32_t rows, uint32_t height) {
    constexpr uint32_t kPer = (kMostExperts + THREADS - 1) / THREADS, kWaves = THREADS / kWave;
    const uint32_t per = (experts + THREADS - 1) / THREADS;
    uint32_t own[kPer], tiles = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) {
      const uint32_t e = threadIdx.x * per + j;
      own[j] = 0;
      if (j < per && e < experts) {
        const uint2 r = rows_of(indptr, e, experts, rows);
        own[j] = (r.y - r.x + height - 1) / height;
      }
      tiles += own[j];
    }
    const uint32_t upto = wave_inclusive_scan_u32(tiles);
    if (threadIdx.x % kWave == kWave - 1) wave_total[threadIdx.x / kWave] = upto;
    __syncthreads();
    uint32_t at = upto - tiles, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      at += w < threadIdx.x / kWave ? wave_total[w] : 0u;
      total += wave_total[w];
    }
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) {
      const uint32_t e = threadIdx.x * per + j;
      if (j < per && e < experts) start[e] = at;
      at += own[j];
    }
    __syncthreads();
    return uniform(total);
  }

  // index < the number of tiles; every wave by itself: the last expert that begins at or before it (those without tiles begin
  // where the next one does), 64 places and then 16 at a time
  __device__ __forceinline__ Tile find(const uint32_t *__restrict__ indptr, uint32_t index, uint32_t experts, uint32_t rows,
                                       uint32_t height) const {
    static_assert(kMostExperts <= 64 * 16, "two looks are enough");
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t coarse = __popcll(__ballot(lane * 16 < experts && start[lane * 16 < experts ? lane * 16 : 0] <= index));
    const uint32_t e = (coarse - 1) * 16 + lane;
    const uint32_t fine = __popcll(__ballot(lane < 16 && e < experts && start[e < experts ? e : 0] <= index));
    const uint32_t expert = uniform((coarse - 1) * 16 + fine - 1);
    const uint2 r = rows_of(indptr, expert, experts, rows);
    const uint32_t first = uniform(r.x) + (index - uniform(start[expert])) * height, end = uniform(r.y);
    return Tile{expert, first, end - first < height ? end : first + height};
  }
};

uint64_t most_tiles(uint32_t rows, uint32_t experts, uint32_t height) {
  // every expert has at most one tile that is not full
  return static_cast<uint64_t>(rows) / height + (experts < rows ? experts : rows);
}

// ---- tiles --------------------------------------------------------------------------------------------------------
// One product kernel body for the three products.  C[m][n] = sum over k of A[m][k] B[n][k], tiles of BM x BN, kDepth (128 bytes
// of a row) of k at a time through two buffers in LDS.  An operand lies in memory with its k side by side ("along": rows of
// tokens, out-major weights) or with its m or n side by side ("across": the others).
//   along:  LDS holds [m][k], 128 bytes a row; a lane reads the 16 bytes of k that its matrix instruction takes.
//   across: LDS holds [k][m]; 16-bit types are transposed by the LDS's transposing read (16 lanes read 4 rows of 16
//           elements and get a column of 4 each), 32-bit ones are read one by one.
// 16-byte pieces are placed so that the lanes of a read meet different banks (place()).
template <typename T>
struct Unit;  // the matrix instructions of a type: one piece of k (kPieceK elements) of 32 x 32 results
template <>
struct Unit<half_t> {
  typedef half_t frag __attribute__((ext_vector_type(8)));
  typedef float acc __attribute__((ext_vector_type(16)));
  static __device__ __forceinline__ acc mul(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Unit<bfloat_t> {
  typedef bfloat_t frag __attribute__((ext_vector_type(8)));
  typedef float acc __attribute__((ext_vector_type(16)));
  static __device__ __forceinline__ acc mul(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Unit<float> {
  typedef float frag __attribute__((ext_vector_type(4)));
  typedef float acc __attribute__((ext_vector_type(16)));
  // (four steps of k = 2: the lower lanes hold k 0 to 3 of the piece, the upper 4 to 7; both operands alike)
  static __device__ __forceinline__ acc mul(frag a, frag b, acc c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

constexpr uint32_t kDepthBytes = 128;
template <typename T>
constexpr uint32_t kDepth = kDepthBytes / sizeof(T);

// Where piece `piece` of row `row` lies, in pieces of 16 bytes.  along: rows of DEPTH (4 or 8) pieces.  across: rows of WIDTH elements; the
// 16-bit transposing read takes two neighbouring pieces of four rows.
template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t DEPTH>
__device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
  if (!ACROSS) return row * DEPTH + (piece ^ ((row / (16 / DEPTH)) & (DEPTH - 1u)));
  constexpr uint32_t kPieces = WIDTH / Piece<T>::kElems;
  if (sizeof(T) == 4) return row * kPieces + piece;
  constexpr uint32_t kPairs = kPieces / 2;  // pairs of pieces in a row: a power of two
  constexpr uint32_t kSpread = kPairs >= 8 ? 2u : 1u;
  return row * kPieces + (piece ^ ((((row & 3u) * kSpread) & (kPairs - 1u)) << 1));
}

// The piece of an operand that a thread brings: `first` .. `end`, the rows (m or n) that there are.
template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t THREADS>
struct Loader {
  static constexpr uint32_t kElems = Piece<T>::kElems;
  static constexpr uint32_t kPieces = WIDTH * kDepthBytes / 16 / THREADS;
  static constexpr uint32_t kRowPieces = ACROSS ? WIDTH / kElems : 8u;
  static_assert(WIDTH * kDepthBytes / 16 % THREADS == 0, "whole rounds");
  typename Piece<T>::type held[kPieces];

  // base: element (k = 0, first row) of the operand; `rows` of it are there, `stride` elements from one line to the next
  __device__ __forceinline__ void load(const T *__restrict__ base, uint32_t rows, size_t stride, uint32_t k0, uint32_t depth) {
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
      const uint32_t at = threadIdx.x + i * THREADS, line = at / kRowPieces, piece = at % kRowPieces;
      held[i] = typename Piece<T>::type{};
      if (ACROSS) {
        if (k0 + line < depth && piece * kElems < rows) held[i] = load_piece<T>(base + (k0 + line) * stride, piece * kElems, rows);
      } else {
        if (line < rows && k0 + piece * kElems < depth) held[i] = load_piece<T>(base + line * stride, k0 + piece * kElems, depth);
      }
    }
  }
  __device__ __forceinline__ void store(T *lds) const {
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
      const uint32_t at = threadIdx.x + i * THREADS;
      reinterpret_cast<float4 *>(lds)[place<T, ACROSS, WIDTH, 8>(at / kRowPieces, at % kRowPieces)] =
          __builtin_bit_cast(float4, held[i]);
    }
  }
};

// What a lane gives the matrix unit: of row `row0` + lane % 32, piece 2 * step + lane / 32 of k.
template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t DEPTH>
__device__ __forceinline__ typename Unit<T>::frag fragment(const T *lds, uint32_t row0, uint32_t step) {
  typedef typename Unit<T>::frag frag;
  const uint32_t lane = threadIdx.x % kWave;
  if constexpr (!ACROSS) {
    return __builtin_bit_cast(frag, reinterpret_cast<const float4 *>(lds)[place<T, false, WIDTH, DEPTH>(row0 + lane % 32, 2 * step + lane / 32)]);
  } else if constexpr (sizeof(T) == 4) {
    frag f;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) f[j] = lds[(step * 8 + lane / 32 * 4 + j) * WIDTH + row0 + lane % 32];
    return f;
  } else {
    typedef short quad __attribute__((ext_vector_type(4)));
    quad half[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t k = step * 16 + lane / 32 * 8 + j * 4 + lane % 16 / 4, col = row0 + lane % 32 / 16 * 16 + lane % 4 * 4;
      const T *from = lds + place<T, true, WIDTH, DEPTH>(k, col / 8) * 8 + col % 8;
      half[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) quad *)from);
    }
    return __builtin_bit_cast(frag, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// Shape of a tile: BM x BN results, WM x WN waves; kStages: of the ring of loads that go straight to LDS, 0: staged through
// registers into two buffers.
template <uint32_t BM_, uint32_t BN_, uint32_t WM_, uint32_t WN_, uint32_t STAGES>
struct Shape {
  static constexpr uint32_t kStages = STAGES;
  // (a wave's room for its results: 32 rows of 64 columns in 16 bits; of 32 where two workgroups are to share a CU)
  static constexpr uint32_t kRoom = BM_ * BN_ >= 256 * 256 ? 4096u : 2048u;
  static constexpr uint32_t kRingBytes = (BM_ + BN_) * (STAGES != 0 ? STAGES : 2u) * kDepthBytes;
  static constexpr uint32_t kLdsBytes = kRingBytes + (STAGES != 0 ? WM_ * WN_ * kRoom : 0u);
  static constexpr uint32_t BM = BM_, BN = BN_, WM = WM_, WN = WN_, kThreads = WM * WN * kWave;
  static constexpr uint32_t kFragsM = BM / WM / 32, kFragsN = BN / WN / 32;
};

template <typename T, typename S>
using Sums = typename Unit<T>::acc[S::kFragsM][S::kFragsN];

// A wave's results to memory by way of a piece of LDS of its own, so that whole pieces of a row go side by side: a lane holds,
// of row lane % 32, 4 neighbouring columns at a time.  ROOM bytes hold 32 rows of so many of the wave's columns.  True: all of
// the wave's results are there, and were stored in whole pieces.
template <typename T, typename S, uint32_t ROOM>
__device__ __forceinline__ bool store_tile(const Sums<T, S> &sum, uint32_t m0, uint32_t n0, uint32_t rows, uint32_t cols,
                                           T *__restrict__ out, size_t out_stride, T *room) {
  constexpr uint32_t kElems = Piece<T>::kElems, kWide = S::BN / S::WN;
  constexpr uint32_t kCols = ROOM / 32 / sizeof(T) < kWide ? ROOM / 32 / sizeof(T) : kWide, kRow = kCols / kElems;
  static_assert(kCols % 8 == 0 && kWide % kCols == 0 && (kRow & (kRow - 1)) == 0, "whole groups of 8 columns");
  typedef T quad __attribute__((ext_vector_type(4)));
  const uint32_t lane = threadIdx.x % kWave;
  const bool whole = m0 + S::BM / S::WM <= rows && n0 + kWide <= cols;
#pragma unroll
  for (uint32_t i = 0; i < S::kFragsM; ++i) {
#pragma unroll
    for (uint32_t c0 = 0; c0 < kWide; c0 += kCols) {
#pragma unroll
      for (uint32_t g = 0; g < kCols / 8; ++g) {
        const uint32_t j = (c0 / 8 + g) / 4, r = (c0 / 8 + g) % 4;
        quad v;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) v[c] = static_cast<T>(sum[i][j][r * 4 + c]);
        const uint32_t row = lane % 32, col = g * 8 + lane / 32 * 4;
        // (pieces are placed by the row, against bank conflicts)
        *reinterpret_cast<quad *>(room + (row * kRow + ((col / kElems) ^ (row & (kRow - 1)))) * kElems + col % kElems) = v;
      }
      // (a wave's LDS instructions are carried out in order)
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_sched_barrier(0);  // (or the compiler fetches the sums of all turns first, and spills them)
      constexpr uint32_t kRows = kWave / kRow;  // that the lanes hold at a time
      const uint32_t row0 = lane / kRow, piece = lane % kRow, n = n0 + c0 + piece * kElems;
      const auto held = [&](uint32_t row) {
        return __builtin_bit_cast(typename Piece<T>::type, reinterpret_cast<const float4 *>(room)[row * kRow + (piece ^ (row & (kRow - 1)))]);
      };
      T *const to = out + (m0 + i * 32 + row0) * out_stride + n;
      if (whole) {
#pragma unroll
        for (uint32_t p = 0; p < 32; p += kRows) *reinterpret_cast<typename Piece<T>::type *>(to + p * out_stride) = held(p + row0);
      } else {
#pragma unroll 1
        for (uint32_t p = 0; p < 32; p += kRows)
          if (m0 + i * 32 + p + row0 < rows && n < cols) store_piece<T>(to + p * out_stride - n, n, cols, held(p + row0));
      }
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  return whole;
}

// The tile's results to `out` (row-major, `stride` elements a row): `rows` x `cols` of it are there.
template <typename T, bool A_ACROSS, bool B_ACROSS, typename S>
__device__ __forceinline__ void tile_product(const T *__restrict__ a, uint32_t rows, size_t a_stride, const T *__restrict__ b,
                                             uint32_t cols, size_t b_stride, uint32_t depth, T *__restrict__ out,
                                             size_t out_stride, float4 *lds) {
  constexpr uint32_t kA = S::BM * kDepth<T>, kB = S::BN * kDepth<T>, kSteps = 4;
  T *const buffer = reinterpret_cast<T *>(lds);  // A, B of one buffer, then of the other
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t m0 = wave / S::WN * (S::BM / S::WM), n0 = wave % S::WN * (S::BN / S::WN);
  typename Unit<T>::acc sum[S::kFragsM][S::kFragsN] = {};
  Loader<T, A_ACROSS, S::BM, S::kThreads> load_a;
  Loader<T, B_ACROSS, S::BN, S::kThreads> load_b;
  if (depth != 0) {
    load_a.load(a, rows, a_stride, 0, depth);
    load_b.load(b, cols, b_stride, 0, depth);
    load_a.store(buffer);
    load_b.store(buffer + kA);
  }
  __syncthreads();
  uint32_t turn = 0;
  for (uint32_t k0 = 0; k0 < depth; k0 += kDepth<T>, turn ^= 1u) {
    const bool more = k0 + kDepth<T> < depth;
    if (more) {
      load_a.load(a, rows, a_stride, k0 + kDepth<T>, depth);
      load_b.load(b, cols, b_stride, k0 + kDepth<T>, depth);
    }
    const T *const at = buffer + turn * (kA + kB);
#pragma unroll
    for (uint32_t step = 0; step < kSteps; ++step) {
      typename Unit<T>::frag fa[S::kFragsM], fb[S::kFragsN];
#pragma unroll
      for (uint32_t i = 0; i < S::kFragsM; ++i) fa[i] = fragment<T, A_ACROSS, S::BM, 8>(at, m0 + i * 32, step);
#pragma unroll
      for (uint32_t j = 0; j < S::kFragsN; ++j) fb[j] = fragment<T, B_ACROSS, S::BN, 8>(at + kA, n0 + j * 32, step);
#pragma unroll
      for (uint32_t i = 0; i < S::kFragsM; ++i)
#pragma unroll
        for (uint32_t j = 0; j < S::kFragsN; ++j) sum[i][j] = Unit<T>::mul(fb[j], fa[i], sum[i][j]);
    }
    if (more) {
      T *const to = buffer + (turn ^ 1u) * (kA + kB);
      load_a.store(to);
      load_b.store(to + kA);
    }
    __syncthreads();
  }
  store_tile<T, S, S::kRoom>(sum, m0, n0, rows, cols, out, out_stride, buffer + wave * (S::kRoom / sizeof(T)));
}

// ---- the same, with loads that go straight to LDS -----------------------------------------------------------------
// For operands whose lines begin at multiples of 16 bytes.  A workgroup takes one tile after the other, and their stages
// (128 bytes of a row of k each, four steps of the matrix unit) are one stream through a ring of S::kStages places in LDS.
//   step 0, 1   the fragments of the stage's other steps are read; then every wave holds all of the stage,
//   step 2, 3   its place is filled with the stage that is kStages later, perhaps the next tile's,
//   step 3      the next stage is waited for, with the later ones under way, and its first fragments are read.
// Loads and reads go between the matrix instructions, evenly: loads in one go hold up the wave that issues them, and a SIMD
// may have no other.  (Stages of 64 bytes with four places leave the loads the same time, but ask the L2 twice as often.)
// A tile's results go out by way of room of their own while the next tile's stages come in.
//
// The compiler knows nothing of these loads (its own form waits for every one of them before any read of LDS): it only
// counts its own, and waits that count more loads than it knows are longer, never shorter.
constexpr uint32_t kStageDepth = 8;  // pieces of 16 bytes
template <typename T>
constexpr uint32_t kStageK = kStageDepth * Piece<T>::kElems;

__device__ __forceinline__ void load_to_lds(uint32_t lds_bytes, uint32_t offset, const void *base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_bytes), "v"(offset), "s"(base) : "memory");
}
template <uint32_t UNDER_WAY>
__device__ __forceinline__ void wait_for_loads() {
  static_assert(UNDER_WAY < 64, "what the counter holds");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(UNDER_WAY) : "memory");
}

template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t THREADS>
struct DirectLoader {
  static constexpr uint32_t kElems = Piece<T>::kElems;
  static constexpr uint32_t kPieces = WIDTH * kStageDepth / THREADS;
  static constexpr uint32_t kRowPieces = ACROSS ? WIDTH / kElems : kStageDepth;
  static_assert(WIDTH * kStageDepth % THREADS == 0, "whole rounds");
  uint32_t offset[kPieces];  // bytes from the operand's element (k0, first row)

  // Lane by lane the pieces of LDS are filled in order; place() is its own inverse, so what belongs at place p of a row is
  // the row's piece place(p).
  __device__ __forceinline__ void begin(uint32_t rows, uint32_t stride) {
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
      const uint32_t at = threadIdx.x + i * THREADS, line = at / kRowPieces;
      const uint32_t piece = place<T, ACROSS, WIDTH, kStageDepth>(line, at % kRowPieces) - line * kRowPieces;
      if (ACROSS) {  // (columns beyond the last whole piece are not stored: any will do)
        const uint32_t last = (rows - 1) / kElems;
        offset[i] = (line * stride + (piece < last ? piece : last) * kElems) * static_cast<uint32_t>(sizeof(T));
      } else {
        offset[i] = ((line < rows ? line : rows - 1) * stride + piece * kElems) * static_cast<uint32_t>(sizeof(T));
      }
    }
  }
  __device__ __forceinline__ void load(uint32_t i, const T *base, uint32_t lds_bytes, uint32_t wave) const {
    load_to_lds(lds_bytes + (i * THREADS + wave * kWave) * 16u, offset[i], base);
  }
  // The last stage, of which only `depth` of k are there: by way of registers, with zeros behind.
  static __device__ __forceinline__ void load_partial(const T *__restrict__ base, uint32_t rows, size_t stride, uint32_t depth, T *lds) {
#pragma unroll 1
    for (uint32_t i = 0; i < kPieces; ++i) {
      const uint32_t at = threadIdx.x + i * THREADS, line = at / kRowPieces, piece = at % kRowPieces;
      typename Piece<T>::type v{};
      if (ACROSS) {
        if (line < depth && piece * kElems < rows) v = load_piece<T>(base + line * stride, piece * kElems, rows);
      } else {
        if (line < rows && piece * kElems < depth) v = load_piece<T>(base + line * stride, piece * kElems, depth);
      }
      reinterpret_cast<float4 *>(lds)[place<T, ACROSS, WIDTH, kStageDepth>(line, piece)] = __builtin_bit_cast(float4, v);
    }
  }
};

// A tile of a product: its operands' first elements, its extent and depth, and where its results go.
template <typename T>
struct Job {
  const T *a, *b;
  T *out;
  uint32_t rows, cols, depth;
};

// job(n, &j): the workgroup's n-th tile; false: there are no more.
template <typename T, bool A_ACROSS, bool B_ACROSS, typename S, typename JOBS>
__device__ __forceinline__ void stream_products(const JOBS &jobs, uint32_t a_stride, uint32_t b_stride, size_t out_stride,
                                                float4 *lds) {
  constexpr uint32_t kA = S::BM * kStageK<T>, kB = S::BN * kStageK<T>, kSteps = kStageDepth / 2, kRing = S::kStages;
  constexpr uint32_t kStageBytes = (kA + kB) * sizeof(T);
  static_assert(kSteps == 4 && (kRing & (kRing - 1)) == 0 && kRing >= 2, "what work() goes by");
  T *const buffer = reinterpret_cast<T *>(lds);
  const uint32_t wave = uniform(threadIdx.x / kWave);
  const uint32_t m0 = wave / S::WN * (S::BM / S::WM), n0 = wave % S::WN * (S::BN / S::WN);
  const uint32_t lds_base = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) float4 *)lds)));
  typedef DirectLoader<T, A_ACROSS, S::BM, S::kThreads> LoaderA;
  typedef DirectLoader<T, B_ACROSS, S::BN, S::kThreads> LoaderB;
  constexpr uint32_t kLoads = LoaderA::kPieces + LoaderB::kPieces;
  const size_t a_step = (A_ACROSS ? static_cast<size_t>(a_stride) : 1u) * kStageK<T>;
  const size_t b_step = (B_ACROSS ? static_cast<size_t>(b_stride) : 1u) * kStageK<T>;

  // what is filled: tile `filling`, from its stage `left` of `to_fill` on; `filled` and `done` count the stream's stages
  Job<T> from;
  LoaderA load_a;
  LoaderB load_b;
  uint32_t filling = 0, depth_left = 0, filled = 0, done = 0;
  bool more = jobs(0, &from);
  const auto begin = [&] {
    load_a.begin(from.rows, a_stride);
    load_b.begin(from.cols, b_stride);
    depth_left = from.depth;
  };
  if (more) begin();
  const auto load_one = [&](uint32_t i) {
    const uint32_t to = lds_base + (filled & (kRing - 1)) * kStageBytes;
    if (i < LoaderA::kPieces)
      load_a.load(i, from.a, to, wave);
    else
      load_b.load(i - LoaderA::kPieces, from.b, to + kA * static_cast<uint32_t>(sizeof(T)), wave);
  };
  const auto filled_one = [&] {
    from.a += a_step;
    from.b += b_step;
    depth_left -= kStageK<T> < depth_left ? kStageK<T> : depth_left;
    ++filled;
  };
  const auto next_job = [&] {  // the next tile that has anything to fill
    while (more && depth_left == 0) {
      more = jobs(++filling, &from);
      if (more) begin();
    }
  };
  const auto fill_partial = [&] {
    T *const to = buffer + (filled & (kRing - 1)) * (kA + kB);
    LoaderA::load_partial(from.a, from.rows, a_stride, depth_left, to);
    LoaderB::load_partial(from.b, from.cols, b_stride, depth_left, to + kA);
    filled_one();
  };

  Sums<T, S> sum = {};
  typename Unit<T>::frag fa[kSteps][S::kFragsM], fb[kSteps][S::kFragsN];
  constexpr uint32_t kReads = S::kFragsM + S::kFragsN, kMuls = S::kFragsM * S::kFragsN;
  const auto read_one = [&](uint32_t stage, uint32_t step, uint32_t i) {
    const T *const at = buffer + (stage & (kRing - 1)) * (kA + kB);
    // (in the order in which the products need them)
    if (i == 0)
      fb[step][0] = fragment<T, B_ACROSS, S::BN, kStageDepth>(at + kA, n0, step);
    else if (i <= S::kFragsM)
      fa[step][i - 1] = fragment<T, A_ACROSS, S::BM, kStageDepth>(at, m0 + (i - 1) * 32, step);
    else
      fb[step][i - S::kFragsM] = fragment<T, B_ACROSS, S::BN, kStageDepth>(at + kA, n0 + (i - S::kFragsM) * 32, step);
  };
  // Stage `done`, whose first fragments are held; FILL: there is a whole one to be filled.  `after`: stores that were issued
  // after the loads of the next stage (the counter counts both, in the order in which they were issued).  Behind the stream's
  // last stage something is read as well, which nothing uses.
  constexpr uint32_t kStores = S::BM / S::WM * (S::BN / S::WN) / kWave / Piece<T>::kElems;  // of a wave's tile
  bool after = false;
  const auto work = [&](auto FILL) {
#pragma unroll
    for (uint32_t step = 0; step < kSteps; ++step) {
      if (step == 2) __syncthreads();  // every wave holds all of the stage
      if (step == 2 && !FILL.value && more) fill_partial();
      if (step == 3) {  // the next stage is there
        constexpr uint32_t kUnderWay = FILL.value ? (kRing - 2) * kLoads + kLoads / 2 : 0;
        if (FILL.value && after)
          wait_for_loads<(kUnderWay + kStores < 63 ? kUnderWay + kStores : kUnderWay)>();
        else
          wait_for_loads<kUnderWay>();
        after = false;
        __syncthreads();
      }
#pragma unroll
      for (uint32_t q = 0; q < kMuls; ++q) {
        const uint32_t i = q % S::kFragsM, j = q / S::kFragsM;
        sum[i][j] = Unit<T>::mul(fb[step][j], fa[step][i], sum[i][j]);
        const uint32_t reads = step == 0 ? 2 * kReads : step == 2 ? 0 : kReads;
#pragma unroll
        for (uint32_t r = q * reads / kMuls; r < (q + 1) * reads / kMuls; ++r) {
          if (step == 0)
            read_one(done, 1 + r / kReads, r % kReads);
          else
            read_one(step == 1 ? done : done + 1, step == 1 ? 3 : 0, r);
        }
        constexpr uint32_t kShare = kLoads / 2;
        static_assert(kLoads % 2 == 0, "an equal share to a step");
        if (FILL.value && step >= 2) {
#pragma unroll
          for (uint32_t r = q * kShare / kMuls; r < (q + 1) * kShare / kMuls; ++r) load_one((step - 2) * kShare + r);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (FILL.value) filled_one();
    ++done;
  };

  for (uint32_t g = 0; g < kRing; ++g) {
    next_job();
    if (!more) break;
    if (depth_left >= kStageK<T>) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) load_one(i);
      filled_one();
    } else {
      fill_partial();
    }
  }
  wait_for_loads<0>();
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kReads; ++i) read_one(0, 0, i);
  Job<T> now;
  for (uint32_t n = 0; jobs(n, &now); ++n) {
    uint32_t left = (now.depth + kStageK<T> - 1) / kStageK<T>;
    while (left != 0) {
      next_job();
      uint32_t turns = depth_left / kStageK<T>;  // stages with a whole one to fill
      turns = turns < left ? turns : left;
      left -= turns;
      for (; turns != 0; --turns) work(std::true_type());
      if (left != 0 && (!more || depth_left != 0)) {
        work(std::false_type());
        --left;
      }
    }
    after = store_tile<T, S, S::kRoom>(sum, m0, n0, now.rows, now.cols, now.out, out_stride,
                                       buffer + kRing * (kA + kB) + wave * (S::kRoom / sizeof(T)));
#pragma unroll
    for (uint32_t i = 0; i < S::kFragsM; ++i)
#pragma unroll
      for (uint32_t j = 0; j < S::kFragsN; ++j) sum[i][j] = typename Unit<T>::acc{};
  }
}

// Tiles of a product: the run of XCD x of the eight (workgroups go round them) lies together, so that its tiles share an
// L2; the XCD's workgroups take the run's tiles in turn.
struct Turn {
  uint32_t index, end, step;
};
__device__ __forceinline__ Turn turn_of(uint64_t tiles) {
  const uint32_t share = static_cast<uint32_t>((tiles + 7) / 8), xcd = blockIdx.x % 8, n = static_cast<uint32_t>(tiles);
  const uint32_t begin = xcd * share < n ? xcd * share : n;
  return Turn{begin + blockIdx.x / 8, begin + share < n ? begin + share : n, gridDim.x / 8};
}

// Rows from `first` on are zero: a workgroup takes a run of pieces of them.
template <typename T>
__device__ __forceinline__ void zero_from(T *__restrict__ out, uint32_t first, uint32_t rows, uint32_t cols, uint32_t threads) {
  if (first >= rows) return;
  const typename Piece<T>::type zero{};
  T *const from = out + static_cast<size_t>(first) * cols;
  const size_t n = static_cast<size_t>(rows - first) * cols;
  const size_t step = static_cast<size_t>(gridDim.x) * threads * Piece<T>::kElems;
  for (size_t at = (static_cast<size_t>(blockIdx.x) * threads + threadIdx.x) * Piece<T>::kElems; at < n; at += step) {
    if (at + Piece<T>::kElems <= n) {
      *reinterpret_cast<typename Piece<T>::type *>(from + at) = zero;
    } else {
      for (size_t j = at; j < n; ++j) from[j] = static_cast<T>(0.f);
    }
  }
}

template <typename T, bool OUT_MAJOR, typename S>
__global__ __launch_bounds__(S::kThreads) void product_kernel(const T *__restrict__ rows, const T *__restrict__ weight,
                                                              const uint32_t *__restrict__ indptr, T *__restrict__ out,
                                                              uint32_t n_rows, uint32_t experts, uint32_t inner,
                                                              uint32_t cols) {
  extern __shared__ float4 lds[];
  __shared__ TileTable table;
  const uint32_t across = (cols + S::BN - 1) / S::BN;
  const uint32_t total = table.build<S::kThreads>(indptr, experts, n_rows, S::BM);
  const Turn turn = turn_of(static_cast<uint64_t>(total) * across);
  const auto jobs = [&](uint32_t n, Job<T> *j) {
    const uint32_t index = turn.index + n * turn.step;
    if (index >= turn.end) return false;
    const uint32_t down = uniform(index / across), col0 = (index - down * across) * S::BN;
    const Tile tile = table.find(indptr, down, experts, n_rows, S::BM);
    const T *const w = weight + static_cast<size_t>(tile.expert) * inner * cols;
    j->a = uniform(rows + static_cast<size_t>(tile.first) * inner);
    j->b = uniform(OUT_MAJOR ? w + static_cast<size_t>(col0) * inner : w + col0);
    j->out = out + static_cast<size_t>(tile.first) * cols + col0;
    j->rows = tile.end - tile.first;
    j->cols = cols - col0 < S::BN ? cols - col0 : S::BN;
    j->depth = inner;
    return true;
  };
  if constexpr (S::kStages != 0) {
    stream_products<T, false, !OUT_MAJOR, S>(jobs, inner, OUT_MAJOR ? inner : cols, cols, lds);
  } else {
    Job<T> j;
    for (uint32_t n = 0; jobs(n, &j); ++n) {
      tile_product<T, false, !OUT_MAJOR, S>(j.a, j.rows, inner, j.b, j.cols, OUT_MAJOR ? inner : cols, inner, j.out, cols, lds);
      __syncthreads();
    }
  }
  const uint32_t behind = indptr[experts];
  zero_from(out, behind < n_rows ? behind : n_rows, n_rows, cols, S::kThreads);
}

// d_weight[expert] = left_e^T @ right_e over the expert's rows; (left, right) = (rows, ct), or (ct, rows) where the weight is
// stored out-major.
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void gradient_kernel(const T *__restrict__ left, const T *__restrict__ right,
                                                               const uint32_t *__restrict__ indptr, T *__restrict__ d_weight,
                                                               uint32_t n_rows, uint32_t experts, uint32_t n_left,
                                                               uint32_t n_right) {
  extern __shared__ float4 lds[];
  const uint32_t down = (n_left + S::BM - 1) / S::BM, across = (n_right + S::BN - 1) / S::BN;
  // An eighth of every expert's tiles to an XCD, neighbouring ones: the XCDs' work is the same however long the experts are.
  const uint32_t tiles = down * across, share = (tiles + 7) / 8;
  const auto jobs = [&](uint32_t n, Job<T> *j) {
    const uint32_t expert = uniform(blockIdx.x / 8 / share);
    const uint32_t in = (blockIdx.x + expert * tiles) % 8 * share + blockIdx.x / 8 % share;
    if (n != 0 || in >= tiles) return false;
    const uint32_t p0 = uniform(in / across) * S::BM, q0 = uniform(in % across) * S::BN;
    uint2 range = rows_of(indptr, expert, experts, n_rows);
    range = make_uint2(uniform(range.x), uniform(range.y));
    j->a = uniform(left + static_cast<size_t>(range.x) * n_left + p0);
    j->b = uniform(right + static_cast<size_t>(range.x) * n_right + q0);
    j->out = d_weight + (static_cast<size_t>(expert) * n_left + p0) * n_right + q0;
    j->rows = n_left - p0 < S::BM ? n_left - p0 : S::BM;
    j->cols = n_right - q0 < S::BN ? n_right - q0 : S::BN;
    j->depth = range.y - range.x;
    return true;
  };
  if constexpr (S::kStages != 0) {
    stream_products<T, true, true, S>(jobs, n_left, n_right, n_right, lds);
  } else {
    Job<T> j;
    for (uint32_t n = 0; jobs(n, &j); ++n) {
      tile_product<T, true, true, S>(j.a, j.rows, n_left, j.b, j.cols, n_right, j.depth, j.out, n_right, lds);
      __syncthreads();
    }
  }
}

bool refuse_grid(const char *target, uint64_t tiles) {
  if (tiles < (1u << 22)) return false;  // (threads of a launch are counted in 32 bits)
  set_error("%s: a product of %llu tiles is too large for one call", target, static_cast<unsigned long long>(tiles));
  return true;
}

// More than 64 KB of LDS has to be asked for, once a kernel and device.
template <typename K>
bool allow_lds(const char *target, K kernel, uint32_t bytes) {
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(bytes));
  if (e == hipSuccess) return true;
  (void)hipGetLastError();
  set_error("%s: %u bytes of LDS: %s", target, bytes, hipGetErrorString(e));
  return false;
}

// Loads that go straight to LDS need lines at multiples of 16 bytes, and offsets within a tile in 32 bits.
template <typename T>
bool whole_pieces(const void *p, uint32_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % Piece<T>::kElems == 0 && stride < (1u << 20);
}

// Shapes for operands in whole pieces, and for others
struct Direct {
  using Large = Shape<256, 256, 2, 2, 2>;
  using Middle = Shape<128, 128, 2, 2, 2>;
  using Small = Shape<64, 64, 2, 2, 4>;
};
struct Staged {
  using Large = Shape<256, 256, 2, 4, 0>;
  using Middle = Shape<128, 128, 2, 2, 0>;
  using Small = Shape<64, 64, 2, 2, 0>;
};

template <typename T, typename S>
void launch_product(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, void **buffers) {
  const uint64_t tiles = most_tiles(d.rows, d.experts, S::BM) * div_up(d.out, S::BN);
  if (tiles >= 1ull << 32) {
    set_error("%s: a product of %llu tiles is too large for one call", target, static_cast<unsigned long long>(tiles));
    return;
  }
  // one workgroup to each place that the LDS leaves
  const uint64_t places = static_cast<uint64_t>(device_info().num_cu) * (160u * 1024u / (S::kLdsBytes + sizeof(TileTable) + 1024u));
  const unsigned grid = static_cast<unsigned>(((tiles < places ? tiles : places) + 7) / 8 * 8);
  const auto launch = [&](auto *kernel) {
    if (!allow_lds(target, kernel, S::kLdsBytes)) return;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::kThreads), S::kLdsBytes, stream,
                       static_cast<const T *>(buffers[0]), static_cast<const T *>(buffers[1]),
                       static_cast<const uint32_t *>(buffers[2]), static_cast<T *>(buffers[3]), d.rows, d.experts, d.width,
                       d.out);
    check_launch(target);
  };
  if (d.flags & BPL_EXPERT_OUT_MAJOR)
    launch(product_kernel<T, true, S>);
  else
    launch(product_kernel<T, false, S>);
}

template <typename T, typename SHAPES>
void choose_product(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, void **buffers) {
  const uint32_t mean = d.rows / d.experts;
  if constexpr (sizeof(T) == 2) {
    if (mean >= 192) return launch_product<T, typename SHAPES::Large>(target, stream, d, buffers);
  }
  if (mean >= 48)
    launch_product<T, typename SHAPES::Middle>(target, stream, d, buffers);
  else
    launch_product<T, typename SHAPES::Small>(target, stream, d, buffers);
}

template <typename T>
void matmul(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.rows == 0 || d.out == 0) return;
  const bool out_major = (d.flags & BPL_EXPERT_OUT_MAJOR) != 0;
  if (whole_pieces<T>(buffers[0], d.width) && whole_pieces<T>(buffers[1], out_major ? d.width : d.out))
    choose_product<T, Direct>(target, stream, d, buffers);
  else
    choose_product<T, Staged>(target, stream, d, buffers);
}

template <typename T, typename S>
void launch_gradient(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, const void *left, const void *right,
                     uint32_t n_left, uint32_t n_right, void **buffers) {
  const uint64_t blocks = 8 * ((static_cast<uint64_t>(div_up(n_left, S::BM)) * div_up(n_right, S::BN) + 7) / 8) * d.experts;
  if (refuse_grid(target, blocks) || !allow_lds(target, gradient_kernel<T, S>, S::kLdsBytes)) return;
  hipLaunchKernelGGL((gradient_kernel<T, S>), dim3(static_cast<unsigned>(blocks)), dim3(S::kThreads), S::kLdsBytes, stream,
                     static_cast<const T *>(left), static_cast<const T *>(right), static_cast<const uint32_t *>(buffers[2]),
                     static_cast<T *>(buffers[3]), d.rows, d.experts, n_left, n_right);
  check_launch(target);
}

template <typename T, typename SHAPES>
void choose_gradient(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, const void *left, const void *right,
                     uint32_t n_left, uint32_t n_right, void **buffers) {
  if constexpr (sizeof(T) == 2) {
    if (static_cast<uint64_t>(d.experts) * div_up(n_left, 256) * div_up(n_right, 256) >= 256)
      return launch_gradient<T, typename SHAPES::Large>(target, stream, d, left, right, n_left, n_right, buffers);
  }
  launch_gradient<T, typename SHAPES::Middle>(target, stream, d, left, right, n_left, n_right, buffers);
}

template <typename T>
void matmul_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.width == 0 || d.out == 0) return;
  const bool out_major = (d.flags & BPL_EXPERT_OUT_MAJOR) != 0;
  const uint32_t n_left = out_major ? d.out : d.width, n_right = out_major ? d.width : d.out;
  const void *const left = buffers[out_major ? 1 : 0], *const right = buffers[out_major ? 0 : 1];
  if (whole_pieces<T>(left, n_left) && whole_pieces<T>(right, n_right))
    choose_gradient<T, Direct>(target, stream, d, left, right, n_left, n_right, buffers);
  else
    choose_gradient<T, Staged>(target, stream, d, left, right, n_left, n_right, buffers);
}

}  // namespace

extern "C" {

BPL_EXPERT_DEFINE(expert_matmul, matmul)
BPL_EXPERT_DEFINE(expert_matmul_gradient, matmul_gradient)

}  // extern "C"
