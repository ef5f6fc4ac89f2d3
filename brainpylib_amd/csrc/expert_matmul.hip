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

// The most tiles of `height` rows that any split of the rows into experts has: every expert has at most one that is not full.
__host__ __device__ constexpr uint64_t most_tiles(uint32_t rows, uint32_t experts, uint32_t height) {
  return static_cast<uint64_t>(rows) / height + (experts < rows ? experts : rows);
}

// The experts' rows and where their tiles of `height` rows begin, counted over the experts in their order: in LDS, built
// by all threads of the workgroup (one barrier, and one for the caller to see it).
struct Tile {
  uint32_t expert, first, end;  // the rows of the tile: [first, end)
};
struct TileTable {
  uint32_t start[kMostExperts];
  uint32_t wave_total[16];

  // the number of tiles: of an indptr that is none, no more than the host has counted with (rows that many experts claim would be
  // worked on again and again, and places beyond 32 bits would never end)
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
    const uint64_t most = most_tiles(rows, experts, height);
    return uniform(total < most ? total : static_cast<uint32_t>(most));
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
    // (of an indptr that is none, more tiles than 32 bits count may leave one beyond the rows: it is empty)
    const uint64_t from = uniform(r.x) + static_cast<uint64_t>(index - uniform(start[expert])) * height;
    const uint32_t end = uniform(r.y), first = from < end ? static_cast<uint32_t>(from) : end;
    return Tile{expert, first, end - first < height ? end : first + height};
  }
};

// ---- tiles --------------------------------------------------------------------------------------------------------
// One product kernel body for the three products.  C[m][n] = sum over k of A[m][k] B[n][k], tiles of BM x BN, kDepth (128 bytes
// of a row) of k at a time through buffers in LDS.  An operand lies in memory with its k side by side ("along": rows of
// tokens, out-major weights) or with its m or n side by side ("across": the others).
//   along:  LDS holds [m][k], 128 bytes a row; a lane reads the 16 bytes of k that its matrix instruction takes.
//   across: LDS holds [k][m]; 16-bit types are transposed by the LDS's transposing read (16 lanes read 4 rows of 16
//           elements and get a column of 4 each), 32-bit ones are read one by one.
// 16-byte pieces are placed so that the lanes of a read meet different banks (place()).
template <typename T, uint32_t SIDE>
struct Unit;  // the matrix instructions of a type: SIDE x SIDE results, a piece (16 bytes) of k from each of a row's 64 / SIDE lanes
#define BPL_UNIT16(TYPE, SIDE, LENGTH, INSTRUCTION)                                                                        \
  template <>                                                                                                              \
  struct Unit<TYPE, SIDE> {                                                                                                \
    typedef TYPE frag __attribute__((ext_vector_type(8)));                                                                 \
    typedef float acc __attribute__((ext_vector_type(LENGTH)));                                                            \
    static __device__ __forceinline__ acc mul(frag a, frag b, acc c) { return INSTRUCTION(a, b, c, 0, 0, 0); }             \
  };
BPL_UNIT16(half_t, 32, 16, __builtin_amdgcn_mfma_f32_32x32x16_f16)
BPL_UNIT16(half_t, 16, 4, __builtin_amdgcn_mfma_f32_16x16x32_f16)
BPL_UNIT16(bfloat_t, 32, 16, __builtin_amdgcn_mfma_f32_32x32x16_bf16)
BPL_UNIT16(bfloat_t, 16, 4, __builtin_amdgcn_mfma_f32_16x16x32_bf16)
// (in 32 bits four instructions of one k a lane each; which k a lane holds is the same for both operands, and no matter else)
#define BPL_UNIT32(SIDE, LENGTH, INSTRUCTION)                                    \
  template <>                                                                    \
  struct Unit<float, SIDE> {                                                     \
    typedef float frag __attribute__((ext_vector_type(4)));                      \
    typedef float acc __attribute__((ext_vector_type(LENGTH)));                  \
    static __device__ __forceinline__ acc mul(frag a, frag b, acc c) {           \
      _Pragma("unroll") for (int j = 0; j < 4; ++j) c = INSTRUCTION(a[j], b[j], c, 0, 0, 0); \
      return c;                                                                  \
    }                                                                            \
  };
BPL_UNIT32(32, 16, __builtin_amdgcn_mfma_f32_32x32x2f32)
BPL_UNIT32(16, 4, __builtin_amdgcn_mfma_f32_16x16x4f32)

constexpr uint32_t kDepthBytes = 128;
template <typename T>
constexpr uint32_t kDepth = kDepthBytes / sizeof(T);

// Where piece `piece` of row `row` lies, in pieces of 16 bytes.  along: rows of kDepthPieces.  across: rows of WIDTH elements; the
// 16-bit transposing read takes two neighbouring pieces of four rows.
constexpr uint32_t kDepthPieces = kDepthBytes / 16;
template <typename T, bool ACROSS, uint32_t WIDTH>
__device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
  if (!ACROSS) return row * kDepthPieces + (piece ^ ((row >> 1) & (kDepthPieces - 1u)));
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
  static constexpr uint32_t kPieces = WIDTH * kDepthPieces / THREADS;
  static constexpr uint32_t kRowPieces = ACROSS ? WIDTH / kElems : kDepthPieces;
  static_assert(WIDTH * kDepthPieces % THREADS == 0, "whole rounds");
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
      reinterpret_cast<float4 *>(lds)[place<T, ACROSS, WIDTH>(at / kRowPieces, at % kRowPieces)] =
          __builtin_bit_cast(float4, held[i]);
    }
  }
};

// What a lane gives the matrix unit: of row `row0` + lane % SIDE, piece (64 / SIDE) * step + lane / SIDE of k.
template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t SIDE>
__device__ __forceinline__ typename Unit<T, SIDE>::frag fragment(const T *lds, uint32_t row0, uint32_t step) {
  typedef typename Unit<T, SIDE>::frag frag;
  const uint32_t lane = threadIdx.x % kWave, piece = kWave / SIDE * step + lane / SIDE;
  if constexpr (!ACROSS) {
    return __builtin_bit_cast(frag, reinterpret_cast<const float4 *>(lds)[place<T, false, WIDTH>(row0 + lane % SIDE, piece)]);
  } else if constexpr (sizeof(T) == 4) {
    frag f;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) f[j] = lds[(piece * 4 + j) * WIDTH + row0 + lane % SIDE];
    return f;
  } else {
    typedef short quad __attribute__((ext_vector_type(4)));
    quad half[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t k = piece * 8 + j * 4 + lane % 16 / 4, col = row0 + lane % SIDE / 16 * 16 + lane % 4 * 4;
      const T *from = lds + place<T, true, WIDTH>(k, col / 8) * 8 + col % 8;
      half[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) quad *)from);
    }
    return __builtin_bit_cast(frag, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// Shape of a tile: BM x BN results, WM x WN waves, matrix instructions of SIDE x SIDE; kStages: of the ring of loads that go
// straight to LDS, 0: staged through registers into two buffers.
template <uint32_t BM_, uint32_t BN_, uint32_t WM_, uint32_t WN_, uint32_t SIDE, uint32_t STAGES, uint32_t LOAD_BYTES = 16>
struct Shape {
  static constexpr uint32_t kLoadBytes = LOAD_BYTES;
  static constexpr uint32_t kWavesWanted = BM_ * BN_ >= 256 * 256 ? 1u : 2u;  // to a SIMD, at least
  static constexpr uint32_t kSide = SIDE, kSteps = kDepthBytes / 16 / (kWave / SIDE);
  static constexpr uint32_t kStages = STAGES;
  // (a wave's room for its results: SIDE rows of 64 columns in 16 bits; of 32 where workgroups are to share a CU)
  static constexpr uint32_t kRoom = BM_ * BN_ >= 256 * 256 ? 4096u : SIDE * 64u;
  static constexpr uint32_t kRingBytes = (BM_ + BN_) * (STAGES != 0 ? STAGES : 2u) * kDepthBytes;
  static constexpr uint32_t kLdsBytes = kRingBytes + (STAGES != 0 ? WM_ * WN_ * kRoom : 0u);
  static constexpr uint32_t BM = BM_, BN = BN_, WM = WM_, WN = WN_, kThreads = WM * WN * kWave;
  static constexpr uint32_t kFragsM = BM / WM / SIDE, kFragsN = BN / WN / SIDE;
};

template <typename T, typename S>
using Sums = typename Unit<T, S::kSide>::acc[S::kFragsM][S::kFragsN];

typedef uint32_t quad32 __attribute__((ext_vector_type(4)));
// Past the caches.  (As an instruction of its own: of a nontemporal store and a plain one that a branch chooses between, the
// compiler makes one plain one.  The two wait states are for a vector instruction that overwrites the data's registers next:
// a store of more than 64 bits reads them late, and the compiler does not know of one that it does not see.)
__device__ __forceinline__ void store_past(void *to, quad32 v) {
  asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1" ::"v"(to), "v"(v) : "memory");
}

// A wave's results to memory by way of a piece of LDS of its own, so that whole pieces of a row go side by side: a lane holds,
// of row lane % kSide, 4 neighbouring columns at a time.  ROOM bytes hold kSide rows of so many of the wave's columns.  True: all of
// the wave's results are there, and were stored in whole pieces.
template <typename T, typename S, uint32_t ROOM, typename O>
__device__ __forceinline__ bool store_tile(const Sums<T, S> &sum, uint32_t m0, uint32_t n0, uint32_t rows, uint32_t cols,
                                           O *__restrict__ out, size_t out_stride, O *room, bool past) {
  constexpr uint32_t kElems = Piece<O>::kElems, kWide = S::BN / S::WN, kSide = S::kSide, kGroup = kWave / kSide * 4;
  constexpr uint32_t kCols = ROOM / kSide / sizeof(O) < kWide ? ROOM / kSide / sizeof(O) : kWide, kRow = kCols / kElems;
  static_assert(kCols % kGroup == 0 && kWide % kCols == 0 && (kRow & (kRow - 1)) == 0 && kWave % kRow == 0, "whole groups of columns");
  typedef O quad __attribute__((ext_vector_type(4)));
  const uint32_t lane = threadIdx.x % kWave;
  const bool whole = m0 + S::BM / S::WM <= rows && n0 + kWide <= cols;
#pragma unroll
  for (uint32_t i = 0; i < S::kFragsM; ++i) {
#pragma unroll
    for (uint32_t c0 = 0; c0 < kWide; c0 += kCols) {
#pragma unroll
      for (uint32_t g = 0; g < kCols / kGroup; ++g) {
        const uint32_t j = (c0 / kGroup + g) * kGroup / kSide, r = (c0 / kGroup + g) % (kSide / kGroup);
        quad v;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) v[c] = static_cast<O>(sum[i][j][r * 4 + c]);
        const uint32_t row = lane % kSide, col = g * kGroup + lane / kSide * 4;
        // (pieces are placed by the row, against bank conflicts)
        *reinterpret_cast<quad *>(room + (row * kRow + ((col / kElems) ^ (row & (kRow - 1)))) * kElems + col % kElems) = v;
      }
      // (a wave's LDS instructions are carried out in order)
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_sched_barrier(0);  // (or the compiler fetches the sums of all turns first, and spills them)
      constexpr uint32_t kRows = kWave / kRow;  // that the lanes hold at a time
      const uint32_t row0 = lane / kRow, piece = lane % kRow, n = n0 + c0 + piece * kElems;
      const auto held = [&](uint32_t row) {
        return __builtin_bit_cast(typename Piece<O>::type, reinterpret_cast<const float4 *>(room)[row * kRow + (piece ^ (row & (kRow - 1)))]);
      };
      O *const to = out + (m0 + i * kSide + row0) * out_stride + n;
      if (whole && past) {
#pragma unroll
        for (uint32_t p = 0; p < kSide; p += kRows) store_past(to + p * out_stride, __builtin_bit_cast(quad32, held(p + row0)));
      } else if (whole) {
#pragma unroll
        for (uint32_t p = 0; p < kSide; p += kRows) *reinterpret_cast<typename Piece<O>::type *>(to + p * out_stride) = held(p + row0);
      } else {
#pragma unroll 1
        for (uint32_t p = 0; p < kSide; p += kRows)
          if (m0 + i * kSide + p + row0 < rows && n < cols) store_piece<O>(to + p * out_stride - n, n, cols, held(p + row0));
      }
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  return whole;
}

// The tile's results to `out` (row-major, `stride` elements a row): `rows` x `cols` of it are there.
template <typename T, bool A_ACROSS, bool B_ACROSS, typename S, typename O>
__device__ __forceinline__ void tile_product(const T *__restrict__ a, uint32_t rows, size_t a_stride, const T *__restrict__ b,
                                             uint32_t cols, size_t b_stride, uint32_t depth, O *__restrict__ out,
                                             size_t out_stride, float4 *lds) {
  constexpr uint32_t kA = S::BM * kDepth<T>, kB = S::BN * kDepth<T>, kSteps = S::kSteps, kSide = S::kSide;
  T *const buffer = reinterpret_cast<T *>(lds);  // A, B of one buffer, then of the other
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t m0 = wave / S::WN * (S::BM / S::WM), n0 = wave % S::WN * (S::BN / S::WN);
  typename Unit<T, S::kSide>::acc sum[S::kFragsM][S::kFragsN] = {};
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
      typename Unit<T, S::kSide>::frag fa[S::kFragsM], fb[S::kFragsN];
#pragma unroll
      for (uint32_t i = 0; i < S::kFragsM; ++i) fa[i] = fragment<T, A_ACROSS, S::BM, kSide>(at, m0 + i * kSide, step);
#pragma unroll
      for (uint32_t j = 0; j < S::kFragsN; ++j) fb[j] = fragment<T, B_ACROSS, S::BN, kSide>(at + kA, n0 + j * kSide, step);
#pragma unroll
      for (uint32_t i = 0; i < S::kFragsM; ++i)
#pragma unroll
        for (uint32_t j = 0; j < S::kFragsN; ++j) sum[i][j] = Unit<T, S::kSide>::mul(fb[j], fa[i], sum[i][j]);
    }
    if (more) {
      T *const to = buffer + (turn ^ 1u) * (kA + kB);
      load_a.store(to);
      load_b.store(to + kA);
    }
    __syncthreads();
  }
  store_tile<T, S, S::kRoom, O>(sum, m0, n0, rows, cols, out, out_stride,
                             reinterpret_cast<O *>(buffer) + wave * (S::kRoom / sizeof(O)), false);
}

// ---- the same, with loads that go straight to LDS -----------------------------------------------------------------
// For operands whose lines begin at multiples of 16 bytes.  A workgroup takes one tile after the other, and their stages
// (128 bytes of a row of k each, four steps of the matrix unit) are one stream through a ring of S::kStages places in LDS.
//   step 0, 1   the fragments of the stage's other steps are read; then every wave holds all of the stage,
//   step 2, 3   its place is filled with the stage that is kStages later, perhaps the next tile's,
//   step 3      the next stage is waited for, with the later ones under way, and its first fragments are read.
// (Instructions of 16 x 16 take the stage in two steps, each twice as deep.)
// Loads and reads go between the matrix instructions, evenly: loads in one go hold up the wave that issues them, and a SIMD
// may have no other.  (Stages of 64 bytes with four places leave the loads the same time, but ask the L2 twice as often.)
// A tile's results go out by way of room of their own while the next tile's stages come in.  The 256 x 256 tiles do so in part only:
// the compiler works out the addresses there ahead of the loop over the tiles and has no registers for them (57 to 112 a lane are
// spilled, none in the loop over the stages), and what is fetched back waits for every load and store before it.
//
// Why these tiles: a wave of 128 x 128 results reads 64 bytes of LDS a cycle and CU for what the matrix unit does, of the 128
// that LDS gives (64 x 64: 128, which is why smaller tiles are slower: 1,140 / 850 / 480 TFLOP/s for 256 / 128 / 64 squared,
// 32,768 rows, 8 experts of 2,048 x 2,048, bfloat16, out-major; at an inner dimension of 4,096 1,260, a library's plain product
// 1,470).  Counters of the large one: the matrix units work 60 to 66 % of the cycles (at 1.7 to 1.8 GHz, which is what the
// card's power allows), waits for stages and for results that go out 20 %; bank conflicts 5 % of LDS cycles.
//
// The compiler knows nothing of these loads (its own form waits for every one of them before any read of LDS): it only
// counts its own, and waits that count more loads than it knows are longer, never shorter.

// BYTES (16, or 4 where lines begin at any element of 32 bits) a lane, side by side in LDS.  ONCE: read once, and to take no
// room in the caches from what is not.
template <uint32_t BYTES, bool ONCE>
__device__ __forceinline__ void load_to_lds(uint32_t lds_bytes, uint32_t offset, const void *base) {
  if constexpr (BYTES == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_bytes), "v"(offset), "s"(base) : "memory");
  else if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_bytes), "v"(offset), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_bytes), "v"(offset), "s"(base) : "memory");
}
template <uint32_t UNDER_WAY>
__device__ __forceinline__ void wait_for_loads() {
  static_assert(UNDER_WAY < 64, "what the counter holds");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(UNDER_WAY) : "memory");
}

template <typename T, bool ACROSS, uint32_t WIDTH, uint32_t THREADS, uint32_t BYTES, bool ONCE>
struct DirectLoader {
  static constexpr uint32_t kElems = Piece<T>::kElems, kParts = 16 / BYTES;  // loads to a piece
  static constexpr uint32_t kPieces = WIDTH * kDepthPieces / THREADS, kLoads = kPieces * kParts;
  static constexpr uint32_t kRowPieces = ACROSS ? WIDTH / kElems : kDepthPieces;
  static_assert(WIDTH * kDepthPieces % THREADS == 0, "whole rounds");
  static_assert(BYTES == 16 || BYTES == sizeof(T), "whole elements");
  uint32_t offset[kLoads];  // bytes from the operand's element (k0, first row)

  // Lane by lane LDS is filled in order; place() is its own inverse, so what belongs at place p of a row is the row's piece
  // place(p).
  __device__ __forceinline__ void begin(uint32_t rows, uint32_t stride) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t at = (threadIdx.x + i * THREADS) / kParts, within = (threadIdx.x + i * THREADS) % kParts;
      const uint32_t line = at / kRowPieces;
      const uint32_t piece = place<T, ACROSS, WIDTH>(line, at % kRowPieces) - line * kRowPieces;
      if (ACROSS) {  // (what is beyond the columns is not stored: any will do)
        const uint32_t unit = kElems / kParts, last = (rows - 1) / unit, col = piece * kParts + within;
        offset[i] = (line * stride + (col < last ? col : last) * unit) * static_cast<uint32_t>(sizeof(T));
      } else {
        offset[i] = ((line < rows ? line : rows - 1) * stride + piece * kElems) * static_cast<uint32_t>(sizeof(T)) + within * BYTES;
      }
    }
  }
  __device__ __forceinline__ void load(uint32_t i, const T *base, uint32_t lds_bytes, uint32_t wave) const {
    load_to_lds<BYTES, ONCE>(lds_bytes + (i * THREADS + wave * kWave) * BYTES, offset[i], base);
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
      reinterpret_cast<float4 *>(lds)[place<T, ACROSS, WIDTH>(line, piece)] = __builtin_bit_cast(float4, v);
    }
  }
};

// A tile of a product: its operands' first elements, its extent and depth, and where its results go.
template <typename T, typename O>
struct Job {
  const T *a, *b;
  O *out;
  uint32_t rows, cols, depth;
};

// jobs(at, &j): the workgroup's next tile from its place `at` on, which begins at 0; false: there are no more.
// ONCE: b is read by one tile.
template <typename T, typename O, bool A_ACROSS, bool B_ACROSS, typename S, bool ONCE, typename JOBS>
__device__ __forceinline__ void stream_products(const JOBS &jobs, uint32_t a_stride, uint32_t b_stride, size_t out_stride,
                                                float4 *lds, bool past) {
  constexpr uint32_t kA = S::BM * kDepth<T>, kB = S::BN * kDepth<T>, kSteps = S::kSteps, kSide = S::kSide, kRing = S::kStages;
  constexpr uint32_t kStageBytes = (kA + kB) * sizeof(T);
  static_assert((kSteps == 4 || kSteps == 2) && (kRing & (kRing - 1)) == 0 && kRing >= 2, "what work() goes by");
  T *const buffer = reinterpret_cast<T *>(lds);
  const uint32_t wave = uniform(threadIdx.x / kWave);
  const uint32_t m0 = wave / S::WN * (S::BM / S::WM), n0 = wave % S::WN * (S::BN / S::WN);
  const uint32_t lds_base = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) float4 *)lds)));
  typedef DirectLoader<T, A_ACROSS, S::BM, S::kThreads, S::kLoadBytes, false> LoaderA;
  typedef DirectLoader<T, B_ACROSS, S::BN, S::kThreads, S::kLoadBytes, ONCE> LoaderB;
  constexpr uint32_t kLoads = LoaderA::kLoads + LoaderB::kLoads;
  const size_t a_step = (A_ACROSS ? static_cast<size_t>(a_stride) : 1u) * kDepth<T>;
  const size_t b_step = (B_ACROSS ? static_cast<size_t>(b_stride) : 1u) * kDepth<T>;

  // what is filled: the tile before `filling`, of which `depth_left` of k is left; `filled` and `done` count the stream's stages
  Job<T, O> from;
  LoaderA load_a;
  LoaderB load_b;
  uint32_t filling = 0, depth_left = 0, filled = 0, done = 0;
  bool more = jobs(filling, &from);
  const auto begin = [&] {
    load_a.begin(from.rows, a_stride);
    load_b.begin(from.cols, b_stride);
    depth_left = from.depth;
  };
  if (more) begin();
  const auto load_one = [&](uint32_t i) {
    const uint32_t to = lds_base + (filled & (kRing - 1)) * kStageBytes;
    if (i < LoaderA::kLoads)
      load_a.load(i, from.a, to, wave);
    else
      load_b.load(i - LoaderA::kLoads, from.b, to + kA * static_cast<uint32_t>(sizeof(T)), wave);
  };
  const auto filled_one = [&] {
    from.a += a_step;
    from.b += b_step;
    depth_left -= kDepth<T> < depth_left ? kDepth<T> : depth_left;
    ++filled;
  };
  const auto next_job = [&] {  // the next tile that has anything to fill
    while (more && depth_left == 0) {
      more = jobs(filling, &from);
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
  typename Unit<T, S::kSide>::frag fa[kSteps][S::kFragsM], fb[kSteps][S::kFragsN];
  constexpr uint32_t kReads = S::kFragsM + S::kFragsN, kMuls = S::kFragsM * S::kFragsN;
  const auto read_one = [&](uint32_t stage, uint32_t step, uint32_t i) {
    const T *const at = buffer + (stage & (kRing - 1)) * (kA + kB);
    // (in the order in which the products need them)
    if (i == 0)
      fb[step][0] = fragment<T, B_ACROSS, S::BN, kSide>(at + kA, n0, step);
    else if (i <= S::kFragsM)
      fa[step][i - 1] = fragment<T, A_ACROSS, S::BM, kSide>(at, m0 + (i - 1) * kSide, step);
    else
      fb[step][i - S::kFragsM] = fragment<T, B_ACROSS, S::BN, kSide>(at + kA, n0 + (i - S::kFragsM) * kSide, step);
  };
  // Stage `done`, whose first fragments are held; FILL: there is a whole one to be filled.  `after`: stores that were issued
  // after the loads of the next stage (the counter counts both, in the order in which they were issued).  A partial stage is no
  // load under way; the wait beside its fill is for all of them, so that none older is left where the counts take it for one.
  // Behind the stream's last stage something is read as well, which nothing uses.
  constexpr uint32_t kStores = S::BM / S::WM * (S::BN / S::WN) / kWave / Piece<O>::kElems;  // of a wave's tile
  bool after = false;
  const auto work = [&](auto FILL) {
#pragma unroll
    for (uint32_t step = 0; step < kSteps; ++step) {
      const bool last = step + 1 == kSteps;
      if (step == kSteps / 2) {
        if (!last) __syncthreads();  // every wave holds all of the stage
      }
      if (last) {  // the next stage is there (and, of two steps, every wave holds all of this one)
        constexpr uint32_t kUnderWay = FILL.value ? (kRing - 2) * kLoads + (kSteps == 4 ? kLoads / 2 : 0) : 0;
        if (FILL.value && after)
          wait_for_loads<(kUnderWay + kStores < 63 ? kUnderWay + kStores : kUnderWay)>();
        else
          wait_for_loads<kUnderWay>();
        after = false;
        __syncthreads();
      }
      if (step == kSteps / 2 && !FILL.value && more) fill_partial();
#pragma unroll
      for (uint32_t q = 0; q < kMuls; ++q) {
        const uint32_t i = q % S::kFragsM, j = q / S::kFragsM;
        sum[i][j] = Unit<T, S::kSide>::mul(fb[step][j], fa[step][i], sum[i][j]);
        // of four steps: 1 and 2 are read in 0, 3 in 1, the next stage's 0 in 3; of two: 1 in 0, the next stage's 0 in 1
        const uint32_t reads = kSteps == 4 ? (step == 0 ? 2 * kReads : step == 2 ? 0 : kReads) : kReads;
#pragma unroll
        for (uint32_t r = q * reads / kMuls; r < (q + 1) * reads / kMuls; ++r) {
          if (last)
            read_one(done + 1, 0, r);
          else if (step == 0)
            read_one(done, 1 + r / kReads, r % kReads);
          else
            read_one(done, 3, r);
        }
        if (FILL.value && step >= kSteps / 2) {
          constexpr uint32_t kShare = kLoads / (kSteps / 2);
          static_assert(kLoads % (kSteps / 2) == 0, "an equal share to a step");
#pragma unroll
          for (uint32_t r = q * kShare / kMuls; r < (q + 1) * kShare / kMuls; ++r) load_one((step - kSteps / 2) * kShare + r);
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
    if (depth_left >= kDepth<T>) {
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
  Job<T, O> now;
  for (uint32_t at = 0; jobs(at, &now);) {
    uint32_t left = (now.depth + kDepth<T> - 1) / kDepth<T>;
    while (left != 0) {
      next_job();
      uint32_t turns = depth_left / kDepth<T>;  // stages with a whole one to fill
      turns = turns < left ? turns : left;
      left -= turns;
      for (; turns != 0; --turns) work(std::true_type());
      if (left != 0 && (!more || depth_left != 0)) {
        work(std::false_type());
        --left;
      }
    }
    after = store_tile<T, S, S::kRoom, O>(sum, m0, n0, now.rows, now.cols, now.out, out_stride,
                                       reinterpret_cast<O *>(buffer + kRing * (kA + kB)) + wave * (S::kRoom / sizeof(O)), past);
#pragma unroll
    for (uint32_t i = 0; i < S::kFragsM; ++i)
#pragma unroll
      for (uint32_t j = 0; j < S::kFragsN; ++j) sum[i][j] = typename Unit<T, S::kSide>::acc{};
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

// Tiles are counted in those of `COARSE`.  S = COARSE takes all of them, or, `split` (in workgroups that the card holds at once),
// as many as fill the card a whole number of times, if those left over fill it at most half; a second launch with a smaller S
// then takes the smaller tiles of what is left over, on all of the card.
// Where there are few tiles the inner dimension is split into `parts`: O = float, part after part, and join_kernel adds them.
template <typename T, typename O, bool OUT_MAJOR, typename S, typename COARSE>
__global__ __launch_bounds__(S::kThreads, S::kWavesWanted) void product_kernel(const T *__restrict__ rows, const T *__restrict__ weight,
                                                              const uint32_t *__restrict__ indptr, O *__restrict__ out,
                                                              uint32_t n_rows, uint32_t experts, uint32_t inner,
                                                              uint32_t cols, uint32_t split, uint32_t parts, bool past) {
  constexpr bool kRest = !std::is_same<S, COARSE>::value;
  constexpr uint32_t kDown = COARSE::BM / S::BM, kAcross = COARSE::BN / S::BN;
  extern __shared__ float4 lds[];
  __shared__ TileTable table;
  const uint32_t across = (cols + COARSE::BN - 1) / COARSE::BN;
  const uint32_t total = table.build<S::kThreads>(indptr, experts, n_rows, COARSE::BM);
  const uint64_t tiles = static_cast<uint64_t>(total) * across;
  uint32_t rest = split != 0 ? static_cast<uint32_t>(tiles % split) : 0u;
  if (rest > split / 2) rest = 0;
  const Turn turn = turn_of(kRest ? static_cast<uint64_t>(rest) * (kDown * kAcross) : (tiles - rest) * parts);
  const uint32_t length = parts == 1 ? inner : ((inner + parts - 1) / parts + kDepth<T> - 1) / kDepth<T> * kDepth<T>;
  const auto jobs = [&](uint32_t &at, Job<T, O> *j) {
    for (;;) {
      uint32_t index = turn.index + at * turn.step, in = 0, k0 = 0;
      if (index >= turn.end) return false;
      ++at;
      if (kRest) {
        in = index % (kDown * kAcross);
        index = static_cast<uint32_t>(tiles - rest) + index / (kDown * kAcross);
      }
      uint32_t part = 0;
      if (parts != 1) {  // (whole stages to a part; the last ones may have none)
        part = uniform(index % parts);
        index /= parts;
        k0 = length * part < inner ? length * part : inner;
      }
      const uint32_t down = uniform(index / across);
      const uint32_t col0 = (index - down * across) * COARSE::BN + in % kAcross * S::BN;
      const Tile tile = table.find(indptr, down, experts, n_rows, COARSE::BM);
      const uint32_t first = tile.first + in / kAcross * S::BM;
      if (first >= tile.end || col0 >= cols) continue;  // (a quarter beyond the tile's rows or columns)
      const T *const w = weight + static_cast<size_t>(tile.expert) * inner * cols;
      j->a = uniform(rows + static_cast<size_t>(first) * inner + k0);
      j->b = uniform(OUT_MAJOR ? w + static_cast<size_t>(col0) * inner + k0 : w + static_cast<size_t>(k0) * cols + col0);
      j->out = out + (static_cast<size_t>(part) * n_rows + first) * cols + col0;
      j->rows = tile.end - first < S::BM ? tile.end - first : S::BM;
      j->cols = cols - col0 < S::BN ? cols - col0 : S::BN;
      j->depth = inner - k0 < length ? inner - k0 : length;
      return true;
    }
  };
  // (shapes of few rows are taken where an expert has few: its weights are read once.  403 MB of weights of 64 experts, 8 rows
  // each: 76 -> 67 us out-major, 84 -> 75 us)
  constexpr bool kOnce = S::kLoadBytes == 16 && (S::BM == 16 || (S::BM == 64 && sizeof(T) == 2));
  if constexpr (S::kStages != 0) {
    stream_products<T, O, false, !OUT_MAJOR, S, kOnce>(jobs, inner, OUT_MAJOR ? inner : cols, cols, lds, past);
  } else {
    Job<T, O> j;
    for (uint32_t at = 0; jobs(at, &j);) {
      tile_product<T, false, !OUT_MAJOR, S, O>(j.a, j.rows, inner, j.b, j.cols, OUT_MAJOR ? inner : cols, j.depth, j.out, cols, lds);
      __syncthreads();
    }
  }
  if (kRest || parts != 1) return;
  const uint32_t behind = indptr[experts];
  zero_from(out, behind < n_rows ? behind : n_rows, n_rows, cols, S::kThreads);
}

// d_weight[expert] = left_e^T @ right_e over the expert's rows; (left, right) = (rows, ct), or (ct, rows) where the weight is
// stored out-major.  Where there are few tiles an expert's rows are split into `parts`: O = float, part after part, and
// join_kernel adds them in their order.
template <typename T, typename O, typename S>
__global__ __launch_bounds__(S::kThreads, S::kWavesWanted) void gradient_kernel(const T *__restrict__ left, const T *__restrict__ right,
                                                               const uint32_t *__restrict__ indptr, O *__restrict__ d_weight,
                                                               uint32_t n_rows, uint32_t experts, uint32_t n_left,
                                                               uint32_t n_right, uint32_t parts, bool past) {
  extern __shared__ float4 lds[];
  const uint32_t down = (n_left + S::BM - 1) / S::BM, across = (n_right + S::BN - 1) / S::BN;
  // An eighth of every expert's tiles to an XCD, neighbouring ones: the XCDs' work is the same however long the experts are.
  // Of up to 64 experts the longest come first, so that what ends last is short.
  const uint32_t tiles = down * across, share = (tiles + 7) / 8;
  const uint32_t which = uniform(blockIdx.x / 8 / share), part = which % parts;
  const uint32_t in = (blockIdx.x + which * tiles) % 8 * share + blockIdx.x / 8 % share;
  if (in >= tiles) return;
  uint32_t expert = which / parts;
  if (experts <= kWave) {
    const uint32_t lane = threadIdx.x % kWave;
    const uint2 r = lane < experts ? rows_of(indptr, lane, experts, n_rows) : make_uint2(0, 0);
    const uint32_t length = r.y - r.x;
    uint32_t before = 0;
    for (uint32_t e = 0; e < experts; ++e) {
      const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(length), static_cast<int>(e)));
      before += other > length || (other == length && e < lane) ? 1u : 0u;
    }
    expert = __builtin_ctzll(__ballot(lane < experts && before == expert));
  }
  expert = uniform(expert);
  uint2 range = rows_of(indptr, expert, experts, n_rows);
  if (parts != 1) {  // whole stages to a part
    const uint32_t length = ((range.y - range.x + parts - 1) / parts + kDepth<T> - 1) / kDepth<T> * kDepth<T>;
    const uint64_t from = static_cast<uint64_t>(range.x) + static_cast<uint64_t>(length) * part;
    range.x = from < range.y ? static_cast<uint32_t>(from) : range.y;
    range.y = range.y - range.x < length ? range.y : range.x + length;
  }
  range = make_uint2(uniform(range.x), uniform(range.y));
  const uint32_t p0 = uniform(in / across) * S::BM, q0 = uniform(in % across) * S::BN;
  const auto jobs = [&](uint32_t &at, Job<T, O> *j) {
    if (at++ != 0) return false;
    j->a = uniform(left + static_cast<size_t>(range.x) * n_left + p0);
    j->b = uniform(right + static_cast<size_t>(range.x) * n_right + q0);
    j->out = d_weight + ((static_cast<size_t>(part) * experts + expert) * n_left + p0) * n_right + q0;
    j->rows = n_left - p0 < S::BM ? n_left - p0 : S::BM;
    j->cols = n_right - q0 < S::BN ? n_right - q0 : S::BN;
    j->depth = range.y - range.x;
    return true;
  };
  if constexpr (S::kStages != 0) {
    stream_products<T, O, true, true, S, false>(jobs, n_left, n_right, n_right, lds, past);
  } else {
    Job<T, O> j;
    for (uint32_t at = 0; jobs(at, &j);) {
      tile_product<T, true, true, S, O>(j.a, j.rows, n_left, j.b, j.cols, n_right, j.depth, j.out, n_right, lds);
      __syncthreads();
    }
  }
}

// indptr: rows of `cols` from indptr[experts] on are zero, and have no parts; nullptr: there are none such.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ parts, T *__restrict__ out, size_t n, uint32_t count,
                                                   const uint32_t *__restrict__ indptr, uint32_t experts, uint32_t cols) {
  const size_t there = indptr != nullptr ? static_cast<size_t>(indptr[experts]) * cols : n;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * 256) {
    float sum = 0.f;
    if (i < there) {
#pragma unroll 8
      for (uint32_t p = 0; p < count; ++p) sum += parts[p * n + i];
    }
    out[i] = static_cast<T>(sum);
  }
}

bool refuse_tiles(const char *target, uint64_t tiles, uint64_t most) {
  if (tiles < most) return false;
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

// Loads of so many bytes that go straight to LDS need lines at multiples of them, and offsets within a tile in 32 bits.
template <typename T>
bool straight(const void *p, uint32_t stride, uint32_t bytes = 16) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * sizeof(T) % bytes == 0 && stride < (1u << 20);
}

// Results of 64 MB and more in whole lines are stored past the caches (32,768 rows, 8 experts of 2,048 x 2,048, bfloat16: 262 ->
// 241 us out-major, 248 -> 229 us; the gradient of such weights 240 -> 232).
bool past_caches(const void *out, uint64_t rows, uint32_t cols, uint32_t element_bytes) {
  const uint64_t line = static_cast<uint64_t>(cols) * element_bytes;
  return rows * line >= 64ull << 20 && line % 128 == 0 && reinterpret_cast<uintptr_t>(out) % 128 == 0;
}

// Shapes for operands in whole pieces, and for others
struct Direct {
  using Large = Shape<256, 256, 2, 2, 32, 2>;
  using Middle = Shape<128, 128, 2, 2, 32, 2>;
  using Small = Shape<64, 64, 2, 2, 32, 4>;
};
// In 32 bits: the matrix unit takes longer than loads do, and a third workgroup on a CU is worth more than two stages.
struct Direct32 {
  using Middle = Shape<128, 128, 2, 2, 32, 2>;
  using Small = Shape<64, 64, 2, 2, 32, 2>;
  using Thin = Shape<16, 64, 1, 2, 16, 4>;
};
// The same for lines that begin at any element: four loads for one.
struct DirectWords {
  using Middle = Shape<128, 128, 2, 2, 32, 2, 4>;
  using Small = Shape<64, 64, 2, 2, 32, 2, 4>;
  using Thin = Shape<16, 64, 1, 2, 16, 4, 4>;
};
template <typename T>
using DirectOf = std::conditional_t<sizeof(T) == 4, Direct32, Direct>;
struct Staged {
  using Large = Shape<256, 256, 2, 4, 32, 0>;
  using Middle = Shape<128, 128, 2, 2, 32, 0>;
  using Small = Shape<64, 64, 2, 2, 32, 0>;
  using Thin = Shape<16, 64, 1, 2, 16, 0>;
};

template <typename T>
bool join(const char *target, hipStream_t stream, const void *parts, void *out, size_t n, uint32_t count, const void *indptr,
          uint32_t experts, uint32_t cols) {
  hipLaunchKernelGGL(join_kernel<T>, dim3(div_up(n, 256) < 4096 ? div_up(n, 256) : 4096), dim3(256), 0, stream,
                     static_cast<const float *>(parts), static_cast<T *>(out), n, count, static_cast<const uint32_t *>(indptr),
                     experts, cols);
  return check_launch(target);
}

// A product as it is launched.  split: what is left over of COARSE's tiles, when they have filled the card, is for S.
template <typename O>
struct Product {
  const bpl_expert_descriptor &d;
  void **buffers;
  O *out;
  uint32_t parts;
  bool split;
};
template <typename T, typename S, typename COARSE = S, typename O>
bool launch_product(const char *target, hipStream_t stream, const Product<O> &p) {
  const bpl_expert_descriptor &d = p.d;
  constexpr uint32_t kDown = COARSE::BM / S::BM * (COARSE::BN / S::BN);
  const uint64_t tiles = most_tiles(d.rows, d.experts, COARSE::BM) * div_up(d.out, COARSE::BN) * kDown * p.parts;
  if (refuse_tiles(target, tiles, 1ull << 31)) return false;
  // one workgroup to each place that the LDS leaves
  const auto held = [](uint32_t lds_bytes) {
    return static_cast<uint32_t>(device_info().num_cu) * (160u * 1024u / (lds_bytes + static_cast<uint32_t>(sizeof(TileTable)) + 1024u));
  };
  const uint64_t places = held(S::kLdsBytes);
  const unsigned grid = static_cast<unsigned>(((tiles < places ? tiles : places) + 7) / 8 * 8);
  const auto launch = [&](auto *kernel) {
    if (!allow_lds(target, kernel, S::kLdsBytes)) return false;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::kThreads), S::kLdsBytes, stream, static_cast<const T *>(p.buffers[0]),
                       static_cast<const T *>(p.buffers[1]), static_cast<const uint32_t *>(p.buffers[2]), p.out, d.rows,
                       d.experts, d.width, d.out, p.split ? held(COARSE::kLdsBytes) : 0u, p.parts,
                       past_caches(p.out, d.rows, d.out, sizeof(O)));
    return check_launch(target);
  };
  return d.flags & BPL_EXPERT_OUT_MAJOR ? launch(product_kernel<T, O, true, S, COARSE>) : launch(product_kernel<T, O, false, S, COARSE>);
}

// Which shape: the least time by the turns in which the card, full of them, works through a shape's tiles.  A turn's time, in us:
// `fixed` and, for 2,048 of the inner dimension (in the gradient: of rows to an expert), `deep`; the large shape has one
// workgroup to a CU, so that nothing goes on there while a tile begins and ends, and spilled registers hold up its results (the
// results' 33 MB of a turn take 7 of the 24 us).  `alone`: of a turn that leaves every CU at most
// one workgroup where two could share it; of a fuller one the share that its tiles have.
// Fitted to 528 products in 16 bits (32 and 128 experts, inner dimensions of 1,024 to 8,192, 768 to 2,048 columns, both
// storages, 4 to 800 rows to an expert) and 144 gradients (8 to 128 experts, 16 to 4,096 rows to one), every shape timed at each:
// the chosen one takes less than 1 % longer than the best on average (5 % and up to 1.67 times, with a time by turns alone), at
// most 1.28 times, where experts' last tiles fill up a turn or do not.  Times of large / middle / small: 128 experts of 448 rows, 8,192 x 1,536, bfloat16, in-major 1,580 / 2,436; 32 experts of
// 320 rows, 1,024 x 768 51 / 30; of 16 rows, 2,048 x 1,536 119 / 86 / 78 (64 experts).
// In 32 bits 356 products (7 to 128 experts, 512 to 4,096 x 512 to 1,536, both storages, odd ones, 2 to 700 rows): half a percent
// over the best on average, at most 1.2 times (4 % and 1.75 by turns alone); 168 gradients by turns alone, 2 % and 1.14.
// Middle / small / thin: 128 experts of 32 rows, 2,048 x 1,536 729 / 440 / 677, 7 of 8, 1,024 x 1,024 67 / 23 / 16.
enum Form { kLarge, kMiddle, kSmall, kThin };
struct FormTime {
  Form form;
  uint32_t height, width, share;  // share: workgroups that share a CU
  float fixed, deep, alone;
};
constexpr FormTime kProduct16[] = {
    {kLarge, 256, 256, 1, 24.f, 46.f, 1.f}, {kMiddle, 128, 128, 2, 0.f, 40.f, 0.6f}, {kSmall, 64, 64, 2, 2.f, 17.f, 0.6f}};
// (staged through registers: 240 products, 2.5 % over the best on average and at most 1.39 times, 4.7 % and 1.5 by kProduct16)
constexpr FormTime kStaged16[] = {
    {kLarge, 256, 256, 1, 0.f, 100.f, 1.f}, {kMiddle, 128, 128, 2, 0.f, 70.f, 0.75f}, {kSmall, 64, 64, 2, 0.f, 26.f, 0.75f}};
constexpr FormTime kGradient16[] = {
    {kLarge, 256, 256, 1, 8.f, 42.f, 1.f}, {kMiddle, 128, 128, 2, 0.f, 42.f, 1.f}, {kSmall, 64, 64, 2, 1.f, 17.f, 1.f}};
constexpr FormTime kProduct32[] = {
    {kMiddle, 128, 128, 2, 8.f, 244.f, 0.75f}, {kSmall, 64, 64, 2, 2.f, 68.f, 0.75f}, {kThin, 16, 64, 3, 0.f, 66.f, 0.75f}};
constexpr FormTime kGradient32[] = {
    {kMiddle, 128, 128, 2, 0.f, 244.f, 1.f}, {kSmall, 64, 64, 2, 0.f, 68.f, 1.f}, {kThin, 16, 64, 3, 0.f, 68.f, 1.f}};
template <typename TILES>
Form best_form(const FormTime (&forms)[3], uint32_t depth, bool split, TILES tiles) {
  const uint64_t cus = device_info().num_cu;
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < 3; ++i) {
    const uint64_t n = tiles(forms[i].height, forms[i].width), held = cus * forms[i].share, rest = n % held;
    float turns = static_cast<float>(n / held);
    if (rest != 0) {
      const float full = static_cast<float>(rest) / static_cast<float>(held);
      turns += full <= 0.5f ? forms[i].alone : forms[i].alone + (1.f - forms[i].alone) * (2.f * full - 1.f);
    }
    if (split && forms[i].form == kLarge && rest != 0 && rest <= held / 4) turns -= 0.35f;
    const float time = (forms[i].fixed + forms[i].deep * static_cast<float>(depth) / 2048.f) * turns;
    if (i == 0 || time < least) best = i, least = time;
  }
  return forms[best].form;
}

// Whether tiles left over by the large ones are worth a second launch: one takes a whole turn of the card, 60 us at an inner
// dimension of 2,048, in quarters 20 to 40; below 512 of it the launch costs what that saves, and of experts of fewer rows the
// quarters are half empty.
bool worth_quarters(const bpl_expert_descriptor &d) { return d.width >= 512 && d.rows / d.experts >= 512; }

// (an expert's last tile is half full on average, and every expert that has rows has one)
uint64_t likely_tiles(const bpl_expert_descriptor &d, uint32_t height, uint32_t width) {
  const uint64_t met = d.experts < d.rows ? d.experts : d.rows, full = d.rows / height + met / 2;
  return (full > met ? full : met) * div_up(d.out, width);
}

Form product_form(uint32_t element_bytes, bool staged, const bpl_expert_descriptor &d) {
  return best_form(element_bytes == 4 ? kProduct32 : staged ? kStaged16 : kProduct16, d.width, worth_quarters(d),
                   [&](uint32_t height, uint32_t width) { return likely_tiles(d, height, width); });
}

// Into how many parts the inner dimension is split where the tiles leave places on the card free, at least 512 of it to a
// part: where that spares 4 us and the 4 us of the launch that adds them up.  A workgroup's stages come one after the other,
// 0.25 us each in 16 bits and 0.35 in 32, and the weights at 5 TB/s.  (One row, 4,096 x 64, bfloat16 19 -> 8 + 4 us; two rows on
// two experts of 2,048 x 1,024, float32 29 -> 13 + 4, bfloat16 11.3 and left as it is, where it would be 7.7 + 4.)
uint32_t product_parts(uint32_t element_bytes, const bpl_expert_descriptor &d) {
  const Form form = product_form(element_bytes, false, d);
  if (form != kSmall && form != kThin) return 1;
  const uint32_t height = form == kSmall ? 64 : 16, share = form == kSmall && element_bytes == 2 ? 2 : 3;
  const uint64_t met = d.experts < d.rows ? d.experts : d.rows;
  uint64_t parts = static_cast<uint64_t>(share) * device_info().num_cu / likely_tiles(d, height, 64);
  if (parts > d.width / 512) parts = d.width / 512;
  if (parts > 16) parts = 16;
  if (parts < 2) return 1;
  const float whole = (element_bytes == 2 ? 0.25f : 0.35f) * static_cast<float>(d.width / (kDepthBytes / element_bytes));
  const float bytes = static_cast<float>(met) * static_cast<float>(d.width) * static_cast<float>(d.out) *
                      static_cast<float>(element_bytes) / 5e6f;
  // (us, both)
  const float split = whole / static_cast<float>(parts) > bytes ? whole / static_cast<float>(parts) : bytes;
  return whole - split < 8.f ? 1u : static_cast<uint32_t>(parts);
}

template <typename T, typename SHAPES, typename O>
bool choose_product(const char *target, hipStream_t stream, Product<O> p) {
  Form form = product_form(sizeof(T), std::is_same<SHAPES, Staged>::value, p.d);
  p.split = false;
  if (p.parts != 1 && form != kThin) form = kSmall;
  if constexpr (sizeof(T) == 2 && std::is_same<T, O>::value) {
    if (form == kLarge) {
      p.split = worth_quarters(p.d);
      return launch_product<T, typename SHAPES::Large>(target, stream, p) &&
             (!p.split || launch_product<T, typename SHAPES::Middle, typename SHAPES::Large>(target, stream, p));
    }
  }
  if constexpr (sizeof(T) == 4) {
    if (form == kThin) return launch_product<T, typename SHAPES::Thin>(target, stream, p);
  }
  if constexpr (std::is_same<T, O>::value) {
    if (form == kMiddle) return launch_product<T, typename SHAPES::Middle>(target, stream, p);
  }
  return launch_product<T, typename SHAPES::Small>(target, stream, p);
}

template <typename T>
void matmul(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.rows == 0 || d.out == 0) return;
  const uint32_t stride = d.flags & BPL_EXPERT_OUT_MAJOR ? d.width : d.out, parts = d.per_token < 1 ? 1u : d.per_token;
  const auto run = [&](auto *out) {
    const Product<std::remove_pointer_t<decltype(out)>> p{d, buffers, out, parts, false};
    if (straight<T>(buffers[0], d.width) && straight<T>(buffers[1], stride)) return choose_product<T, DirectOf<T>>(target, stream, p);
    if constexpr (sizeof(T) == 4) {
      if (straight<T>(buffers[0], d.width, 4) && straight<T>(buffers[1], stride, 4))
        return choose_product<T, DirectWords>(target, stream, p);
    }
    return choose_product<T, Staged>(target, stream, p);
  };
  if (parts == 1)
    run(static_cast<T *>(buffers[3]));
  else if (run(static_cast<float *>(buffers[4])))
    join<T>(target, stream, buffers[4], buffers[3], static_cast<size_t>(d.rows) * d.out, parts, buffers[2], d.experts, d.out);
}

// The gradient's shape, and into how many parts an expert's rows are split where the tiles leave places on the card free: at
// least 512 rows to a part on average (2 experts of 16,384 rows, 64 x 64 results: 58 us, in 32 parts 7 and 3.4 for their sum).
// How many parts there are is the caller's, who brings the room for them; the shape is chosen here.
struct GradientPlan {
  Form form;
  uint32_t parts;
};
GradientPlan gradient_plan(uint32_t element_bytes, uint32_t rows, uint32_t experts, uint32_t inner, uint32_t out) {
  const auto tiles = [&](uint32_t height, uint32_t width) {
    return static_cast<uint64_t>(experts) * div_up(inner, height) * div_up(out, width);
  };
  GradientPlan p;
  const uint32_t mean = rows / experts;  // (a tile of few rows begins and ends as well)
  p.form = best_form(element_bytes == 2 ? kGradient16 : kGradient32, mean < 64 ? 64 : mean, false, tiles);
  if (p.form == kThin) p.form = kSmall;
  const uint32_t side = p.form == kLarge ? 256 : p.form == kMiddle ? 128 : 64;
  const uint64_t free = 2ull * device_info().num_cu / tiles(side, side), most = rows / experts / 512;
  const uint64_t parts = free < most ? free : most;
  p.parts = parts < 1 || p.form == kLarge ? 1u : parts < kMostPerToken ? static_cast<uint32_t>(parts) : kMostPerToken;
  return p;
}

template <typename T, typename O, typename S>
bool launch_gradient(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, const void *left, const void *right,
                     uint32_t n_left, uint32_t n_right, const void *indptr, O *out, uint32_t parts) {
  const uint64_t blocks = 8 * ((static_cast<uint64_t>(div_up(n_left, S::BM)) * div_up(n_right, S::BN) + 7) / 8) * d.experts * parts;
  // (threads of a launch are counted in 32 bits)
  if (refuse_tiles(target, blocks, (1ull << 32) / S::kThreads) || !allow_lds(target, gradient_kernel<T, O, S>, S::kLdsBytes)) return false;
  hipLaunchKernelGGL((gradient_kernel<T, O, S>), dim3(static_cast<unsigned>(blocks)), dim3(S::kThreads), S::kLdsBytes, stream,
                     static_cast<const T *>(left), static_cast<const T *>(right), static_cast<const uint32_t *>(indptr), out,
                     d.rows, d.experts, n_left, n_right, parts,
                     past_caches(out, static_cast<uint64_t>(d.experts) * n_left * parts, n_right, sizeof(O)));
  return check_launch(target);
}

template <typename T, typename O, typename SHAPES>
bool choose_gradient(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, const void *left, const void *right,
                     uint32_t n_left, uint32_t n_right, const void *indptr, O *out, const GradientPlan &plan) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, O>::value) {
    if (plan.form == kLarge)
      return launch_gradient<T, O, typename SHAPES::Large>(target, stream, d, left, right, n_left, n_right, indptr, out, plan.parts);
  }
  if (plan.form == kMiddle)
    return launch_gradient<T, O, typename SHAPES::Middle>(target, stream, d, left, right, n_left, n_right, indptr, out, plan.parts);
  return launch_gradient<T, O, typename SHAPES::Small>(target, stream, d, left, right, n_left, n_right, indptr, out, plan.parts);
}

template <typename T>
void matmul_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  if (d.width == 0 || d.out == 0) return;
  const bool out_major = (d.flags & BPL_EXPERT_OUT_MAJOR) != 0;
  const uint32_t n_left = out_major ? d.out : d.width, n_right = out_major ? d.width : d.out;
  const void *const left = buffers[out_major ? 1 : 0], *const right = buffers[out_major ? 0 : 1];
  GradientPlan plan = gradient_plan(sizeof(T), d.rows, d.experts, d.width, d.out);
  plan.parts = d.per_token < 1 ? 1u : d.per_token;
  if (plan.parts != 1 && plan.form == kLarge) plan.form = kMiddle;
  const auto run = [&](auto *out) {
    typedef std::remove_pointer_t<decltype(out)> O;
    if (straight<T>(left, n_left) && straight<T>(right, n_right))
      return choose_gradient<T, O, DirectOf<T>>(target, stream, d, left, right, n_left, n_right, buffers[2], out, plan);
    if constexpr (sizeof(T) == 4) {
      if (straight<T>(left, n_left, 4) && straight<T>(right, n_right, 4))
        return choose_gradient<T, O, DirectWords>(target, stream, d, left, right, n_left, n_right, buffers[2], out, plan);
    }
    return choose_gradient<T, O, Staged>(target, stream, d, left, right, n_left, n_right, buffers[2], out, plan);
  };
  if (plan.parts == 1) {
    run(static_cast<T *>(buffers[3]));
    return;
  }
  if (!run(static_cast<float *>(buffers[4]))) return;
  join<T>(target, stream, buffers[4], buffers[3], static_cast<size_t>(d.experts) * n_left * n_right, plan.parts, nullptr, 0, 0);
}

}  // namespace

extern "C" {

uint32_t bpl_expert_matmul_parts(uint32_t rows, uint32_t experts, uint32_t width, uint32_t out_width, uint32_t element_bytes) {
  if (rows == 0 || experts == 0 || width == 0 || out_width == 0) return 1;
  return product_parts(element_bytes, bpl_expert_descriptor{0, 0, experts, rows, width, out_width, 0});
}
uint32_t bpl_expert_matmul_gradient_parts(uint32_t rows, uint32_t experts, uint32_t width, uint32_t out_width,
                                          uint32_t element_bytes) {
  if (experts == 0 || width == 0 || out_width == 0) return 1;
  return gradient_plan(element_bytes, rows, experts, width, out_width).parts;
}

BPL_EXPERT_DEFINE(expert_matmul, matmul)
BPL_EXPERT_DEFINE(expert_matmul_gradient, matmul_gradient)

}  // extern "C"
