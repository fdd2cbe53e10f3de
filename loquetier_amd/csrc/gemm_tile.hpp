// The product of two 16-bit matrices, a tile of 256 x 256 (or 256 x 64) sums a workgroup of four waves, for the loss over the
// vocabulary: D[a, b] = sum_k A[a, k] B[b, k], sums in float.
//
// Bound by the matrix cores where there are rows enough, so the tile is as large as the registers: a wave holds 128 x 128 sums (256
// registers) and reads 16 KB of operands out of LDS for each 1024 cycles of products (32 of k), half of what LDS gives; eight waves
// of 128 x 64 would read all of it.  Two stages of 64 of k lie in LDS: one is multiplied while the other's loads, straight to LDS
// and a row's whole line at a time, are on their way; operands of the next 16 of k are read while those at hand are multiplied;
// one barrier a stage.  (Four stages of 32, half lines: 1.18 PFLOP/s for 1.23 at 32000 x 4096 x 4096, whatever the loads' lead; the L2
// serves a half line as slowly as a whole one.)
// With one wave a SIMD nothing hides what the wave does besides: a product takes 32 cycles, and five or six other instructions
// cost as many.  So the loop holds products, reads, loads and their LDS addresses, and little else: lanes' offsets stay, k moves in a
// scalar, and the ends of k go through a second form of the loads.
// 32 x 32 x 16 products: fewer register reads an operation than 16 x 16 x 32, and the card's power is the bound of long products.
//
// An operand lies in memory either with k next to each other (rows of the tile are rows in memory) or with its tile dimension
// next to each other ("across": a row in memory is one k).  The first goes through LDS as rows of 64 of k, 16-byte pieces turned by the
// row's number so that the reads of sixteen neighbouring rows meet all banks.  The second goes as it lies: a lane reads four (two)
// neighbouring columns of each k and joins pairs of k with byte permutes, so its columns belong to the wave's four (two) blocks: block i
// has the columns 4 m + i.  (The transposing read of LDS takes four times as long a byte: 256 x 256 x 16384 by one workgroup, both
// operands across, 528 us with it, 246 plain.)
//
// Loads go through a buffer resource: what lies past the matrix, or past the end of k, has an offset past the resource's end and
// is zeros.
#pragma once
#include <type_traits>

#include "smlm_common.hpp"

namespace smlm {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGemmK = 64;                  // of k a stage: a row's whole line of 128 bytes
constexpr int kGemmStages = 2;
constexpr uint32_t kGemmFar = 0xf8000000u;  // an offset past every resource's end
constexpr uint32_t kGemmSpan = 0xf0000000u;

template <int DT>
__device__ __forceinline__ f32x16 gemm_mfma(u32x4 a, u32x4 b, f32x16 c) {
  if (DT == SMLM_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A matrix operand: `rows` rows in memory of `ld` elements (a multiple of 8; 256 of them lie within 2^32 bytes).
struct GemmOperand {
  const uint16_t* base;
  int64_t ld;
  int64_t rows;
};

// The tile's side of an operand in LDS: ROWS rows of kGemmK (plain), or kGemmK rows of ROWS (across).
template <int ROWS, bool ACROSS>
struct GemmSide {
  static constexpr int kElems = ROWS * kGemmK;
  static constexpr int kLoads = ROWS / 32;                // a wave's loads of 1 KB a stage
  static constexpr int kLanes = ACROSS ? ROWS / 8 : 8;    // of a row in LDS
  uint32_t off[kLoads];                                   // a lane's bytes from the stage's first element
  const uint16_t* at;                                     // that element
  uint32_t span, step;                                    // bytes of the resource, from stage to stage

  static __device__ __forceinline__ int place(int row, int piece) {
    return ACROSS ? row * ROWS + piece * 8 : row * kGemmK + ((piece ^ ((row >> 1) & 7)) << 3);
  }
  static __device__ __forceinline__ int load_row(int i, int wave, int lane) {
    return (wave * kLoads + i) * (64 / kLanes) + lane / kLanes;
  }
  // (the turn undoes itself: the piece that belongs into the lane's place)
  static __device__ __forceinline__ int load_piece(int row, int lane) {
    return (place(row, lane % kLanes) - row * (ACROSS ? ROWS : kGemmK)) >> 3;
  }
  // first: the tile's first row (plain) or column; k0: where k starts
  __device__ __forceinline__ void start(const GemmOperand& m, int64_t first, int k0, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = load_row(i, wave, lane), piece = load_piece(row, lane);
      off[i] = (uint32_t)row * (uint32_t)(m.ld * 2) + (uint32_t)piece * 16u;
      if (ACROSS && first + piece * 8 >= m.ld) off[i] = kGemmFar;
    }
    const int64_t left = m.rows - first;  // (plain; the others' rows are k)
    span = ACROSS ? kGemmSpan : left < ROWS ? (uint32_t)(left < 0 ? 0 : left) * (uint32_t)(m.ld * 2) : kGemmSpan;
    at = m.base + (ACROSS ? (int64_t)k0 * m.ld + first : first * m.ld + k0);
    step = ACROSS ? (uint32_t)(kGemmK * m.ld * 2) : kGemmK * 2;
  }
  __device__ __forceinline__ void load(uint16_t* lds, int ahead, int wave) const {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), 0, span, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + (wave * kLoads + i) * 512), 16,
                                               off[i], ahead * step, 0, 0);
  }
  // The same where k ends: k_left of it from that stage on.
  __device__ __forceinline__ void load_end(uint16_t* lds, int ahead, int k_left, int wave, int lane) const {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), 0, span, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = load_row(i, wave, lane), k = ACROSS ? row : load_piece(row, lane) * 8;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + (wave * kLoads + i) * 512), 16,
                                               k < k_left ? off[i] : kGemmFar, k_left > 0 ? ahead * step : 0, 0, 0);
    }
  }
  __device__ __forceinline__ void advance(int stages) {
    at = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(at) + (uint64_t)stages * step);
  }
};

// A wave's operands of 16 of k, BLOCKS blocks of 32 rows: as they come from LDS, and as the products take them.
template <int ROWS, bool ACROSS, int BLOCKS>
struct GemmReader;

template <int ROWS, int BLOCKS>
struct GemmReader<ROWS, false, BLOCKS> {
  static constexpr int kReads = BLOCKS, kTurns = 0;
  struct Raw {
    u32x4 of[BLOCKS];
  };
  int at[kGemmK / 16];  // a lane's place in each step (blocks are constants apart)
  __device__ __forceinline__ void start(int first, int lane) {  // first: row of the tile of the wave's first block
#pragma unroll
    for (int s = 0; s < kGemmK / 16; ++s) at[s] = GemmSide<ROWS, false>::place(first + (lane & 31), s * 2 + (lane >> 5));
  }
  __device__ __forceinline__ void read(const uint16_t* lds, int s, Raw& r) const {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) r.of[b] = *(const u32x4*)(lds + at[s] + b * 32 * kGemmK);
  }
  static __device__ __forceinline__ u32x4 block(const Raw& r, int b) { return r.of[b]; }
};

template <int ROWS, int BLOCKS>
struct GemmReader<ROWS, true, BLOCKS> {
  static_assert(BLOCKS == 2 || BLOCKS == 4, "");
  static constexpr int kReads = 8, kTurns = 4 * BLOCKS;
  typedef uint32_t words __attribute__((ext_vector_type(BLOCKS / 2)));
  struct Raw {
    words of[8];  // columns of each k
  };
  int at;
  __device__ __forceinline__ void start(int first, int lane) { at = (lane >> 5) * 8 * ROWS + first + (lane & 31) * BLOCKS; }
  __device__ __forceinline__ void read(const uint16_t* lds, int s, Raw& r) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) r.of[k] = *(const words*)(lds + at + (s * 16 + k) * ROWS);
  }
  static __device__ __forceinline__ u32x4 block(const Raw& r, int b) {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = __builtin_amdgcn_perm(r.of[2 * e + 1][b >> 1], r.of[2 * e][b >> 1], b & 1 ? 0x07060302u : 0x05040100u);
    return o;
  }
};

// WA x WB waves of IA x JB blocks of 32 x 32.
template <int WA, int IA, bool XA, int WB, int JB, bool XB>
struct GemmShape {
  static constexpr int kA = WA * IA * 32, kB = WB * JB * 32;
  static constexpr int kStage = (kA + kB) * kGemmK;  // elements of LDS
};

// The order of a step: ITEMS reads and loads, the reads first, and TURNS permutes of what was read before, shared out over PRODUCTS
// products; the first blocks' permutes come before the first of them.
template <int I, int READS, int ITEMS, int TURNS, int PRODUCTS>
__device__ __forceinline__ void gemm_order() {
  if constexpr (I < PRODUCTS) {
    constexpr int from = I * ITEMS / PRODUCTS, to = (I + 1) * ITEMS / PRODUCTS;
    constexpr int reads = (to < READS ? to : READS) - (from < READS ? from : READS), loads = to - from - reads;
    constexpr int turns = I == 0 ? (TURNS + 3) / 4 : (TURNS * 3 / 4 * I / (PRODUCTS - 1)) - (TURNS * 3 / 4 * (I - 1) / (PRODUCTS - 1));
    if constexpr (turns > 0) __builtin_amdgcn_sched_group_barrier(0x2, turns, 0);
    if constexpr (reads > 0) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if constexpr (loads > 0) __builtin_amdgcn_sched_group_barrier(0x10, loads, 0);
    gemm_order<I + 1, READS, ITEMS, TURNS, PRODUCTS>();
  }
}

// Row m of the wave's block i of an operand: the tile's row (or column, across) from the wave's first on.
template <bool ACROSS, int BLOCKS>
__device__ __forceinline__ constexpr int gemm_row(int i, int m) {
  return ACROSS ? BLOCKS * m + i : 32 * i + m;
}
// Row m (of A) in a block that a lane's sum e belongs to; its column (of B) is the lane's number modulo 32.
__device__ __forceinline__ int gemm_sum_row(int e, int lane) { return 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }

// acc[i][j] += the tile's sums over k in [k0, k1).  lds: kGemmStages * kStage elements.
template <int DT, int WA, int IA, bool XA, int WB, int JB, bool XB>
struct GemmTile {
  static __device__ __forceinline__ void run(f32x16 (&acc)[IA][JB], uint16_t* lds, const GemmOperand& ma, int64_t a0,
                                             const GemmOperand& mb, int64_t b0, int k0, int k1) {
    typedef GemmShape<WA, IA, XA, WB, JB, XB> S;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    GemmSide<S::kA, XA> sa;
    GemmSide<S::kB, XB> sb;
    sa.start(ma, a0, k0, wave, lane);
    sb.start(mb, b0, k0, wave, lane);
    typedef GemmReader<S::kA, XA, IA> RA;
    typedef GemmReader<S::kB, XB, JB> RB;
    RA ra;
    RB rb;
    ra.start((wave / WB) * IA * 32, lane);
    rb.start((wave % WB) * JB * 32, lane);
    typename RA::Raw fa[2];
    typename RB::Raw fb[2];
    auto read = [&](int slot, int s, int to) {
      const uint16_t* st = lds + slot * S::kStage;
      ra.read(st, s, fa[to]);
      rb.read(st + S::kA * kGemmK, s, fb[to]);
    };
    auto multiply = [&](int from) {
      u32x4 b[JB];
#pragma unroll
      for (int j = 0; j < JB; ++j) b[j] = RB::block(fb[from], j);
#pragma unroll
      for (int i = 0; i < IA; ++i) {
        const u32x4 a = RA::block(fa[from], i);
#pragma unroll
        for (int j = 0; j < JB; ++j) acc[i][j] = gemm_mfma<DT>(a, b[j], acc[i][j]);
      }
    };
    constexpr int kLoadsA = GemmSide<S::kA, XA>::kLoads, kLoadsB = GemmSide<S::kB, XB>::kLoads;
    constexpr int kLanded = 0x0070;  // s_waitcnt vmcnt(0) lgkmcnt(0): a barrier waits for neither by itself
    __syncthreads();  // (whoever used the LDS before is done)
    if (k0 >= k1) return;
    int left = k1 - k0;  // of k, from the stage that is multiplied next on
    auto load_a = [&](auto end, int slot, int ahead) {
      uint16_t* to = lds + slot * S::kStage;
      if constexpr (decltype(end)::value) sa.load_end(to, ahead, left - ahead * kGemmK, wave, lane);
      else sa.load(to, ahead, wave);
    };
    auto load_b = [&](auto end, int slot, int ahead) {
      uint16_t* to = lds + slot * S::kStage + S::kA * kGemmK;
      if constexpr (decltype(end)::value) sb.load_end(to, ahead, left - ahead * kGemmK, wave, lane);
      else sb.load(to, ahead, wave);
    };
    load_a(std::true_type{}, 0, 0);
    load_b(std::true_type{}, 0, 0);
    __builtin_amdgcn_s_waitcnt(kLanded);
    asm volatile("s_barrier" ::: "memory");
    load_a(std::true_type{}, 1, 1);
    read(0, 0, 0);
    // One read of the next step's operands, and then one load, between two products: left to itself the compiler has each product wait for
    // a read, and a wave that gives all its loads at once waits for the address unit with the matrix core idle.  (Loads come after the
    // reads: the compiler takes a load to LDS to be a write that a read might meet, and keeps their order.)
    constexpr int kReads = RA::kReads + RB::kReads, kTurns = RA::kTurns + RB::kTurns, kProducts = IA * JB;
    auto stage = [&](auto end, auto slot_, int ahead) {
      constexpr int slot = decltype(slot_)::value;
      read(slot, 1, 1);
      load_b(end, slot ^ 1, ahead + 1);
      multiply(0);
      gemm_order<0, kReads, kReads + kLoadsB, kTurns, kProducts>();
      read(slot, 2, 0);
      multiply(1);
      gemm_order<0, kReads, kReads, kTurns, kProducts>();
      read(slot, 3, 1);
      multiply(0);
      gemm_order<0, kReads, kReads, kTurns, kProducts>();
      __builtin_amdgcn_s_waitcnt(kLanded);
      asm volatile("s_barrier" ::: "memory");  // the next stage has landed, and everybody has read this one
      read(slot ^ 1, 0, 0);
      load_a(end, slot, ahead + 2);
      multiply(1);
      gemm_order<0, kReads, kReads + kLoadsA, kTurns, kProducts>();
    };
    typedef std::integral_constant<int, 0> zero;
    typedef std::integral_constant<int, 1> one;
    auto next = [&] {
      sa.advance(2);
      sb.advance(2);
      left -= 2 * kGemmK;
    };
#pragma unroll 1
    for (; left >= 4 * kGemmK; next()) {
      stage(std::false_type{}, zero{}, 0);
      stage(std::false_type{}, one{}, 1);
    }
#pragma unroll 1
    for (; left > 0; next()) {
      stage(std::true_type{}, zero{}, 0);
      if (left > kGemmK) stage(std::true_type{}, one{}, 1);
    }
  }
};

}  // namespace smlm
