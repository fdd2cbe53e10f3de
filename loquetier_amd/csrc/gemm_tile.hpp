// The product of two 16-bit matrices, a tile of 256 x 256 (or 256 x 64) sums a workgroup of four waves, for the loss over the
// vocabulary: D[a, b] = sum_k A[a, k] B[b, k], sums in float.
//
// Bound by the matrix cores where there are rows enough, so the tile is as large as the registers: a wave holds 128 x 128 sums (256
// registers) and reads 16 KB of operands out of LDS for each 1024 cycles of products (32 of k), half of what LDS gives; eight waves
// of 128 x 64 would read all of it.  Two stages of 64 of k in LDS, 128 KB: one is multiplied while the other's loads, straight to
// LDS, are on their way; operands of the next 16 of k are read while those at hand are multiplied; one barrier for 64 of k.
// 32 x 32 x 16 products: fewer register reads an operation than 16 x 16 x 32, and the card's power is the bound of long products.
//
// An operand lies in memory either with k next to each other (rows of the tile are rows in memory) or with its tile dimension
// next to each other ("across": a row in memory is one k).  The first goes through LDS as rows of 64 of k, the second as it lies,
// turned by the transposing read.  In both the 16-byte pieces of a row are turned by the row's number, so that the lanes of a read
// meet all banks: the first as attn_place's rows of 64, the second as attn_place_v's, the turn's low bit from the row's bit 3
// because the two halves of a wave here read rows 8 apart.
//
// Loads go through a buffer resource that ends where the matrix ends: rows past it are zeros, and cost no branch.  Pieces of k past
// the end of a row (not past the matrix) are given an offset past any end.
#pragma once
#include "smlm_common.hpp"

namespace smlm {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGemmK = 64;                          // of k a stage
constexpr uint32_t kGemmFar = 0xf8000000u;          // an offset past every resource's end
constexpr int64_t kGemmMostBytes = 0xf0000000ll;    // that a resource may span

template <int DT>
__device__ __forceinline__ f32x16 gemm_mfma(u32x4 a, u32x4 b, f32x16 c) {
  if (DT == SMLM_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A matrix operand: `rows` rows in memory of `ld` elements, and the first row or column of the tile.
struct GemmOperand {
  const uint16_t* base;
  int64_t ld;    // elements from row to row
  int64_t rows;  // rows in memory
};

// The tile's side of an operand in LDS: ROWS rows of kGemmK (plain), or kGemmK rows of ROWS (across).
template <int ROWS, bool ACROSS>
struct GemmSide {
  static constexpr int kElems = ROWS * kGemmK;
  static constexpr int kLoads = ROWS / 32;  // a wave's loads of 1 KB a stage
  uint32_t off[kLoads];                     // bytes from the stage's first element
  const uint16_t* at;                       // the stage's first element
  int64_t left;                             // bytes from there to the matrix's end

  static __device__ __forceinline__ int place(int row, int piece) {
    if (!ACROSS) return row * kGemmK + ((piece ^ ((row >> 1) & 7)) << 3);
    return row * ROWS + ((piece ^ ((((row & 3) << 1) | ((row >> 3) & 1)) << 1)) << 3);
  }
  __device__ __forceinline__ void start(const GemmOperand& m, int64_t first, int k0, int wave, int lane) {
    constexpr int kLanes = ACROSS ? ROWS / 8 : 8;  // of a row in LDS
    constexpr int kStep = 64 / kLanes;             // rows a load
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave * kLoads + i) * kStep + lane / kLanes, slot = lane % kLanes;
      // (the turn undoes itself: the piece that belongs into the lane's place)
      const int piece = (place(row, slot) - row * (ACROSS ? ROWS : kGemmK)) >> 3;
      off[i] = (uint32_t)row * (uint32_t)(m.ld * 2) + (uint32_t)piece * 16u;
    }
    const int64_t e = ACROSS ? (int64_t)k0 * m.ld + first : first * m.ld + k0;
    at = m.base + e;
    left = (m.rows * m.ld - e) * 2;
  }
  // k_left: of k, what is left of the rows from this stage on (plain)
  __device__ __forceinline__ void load(uint16_t* lds, const GemmOperand& m, int k_left, int wave, int lane) {
    const uint32_t span = (uint32_t)(left < 0 ? 0 : left < kGemmMostBytes ? left : kGemmMostBytes);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), 0, span, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t o = off[i];
      if (!ACROSS && k_left < kGemmK) {
        const int row = (wave * kLoads + i) * 8 + lane / 8;
        if (((place(row, lane % 8) - row * kGemmK) >> 3) * 8 >= k_left) o = kGemmFar;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (wave * kLoads + i) * 512), 16, o, 0, 0, 0);
    }
    const int64_t step = ACROSS ? (int64_t)kGemmK * m.ld : kGemmK;
    at += step;
    left -= step * 2;
  }
};

// Where a lane reads its operands: one place for each 16 of k of a stage (plain; the blocks of 32 rows are constants apart), or one
// for each block of 32 (across; steps of 16 of k are constants apart).
template <int ROWS, bool ACROSS, int BLOCKS>
struct GemmReader {
  static constexpr int kPlaces = ACROSS ? BLOCKS : kGemmK / 16;
  int at[kPlaces];
  __device__ __forceinline__ void start(int first, int lane) {  // first: row of the tile of the wave's first block
    const int h = lane >> 5;
    if (!ACROSS) {
#pragma unroll
      for (int s = 0; s < kPlaces; ++s) at[s] = GemmSide<ROWS, false>::place(first + (lane & 31), s * 2 + h);
    } else {
      const int l = lane & 15;
#pragma unroll
      for (int b = 0; b < kPlaces; ++b) {
        const int d = first + b * 32 + ((lane >> 4) & 1) * 16 + (l & 3) * 4;
        at[b] = GemmSide<ROWS, true>::place(h * 8 + (l >> 2), d >> 3) + (d & 7);
      }
    }
  }
  __device__ __forceinline__ u32x4 read(const uint16_t* lds, int b, int s) const {
    if (!ACROSS) return *(const u32x4*)(lds + at[s] + b * 32 * kGemmK);
    const uint16_t* p = lds + at[b] + s * 16 * ROWS;
    const u32x2 x = lds_read_tr16(p), y = lds_read_tr16(p + 4 * ROWS);  // (four rows on: the same turn)
    return u32x4{x[0], x[1], y[0], y[1]};
  }
};

// WA x WB waves of IA x JB blocks of 32 x 32.
template <int WA, int IA, bool XA, int WB, int JB, bool XB>
struct GemmShape {
  static constexpr int kA = WA * IA * 32, kB = WB * JB * 32;
  static constexpr int kStage = (kA + kB) * kGemmK;  // elements of LDS
};

// acc[i][j] += the tile's sums over k in [k0, k1).  lds: 2 * kStage elements.
template <int DT, int WA, int IA, bool XA, int WB, int JB, bool XB>
__device__ __forceinline__ void gemm_tile(f32x16 (&acc)[IA][JB], uint16_t* lds, const GemmOperand& ma, int64_t a0,
                                          const GemmOperand& mb, int64_t b0, int k0, int k1) {
  typedef GemmShape<WA, IA, XA, WB, JB, XB> S;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  GemmSide<S::kA, XA> sa;
  GemmSide<S::kB, XB> sb;
  sa.start(ma, a0, k0, wave, lane);
  sb.start(mb, b0, k0, wave, lane);
  GemmReader<S::kA, XA, IA> ra;
  GemmReader<S::kB, XB, JB> rb;
  ra.start((wave / WB) * IA * 32, lane);
  rb.start((wave % WB) * JB * 32, lane);
  uint16_t* const st0 = lds;
  uint16_t* const st1 = lds + S::kStage;
  auto load = [&](uint16_t* st, int k) {
    sa.load(st, ma, k1 - k, wave, lane);
    sb.load(st + S::kA * kGemmK, mb, k1 - k, wave, lane);
  };
  u32x4 fa[2][IA], fb[2][JB];
  auto read = [&](const uint16_t* st, int s, u32x4 (&a)[IA], u32x4 (&b)[JB]) {
#pragma unroll
    for (int i = 0; i < IA; ++i) a[i] = ra.read(st, i, s);
#pragma unroll
    for (int j = 0; j < JB; ++j) b[j] = rb.read(st + S::kA * kGemmK, j, s);
  };
  auto multiply = [&](const u32x4 (&a)[IA], const u32x4 (&b)[JB]) {
#pragma unroll
    for (int i = 0; i < IA; ++i)
#pragma unroll
      for (int j = 0; j < JB; ++j) acc[i][j] = gemm_mfma<DT>(a[i], b[j], acc[i][j]);
  };
  __syncthreads();  // (whoever used the LDS before is done)
  if (k0 >= k1) return;
  load(st0, k0);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): a barrier does not wait for loads to LDS
  __syncthreads();
  load(st1, k0 + kGemmK);  // (past the end: zeros, and no access to memory)
  read(st0, 0, fa[0], fb[0]);
  // One read or two of the next step's operands between two products: left to itself the compiler has each product wait for a read.
  constexpr int kReads = (XA ? 2 : 1) * IA + (XB ? 2 : 1) * JB, kProducts = IA * JB;
  auto turn = [&] {
    constexpr int kPer = (kReads + kProducts - 1) / kProducts;
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      if (i < kReads / kPer) __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
  };
  auto stage = [&](const uint16_t* st, uint16_t* next, uint16_t* mine, int k) {
    read(st, 1, fa[1], fb[1]);
    multiply(fa[0], fb[0]);
    turn();
    read(st, 2, fa[0], fb[0]);
    multiply(fa[1], fb[1]);
    turn();
    read(st, 3, fa[1], fb[1]);
    multiply(fa[0], fb[0]);
    turn();
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();  // the next stage has landed, and everybody has read this one
    load(mine, k + 2 * kGemmK);
    read(next, 0, fa[0], fb[0]);
    multiply(fa[1], fb[1]);
    turn();
  };
  int k = k0;
#pragma unroll 1
  for (; k + kGemmK < k1; k += 2 * kGemmK) {
    stage(st0, st1, st0, k);
    stage(st1, st0, st1, k + kGemmK);
  }
  if (k < k1) stage(st0, st1, st0, k);
}

}  // namespace smlm
