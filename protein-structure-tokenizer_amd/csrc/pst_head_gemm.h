// pst_head_gemm.h — the matrix product under the token head's operators (gfx950 / CDNA4).
//
// D[m][n] = sum_k A[m][k] B[n][k] on a BM x BN tile, 16-bit floats (f32 sums) or 8-bit integers (i32 sums),
// by v_mfma_*_32x32x16 / 32x32x32. Lane l of a wave holds, of each 32x32 block, column n = l & 31 and rows
// m = 8 (r >> 2) + 4 (l >> 5) + (r & 3), r = 0..15: the operand whose index runs along the outputs' contiguous
// axis is A (four neighbours in one lane), and a reduction over that axis stays inside a lane.
//
// A K-step is 128 bytes of k (64 16-bit values, 128 8-bit ones) of every tile row. Operands are staged by
// global_load_lds_dwordx4 (global memory to LDS without registers: lane i of the instruction fills 16 bytes
// at base + 16 i, so what is permuted is the global address each lane reads) in two forms:
//   ROWS  memory holds k contiguous in each row. LDS: [row][8 chunks of 16 bytes], chunk c of row r at place
//         c ^ (r & 7): the 32 rows that a fragment read touches at one c lie in all banks.
//   COLS  memory holds the tile's rows as columns: [k][m]. LDS: [k][m], 64-byte pieces of row k at place
//         p ^ (k & 3) (p ^ (k >> 1 & 1) for 128-byte rows); ds_read_b64_tr_b16 turns four k-rows of 16 columns
//         into four consecutive k of one column per lane, so no transposed copy of a matrix is ever made.
// k that passes the end: the last K-step reads the last valid chunk or row again; the caller sees to it that
// the other operand holds zeros there.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pst_head {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Elem { BF16 = 0, F16 = 1, I8 = 2 };

template <int E>
struct Mma;
template <>
struct Mma<BF16> {
  typedef f32x16 Acc;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<F16> {
  typedef f32x16 Acc;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<I8> {
  typedef i32x16 Acc;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};

// One operand in memory. ROWS: `rows` rows of `bytes` valid bytes (a multiple of 16). COLS: `rows` k-rows of
// `bytes` valid bytes. ld in bytes, a multiple of 16 (and p 16-byte aligned). Plane q (a 32-bit float split
// into 16-bit ones has two) starts at p + q * plane.
struct Operand {
  const char* p;
  int64_t plane;
  int64_t ld;
  int32_t rows;
  int32_t bytes;
};

// The product's K loop: `segs` passes over the same k range with the operands' planes seg_a / seg_b (2 bits a
// pass), K-steps [step0, step1) of each.
struct KLoop {
  int32_t segs;
  uint32_t seg_a, seg_b;
};

constexpr int STEP = 128;  // bytes of k in a K-step

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// 16 bytes a lane from base + off to LDS at `lds` + 16 lane; nothing returns to registers. The M0 write needs a
// wait state before the load reads it.
__device__ __forceinline__ void load_lds(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}

// Everything this wave has loaded has landed and everything it read from LDS has been read, then all waves meet.
__device__ __forceinline__ void landed_and_met() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// R: tile rows (m or n); NW: waves that share the loading
template <int R, bool COLS, int NW>
struct Stager {
  static constexpr int NI = R * STEP / 1024 / NW;  // instructions a wave and K-step
  static constexpr int RT = COLS ? R * 2 : STEP;   // bytes of an LDS row
  static constexpr int PER = 1024 / RT;            // LDS rows an instruction fills
  static_assert(NI >= 1 && NI * NW * 1024 == R * STEP, "tile and waves do not fit");
  uint32_t off[NI];
  const char* base;  // of the current plane's tile
  int32_t k_bytes;   // ROWS: valid bytes of a row; COLS: valid k-rows
  int64_t ld;

  // swizzle of LDS row k's 64-byte pieces
  static __device__ __forceinline__ int sw(int k) { return RT == 128 ? (k >> 1) & 1 : k & 3; }

  __device__ __forceinline__ void init(const Operand& o, int row0, int lane, int wave) {
    ld = o.ld;
    // a tile behind the last row (a column of zeros in the output) reads the last one
    const int first = COLS ? min(row0 * 2, o.bytes - 16) : min(row0, o.rows - 1);
    base = o.p + (COLS ? (int64_t)first : (int64_t)first * o.ld);
    k_bytes = COLS ? o.rows : o.bytes;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = (wave * NI + j) * PER + lane / (RT / 16);  // LDS row
      const int c = lane % (RT / 16);                          // 16-byte place in it
      if (COLS) {
        const int col = (((c >> 2) ^ sw(r)) << 6) | ((c & 3) << 4);
        off[j] = (uint32_t)(r * (int64_t)o.ld) + (uint32_t)min(col, o.bytes - 16 - first);
      } else {
        off[j] = (uint32_t)(min(r, o.rows - 1 - first) * o.ld) + (uint32_t)((c ^ (r & 7)) << 4);
      }
    }
  }
  // loads K-step `step` of plane `plane_off` into the LDS tile at `lds`
  __device__ __forceinline__ void issue(int64_t plane_off, int step, uint32_t lds, int lane, int wave) {
    const char* b = base + plane_off + (COLS ? (int64_t)min(step * 64, k_bytes - 1) * ld : (int64_t)step * STEP);
    const int left = COLS ? k_bytes - step * 64 : k_bytes - step * STEP;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (uint32_t)wave * (NI * 1024));
    if (left >= (COLS ? 64 : STEP)) {
#pragma unroll
      for (int j = 0; j < NI; ++j) load_lds(b, off[j], to + j * 1024);
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int r = (wave * NI + j) * PER + lane / (RT / 16);
        const int c = lane % (RT / 16);
        uint32_t o = off[j];
        if (COLS) {
          o -= (uint32_t)((int64_t)max(0, r - max(0, left - 1)) * ld);
        } else {
          o -= (uint32_t)max(0, ((c ^ (r & 7)) << 4) - (left - 16));
        }
        load_lds(b, o, to + j * 1024);
      }
    }
  }
};

// Fragment addresses of one wave: NB 32-row blocks from block `blk0` of the tile
template <int R, bool COLS, int NB>
struct Reader {
  uint32_t at[COLS ? NB : 4];
  __device__ __forceinline__ void init(int blk0, int lane) {
    if (COLS) {
      constexpr int RT = R * 2;
      const int g = lane >> 4, i = lane & 15;
      const int k = 8 * (g >> 1) + (i >> 2);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        at[b] = k * RT + (((blk0 + b) ^ Stager<R, true, R * STEP / 1024>::sw(k)) << 6) + ((g & 1) << 5) + ((i & 3) << 3);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        at[s] = (blk0 * 32 + (lane & 31)) * STEP + (((2 * s + (lane >> 5)) ^ (lane & 7)) << 4);
    }
  }
  // block b, 16-byte k piece s of the K-step whose tile is at `tile`
  __device__ __forceinline__ i32x4 get(const char* tile, int b, int s) const {
    if (COLS) {
      constexpr int RT = R * 2;
      typedef __attribute__((address_space(3))) s16x4* P;
      const char* q = tile + at[b] + s * 16 * RT;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(q + 4 * RT));
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *(const i32x4*)(tile + at[s] + b * 32 * STEP);
  }
};

template <int BM_, int BN_, int WM_, int WN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM_ * WN_, THREADS = NW * 64;
  static constexpr int MI = BM_ / WM_ / 32, NI = BN_ / WN_ / 32;
  static constexpr int STAGE = (BM_ + BN_) * STEP, LDS = 2 * STAGE;
};

// The K loop: acc[MI][NI] of this wave. Two LDS stages; the loads of K-step t + 1 fly while t is multiplied.
template <int E, class T, bool ACOLS, bool BCOLS>
__device__ __forceinline__ void multiply(typename Mma<E>::Acc (&acc)[T::MI][T::NI], const Operand& A, const Operand& B,
                                         const KLoop& kl, int m0, int n0, int step0, int step1, char* smem) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  Stager<T::BM, ACOLS, T::NW> sa;
  Stager<T::BN, BCOLS, T::NW> sb;
  sa.init(A, m0, lane, wave);
  sb.init(B, n0, lane, wave);
  Reader<T::BM, ACOLS, T::MI> ra;
  Reader<T::BN, BCOLS, T::NI> rb;
  ra.init(wm * T::MI, lane);
  rb.init(wn * T::NI, lane);
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  const uint32_t lds0 = lds_addr(smem);
  const int steps = step1 - step0, total = steps * kl.segs;
  int seg = 0, step = step0;  // what is loaded next
  auto issue = [&](int stage) {
    const uint32_t to = lds0 + stage * T::STAGE;
    sa.issue((int64_t)((kl.seg_a >> (2 * seg)) & 3) * A.plane, step, to, lane, wave);
    sb.issue((int64_t)((kl.seg_b >> (2 * seg)) & 3) * B.plane, step, to + T::BM * STEP, lane, wave);
    if (++step == step1) {
      step = step0;
      ++seg;
    }
  };
  if (total > 0) issue(0);
  for (int t = 0; t < total; ++t) {
    landed_and_met();
    if (t + 1 < total) issue((t + 1) & 1);
    const char* ta = smem + (t & 1) * T::STAGE;
    const char* tb = ta + T::BM * STEP;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      i32x4 a[T::MI], b[T::NI];
#pragma unroll
      for (int i = 0; i < T::MI; ++i) a[i] = ra.get(ta, i, s);
#pragma unroll
      for (int j = 0; j < T::NI; ++j) b[j] = rb.get(tb, j, s);
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int j = 0; j < T::NI; ++j) acc[i][j] = Mma<E>::mma(a[i], b[j], acc[i][j]);
    }
  }
  landed_and_met();  // the stages are free for the epilogue
}

// Tiles of a grid in the order that keeps an XCD's L2 warm: workgroup b runs on XCD b % 8, each XCD takes one
// contiguous range of the tiles, and within it `gm` tiles along m share each tile along n.
__device__ __forceinline__ void place(int b, int total, int nm, int nn, int gm, int& m, int& n, int& z) {
  const int x = b & 7, q = total >> 3, r = total & 7;
  int lin = x * q + min(x, r) + (b >> 3);
  const int per = nm * nn;
  z = lin / per;
  lin -= z * per;
  const int g = lin / (gm * nn), rem = lin - g * (gm * nn), sz = min(gm, nm - g * gm);
  n = rem / sz;
  m = g * gm + rem - n * sz;
}

}  // namespace pst_head
