// pst_head_gemm.h — the matrix product under the token head's operators (gfx950 / CDNA4).
//
// D[m][n] = sum_k A[m][k] B[n][k] on a BM x BN tile, 16-bit or 32-bit floats (f32 sums) or 8-bit integers (i32 sums), by
// v_mfma_*_16x16x32 / 16x16x4 / 16x16x64. Lane l of a wave holds, of each 16x16 block, column n = l & 15 and rows
// m = 4 (l >> 4) + r, r = 0..3: the operand whose index runs along the outputs' contiguous axis is A (four
// neighbours in one lane), and a reduction over that axis is 32 values in a lane and two lane exchanges.
//
// What bounds the large products is power: with operands of random bits the card sustains 2.06 PFLOP/s of bf16
// 16x16x32 and 1.77 of 32x32x16 (whose sums move twice the bits for each product; 8-bit: 4.04 and 3.40), all from
// registers. So the small block is used, and bytes are moved as rarely as the registers allow: 128 x 64 a wave. What the
// loop waits for was taken from a launch of dW alone, in one plane (8192 x 16128 x 1024 bf16, 216 us, 1.25 PFLOP/s): matrix
// cores busy 2/3 of the time at 1.87 GHz; without the loads to LDS (leaving all else) 155 us, without the LDS reads 195:
// what remains is moving operands. 80 % of the loads hit L2, whose share of the rest is what the tile order leaves: each
// matrix once from behind it. 32-bit products are bound by their instructions: 0.14 PFLOP/s of 0.157.
//
// A K-step is 128 bytes of k (64 16-bit values, 32 32-bit ones, 128 8-bit ones) of every tile row. Operands are staged by
// global_load_lds_dwordx4 (global memory to LDS without registers: lane i of the instruction fills 16 bytes
// at base + 16 i, so what is permuted is the global address each lane reads) in two forms:
//   ROWS  memory holds k contiguous in each row. LDS: [row][8 chunks of 16 bytes], chunk c of row r at place
//         c ^ (r >> 1 & 7): 16 rows read at one c fill the 64 banks once.
//   COLS  memory holds the tile's rows as columns: [k][m]. LDS: [k][m], pieces of 16 values of row k permuted by swizzle(k)
//         so that the 16 k-rows of a read spread over the banks; ds_read_b64_tr_b16 turns four k-rows of 16
//         columns into four consecutive k of one column per lane (32-bit values are read one by one): no transposed copy
//         of a matrix is ever made.
// k that passes the end: the last K-step reads the last valid chunk or row again, against zeros that the caller sees to in
// the other operand; of ROWS of floats in A what was read again is cleared.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pst_head {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Elem { BF16 = 0, F16 = 1, I8 = 2, F32 = 3 };
constexpr int bytes_of(int elem) { return elem == I8 ? 1 : elem == F32 ? 4 : 2; }

template <int E>
struct Mma;
template <>
struct Mma<BF16> {
  typedef f32x4 Acc;
  static constexpr int PARTS = 1;  // instructions for the 16 bytes of k a lane holds
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<F16> {
  typedef f32x4 Acc;
  static constexpr int PARTS = 1;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<I8> {
  typedef i32x4 Acc;
  static constexpr int PARTS = 1;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c, int) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
// 32-bit floats: of the four k a lane holds, each instruction takes one of each 16-lane group
template <>
struct Mma<F32> {
  typedef f32x4 Acc;
  static constexpr int PARTS = 4;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c, int part) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[part], __builtin_bit_cast(f32x4, b)[part], c, 0, 0, 0);
  }
};

// One operand in memory. ROWS: `rows` rows of `bytes` valid bytes (a multiple of 16). COLS: `rows` k-rows of
// `bytes` valid bytes. ld in bytes, a multiple of 16 (and p 16-byte aligned). Sums of two 16-bit floats have two planes,
// hi at p and lo at p + plane.
struct Operand {
  const char* p;
  int64_t plane;
  int64_t ld;
  int32_t rows;
  int32_t bytes;
};

constexpr int STEP = 128;  // bytes of k in a K-step

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// 16 bytes a lane from base + off to LDS at `lds` + 16 lane; nothing returns to registers. The M0 write needs a
// wait state before the load reads it. (M0 is named as clobbered, so that no value of the compiler's is taken to outlive it
// there; that it is a reserved register is what the warning would say.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0", "memory");
}
#pragma clang diagnostic pop

// All but the last N of this wave's loads have landed (they return in the order of their issue) and everything it read
// from LDS has been read, then all waves meet.
template <int N>
__device__ __forceinline__ void landed_but() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// All waves meet, with what they wrote to LDS and whatever loads in flight.
__device__ __forceinline__ void met() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// COLS: LDS row k is made of pieces of 16 values (a block's rows), and this is what a piece's number is xored with, of B-byte
// values in rows of RT bytes. 16 bits: a read takes k-rows 8 g + i (g, i = 0..3) and one piece of each: eight places
// of the 256-byte bank row, each twice. 32 bits: k-rows 4 g + e, each e a read of its own: four places, each once.
template <int RT, int B>
__device__ __forceinline__ int swizzle(int k) {
  if (B == 4) return k >> 2 & 3;
  return RT == 128 ? (k >> 1 & 1) | (k >> 2 & 2) : (k & 3) | (k >> 1 & 4);
}

// R: tile rows (m or n); NW: waves that share the loading; B: bytes of a value
template <int R, bool COLS, int NW, int B>
struct Stager {
  static constexpr int NI = R * STEP / 1024 / NW;  // instructions a wave and K-step
  static constexpr int RT = COLS ? R * B : STEP;   // bytes of an LDS row
  static constexpr int KS = STEP / B;              // k-rows of a K-step
  static constexpr int PER = 1024 / RT;            // LDS rows an instruction fills
  static_assert(NI >= 1 && NI * NW * 1024 == R * STEP, "tile and waves do not fit");
  uint32_t off[NI];
  const char* base;  // of the tile
  int32_t k_bytes;   // ROWS: valid bytes of a row; COLS: valid k-rows
  int64_t ld;
  int64_t plane;
  const char* src;   // the K-step being loaded, what is valid of it, and where it goes
  int32_t left;
  uint32_t to;

  __device__ __forceinline__ void init(const Operand& o, int row0, int lane, int wave) {
    ld = o.ld;
    plane = o.plane;
    left = 1 << 30;
    // a tile behind the last row (a column of zeros in the output) reads the last one
    const int first = COLS ? min(row0 * B, o.bytes - 16) : min(row0, o.rows - 1);
    base = o.p + (COLS ? (int64_t)first : (int64_t)first * o.ld);
    k_bytes = COLS ? o.rows : o.bytes;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = (wave * NI + j) * PER + lane / (RT / 16);  // LDS row
      const int c = lane % (RT / 16);                          // 16-byte place in it
      if (COLS) {
        const int col = ((c / B) ^ swizzle<RT, B>(r)) * (16 * B) + c % B * 16;
        off[j] = (uint32_t)(r * (int64_t)o.ld) + (uint32_t)min(col, o.bytes - 16 - first);
      } else {
        off[j] = (uint32_t)(min(r, o.rows - 1 - first) * o.ld) + (uint32_t)((c ^ (r >> 1 & 7)) << 4);
      }
    }
  }
  // K-step `step` goes to the LDS tile at `lds`, by one(0) ... one(NI - 1).
  // AGAIN: the K range comes more than once, from plane `q`
  template <bool AGAIN>
  __device__ __forceinline__ void aim(int step, int q, uint32_t lds, int lane, int wave) {
    constexpr int WHOLE = COLS ? KS : STEP;
    if (AGAIN && left < WHOLE) shift<-1>(left, lane, wave);  // back from the last step of the range
    src = base + (COLS ? (int64_t)min(step * KS, k_bytes - 1) * ld : (int64_t)step * STEP);
    if (AGAIN) src += q * plane;
    left = COLS ? k_bytes - step * KS : k_bytes - step * STEP;
    if (left < WHOLE) shift<1>(left, lane, wave);  // the last step of the range
    to = __builtin_amdgcn_readfirstlane(lds + (uint32_t)wave * (NI * 1024));
  }
  // a K-step of which `valid` (k-rows or bytes) exist: what lies behind reads the last of them (SIGN -1: no more)
  template <int SIGN>
  __device__ __forceinline__ void shift(int valid, int lane, int wave) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = (wave * NI + j) * PER + lane / (RT / 16);
      const int c = lane % (RT / 16);
      off[j] -= SIGN * (COLS ? (uint32_t)((int64_t)max(0, r - max(0, valid - 1)) * ld) : (uint32_t)max(0, ((c ^ (r >> 1 & 7)) << 4) - (valid - 16)));
    }
  }
  __device__ __forceinline__ void one(int j) const {
    load_lds(src, off[j], to + j * 1024);
  }
};

// Fragments of one wave, 16 rows x 64 bytes of k each: block b (from block blk0 of the tile), half s of the K-step
template <int R, bool COLS, int B>
struct Reader {
  uint32_t at[2];
  __device__ __forceinline__ void init(int blk0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    if (COLS) {
      constexpr int RT = R * B;
      const int k = B == 4 ? 4 * g : 8 * g + (i >> 2);
      at[0] = k * RT + (blk0 ^ swizzle<RT, B>(k)) * (16 * B) + (B == 4 ? i << 2 : (i & 3) << 3);
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (blk0 * 16 + i) * STEP + (((4 * s + g) ^ (i >> 1)) << 4);
    }
  }
  __device__ __forceinline__ i32x4 get(const char* tile, int b, int s) const {
    if (COLS && B == 4) {
      constexpr int RT = R * B;
      const char* q = tile + (at[0] ^ (uint32_t)(b << 6)) + s * 16 * RT;
      i32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *(const int*)(q + e * RT);
      return v;
    }
    if (COLS) {
      constexpr int RT = R * 2;
      typedef __attribute__((address_space(3))) s16x4* P;
      const char* q = tile + (at[0] ^ (uint32_t)(b << 5)) + s * 32 * RT;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(q + 4 * RT));
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *(const i32x4*)(tile + at[s] + b * 16 * STEP);
  }
};

template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM_ * WN_, THREADS = NW * 64;
  static constexpr int MI = BM_ / WM_ / 16, NI = BN_ / WN_ / 16;  // a wave's 16x16 blocks
  static constexpr int WAVES = 2;  // on each SIMD at least: what a workgroup's registers leave room for
  static constexpr int STAGES = STAGES_;
  static constexpr int STAGE = (BM_ + BN_) * STEP, LDS = STAGES * STAGE;  // (an epilogue's own LDS lies behind)
};

// The K loop of one tile after another: begin() starts the loads of a tile's first K-steps, run() leaves the tile's sums in
// acc[MI][NI] of this wave. Between them a workgroup can store the tile before.
// A ring of S LDS stages: the loads of K-step t + S start when all waves have read the last of step t, and fly while the
// steps between are multiplied. A K-step is four parts, (k half, half of the wave's rows): each part's fragments are read
// from LDS while the part before is multiplied, also across the one barrier of a K-step.
// Measured on that launch of dW (210 - 216 us as it is): K-steps of 64 bytes in rings of 3, 4 and 5 stages
// 226 - 228 (twice the barriers; deeper prefetch gains nothing), two 256 x 128 workgroups a unit 252 (half as much again
// through LDS), four waves of 128 x 128 224, blocks of 32 x 32 227, loads in one burst 222.
// HALVES: operands that are sums of two planes, hi and lo, come in `products` runs through the same `range` of K-steps: of B alone
// lo, hi (2 products); of both hi lo, lo hi, hi hi (3; lo lo, 2^-16 of the whole, is left out). The small ones first. More
// of the K loop, where both planes in LDS would take as much room as a tile twice as large.
template <int E, class T, bool ACOLS, bool BCOLS, bool HALVES = false>
struct Loop {
  typedef typename Mma<E>::Acc Acc;
  static constexpr int HI = T::MI / 2;
  // blocks of a wave start at a multiple of their number, so that a COLS read can xor the block into its address
  static_assert((T::MI & (T::MI - 1)) == 0 && (T::NI & (T::NI - 1)) == 0 && T::MI >= 2, "wave tile");
  static constexpr int S = T::STAGES, B = bytes_of(E);
  static constexpr int LA = Stager<T::BM, ACOLS, T::NW, B>::NI, LB = Stager<T::BN, BCOLS, T::NW, B>::NI, L = LA + LB;
  static_assert((S & (S - 1)) == 0 && S >= 2, "ring of stages");
  Stager<T::BM, ACOLS, T::NW, B> sa;
  Stager<T::BN, BCOLS, T::NW, B> sb;
  Reader<T::BM, ACOLS, B> ra;
  Reader<T::BN, BCOLS, B> rb;
  char* smem;
  uint32_t lds0;
  int lane, wave;
  int step, total;  // step: what is loaded next
  int range, products;

  __device__ __forceinline__ explicit Loop(char* smem_) : smem(smem_), lds0(lds_addr(smem_)) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ra.init(wave / T::WN * T::MI, lane);
    rb.init(wave % T::WN * T::NI, lane);
  }
  __device__ __forceinline__ void aim(int stage) {
    const uint32_t to = lds0 + stage * T::STAGE;
    int c = 0;
    if (HALVES) c = step >= 2 * range ? 2 : step >= range ? 1 : 0;
    const int s = HALVES ? step - c * range : step;
    sa.template aim<HALVES>(s, products == 3 && c == 1, to, lane, wave);
    sb.template aim<HALVES>(s, products > 1 && c == 0, to + T::BM * STEP, lane, wave);
    ++step;
  }
  __device__ __forceinline__ void load(int i) const {
    if (i < LA) sa.one(i);
    else sb.one(i - LA);
  }
  __device__ __forceinline__ void issue(int stage) {
    aim(stage);
#pragma unroll
    for (int i = 0; i < L; ++i) load(i);
  }
  // K-steps [from, to) of all products'; all waves have left the stages
  __device__ __forceinline__ void begin(const Operand& A, const Operand& B, int m0, int n0, int from, int to, int range_ = 0, int products_ = 1) {
    sa.init(A, m0, lane, wave);
    sb.init(B, n0, lane, wave);
    step = from;
    total = to - from;
    range = range_;
    products = products_;
    for (int t = 0; t < min(S, total); ++t) issue(t);
  }

  // at most `steps` K-steps' loads are in flight behind this
  template <int MOST = S - 1>
  __device__ __forceinline__ void landed_but_steps(int steps) const {
    if constexpr (MOST == 0) {
      landed_but<0>();
    } else {
      if (steps >= MOST) return landed_but<MOST * L>();
      landed_but_steps<MOST - 1>(steps);
    }
  }
  __device__ __forceinline__ void clear(Acc (&acc)[T::MI][T::NI]) {
#pragma unroll
    for (int i = 0; i < T::MI; ++i)
#pragma unroll
      for (int j = 0; j < T::NI; ++j) acc[i][j] = {0, 0, 0, 0};
  }
  // the loads of a K-step between `count` multiplications, behind the q-th: the unit that takes them accepts one in 16
  // clocks of the whole workgroup, and a wave behind it would wait with idle matrix cores
  template <int COUNT>
  __device__ __forceinline__ void load_behind(int q) const {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int l = q * L / COUNT; l < (q + 1) * L / COUNT; ++l) load(l);
    __builtin_amdgcn_sched_barrier(0);
  }

  i32x4 a[2][HI], b[2][T::NI];
  // fragments of part p of the K-step in `stage`
  __device__ __forceinline__ void fetch(int stage, int p) {
    const char* ta = smem + stage * T::STAGE;
    const char* tb = ta + T::BM * STEP;
#pragma unroll
    for (int i = 0; i < HI; ++i) a[p & 1][i] = ra.get(ta, (p & 1) * HI + i, p >> 1);
    if ((p & 1) == 0) {
#pragma unroll
      for (int j = 0; j < T::NI; ++j) b[p >> 1][j] = rb.get(tb, j, p >> 1);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // multiplies part p; MORE: with the loads of a K-step
  template <bool MORE>
  __device__ __forceinline__ void mult(Acc (&acc)[T::MI][T::NI], int p) {
    constexpr int ONE = HI * T::NI, COUNT = ONE * Mma<E>::PARTS;
#pragma unroll
    for (int q = 0; q < COUNT; ++q) {
      const int i = q % ONE / T::NI, j = q % T::NI;
      acc[(p & 1) * HI + i][j] = Mma<E>::mma(a[p & 1][i], b[p >> 1][j], acc[(p & 1) * HI + i][j], q / ONE);
      if constexpr (MORE) load_behind<COUNT>(q);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // the first three parts of K-step t, and the fragments of its last
  __device__ __forceinline__ void most(Acc (&acc)[T::MI][T::NI], int t) {
    const int stage = t & (S - 1);
    fetch(stage, 1);
    mult<false>(acc, 0);
    fetch(stage, 2);
    mult<false>(acc, 1);
    fetch(stage, 3);
    mult<false>(acc, 2);
  }

  // The last K-step of rows that end inside it holds their last 16 bytes again, against zeros of B. Zeros take their place,
  // since zero times an infinity is none (integers cannot spoil anything). All waves are past the wait for the step. Costs the
  // 256 x 256 loop two registers: 8192 x 64003 x 1024 bf16 859 -> 870 us.
  __device__ __forceinline__ void clear_tail(int stage) const {
    if (ACOLS || E == I8 || sa.left >= STEP) return;
    for (int i = threadIdx.x; i < T::BM * (STEP / 16); i += T::THREADS) {
      const int r = i / (STEP / 16), c = i % (STEP / 16);
      if ((c ^ (r >> 1 & 7)) * 16 >= sa.left) *(i32x4*)(smem + stage * T::STAGE + r * STEP + c * 16) = {0, 0, 0, 0};
    }
    met();
  }

  __device__ __forceinline__ void run(Acc (&acc)[T::MI][T::NI]) {
    clear(acc);
    int t = 0;
    // (what this wave stored since begin() counts as loads in flight do, so the first wait may be for some of it)
    if (total > 0) {
      landed_but_steps(min(S, total) - 1);
      if (total == 1) clear_tail(0);
      fetch(0, 0);
    }
    for (; t + S < total; ++t) {
      most(acc, t);
      // the last fragments of step t are in registers: its stage is free once all waves are here
      landed_but<(S - 2) * L>();
      fetch((t + 1) & (S - 1), 0);
      aim(t & (S - 1));
      mult<true>(acc, 3);
    }
    for (; t + 1 < total; ++t) {
      most(acc, t);
      landed_but_steps(total - t - 2);
      if (t + 2 == total) clear_tail((t + 1) & (S - 1));
      fetch((t + 1) & (S - 1), 0);
      mult<false>(acc, 3);
    }
    if (t < total) {
      most(acc, t);
      mult<false>(acc, 3);
    }
    landed_but<0>();  // the stages are free
  }
};

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
