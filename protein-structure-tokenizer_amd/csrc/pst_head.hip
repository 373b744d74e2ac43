// pst_head.hip — the token head: operators over a learned table weight [V, d], one row per token id.
//
//   token loss        lse[n] = log sum_v exp(<x_n, w_v>), loss[n] = lse[n] - <x_n, w_t>     (t = target of n)
//   its gradient      D[n][v] = g_n (exp(<x_n, w_v> - lse_n) - [v = t]),  dx = D W,  dW = D^T x
//   8-bit scores      s_n s_v sum_k q_nk q_vk, q_nk = rint(x_nk / s_n), s_n = max_k |x_nk| * (1/127)
//
// The logits never reach memory: the loss keeps per tile of the vocabulary a running maximum and sum for each
// row (k_loss) and joins them (k_join); the gradient makes D for a piece of the vocabulary at a time, as sums of two
// 16-bit floats in a workspace that the last-level cache holds, and multiplies it in both directions from there.
//
// 32-bit inputs are multiplied by the 32-bit matrix instructions (0.157 PFLOP/s at most): every value keeps its 24 bits and
// its exponent, whatever else its row or tensor holds, and an infinity in one place stays there. Splits into 16-bit
// floats are two to three times as fast and have neither: their halves share a scale, and infinity times a half that is
// zero is NaN.
//
// Times in this file: one MI355X, median of 40 - 600 calls in a row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <string>

#include "../../include/pst.h"
#include "pst_head_gemm.h"

namespace pst_head {
namespace {

// Tiles of the products. A remainder of up to 64 vocabulary rows (the marks behind a codebook of 4096 or 64000) or
// positions behind the whole tiles goes to thin tiles of the same launch instead of a round of nearly empty ones.
struct T64 : Tile<64, 64, 2, 2, 2> {
  static constexpr bool HAS_THIN = false;
};
struct T128 : Tile<128, 128, 2, 2, 2> {
  static constexpr bool HAS_THIN = true;
  typedef T64 Thin;
};
struct T256 : Tile<256, 256, 2, 4, 2> {
  static constexpr bool HAS_THIN = true;
  struct Thin : Tile<64, 64, 2, 4, 4> {};
};
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float load1(const void* p, int type, int64_t i) {
  if (type == PST_F32) return ((const float*)p)[i];
  if (type == PST_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ uint32_t bits16(float v, int type) {  // (type: a constant where it counts)
  if (type == PST_BF16) return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int type) { return bits16(a, type) | bits16(b, type) << 16; }
// what a bf16 leaves of v (of an infinity or NaN, and of what rounds to one, nothing)
__device__ __forceinline__ float rest(float v) { return fabsf(v) <= 3.3895313892515355e38f ? v - (float)(__bf16)v : 0.0f; }
// four neighbours of an output row, `n` of them valid
__device__ __forceinline__ void store4(void* p, int type, int64_t i, const float* v, int n, bool wide) {
  if (type == PST_F32) {
    float* q = (float*)p + i;
    if (wide && n >= 4) {
      *(f32x4*)q = (f32x4){v[0], v[1], v[2], v[3]};
    } else {
      for (int j = 0; j < 4; ++j)
        if (j < n) q[j] = v[j];
    }
  } else {
    uint16_t* q = (uint16_t*)p + i;
    const uint32_t a = bits16(v[0], type) | bits16(v[1], type) << 16, b = bits16(v[2], type) | bits16(v[3], type) << 16;
    if (wide && n >= 4) {
      *(uint2*)q = make_uint2(a, b);
    } else {
      for (int j = 0; j < 4; ++j)
        if (j < n) q[j] = (uint16_t)(j < 2 ? a >> (16 * j) : b >> (16 * (j - 2)));
    }
  }
}

struct Targets {
  const void* p;
  int64_t ignore;
  int32_t bits;   // 32 or 64
  int32_t vocab;
};
// the target row, -1 where there is none to find (ignored, or out of range), and whether the position counts
__device__ __forceinline__ int target_of(const Targets& t, int64_t n, bool& counts) {
  const int64_t v = t.bits == 64 ? ((const int64_t*)t.p)[n] : (int64_t)((const int32_t*)t.p)[n];
  counts = v != t.ignore;
  return counts && v >= 0 && v < t.vocab ? (int)v : -1;
}

// The pieces of a matrix's rows over workgroups of 256 threads, without a division: a power of two of threads, at most 64,
// takes a row.
struct Spread {
  int64_t row, rows;  // this thread's first row, and how far its next is
  int piece, pieces;  // the same of the pieces within a row
  __device__ __forceinline__ Spread(int block, int blocks, int per_row) {
    const int shift = per_row >= 64 ? 6 : per_row <= 1 ? 0 : 32 - __builtin_clz(per_row - 1);
    row = ((int64_t)block * 256 + threadIdx.x) >> shift;
    rows = ((int64_t)blocks * 256) >> shift;
    pieces = 1 << shift;
    piece = threadIdx.x & (pieces - 1);
  }
};

// A matrix copied into rows of whole K-steps with zeros behind. Bound by its bytes where they are many: 8192 x 1024 bf16 8.3 us,
// 1023 + 4099 odd rows of 333 f32, read four bytes at a time, 8.4; 8192 + 64003 rows of 1024 f16 into halves 73 (6.3 TB/s).
struct PackJob {
  const char* src;
  int64_t ld;              // bytes
  int64_t rows, rows_pad;  // rows beyond `rows` are zeros
  char* dst;               // [rows_pad][width_pad]; null (wide sources): only `halves` are made
  char* halves;            // f16: two bf16 planes, hi and lo, whose sum is the value (8 + 3 bits); null: not needed
  int32_t zero_rows;       // rows whose position does not count are zeros
  int32_t wide;            // the source allows 16-byte loads
};
struct PackArgs {
  PackJob job[2];
  int32_t blocks[2];       // workgroups of each job
  int32_t bytes, bytes_pad, type;  // of a row
  Targets targets;
};
// pairs of f16 values as pairs of bf16 ones, hi and lo
template <int N>
__device__ __forceinline__ void halves_of(const uint32_t (&h)[N], uint32_t (&hi)[N], uint32_t (&lo)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float x = (float)__builtin_bit_cast(_Float16, (uint16_t)h[j]), y = (float)__builtin_bit_cast(_Float16, (uint16_t)(h[j] >> 16));
    hi[j] = pack2(x, y, PST_BF16);
    lo[j] = pack2(rest(x), rest(y), PST_BF16);
  }
}
// four bytes of a row from byte c, zeros behind the last: a 32-bit value or two 16-bit ones, without a branch
__device__ __forceinline__ uint32_t load_word(const char* row, int c, int bytes, bool f32) {
  if (f32) {
    const uint32_t v = *(const uint32_t*)(row + min(c, bytes - 4));
    return c < bytes ? v : 0;
  }
  const uint32_t x = *(const uint16_t*)(row + min(c, bytes - 2)), y = *(const uint16_t*)(row + min(c + 2, bytes - 2));
  return (c < bytes ? x : 0) | (c + 2 < bytes ? y : 0) << 16;
}
__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  const int which = (int)blockIdx.x < a.blocks[0] ? 0 : 1;
  const int block = (int)blockIdx.x - (which ? a.blocks[0] : 0);
  const PackJob& p = a.job[which];
  const bool f32 = a.type == PST_F32;
  if (!p.wide) {  // four bytes a thread; four pieces' loads before the first store
    const Spread at_row(block, a.blocks[which], a.bytes_pad / 4);
    for (int64_t r = at_row.row; r < p.rows_pad; r += at_row.rows) {
      bool keep = r < p.rows;
      if (keep && p.zero_rows) (void)target_of(a.targets, r, keep);
      const char* row = p.src + r * p.ld;
      const int64_t to = r * a.bytes_pad;
      for (int c0 = at_row.piece * 4; c0 < a.bytes_pad; c0 += at_row.pieces * 16) {
        uint32_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = keep ? load_word(row, c0 + at_row.pieces * 4 * u, a.bytes, f32) : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + at_row.pieces * 4 * u;
          if (c >= a.bytes_pad) break;
          *(uint32_t*)(p.dst + to + c) = v[u];
          if (p.halves) {
            const uint32_t h[1] = {v[u]};
            uint32_t hi[1], lo[1];
            halves_of(h, hi, lo);
            *(uint32_t*)(p.halves + to + c) = hi[0];
            *(uint32_t*)(p.halves + p.rows_pad * a.bytes_pad + to + c) = lo[0];
          }
        }
      }
    }
    return;
  }
  const Spread at_row(block, a.blocks[which], a.bytes_pad / 16);
  for (int64_t r = at_row.row; r < p.rows_pad; r += at_row.rows) {
    bool keep = r < p.rows;
    if (keep && p.zero_rows) (void)target_of(a.targets, r, keep);
    const char* row = p.src + r * p.ld;
    for (int c = at_row.piece * 16; c < a.bytes_pad; c += at_row.pieces * 16) {
      const int64_t to = r * a.bytes_pad + c;
      uint32_t h[4] = {0, 0, 0, 0};
      if (keep && c + 16 <= a.bytes) {
        const uint4 v = *(const uint4*)(row + c);
        h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
      } else if (keep) {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = load_word(row, c + 4 * j, a.bytes, f32);
      }
      if (p.dst) *(uint4*)(p.dst + to) = make_uint4(h[0], h[1], h[2], h[3]);
      if (p.halves) {
        uint32_t hi[4], lo[4];
        halves_of(h, hi, lo);
        *(uint4*)(p.halves + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *(uint4*)(p.halves + p.rows_pad * a.bytes_pad + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }
}

// ------------------------------------------------------------------ products with their epilogues
struct GemmArgs {
  Operand A, B;
  int32_t M, N;        // rows of A and of B that exist
  int32_t nm, nn, nz;  // tiles along m and n, parts of the K loop
  int32_t blocks;      // workgroups that share the nm nn tiles; those behind them take the `thins` thin tiles of the last rows
  int32_t thins;
  int32_t steps;       // K-steps of the whole range
  int32_t range, products;  // gradients: K-steps of one product, and how many (see Loop); steps is of all of them
  int32_t gm;
  // loss and logit gradient: n = position, m = vocabulary row (from v0)
  Targets targets;
  float2* part;        // loss: [nm][N] (maximum, sum)
  float* tlogit;       // loss: [N]
  const float *lse, *gloss;
  char* D;             // [2][rows][ldd] 16-bit: hi and lo; 32-bit operands: [rows][ldd] 32-bit
  int64_t dplane, ldd; // bytes, elements
  int32_t v0;
  // matrix outputs
  void* out;
  int64_t ldo;
  int32_t otype, wide;
  // outputs in parts of the K loop: 32-bit [nz][..][ldp], added to what is there with `add`
  float* part_out;
  int64_t ldp, zstride;
  int32_t add;
  const float *sn, *sm; // scores: scales of the rows of B and of A
};

struct GradArgs {
  GemmArgs dx, dw;
  int32_t blocks[4];
};

enum Kind { LOSS, DLOGIT, SCORES };

// Where a tile lies, and this wave and lane in it. `nm` x `nn` tiles start at row m_base and column n_base.
template <class T>
struct Place {
  static constexpr int BM = T::BM, BN = T::BN;
  int m0, n0, z, mtile, lane, col, wrow, mwave, mw, nw;  // mwave, nw: this wave's first row and column, mw: this lane's first row
  __device__ __forceinline__ Place(const GemmArgs& g, int tile, int nm, int nn, int m_base, int n_base) {
    int m, n;
    place(tile, nm * nn * g.nz, nm, nn, g.gm, m, n, z);
    m0 = m_base + m * T::BM;
    n0 = n_base + n * T::BN;
    mtile = m_base ? g.nm : m;
    lane = threadIdx.x & 63;
    col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wrow = wave / T::WN;
    mwave = m0 + wrow * T::MI * 16;
    mw = mwave + 4 * (lane >> 4);
    nw = n0 + (wave % T::WN) * T::NI * 16;
  }
};

// Two blocks' packed 16-bit values (w[u][q]: block u, the lane's values 2q and 2q + 1) to 32 consecutive columns of the
// lane's row, whose first is at `to`: the exchange of odd and even 16-lane groups leaves 16 consecutive bytes in a lane.
__device__ __forceinline__ void store_pair(char* to, const uint32_t (&w)[2][2], int lane, bool row = true) {
  const auto x = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
  const int g = lane >> 4;
  if (row) *(uint4*)(to + (g & 1) * 32 + (g >> 1) * 16) = make_uint4(x[0], y[0], x[1], y[1]);
}

// sums over the four lanes that hold a column
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// LDS behind a tile's stages: 4 KB for what an epilogue needs of the tile's rows and columns
template <class T>
__device__ __forceinline__ float* epilogue_lds(char* smem) {
  return (float*)(smem + T::LDS);
}
constexpr int EPILOGUE_LDS = 4096;

// A workgroup's tiles: tile, tile + stride, ... of the nm x nn of type T from row m_base. The next tile's loads fly during the
// epilogue of the last; what the epilogue needs from memory is loaded during the K loop (column and row of this thread),
// since waiting for a load is waiting for all that were started before it.
template <int E, class T, bool MANY, class Epilogue>
__device__ __forceinline__ void tiles(const GemmArgs& g, int tile, int stride, int nm, int nn, int m_base, char* smem, Epilogue epilogue) {
  Loop<E, T, false, false> loop(smem);
  const int total = nm * nn;
  if (tile >= total) return;
  Place<T> p(g, tile, nm, nn, m_base, 0);
  loop.begin(g.A, g.B, p.m0, p.n0, 0, g.steps);
  for (;;) {
    typename Mma<E>::Acc acc[T::MI][T::NI];
    auto inputs = epilogue.load(g, p);
    loop.run(acc);
    epilogue.share(inputs, epilogue_lds<T>(smem));
    const Place<T> done = p;
    tile += stride;
    const bool more = MANY && tile < total;
    if (more) {
      p = Place<T>(g, tile, nm, nn, m_base, 0);
      loop.begin(g.A, g.B, p.m0, p.n0, 0, g.steps);
    }
    met();
    epilogue.template store<T>(g, done, acc, epilogue_lds<T>(smem));
    if (!more) return;
  }
}

// The loss: m = vocabulary row, n = position, so a lane holds 32 logits of each of its columns: their maximum and the sum of
// exp(l - maximum) in registers, then over the column's four lanes and the two wave rows, and 8 bytes a tile and position
// go to memory. One exponential a logit (16 clocks of a SIMD for 64 of them) is 1/8 of the matrix work at d = 1024;
// persistent workgroups load the next tile meanwhile.
// 8192 x 64003 x 1024 bf16: 858 us, 1.25 PFLOP/s (the library's product of that shape alone, logits to memory: 961 us);
// 4096 x 4096 x 1024 f32 245 us a call, 0.140 PFLOP/s.
struct LossEpilogue {
  struct Inputs {
    int target;
  };
  template <class P>
  __device__ __forceinline__ Inputs load(const GemmArgs& g, const P& p) const {
    bool counts;
    const int n = p.n0 + (int)threadIdx.x;
    return {(int)threadIdx.x < P::BN && n < g.N ? target_of(g.targets, n, counts) : -1};
  }
  __device__ __forceinline__ void share(const Inputs& in, float* lds) const {
    asm volatile("" ::"v"(in.target));
    if (threadIdx.x < 256) ((int*)lds)[threadIdx.x] = in.target;
  }
  template <class T>
  __device__ __forceinline__ void store(const GemmArgs& g, const Place<T>& p, f32x4 (&acc)[T::MI][T::NI], float* lds) const {
    if (p.mwave + T::MI * 16 > g.M) {  // rows behind the vocabulary's last
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (p.mw + 16 * i + r >= g.M) {
#pragma unroll
            for (int j = 0; j < T::NI; ++j) acc[i][j][r] = -__builtin_inff();
          }
    }
    static_assert(256 * 4 + T::BN * 8 <= EPILOGUE_LDS, "epilogue's LDS");
    float2* sm = (float2*)(lds + 256);  // [WM - 1][BN]: the other waves' maxima and sums
    float mxs[T::NI], sums[T::NI];
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int n = p.nw + 16 * j + p.col;
      float mx = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
      mx = col_max(mx);
      const float base = mx == -__builtin_inff() ? 0.0f : mx;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll  // (the difference first: a rounded mx log2 e is off by more than an exponential's range from 2^31 on)
        for (int r = 0; r < 4; ++r) sum += exp2_fast((acc[i][j][r] - base) * LOG2E);
      sum = col_sum(sum);
      mxs[j] = mx;
      sums[j] = sum;
      // the target's logit, where it is among this wave's rows
      const int t = ((const int*)lds)[n - p.n0];
      if (__any(t >= p.mwave && t < p.mwave + T::MI * 16)) {
        const int at = t < 0 ? -1 : t - p.mw;
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (at == 16 * i + r) g.tlogit[n] = acc[i][j][r];
      }
    }
    // the waves of a column join in wave row 0
    static_assert(T::WM == 2, "two waves a column");
    if (p.wrow == 1 && p.lane < 16) {
#pragma unroll
      for (int j = 0; j < T::NI; ++j) sm[p.nw - p.n0 + 16 * j + p.lane] = make_float2(mxs[j], sums[j]);
    }
    met();
    if (p.wrow == 0 && p.lane < 16) {
#pragma unroll
      for (int j = 0; j < T::NI; ++j) {
        const int n = p.nw + 16 * j + p.lane;
        const float2 o = sm[n - p.n0];
        const float mx = fmaxf(mxs[j], o.x);
        const float safe = mx == -__builtin_inff() ? 0.0f : mx;
        if (n < g.N)
          g.part[(int64_t)p.mtile * g.N + n] = make_float2(mx, sums[j] * exp2_fast((mxs[j] - safe) * LOG2E) + o.y * exp2_fast((o.x - safe) * LOG2E));
      }
    }
  }
};

template <int E, class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES) void k_loss(GemmArgs g) {
  extern __shared__ char smem[];
  if ((int)blockIdx.x < g.blocks) {
    tiles<E, T, true>(g, blockIdx.x, g.blocks, g.nm, g.nn, 0, smem, LossEpilogue{});
  } else if constexpr (T::HAS_THIN) {
    tiles<E, typename T::Thin, false>(g, blockIdx.x - g.blocks, 1 << 30, 1, g.thins, g.nm * T::BM, smem, LossEpilogue{});
  }
}

struct JoinArgs {
  const float2* part;
  const float* tlogit;
  Targets targets;
  float *loss, *lse;
  int32_t n, tiles;
};
// 1024 threads share the vocabulary tiles of COLS positions; 8192 positions of 251 tiles (16 MB): 6.2 us
template <int COLS>
__global__ __launch_bounds__(1024) void k_join(JoinArgs a) {
  constexpr int ROWS = 1024 / COLS;
  __shared__ float2 sm[ROWS][COLS];
  const int col = threadIdx.x % COLS, row = threadIdx.x / COLS;
  const int n = blockIdx.x * COLS + col;
  auto join = [](float2 p, float2 q) {
    const float mx = fmaxf(p.x, q.x);
    const float safe = mx == -__builtin_inff() ? 0.0f : mx;
    return make_float2(mx, p.y * exp2_fast((p.x - safe) * LOG2E) + q.y * exp2_fast((q.x - safe) * LOG2E));
  };
  float2 mine = make_float2(-__builtin_inff(), 0.0f);
  if (n < a.n) {
#pragma unroll 4
    for (int t = row; t < a.tiles; t += ROWS) mine = join(mine, a.part[(int64_t)t * a.n + n]);
  }
  sm[row][col] = mine;
#pragma unroll
  for (int half = ROWS / 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (row < half) sm[row][col] = join(sm[row][col], sm[row + half][col]);
  }
  if (row != 0 || n >= a.n) return;
  const float2 all = sm[0][col];
  const float lse = (all.x == -__builtin_inff() ? 0.0f : all.x) + logf(all.y);
  bool counts;
  const int t = target_of(a.targets, n, counts);
  a.lse[n] = lse;
  a.loss[n] = !counts ? 0.0f : t < 0 ? __builtin_nanf("") : lse - a.tlogit[n];
}
void launch_join(const JoinArgs& j, hipStream_t st) {
  if (j.n <= 1024) hipLaunchKernelGGL(k_join<16>, dim3((unsigned)((j.n + 15) / 16)), dim3(1024), 0, st, j);
  else hipLaunchKernelGGL(k_join<64>, dim3((unsigned)((j.n + 63) / 64)), dim3(1024), 0, st, j);
}

// D of one piece of the vocabulary (columns v0 ...; zeros behind the last row and for positions that do not count), each entry
// as a sum of two bf16 values, hi + lo: off by 2^-16 of the entry whatever its size, since a bf16 has a float's exponents.
// One alone would be off by 2^-8, which the sums over thousands of entries of either sign do not lose; f16 ones, scaled to
// the largest |g|, would drop probabilities and weights far below it. (32-bit operands: D in 32 bits.) The second
// half is a second run of the products (see Loop): 8192 x 64003 x 1024 bf16 4.46 ms, with hi alone 2.71.
// exp(l - lse) as 2^((l - lse) log2 e): the difference first, so that large logits lose nothing in the product. Stores of
// 16 bytes a lane. 8192 x 8192 x 1024 bf16 144 us (0.95 PFLOP/s with 268 MB of halves); f32 1000 x 4096 x 512 39.
template <int E>
struct DlogitEpilogue {
  struct Inputs {
    int target;  // less v0; a position that does not count has a factor of 0
    float lse, c;
  };
  template <class P>
  __device__ __forceinline__ Inputs load(const GemmArgs& g, const P& p) const {
    const int n = p.n0 + (int)threadIdx.x;
    Inputs in = {-1, 0.0f, 0.0f};
    if ((int)threadIdx.x < P::BN && n < g.N) {
      bool counts;
      const int t = target_of(g.targets, n, counts);
      in.target = t < 0 ? -1 : t - g.v0;
      in.lse = counts ? g.lse[n] : 0.0f;
      in.c = !counts ? 0.0f : t < 0 ? __builtin_nanf("") : g.gloss[n];
    }
    return in;
  }
  __device__ __forceinline__ void share(const Inputs& in, float* lds) const {
    asm volatile("" ::"v"(in.target), "v"(in.lse), "v"(in.c));
    if (threadIdx.x < 256) {
      ((int*)lds)[threadIdx.x] = in.target;
      lds[256 + threadIdx.x] = in.lse;
      lds[512 + threadIdx.x] = in.c;
    }
  }
  template <class T>
  __device__ __forceinline__ void store(const GemmArgs& g, const Place<T>& p, f32x4 (&acc)[T::MI][T::NI], float* lds) const {
    const bool edge = p.mwave + T::MI * 16 > g.M;
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int n = p.nw + 16 * j + p.col;
      const int t = ((const int*)lds)[n - p.n0];
      const float lse = lds[256 + n - p.n0], c = lds[512 + n - p.n0];
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = exp2_fast((acc[i][j][r] - lse) * LOG2E);
      if (__any(t >= p.mwave && t < p.mwave + T::MI * 16)) {
        const int at = t - p.mw;
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][j][r] -= at == 16 * i + r ? 1.0f : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] *= c;
      // what does not count is zero whatever its hidden row holds
      if (__any(c == 0.0f)) {
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = c == 0.0f ? 0.0f : acc[i][j][r];
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = p.mw + 16 * i + r < g.M ? acc[i][j][r] : 0.0f;
      }
      if constexpr (E == F32) {
        float* to = (float*)g.D + (int64_t)n * g.ldd + p.mw;
#pragma unroll
        for (int i = 0; i < T::MI; ++i) *(f32x4*)(to + 16 * i) = acc[i][j];
        continue;
      }
      char* to = g.D + ((int64_t)n * g.ldd + p.mwave) * 2;
#pragma unroll
      for (int i = 0; i < T::MI; i += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < 2; ++q) w[u][q] = pack2(acc[i + u][j][2 * q], acc[i + u][j][2 * q + 1], PST_BF16);
        store_pair(to + i * 32, w, p.lane);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < 2; ++q) w[u][q] = pack2(rest(acc[i + u][j][2 * q]), rest(acc[i + u][j][2 * q + 1]), PST_BF16);
        store_pair(to + g.dplane + i * 32, w, p.lane);
      }
    }
  }
};

template <int E, class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES) void k_dlogit(GemmArgs g) {
  extern __shared__ char smem[];
  if ((int)blockIdx.x < g.blocks) {
    tiles<E, T, true>(g, blockIdx.x, g.blocks, g.nm, g.nn, 0, smem, DlogitEpilogue<E>{});
  } else if constexpr (T::HAS_THIN) {
    tiles<E, typename T::Thin, false>(g, blockIdx.x - g.blocks, 1 << 30, 1, g.thins, g.nm * T::BM, smem, DlogitEpilogue<E>{});
  }
}

// a wave's blocks as (a part of) a 32-bit sum: column n of the product is row n of `out`
template <class T>
__device__ __forceinline__ void store_part(const f32x4 (&acc)[T::MI][T::NI], const GemmArgs& g, const Place<T>& p) {
  float* out = (float*)g.part_out + p.z * g.zstride;
#pragma unroll
  for (int j = 0; j < T::NI; ++j) {
    const int n = p.nw + 16 * j + p.col;
    if (n >= g.N) continue;
#pragma unroll
    for (int i = 0; i < T::MI; ++i) {
      const int m = p.mw + 16 * i;
      if (m >= g.ldp) continue;
      f32x4* to = (f32x4*)(out + (int64_t)n * g.ldp + m);
      f32x4 v = acc[i][j];
      if (g.add) {
        const f32x4 o = *to;
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      *to = v;
    }
  }
}

// a gradient from its parts' sums; 4096 and 4099 rows of 512 from theirs (50 MB, in the cache): 11 us
struct FinishJob {
  const float* part;
  int64_t ldp, zstride;
  int64_t rows;
  int32_t nz;
  int32_t rows_count;  // rows are positions: those that do not count become zeros
  void* out;
  int64_t ldo;
  int32_t wide;
};
struct FinishArgs {
  FinishJob job[2];
  int32_t blocks[2];
  int32_t width, otype;
  Targets targets;
};
__global__ __launch_bounds__(256) void k_finish(FinishArgs a) {
  const int which = (int)blockIdx.x < a.blocks[0] ? 0 : 1;
  const int block = (int)blockIdx.x - (which ? a.blocks[0] : 0);
  const FinishJob& f = a.job[which];
  const Spread at_row(block, a.blocks[which], (a.width + 3) / 4);
  for (int64_t n = at_row.row; n < f.rows; n += at_row.rows) {
    bool counts = true;
    if (f.rows_count) (void)target_of(a.targets, n, counts);
    for (int c = at_row.piece * 4; c < a.width; c += at_row.pieces * 4) {
      f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
      for (int z = 0; z < f.nz; ++z) {
        const f32x4 v = *(const f32x4*)(f.part + z * f.zstride + n * f.ldp + c);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const float v[4] = {counts ? s.x : 0.0f, counts ? s.y : 0.0f, counts ? s.z : 0.0f, counts ? s.w : 0.0f};
      store4(f.out, a.otype, n * f.ldo + c, v, a.width - c, f.wide);
    }
  }
}

// A wave's blocks as rows of a matrix of OT: column n of the product is row `row0 + n` of the output, which has M
// columns. `wide`: rows and base allow 16-byte stores (of 16-bit values: two blocks make 16 bytes a lane).
template <int OT, class T>
__device__ __forceinline__ void store_rows_of(const f32x4 (&acc)[T::MI][T::NI], const GemmArgs& g, const Place<T>& p, int64_t row0) {
  const bool whole = g.wide && p.mwave + T::MI * 16 <= g.M;
#pragma unroll
  for (int j = 0; j < T::NI; ++j) {
    const int n = p.nw + 16 * j + p.col;
    const bool row = n < g.N;
    const int64_t at = (row0 + n) * g.ldo;
    if (whole) {
      if (OT == PST_F32) {
        float* to = (float*)g.out + at + p.mw;
        if (row) {
#pragma unroll
          for (int i = 0; i < T::MI; ++i) *(f32x4*)(to + 16 * i) = acc[i][j];
        }
      } else {
        char* to = (char*)g.out + (at + p.mwave) * 2;
#pragma unroll
        for (int i = 0; i < T::MI; i += 2) {
          uint32_t w[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int q = 0; q < 2; ++q) w[u][q] = pack2(acc[i + u][j][2 * q], acc[i + u][j][2 * q + 1], OT);
          store_pair(to + i * 32, w, p.lane, row);
        }
      }
    } else if (row) {
#pragma unroll
      for (int i = 0; i < T::MI; ++i) {
        const int m = p.mw + 16 * i;
        if (m >= g.M) continue;
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        store4(g.out, OT, at + m, v, g.M - m, g.wide);
      }
    }
  }
}
template <class T>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[T::MI][T::NI], const GemmArgs& g, const Place<T>& p, int64_t row0) {
  if (g.otype == PST_BF16) store_rows_of<PST_BF16, T>(acc, g, p, row0);
  else if (g.otype == PST_F16) store_rows_of<PST_F16, T>(acc, g, p, row0);
  else store_rows_of<PST_F32, T>(acc, g, p, row0);
}

// Both gradients of a piece of the vocabulary in one launch, since D feeds both and neither fills the card evenly (4096 x
// 4099 x 512 with one plane of D: 43 us together, 31 and 45 in launches of their own; with both planes 75). 8192 x 8192 x 1024
// bf16: 421 us, 1.31 PFLOP/s of the four products; f16 620 of its six; 1000 x 4096 x 512 f32 71, 0.119 of its two:
// dx's parts (m = column, n = position, k = vocabulary row of the piece, its K loop in nz parts) and rows v0 ... of dW
// (m = column, n = vocabulary row, k = position; in one part straight to the output, or in parts as dx).
template <int E, class T, bool DX>
__device__ __forceinline__ void grad_tile(const GemmArgs& g, int tile, int nm, int nn, int n_base, char* smem) {
  const Place<T> p(g, tile, nm, nn, 0, n_base);
  const int s0 = (int)((int64_t)g.steps * p.z / g.nz), s1 = (int)((int64_t)g.steps * (p.z + 1) / g.nz);
  f32x4 acc[T::MI][T::NI];
  Loop<E, T, true, !DX, E != F32> loop(smem);
  loop.begin(g.A, g.B, p.m0, p.n0, s0, s1, g.range, g.products);
  loop.run(acc);
  if (DX || g.part_out) {
    store_part<T>(acc, g, p);
  } else {
    store_rows<T>(acc, g, p, g.v0);
  }
}
// workgroups: dx's tiles, dW's, then the thin ones of dx and of dW
template <int E, class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES) void k_grads(GradArgs g) {
  extern __shared__ char smem[];
  int b = blockIdx.x;
  if (b < g.blocks[0]) return grad_tile<E, T, true>(g.dx, b, g.dx.nm, g.dx.nn, 0, smem);
  b -= g.blocks[0];
  if (b < g.blocks[1]) return grad_tile<E, T, false>(g.dw, b, g.dw.nm, g.dw.nn, 0, smem);
  if constexpr (T::HAS_THIN) {
    b -= g.blocks[1];
    if (b < g.blocks[2]) return grad_tile<E, typename T::Thin, true>(g.dx, b, g.dx.thins, 1, g.dx.nn * T::BN, smem);
    grad_tile<E, typename T::Thin, false>(g.dw, b - g.blocks[2], g.dw.thins, 1, g.dw.nn * T::BN, smem);
  }
}

// 8-bit scores: m = vocabulary row, n = position. Few positions are bound by the table's bytes: 16 x 64003 x 1024 12.9 us,
// 5.3 TB/s with the scores; many by power, as the other products, and by their stores: 8192 x 64003 x 1024 to bf16 622 us,
// 1.73 POP/s and 1.7 TB/s.
struct ScoresEpilogue {
  struct Inputs {
    float sm, sn;
  };
  template <class P>
  __device__ __forceinline__ Inputs load(const GemmArgs& g, const P& p) const {
    const int i = (int)threadIdx.x & 255;
    return {i < P::BM ? g.sm[min(p.m0 + i, g.M - 1)] : 0.0f, i < P::BN ? g.sn[min(p.n0 + i, g.N - 1)] : 0.0f};
  }
  __device__ __forceinline__ void share(const Inputs& in, float* lds) const {
    asm volatile("" ::"v"(in.sm), "v"(in.sn));
    if (threadIdx.x < 256) {
      lds[threadIdx.x] = in.sm;
      lds[256 + threadIdx.x] = in.sn;
    }
  }
  template <class T>
  __device__ __forceinline__ void store(const GemmArgs& g, const Place<T>& p, i32x4 (&sums)[T::MI][T::NI], float* lds) const {
    f32x4 acc[T::MI][T::NI];
#pragma unroll
    for (int i = 0; i < T::MI; ++i) {
      const f32x4 sv = *(const f32x4*)(lds + p.mw - p.m0 + 16 * i);
#pragma unroll
      for (int j = 0; j < T::NI; ++j) {
        const float sn = lds[256 + p.nw - p.n0 + 16 * j + p.col];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = (float)sums[i][j][r] * sn * sv[r];
      }
    }
    store_rows<T>(acc, g, p, 0);
  }
};
template <class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES) void k_scores(GemmArgs g) {
  extern __shared__ char smem[];
  if ((int)blockIdx.x < g.blocks) {
    tiles<I8, T, true>(g, blockIdx.x, g.blocks, g.nm, g.nn, 0, smem, ScoresEpilogue{});
  } else if constexpr (T::HAS_THIN) {
    tiles<I8, typename T::Thin, false>(g, blockIdx.x - g.blocks, 1 << 30, 1, g.thins, g.nm * T::BM, smem, ScoresEpilogue{});
  }
}

// ------------------------------------------------------------------ the loss of few positions, 32 bits
// With few positions the way of a 32-bit table through memory is all that counts, and the products above are launches of
// many K-steps for tiles that are mostly empty, after a copy of the table where its rows are not aligned. This kernel
// reads it once for 16 NB positions, at any alignment (v_mfma_f32_16x16x4: 32 clocks of a SIMD for 256 bytes of the table,
// 17 TB/s of them all). A call, us: 1 x 64000 x 1024 48 (5.4 TB/s), 16 x 64000 x 1024 67, 16 x 4096 x 2048 16. More
// positions read the table again and again, and each block of the table all their hidden states.
struct FewArgs {
  const float *x, *w;
  int64_t ldx, ldw;
  int32_t wide;          // rows of whole fours, aligned to 16 bytes
  int32_t rows, vocab, width;
  int32_t blocks;        // 16-row blocks of the table a workgroup
  Targets targets;
  float2* part;          // [workgroups][rows]
  float* tlogit;
};
// four neighbours of a row from column k, zeros behind its `width`: loads without a branch, so that many are in flight
__device__ __forceinline__ f32x4 load4(const float* row, bool wide, int k, int width) {
  f32x4 v;
  if (wide) {
    v = *(const f32x4*)(row + min(k, width - 4));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = row[min(k + j, width - 1)];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = k + j < width ? v[j] : 0.0f;
  return v;
}
// `blocks` 16-row blocks of the table and 16 NB positions: the four waves take every fourth 16 columns, and each finishes a
// block of 16 positions
template <int NB>
__global__ __launch_bounds__(256) void k_few(FewArgs a) {
  __shared__ f32x4 sm[4][NB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.y * 16 * NB;
  const float* xrow[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) xrow[j] = a.x + min(n0 + 16 * j + r, a.rows - 1) * a.ldx;
  const bool mine = wave < NB;
  const int n = n0 + 16 * wave + r;
  int target = -1;
  bool counts = false;
  if (mine && n < a.rows) target = target_of(a.targets, n, counts);
  float mx = -__builtin_inff(), sum = 0.0f;
  const int first = blockIdx.x * a.blocks * 16, last = min(first + a.blocks * 16, a.vocab);
  for (int v0 = first; v0 < last; v0 += 16) {
    const float* wrow = a.w + min(v0 + r, a.vocab - 1) * a.ldw;
    f32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = {0, 0, 0, 0};
    constexpr int U = NB == 1 ? 4 : 2;
    for (int k0 = wave * 16; k0 < a.width; k0 += 64 * U) {
      f32x4 wv[U], xv[U][NB];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 64 * u + 4 * g;
        wv[u] = load4(wrow, a.wide, k, a.width);
#pragma unroll
        for (int j = 0; j < NB; ++j) xv[u][j] = load4(xrow[j], a.wide, k, a.width);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[u][e], xv[u][j][e], acc[j], 0, 0, 0);
    }
    __syncthreads();  // the block before has been read
#pragma unroll
    for (int j = 0; j < NB; ++j) sm[wave][j][lane] = acc[j];
    __syncthreads();
    if (!mine) continue;
    f32x4 l = {0, 0, 0, 0};
    for (int w = 0; w < 4; ++w) l += sm[w][wave][lane];
    const int v = v0 + 4 * g;
    float m = mx;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (v + q >= a.vocab) l[q] = -__builtin_inff();
      else if (v + q == target) a.tlogit[n] = l[q];
      m = fmaxf(m, l[q]);
    }
    const float safe = m == -__builtin_inff() ? 0.0f : m;
    sum *= exp2_fast((mx - safe) * LOG2E);
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += exp2_fast((l[q] - safe) * LOG2E);
    mx = m;
  }
  if (!mine) return;
  const float top = col_max(mx), safe = top == -__builtin_inff() ? 0.0f : top;
  sum = col_sum(sum * exp2_fast((mx - safe) * LOG2E));
  if (lane < 16 && n < a.rows) a.part[(int64_t)blockIdx.x * a.rows + n] = make_float2(top, sum);
}

struct QuantArgs {
  const void* src;
  int64_t ld, ldq;
  int64_t rows;
  int32_t width, width_pad, type;  // columns width .. width_pad - 1 become zeros
  int8_t* q;
  float* scale;
  int32_t wide_in, wide_out;       // rows allow 16-byte loads, 8-byte stores
};
// eight neighbours of a row from column c, zeros behind the last; `wide`: 16-byte loads
__device__ __forceinline__ void load8(const QuantArgs& a, int64_t row, int c, float* v) {
  if (a.wide_in && c + 8 <= a.width) {
    if (a.type == PST_F32) {
      const f32x4 lo = *(const f32x4*)((const float*)a.src + row + c), hi = *(const f32x4*)((const float*)a.src + row + c + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
    } else {
      const uint4 w = *(const uint4*)((const uint16_t*)a.src + row + c);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t h = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
        v[j] = a.type == PST_BF16 ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < a.width ? load1(a.src, a.type, row + c + j) : 0.0f;
}
// One wave a row: the largest magnitude, then rint(x / s), rows of up to 512 ITERS values read once. A row that holds
// an infinity or a NaN gets the scale NaN and zeros, so that what is computed from it says so. 16 x 1024 4 us, 8192 x 1024
// f16 15 us (25 MB: its launch and two passes of latency; through a reciprocal instead of the division it took as long).
template <int ITERS>
__global__ __launch_bounds__(256) void k_quantize(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const int64_t row = r * a.ld;
  float held[ITERS ? ITERS : 1][8];
  float m = 0.0f;
  bool bad = false;
  auto look = [&](const float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad |= !(fabsf(v[j]) <= 3.4028234663852886e38f);
      m = fmaxf(m, fabsf(v[j]));
    }
  };
  if (ITERS) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) load8(a, row, i * 512 + lane * 8, held[i]);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) look(held[i]);
  } else {
    for (int c = lane * 8; c < a.width; c += 512) {
      load8(a, row, c, held[0]);
      look(held[0]);
    }
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
  bad = __any(bad);
  const float s = m * (1.0f / 127.0f);
  if (lane == 0) a.scale[r] = bad ? __builtin_nanf("") : s;
  const bool zero = bad || !(s > 0.0f);
  auto write = [&](int c, const float* v) {
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)  // (a subnormal scale can make the quotient pass 127)
      q[j] = zero ? 0u : (uint32_t)(int)fminf(fmaxf(rintf(v[j] / s), -127.0f), 127.0f) & 255u;
    int8_t* to = a.q + r * a.ldq + c;
    if (a.wide_out && c + 8 <= a.width_pad) {
      *(uint2*)to = make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.width_pad) to[j] = (int8_t)q[j];
    }
  };
  if (ITERS) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
      if (i * 512 + lane * 8 < a.width_pad) write(i * 512 + lane * 8, held[i]);
  } else {
    for (int c = lane * 8; c < a.width_pad; c += 512) {
      load8(a, row, c, held[0]);
      write(c, held[0]);
    }
  }
}
// 8-bit rows into whole K-steps, four neighbours a thread
__global__ __launch_bounds__(256) void k_pack8(const int8_t* src, int64_t ld, int64_t rows, int32_t width, int32_t width_pad, int8_t* dst) {
  const Spread at_row(blockIdx.x, gridDim.x, width_pad / 4);
  for (int64_t r = at_row.row; r < rows; r += at_row.rows)
    for (int c = at_row.piece * 4; c < width_pad; c += at_row.pieces * 4) {
      uint32_t v = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < width) v |= (uint32_t)(uint8_t)src[r * ld + c + j] << (8 * j);
      *(uint32_t*)(dst + r * width_pad + c) = v;
    }
}

// ------------------------------------------------------------------ host
thread_local std::string g_error;

int fail(int code, const std::string& what) {
  g_error = what;
  return code;
}
// a runtime error is reported here, and not again by the caller's next call
int hip_fail(const std::string& what, hipError_t e) {
  (void)hipGetLastError();
  return fail(PST_E_HIP, what + ": " + hipGetErrorString(e));
}
#define HEADCHK(x)                                       \
  do {                                                   \
    const hipError_t e_ = (x);                           \
    if (e_ != hipSuccess) return hip_fail(#x, e_);       \
  } while (0)

// the calling thread's current device, put back on return
struct OnDevice {
  int old = -1;
  hipError_t e;
  explicit OnDevice(int device) {
    e = hipGetDevice(&old);
    if (e == hipSuccess && old != device) {
      e = hipSetDevice(device);
    } else if (e == hipSuccess) {
      old = -1;
    }
  }
  ~OnDevice() {
    if (e == hipSuccess && old >= 0) (void)hipSetDevice(old);
  }
};

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int size_of(int type) { return type == PST_F32 ? 4 : 2; }
bool is_type(int type) { return type == PST_F32 || type == PST_BF16 || type == PST_F16; }

// offsets in the caller's workspace
struct Bump {
  int64_t n = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = n;
    n += up(bytes, 256);
    return at;
  }
};

// a matrix that the kernels read where it is: 16-byte rows of whole 16-byte pieces
bool in_place(const void* p, int64_t ld_bytes, int64_t row_bytes) {
  return ((uintptr_t)p & 15) == 0 && ld_bytes % 16 == 0 && row_bytes % 16 == 0;
}

enum TileId { TILE64 = 0, TILE128 = 1, TILE256 = 2, FLOAT64 = 3, FLOAT128 = 4 };
constexpr int TILE_M[5] = {64, 128, 256, 64, 128};

// ---- the choice of tiles
// Times of a workgroup in us, fitted to launches on the card (d = 256 ... 1024, 16 ... 8192 positions): BASE and, for
// each K-step of 64, STEP + MORE for each workgroup that shares the compute unit, up to `slots` of them. Over 71 sizes of the
// loss and the scores with each tile forced, what the estimate takes is 0.4 % slower than the fastest (8 % at most). The largest
// tiles reach 1.3 PFLOP/s, those of 128 about 0.95, those of 64 about 0.65; the smaller ones fill the card sooner. The two
// of 32-bit values, whose K-steps are of 32, are bound by their instructions alone (0.14 PFLOP/s of tiles of 128, 0.13 of 64).
constexpr int CUS = 256;  // the card's compute units, whatever device is asked: a workspace's size needs none
constexpr double TILE_BASE[5] = {2.0, 3.0, 4.0, 2.0, 3.0}, TILE_STEP[5] = {0.45, 0.55, 1.5, 0.1, 0.0}, TILE_MORE[5] = {0.1, 0.27, 0.0, 0.45, 1.75};
constexpr int TILE_SLOTS[5] = {4, 2, 1, 4, 2};
constexpr double THIN[5] = {0.0, 0.6, 0.35, 0.0, 0.15};  // a thin tile's time, of a whole one's
double tile_us(int tile, double share, int64_t steps) { return TILE_BASE[tile] + (TILE_STEP[tile] + TILE_MORE[tile] * share) * steps; }
int64_t tiles_of(int64_t m, int64_t n, int tile) { return ceil_div(m, TILE_M[tile]) * ceil_div(n, TILE_M[tile]); }
// rows that thin tiles take
int64_t thin_rows(int64_t m, int tile) {
  const int64_t rest = m % TILE_M[tile];
  return THIN[tile] > 0 && m > rest && rest <= 64 ? rest : 0;
}
// m x n of the loss, the logits' gradient and the scores; a compute unit stores about 20 KB in a us (5 TB/s of all)
int tile_for(int64_t m, int64_t n, int64_t steps, bool f32, int out_bytes, double* estimate = nullptr) {
  int best = TILE64;
  double us = 1e30;
  for (int t = f32 ? FLOAT128 : TILE256; t >= (f32 ? FLOAT64 : TILE64); --t) {
    const int64_t thin = thin_rows(m, t), slots = (int64_t)CUS * TILE_SLOTS[t], full = tiles_of(m - thin, n, t);
    // whole rounds with all slots taken, and a last one whose units have fewer workgroups
    const auto round = [&](int64_t share) { return tile_us(t, share, steps) + (double)TILE_M[t] * TILE_M[t] * out_bytes * share / 20e3; };
    const double whole = round(TILE_SLOTS[t]), last = full % slots ? round(ceil_div(full % slots, CUS)) : whole;
    double e = full / slots * whole + (full % slots ? last : 0.0);
    if (thin && full + ceil_div(n, 64) > ceil_div(full, slots) * slots) e += THIN[t] * last;  // not into what the last round leaves free
    if (e < us) us = e, best = t;
  }
  if (estimate) *estimate = us;
  return best;
}

template <class F, class A>
hipError_t launch(F* f, int64_t grid, int threads, int lds, hipStream_t st, const A& g) {
  if (grid > 0x7fffffff) return hipErrorInvalidConfiguration;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(f, dim3((unsigned)grid), dim3(threads), lds, st, g);
  return hipGetLastError();
}
template <int E, class T>
hipError_t launch_kind(int kind, const GemmArgs& g, int64_t grid, hipStream_t st) {
  constexpr int LDS = T::LDS + EPILOGUE_LDS;
  if constexpr (E == I8) {
    return launch(k_scores<T>, grid, T::THREADS, LDS, st, g);
  } else {
    return kind == LOSS ? launch(k_loss<E, T>, grid, T::THREADS, LDS, st, g) : launch(k_dlogit<E, T>, grid, T::THREADS, LDS, st, g);
  }
}
void set_tiles(GemmArgs& g, int64_t m, int64_t n, int tile) {
  g.nm = (int32_t)ceil_div(m, TILE_M[tile]);
  g.nn = (int32_t)ceil_div(n, TILE_M[tile]);
  g.nz = std::max(g.nz, 1);
  g.gm = 4;
}
template <int E>
hipError_t launch_elem(int kind, int tile, const GemmArgs& g, int64_t grid, hipStream_t st) {
  if constexpr (E == F32) {
    return tile == FLOAT128 ? launch_kind<E, T128>(kind, g, grid, st) : launch_kind<E, T64>(kind, g, grid, st);
  } else {
    return tile == TILE256   ? launch_kind<E, T256>(kind, g, grid, st)
           : tile == TILE128 ? launch_kind<E, T128>(kind, g, grid, st)
                             : launch_kind<E, T64>(kind, g, grid, st);
  }
}
hipError_t launch_gemm(int kind, int elem, int tile, GemmArgs g, hipStream_t st) {
  const int64_t thin = thin_rows(g.M, tile);
  set_tiles(g, g.M - thin, g.N, tile);
  const int64_t tiles = (int64_t)g.nm * g.nn;
  if (tiles > 0x3fffffff) return hipErrorInvalidConfiguration;
  g.blocks = (int32_t)std::min<int64_t>(tiles, (int64_t)CUS * TILE_SLOTS[tile]);
  g.thins = (int32_t)ceil_div(g.N, 64);
  const int64_t grid = g.blocks + (thin ? g.thins : 0);
  return elem == I8     ? launch_elem<I8>(kind, tile, g, grid, st)
         : elem == BF16 ? launch_elem<BF16>(kind, tile, g, grid, st)
         : elem == F32  ? launch_elem<F32>(kind, tile, g, grid, st)
                        : launch_elem<F16>(kind, tile, g, grid, st);
}
hipError_t launch_grads(int tile, GradArgs g, bool dx, bool dw, hipStream_t st) {
  int64_t grid = 0;
  for (int i = 0; i < 2; ++i) {
    GemmArgs& q = i ? g.dw : g.dx;
    const int64_t thin = thin_rows(q.N, tile);
    set_tiles(q, i ? q.M : q.ldp, q.N - thin, tile);
    const bool on = i ? dw : dx;
    q.thins = (int32_t)ceil_div(i ? q.M : q.ldp, 64);
    const int64_t blocks = on ? (int64_t)q.nm * q.nn * q.nz : 0, thins = on && thin ? (int64_t)q.thins * q.nz : 0;
    grid += blocks + thins;
    if (grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    g.blocks[i] = (int32_t)blocks;
    g.blocks[2 + i] = (int32_t)thins;
  }
  return tile == FLOAT64   ? launch(k_grads<F32, T64>, grid, T64::THREADS, T64::LDS, st, g)
         : tile == TILE256 ? launch(k_grads<BF16, T256>, grid, T256::THREADS, T256::LDS, st, g)
         : tile == TILE128 ? launch(k_grads<BF16, T128>, grid, T128::THREADS, T128::LDS, st, g)
                           : launch(k_grads<BF16, T64>, grid, T64::THREADS, T64::LDS, st, g);
}

// What a call on [rows, width] x [vocab, width] needs of its workspace; the same for the query and for the call.
struct Plan {
  int type, elem;
  int products;                                  // of each gradient (see Loop)
  int64_t rows, vocab, width, width_pad, rows_pad;
  bool pack_x, pack_w;
  int64_t x = 0, w = 0;                          // offsets
  int64_t part = 0, tlogit = 0;                  // loss
  int64_t xh = 0, wh = 0, D = 0, dxp = 0, dwp = 0;  // gradient
  int64_t few = 0;                               // k_few: 16-row blocks a workgroup
  int64_t span = 0, piece = 0;                   // positions and vocabulary rows of a piece of D
  int tile = 0, zx = 1, zw = 1;                  // of the two gradients' launch
  int64_t bytes = 0;
};
Plan plan_common(int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width, bool grad, Bump& b) {
  Plan p;
  p.type = type;
  p.elem = type == PST_F32 ? F32 : type == PST_BF16 ? BF16 : F16;
  p.products = type == PST_BF16 ? 2 : type == PST_F16 ? 3 : 1;
  p.rows = rows;
  p.vocab = vocab;
  p.width = width;
  const int e = size_of(type);
  p.width_pad = up(width, STEP / e);
  p.rows_pad = grad ? up(rows, 64) : rows;
  p.pack_w = !in_place(w, ldw * e, width * e);
  // x is the operand with zeros behind the last column; the gradient needs zeros behind the last row too
  p.pack_x = grad || p.width_pad != width || !in_place(x, ldx * e, width * e);
  if (p.pack_x) p.x = b.take(p.rows_pad * p.width_pad * e);
  if (p.pack_w) p.w = b.take(vocab * p.width_pad * e);
  return p;
}
Plan plan_loss(int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width) {
  Bump b;
  Plan p = plan_common(type, x, ldx, w, ldw, rows, vocab, width, false, b);
  // Up to 16 positions of aligned rows, or a product of about what its launches take (see k_few). A call, this kernel and
  // the tiles, us: 1, 16, 32 x 64000 x 1024 48, 67, 96 and 74; 16 x 4096 x 2048 16 and 45; 64 x 4096 x 1024 20 and 26;
  // 256 x 4096 x 256 16 and 15; of 333 columns, whose rows are not aligned, 1, 16 x 64000 57, 87 and 74.
  const bool aligned = in_place(x, ldx * 4, width * 4) && in_place(w, ldw * 4, width * 4);
  if (type == PST_F32 && ((rows <= 16 && aligned) || (rows <= 1024 && rows * vocab * width <= 1 << 28))) {
    b = Bump();
    // about four workgroups a compute unit
    p.few = ceil_div(ceil_div(vocab, 16), 4 * CUS);
    p.part = b.take(ceil_div(vocab, 16 * p.few) * rows * 8);
    p.tlogit = b.take(rows * 4);
    p.bytes = b.n;
    return p;
  }
  p.tile = tile_for(vocab, rows, p.width_pad * size_of(type) / STEP, type == PST_F32, 0);
  p.part = b.take(ceil_div(vocab, TILE_M[p.tile]) * rows * 8);
  p.tlogit = b.take(rows * 4);
  p.bytes = b.n;
  return p;
}
// The tiles of the two gradients' launch and the parts zx, zw of their K loops, for pieces of nv vocabulary rows: the least of
// the estimated launch and of the parts' way back through memory (4.5 TB/s), which is returned. 32-bit operands: tiles of 64
// alone, which fill the card sooner and lose nothing to those of 128 (both gradients, us: 300 x 432 x 512 29 and 36,
// 4096 x 4099 x 512 427 and 455, 2048 x 8192 x 2048 1493 and 1481).
double split_grads(Plan& p, int64_t nv, bool pieces) {
  constexpr int Z[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
  const bool f32 = p.type == PST_F32;
  const int64_t ks = STEP / (f32 ? 4 : 2), sx = p.products * ceil_div(nv, ks), sw = p.products * ceil_div(p.rows, ks), least = 4;
  double best = 1e30;
  for (int t = f32 ? FLOAT64 : TILE256; t >= (f32 ? FLOAT64 : TILE64); --t) {
    const int64_t thin_x = thin_rows(p.rows, t), thin_w = thin_rows(nv, t);
    const double slots = (double)CUS * TILE_SLOTS[t];
    const double one_x = tiles_of(p.width_pad, p.rows - thin_x, t), one_w = tiles_of(p.width, nv - thin_w, t);
    const double thins_x = thin_x ? ceil_div(p.width_pad, 64) : 0, thins_w = thin_w ? ceil_div(p.width, 64) : 0;
    for (int zx : Z)
      for (int zw : Z) {
        if ((zx > 1 && sx < least * zx) || (zw > 1 && (pieces || sw < least * zw))) continue;
        const double n = one_x * zx + one_w * zw, thins = thins_x * zx + thins_w * zw;
        const double share = std::min<double>(TILE_SLOTS[t], std::max(1.0, n / CUS));
        const double tx = tile_us(t, share, ceil_div(sx, zx)), tw = tile_us(t, share, ceil_div(sw, zw)), longest = std::max(tx, tw);
        double us = longest;
        // both kinds share the slots; the last to start ends half its time behind the rest
        if (n > slots) us = std::max((one_x * zx * tx + one_w * zw * tw) / slots + 0.5 * longest, longest + std::min(tx, tw));
        if (n + thins > ceil_div((int64_t)n, (int64_t)slots) * slots) us += THIN[t] * longest;
        us += 4.0 * p.width_pad * (p.rows * (double)zx + (zw > 1 ? nv * (double)zw : 0.0)) / 4.5e6 + 0.3 * (zx + zw);
        if (us < best) best = us, p.tile = t, p.zx = zx, p.zw = zw;
      }
  }
  return best;
}
// The vocabulary rows of a piece, `most` at most, and how its gradients are made: of the fewest pieces and a few more, what is
// estimated to take least, since a piece whose tiles fill the card unevenly, or whose two gradients have K loops of very different
// lengths, costs more than another launch. By a rule that filled whole rounds alone, and so (bf16, ms): 8448 x 64003 x 1024
// 5.8 and 5.0, 2048 x 64003 x 1024 1.46 and 1.22, 8192 x 64003 x 1024 4.55 and 4.55. The last choice
// is kept, by the sizes alone.
void choose_pieces(Plan& p, int64_t most) {
  struct Last {
    int64_t rows = -1, vocab, width, piece;
    int products, tile, zx, zw;
  };
  thread_local Last last;
  if (last.rows != p.rows || last.vocab != p.vocab || last.width != p.width || last.products != p.products) {
    const int64_t fewest = ceil_div(p.vocab, most), steps = p.width_pad * size_of(p.type) / STEP;
    double best = 1e30;
    for (int64_t k = fewest; k <= (fewest > 1 ? fewest + 8 : 1); ++k) {
      const int64_t piece = up(ceil_div(p.vocab, k), 256);
      double us;
      (void)tile_for(std::min(piece, p.vocab), p.rows, steps, p.type == PST_F32, 4, &us);
      us = (us + split_grads(p, std::min(piece, p.vocab), k > 1) + 10.0) * ceil_div(p.vocab, piece);
      if (us < best) best = us, last.piece = piece, last.tile = p.tile, last.zx = p.zx, last.zw = p.zw;
    }
    last.rows = p.rows;
    last.vocab = p.vocab;
    last.width = p.width;
    last.products = p.products;
  }
  p.piece = last.piece;
  p.tile = last.tile;
  p.zx = last.zx;
  p.zw = last.zw;
}
// D is made in pieces of about what the last-level cache (256 MB) holds: of all positions by as many vocabulary rows, or of
// SPAN positions at least, since each piece of the vocabulary adds to the sums of its positions' dx in memory, and each
// span of positions to those of all of dW.
constexpr int64_t PIECE_BYTES = 288ll << 20, SPAN = 8192;
Plan plan_grad(int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width) {
  const int64_t longest = std::max(SPAN, PIECE_BYTES / (4 * up(vocab, 256)) / 256 * 256);
  const int64_t span = rows <= longest ? rows : up(ceil_div(rows, ceil_div(rows, longest)), 256);
  Bump b;
  Plan p = plan_common(type, x, ldx, w, ldw, span, vocab, width, true, b);
  p.span = span;
  if (type == PST_F16) {
    p.xh = b.take(p.rows_pad * p.width_pad * 4);
    p.wh = b.take(vocab * p.width_pad * 4);
  }
  const int64_t drows = up(span, 256);
  choose_pieces(p, PIECE_BYTES / (drows * 4) / 256 * 256);
  p.D = b.take(drows * p.piece * 4);
  p.dxp = b.take(p.zx * span * p.width_pad * 4);
  if (p.zw > 1 || rows > span) p.dwp = b.take(p.zw * vocab * p.width_pad * 4);
  p.bytes = b.n;
  return p;
}

int check_sizes(int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width) {
  if (!is_type(type)) return fail(PST_E_INVALID, "unknown type");
  if (rows < 0 || vocab < 1 || width < 1) return fail(PST_E_INVALID, "rows >= 0, vocab >= 1 and width >= 1 are needed");
  if (rows > (1ll << 30) || vocab > (1ll << 30) || width > (1 << 20)) return fail(PST_E_TOO_LARGE, "rows or vocab over 2^30, or width over 2^20");
  if (ldx < width || ldw < width) return fail(PST_E_INVALID, "a row stride is smaller than the width");
  if (ldx > (1 << 21) || ldw > (1 << 21)) return fail(PST_E_TOO_LARGE, "a row stride over 2^21");
  const int e = size_of(type);
  if (rows && (!x || ((uintptr_t)x % e))) return fail(PST_E_INVALID, "hidden is null or not aligned to its type");
  if (!w || ((uintptr_t)w % e)) return fail(PST_E_INVALID, "weight is null or not aligned to its type");
  return PST_OK;
}
int check_targets(const void* targets, int bits, int64_t rows) {
  if (bits != 32 && bits != 64) return fail(PST_E_INVALID, "targets are 32 or 64 bits wide");
  if (rows && (!targets || ((uintptr_t)targets % (bits / 8)))) return fail(PST_E_INVALID, "targets are null or not aligned");
  return PST_OK;
}
int check_ws(const void* ws, int64_t have, int64_t need) {
  if (have < need) return fail(PST_E_INVALID, "workspace of " + std::to_string(have) + " bytes, " + std::to_string(need) + " are needed");
  if (!ws || ((uintptr_t)ws & 255)) return fail(PST_E_INVALID, "the workspace is null or not aligned to 256 bytes");
  return PST_OK;
}

// workgroups of the kernels that go through rows by a Spread: each thread one row, up to a few workgroups a compute unit
int32_t row_grid(int64_t rows, int64_t per_row) {
  int shift = 0;
  while (shift < 6 && (1 << shift) < per_row) ++shift;
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows << shift, 256), CUS * 16ll));
}

// the operands in a form that the products read: in place, or packed into the workspace; for the gradient (`grad`) of f16
// also their bf16 halves; `table`: the table's too, or they are there. One launch, none where there is nothing to do.
int operands(const Plan& p, const void* x, int64_t ldx, int64_t rows, const void* w, int64_t ldw, bool table, const Targets& t, bool grad, char* ws,
             hipStream_t st, Operand* X, Operand* W) {
  const int e = size_of(p.type);
  PackArgs a{};
  a.bytes = (int32_t)(p.width * e);
  a.bytes_pad = (int32_t)(p.width_pad * e);
  a.type = p.type;
  a.targets = t;
  const bool halves = grad && p.type == PST_F16;
  auto job = [&](int which, const void* src, int64_t ld, int64_t rows, int64_t rows_pad, bool copy, int64_t at, int64_t half) {
    PackJob& j = a.job[which];
    j = {(const char*)src, ld * e, rows, rows_pad, copy ? ws + at : nullptr, halves ? ws + half : nullptr, which == 0 && grad,
         ((uintptr_t)src & 15) == 0 && ld * e % 16 == 0};
    a.blocks[which] = row_grid(rows_pad, a.bytes_pad / (j.wide ? 16 : 4));
  };
  const int64_t rows_pad = grad ? up(std::max<int64_t>(rows, 1), 64) : rows;
  *X = p.pack_x ? Operand{ws + p.x, 0, a.bytes_pad, (int32_t)rows_pad, a.bytes_pad} : Operand{(const char*)x, 0, ldx * e, (int32_t)rows, a.bytes};
  *W = p.pack_w ? Operand{ws + p.w, 0, a.bytes_pad, (int32_t)p.vocab, a.bytes_pad} : Operand{(const char*)w, 0, ldw * e, (int32_t)p.vocab, a.bytes};
  if (p.pack_x) job(0, x, ldx, rows, rows_pad, true, p.x, p.xh);
  if (table && (p.pack_w || halves)) job(1, w, ldw, p.vocab, p.vocab, p.pack_w, p.w, p.wh);
  if (a.blocks[0] + a.blocks[1]) {
    hipLaunchKernelGGL(k_pack, dim3((unsigned)(a.blocks[0] + a.blocks[1])), dim3(256), 0, st, a);
    HEADCHK(hipGetLastError());
  }
  return PST_OK;
}

hipError_t launch_few(const FewArgs& f, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(f.vocab, 16ll * f.blocks), (unsigned)ceil_div(f.rows, 64)), block(256);
  if (f.rows <= 16) hipLaunchKernelGGL(k_few<1>, grid, block, 0, st, f);
  else if (f.rows <= 32) hipLaunchKernelGGL(k_few<2>, grid, block, 0, st, f);
  else hipLaunchKernelGGL(k_few<4>, grid, block, 0, st, f);
  return hipGetLastError();
}

int token_loss(int device, int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width,
               const void* targets, int tbits, int64_t ignore, float* loss, float* lse, void* ws_, int64_t ws_bytes, hipStream_t st) {
  int rc = check_sizes(type, x, ldx, w, ldw, rows, vocab, width);
  if (rc == PST_OK) rc = check_targets(targets, tbits, rows);
  if (rc != PST_OK) return rc;
  if (rows == 0) return PST_OK;
  if (!loss || !lse || ((uintptr_t)loss & 3) || ((uintptr_t)lse & 3)) return fail(PST_E_INVALID, "loss or lse is null or not aligned");
  const Plan p = plan_loss(type, x, ldx, w, ldw, rows, vocab, width);
  rc = check_ws(ws_, ws_bytes, p.bytes);
  if (rc != PST_OK) return rc;
  OnDevice on(device);
  if (on.e != hipSuccess) return hip_fail("device " + std::to_string(device), on.e);
  char* ws = (char*)ws_;
  GemmArgs g{};
  g.targets = {targets, ignore, tbits, (int32_t)vocab};
  if (p.few) {
    const bool wide = in_place(x, ldx * 4, width * 4) && in_place(w, ldw * 4, width * 4);
    const FewArgs f{(const float*)x, (const float*)w, ldx, ldw, wide, (int32_t)rows, (int32_t)vocab, (int32_t)width, (int32_t)p.few, g.targets,
                    (float2*)(ws + p.part), (float*)(ws + p.tlogit)};
    HEADCHK(launch_few(f, st));
    launch_join({f.part, f.tlogit, f.targets, loss, lse, (int32_t)rows, (int32_t)ceil_div(vocab, 16 * p.few)}, st);
    HEADCHK(hipGetLastError());
    return PST_OK;
  }
  rc = operands(p, x, ldx, rows, w, ldw, true, g.targets, false, ws, st, &g.B, &g.A);
  if (rc != PST_OK) return rc;
  g.M = (int32_t)vocab;
  g.N = (int32_t)rows;
  g.steps = (int32_t)(p.width_pad * size_of(type) / STEP);
  g.part = (float2*)(ws + p.part);
  g.tlogit = (float*)(ws + p.tlogit);
  HEADCHK(launch_gemm(LOSS, p.elem, p.tile, g, st));
  JoinArgs j{g.part, g.tlogit, g.targets, loss, lse, (int32_t)rows, (int32_t)ceil_div(vocab, TILE_M[p.tile])};
  launch_join(j, st);
  HEADCHK(hipGetLastError());
  return PST_OK;
}

int token_loss_grad(int device, int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width,
                    const void* targets, int tbits, int64_t ignore, const float* lse, const float* gloss, void* dx, int64_t lddx, void* dw,
                    int64_t lddw, void* ws_, int64_t ws_bytes, hipStream_t st) {
  int rc = check_sizes(type, x, ldx, w, ldw, rows, vocab, width);
  if (rc == PST_OK) rc = check_targets(targets, tbits, rows);
  if (rc != PST_OK) return rc;
  const int e = size_of(type);
  if ((dx && lddx < width) || (dw && lddw < width)) return fail(PST_E_INVALID, "a gradient's row stride is smaller than the width");
  if (((uintptr_t)dx % e) || ((uintptr_t)dw % e)) return fail(PST_E_INVALID, "a gradient is not aligned to its type");
  if (!dx && !dw) return PST_OK;
  if (rows && (!lse || !gloss || ((uintptr_t)lse & 3) || ((uintptr_t)gloss & 3)))
    return fail(PST_E_INVALID, "lse or grad_loss is null or not aligned");
  if (rows == 0 && !dw) return PST_OK;
  const Plan p = plan_grad(type, x, ldx, w, ldw, std::max<int64_t>(rows, 1), vocab, width);
  rc = check_ws(ws_, ws_bytes, p.bytes);
  if (rc != PST_OK) return rc;
  OnDevice on(device);
  if (on.e != hipSuccess) return hip_fail("device " + std::to_string(device), on.e);
  char* ws = (char*)ws_;
  const int de = type == PST_F32 ? 4 : 2, ks = STEP / de;  // bytes of D's values, K-steps' values
  char* D = ws + p.D;
  const bool spans = rows > p.span;
  // no positions: 64 of zeros stand for them, so that dW is written as the zeros that it is
  for (int64_t n0 = 0; n0 < std::max<int64_t>(rows, 1); n0 += p.span) {
    const int64_t n = std::min(p.span, rows - n0), drows = up(std::max<int64_t>(n, 1), 256);
    const bool last = n0 + p.span >= rows, need_dx = dx && n;
    const Targets t{targets ? (const char*)targets + n0 * (tbits / 8) : nullptr, ignore, tbits, (int32_t)vocab};
    Operand X, W;
    rc = operands(p, x ? (const char*)x + n0 * ldx * e : nullptr, ldx, n, w, ldw, n0 == 0, t, true, ws, st, &X, &W);
    if (rc != PST_OK) return rc;
    // what the gradients' products read
    const Operand Xh = type == PST_F16 ? Operand{ws + p.xh, X.rows * X.ld, X.ld, X.rows, X.bytes} : X;
    const Operand Wh = type == PST_F16 ? Operand{ws + p.wh, vocab * X.ld, X.ld, (int32_t)vocab, X.bytes} : W;
    for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
      const int64_t nv = std::min(p.piece, vocab - v0), ldd = up(nv, 256);
      const Operand dop{D, drows * ldd * de, ldd * de, (int32_t)drows, (int32_t)(ldd * de)};
      GemmArgs g{};
      g.A = W;
      g.A.p += v0 * W.ld;
      g.A.rows = (int32_t)nv;
      g.B = X;
      g.M = (int32_t)nv;
      g.N = (int32_t)n;
      g.steps = (int32_t)(p.width_pad * e / STEP);
      g.targets = t;
      g.lse = lse + n0;
      g.gloss = gloss + n0;
      g.D = D;
      g.dplane = dop.plane;
      g.ldd = ldd;
      g.v0 = (int32_t)v0;
      if (n) HEADCHK(launch_gemm(DLOGIT, p.elem, tile_for(nv, n, g.steps, type == PST_F32, 4), g, st));
      GradArgs b{};
      b.dx.A = Wh;
      b.dx.A.p += v0 * Wh.ld;
      b.dx.A.rows = (int32_t)nv;
      b.dw.A = Xh;
      b.dx.B = b.dw.B = dop;
      b.dx.M = b.dw.M = (int32_t)width;
      b.dx.N = (int32_t)n;
      b.dw.N = (int32_t)nv;
      b.dx.range = (int32_t)ceil_div(nv, ks);
      b.dw.range = (int32_t)ceil_div(n, ks);
      b.dx.products = b.dw.products = p.products;
      b.dx.steps = b.dx.range * p.products;
      b.dw.steps = b.dw.range * p.products;
      b.dx.nz = p.zx;
      b.dw.nz = p.zw;
      b.dx.ldp = b.dw.ldp = p.width_pad;
      b.dx.part_out = (float*)(ws + p.dxp);
      b.dx.zstride = n * p.width_pad;
      b.dx.add = v0 > 0;
      if (p.zw > 1 || spans) {
        b.dw.part_out = (float*)(ws + p.dwp) + v0 * p.width_pad;
        b.dw.zstride = vocab * p.width_pad;
        b.dw.add = n0 > 0;
      }
      b.dw.v0 = (int32_t)v0;
      b.dw.out = dw;
      b.dw.ldo = lddw;
      b.dw.otype = type;
      b.dw.wide = lddw % (16 / e) == 0 && ((uintptr_t)dw & 15) == 0;
      HEADCHK(launch_grads(p.tile, b, need_dx, dw != nullptr, st));
    }
    FinishArgs f{};
    f.width = (int32_t)width;
    f.otype = type;
    f.targets = t;
    auto job = [&](int which, int64_t part, int64_t count, int nz, char* out, int64_t ldo) {
      f.job[which] = {(const float*)(ws + part), p.width_pad, count * p.width_pad, count, nz, which == 0, out, ldo,
                      ldo % 4 == 0 && ((uintptr_t)out & (type == PST_F32 ? 15 : 7)) == 0};
      f.blocks[which] = row_grid(count, ceil_div(width, 4));
    };
    if (need_dx) job(0, p.dxp, n, p.zx, (char*)dx + n0 * lddx * e, lddx);
    if (dw && last && (p.zw > 1 || spans)) job(1, p.dwp, vocab, p.zw, (char*)dw, lddw);
    if (f.blocks[0] + f.blocks[1]) {
      hipLaunchKernelGGL(k_finish, dim3((unsigned)(f.blocks[0] + f.blocks[1])), dim3(256), 0, st, f);
      HEADCHK(hipGetLastError());
    }
  }
  return PST_OK;
}

hipError_t launch_quantize(QuantArgs a, hipStream_t st) {
  a.wide_in = in_place(a.src, a.ld * size_of(a.type), 16);
  a.wide_out = ((uintptr_t)a.q & 7) == 0 && a.ldq % 8 == 0;
  const dim3 grid((unsigned)ceil_div(a.rows, 4)), block(256);
  if (a.width_pad <= 512) hipLaunchKernelGGL(k_quantize<1>, grid, block, 0, st, a);
  else if (a.width_pad <= 1024) hipLaunchKernelGGL(k_quantize<2>, grid, block, 0, st, a);
  else if (a.width_pad <= 2048) hipLaunchKernelGGL(k_quantize<4>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_quantize<0>, grid, block, 0, st, a);
  return hipGetLastError();
}

int quantize_rows(int device, int type, const void* x, int64_t ldx, int64_t rows, int64_t width, int8_t* q, int64_t ldq, float* scale,
                  hipStream_t st) {
  if (!is_type(type)) return fail(PST_E_INVALID, "unknown type");
  if (rows < 0 || width < 1) return fail(PST_E_INVALID, "rows >= 0 and width >= 1 are needed");
  if (rows > (1ll << 30) || width > (1 << 20)) return fail(PST_E_TOO_LARGE, "rows over 2^30, or width over 2^20");
  if (ldx < width || ldq < width) return fail(PST_E_INVALID, "a row stride is smaller than the width");
  if (rows == 0) return PST_OK;
  if (!x || ((uintptr_t)x % size_of(type)) || !q || !scale || ((uintptr_t)scale & 3))
    return fail(PST_E_INVALID, "a buffer is null or not aligned to its type");
  OnDevice on(device);
  if (on.e != hipSuccess) return hip_fail("device " + std::to_string(device), on.e);
  HEADCHK(launch_quantize({x, ldx, ldq, rows, (int32_t)width, (int32_t)width, type, q, scale, 0, 0}, st));
  return PST_OK;
}

struct ScorePlan {
  int64_t width_pad;
  bool pack_w;
  int64_t q, scale, w, bytes;
};
ScorePlan plan_scores(const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width) {
  ScorePlan p{};
  Bump b;
  p.width_pad = up(width, STEP);
  p.pack_w = !in_place(w, ldw, width);
  p.q = b.take(rows * p.width_pad);
  p.scale = b.take(rows * 4);
  if (p.pack_w) p.w = b.take(vocab * p.width_pad);
  p.bytes = b.n;
  return p;
}
int check_scores(int type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t width) {
  if (!is_type(type)) return fail(PST_E_INVALID, "unknown type");
  if (rows < 0 || vocab < 1 || width < 1) return fail(PST_E_INVALID, "rows >= 0, vocab >= 1 and width >= 1 are needed");
  // 127 * 127 * width has to stay inside 32 bits
  if (rows > (1ll << 30) || vocab > (1ll << 30) || width > 131072) return fail(PST_E_TOO_LARGE, "rows or vocab over 2^30, or width over 131072");
  if (ldx < width || ldw < width) return fail(PST_E_INVALID, "a row stride is smaller than the width");
  if (ldw > (1 << 23)) return fail(PST_E_TOO_LARGE, "a row stride over 2^23");
  if (rows && (!x || ((uintptr_t)x % size_of(type)))) return fail(PST_E_INVALID, "hidden is null or not aligned to its type");
  if (!w) return fail(PST_E_INVALID, "weight is null");
  return PST_OK;
}
int token_scores_i8(int device, int type, const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const float* wscale, int64_t rows, int64_t vocab,
                    int64_t width, int otype, void* out, int64_t ldo, void* ws_, int64_t ws_bytes, hipStream_t st) {
  int rc = check_scores(type, x, ldx, w, ldw, rows, vocab, width);
  if (rc != PST_OK) return rc;
  if (!is_type(otype)) return fail(PST_E_INVALID, "unknown output type");
  if (rows == 0) return PST_OK;
  if (ldo < vocab) return fail(PST_E_INVALID, "the scores' row stride is smaller than the vocabulary");
  if (!wscale || ((uintptr_t)wscale & 3) || !out || ((uintptr_t)out % size_of(otype)))
    return fail(PST_E_INVALID, "scale or scores is null or not aligned");
  const ScorePlan p = plan_scores(w, ldw, rows, vocab, width);
  rc = check_ws(ws_, ws_bytes, p.bytes);
  if (rc != PST_OK) return rc;
  OnDevice on(device);
  if (on.e != hipSuccess) return hip_fail("device " + std::to_string(device), on.e);
  char* ws = (char*)ws_;
  HEADCHK(launch_quantize(
      {x, ldx, p.width_pad, rows, (int32_t)width, (int32_t)p.width_pad, type, (int8_t*)(ws + p.q), (float*)(ws + p.scale), 0, 0}, st));
  GemmArgs g{};
  if (p.pack_w) {
    hipLaunchKernelGGL(k_pack8, dim3(row_grid(vocab, p.width_pad / 4)), dim3(256), 0, st, w, ldw, vocab, (int32_t)width, (int32_t)p.width_pad,
                       (int8_t*)(ws + p.w));
    HEADCHK(hipGetLastError());
    g.A = {ws + p.w, 0, p.width_pad, (int32_t)vocab, (int32_t)p.width_pad};
  } else {
    g.A = {(const char*)w, 0, ldw, (int32_t)vocab, (int32_t)width};
  }
  g.B = {ws + p.q, 0, p.width_pad, (int32_t)rows, (int32_t)p.width_pad};
  g.M = (int32_t)vocab;
  g.N = (int32_t)rows;
  g.steps = (int32_t)(p.width_pad / STEP);
  g.out = out;
  g.ldo = ldo;
  g.otype = otype;
  g.wide = ldo % (16 / size_of(otype)) == 0 && ((uintptr_t)out & 15) == 0;
  g.sn = (const float*)(ws + p.scale);
  g.sm = wscale;
  HEADCHK(launch_gemm(SCORES, I8, tile_for(vocab, rows, g.steps, false, size_of(otype)), g, st));
  return PST_OK;
}

template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return PST_E_NOMEM;
  } catch (...) {
    return PST_E_INVALID;
  }
}

}  // namespace
}  // namespace pst_head

extern "C" {

const char* pst_head_error(void) { return pst_head::g_error.c_str(); }

int64_t pst_token_loss_workspace(int32_t type, const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int64_t rows,
                                 int64_t vocab, int64_t width) {
  using namespace pst_head;
  const int rc = guarded([&]() -> int { return check_sizes(type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width); });
  return rc == PST_OK ? plan_loss(type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width).bytes : rc;
}

int pst_token_loss(int32_t device, int32_t type, const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int64_t rows,
                   int64_t vocab, int64_t width, const void* d_targets, int32_t target_bits, int64_t ignore, float* d_loss, float* d_lse,
                   void* d_workspace, int64_t workspace_bytes, void* stream) {
  return pst_head::guarded([&] {
    return pst_head::token_loss(device, type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width, d_targets, target_bits, ignore, d_loss,
                                d_lse, d_workspace, workspace_bytes, (hipStream_t)stream);
  });
}

int64_t pst_token_loss_grad_workspace(int32_t type, const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int64_t rows,
                                      int64_t vocab, int64_t width) {
  using namespace pst_head;
  const int rc = guarded([&]() -> int { return check_sizes(type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width); });
  return rc == PST_OK ? plan_grad(type, d_hidden, ld_hidden, d_weight, ld_weight, std::max<int64_t>(rows, 1), vocab, width).bytes : rc;
}

int pst_token_loss_grad(int32_t device, int32_t type, const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int64_t rows,
                        int64_t vocab, int64_t width, const void* d_targets, int32_t target_bits, int64_t ignore, const float* d_lse,
                        const float* d_grad_loss, void* d_grad_hidden, int64_t ld_grad_hidden, void* d_grad_weight, int64_t ld_grad_weight,
                        void* d_workspace, int64_t workspace_bytes, void* stream) {
  return pst_head::guarded([&] {
    return pst_head::token_loss_grad(device, type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width, d_targets, target_bits, ignore,
                                     d_lse, d_grad_loss, d_grad_hidden, ld_grad_hidden, d_grad_weight, ld_grad_weight, d_workspace, workspace_bytes,
                                     (hipStream_t)stream);
  });
}

int pst_quantize_rows(int32_t device, int32_t type, const void* d_x, int64_t ld_x, int64_t rows, int64_t width, int8_t* d_q, int64_t ld_q,
                      float* d_scale, void* stream) {
  return pst_head::guarded(
      [&] { return pst_head::quantize_rows(device, type, d_x, ld_x, rows, width, d_q, ld_q, d_scale, (hipStream_t)stream); });
}

int64_t pst_token_scores_i8_workspace(int32_t type, const void* d_hidden, int64_t ld_hidden, const int8_t* d_weight, int64_t ld_weight, int64_t rows,
                                      int64_t vocab, int64_t width) {
  using namespace pst_head;
  const int rc = guarded([&]() -> int { return check_scores(type, d_hidden, ld_hidden, d_weight, ld_weight, rows, vocab, width); });
  return rc == PST_OK ? plan_scores(d_weight, ld_weight, rows, vocab, width).bytes : rc;
}

int pst_token_scores_i8(int32_t device, int32_t type, const void* d_hidden, int64_t ld_hidden, const int8_t* d_weight, int64_t ld_weight,
                        const float* d_weight_scale, int64_t rows, int64_t vocab, int64_t width, int32_t out_type, void* d_scores, int64_t ld_scores,
                        void* d_workspace, int64_t workspace_bytes, void* stream) {
  return pst_head::guarded([&] {
    return pst_head::token_scores_i8(device, type, d_hidden, ld_hidden, d_weight, ld_weight, d_weight_scale, rows, vocab, width, out_type, d_scores,
                                     ld_scores, d_workspace, workspace_bytes, (hipStream_t)stream);
  });
}

}  // extern "C"
