// The matrix products of a training step: C[M,N] = sum over k of A(m,k) B(n,k), bf16 operands, fp32 sums, where either operand may
// lie with k contiguous (rows of m or n) or with k as its rows.  A projection y = x w^T needs three of them,
//     forward  x w^T      A = x  [m][k],  B = w  [n][k]
//     dx = dz w           A = dz [m][k],  B = w  [k][n]
//     dw = dz^T x         A = dz [k][m],  B = x  [k][n]     (k: the tokens)
// and what a training step keeps or needs beside the product is made in the epilogue:
//   ACT         z = C + bias kept for the backward pass, y = act(z) (+ residual)
//   SWIGLU      [gate | up] kept, h = silu(gate) up
//   SWIGLU_BWD  C = dh: dgate = dh up silu'(gate), dup = dh silu(gate), from the kept [gate | up]
// (dx and dw: plain stores; dw of few tiles is cut along the tokens, fp32 partial sums added in order by another kernel.)
//
// Tiles are staged as k-tiles of 64 by loads that go straight into LDS.  An operand with contiguous k lies there as rows of 128 B
// like in the other GEMMs and is read with ds_read_b128; one with k as rows lies as 64 rows of 128 (64) columns and is read with the
// transposing ds_read_b64_tr_b16, two reads for the 8 k of a lane: no transposed copy is made of anything.  Its 32-byte column pairs
// are XOR-swizzled by the k row so that the eight k rows which half a wave reads at once lie on different banks (counted: no bank conflicts
// in any of the three).
//
// Measured, of the 1480 TFLOP/s that the best plain library product reaches: dx 1230-1270 TFLOP/s (14400 tokens, 12288 x 1536: 430 us), dw 1290
// (the same, 417 us), matrix pipe busy 62 and 74 % of the cycles; epilogues that keep three bytes a value beside the result and run while no
// product does cost a large tile a fifth to a half more: [gate | up] kept 1030 TFLOP/s, dgate and dup 750 (360 us, 232 for the product alone).
#include "common.h"
#include "gemm_common.h"
#include "kernels.h"
#include <type_traits>

namespace aeris {

namespace {

constexpr int BK = 64;

enum GradEpi { EPI_STORE, EPI_ACT, EPI_SWIGLU, EPI_SWIGLU_BWD };

struct GradGemm {
  const uint16_t* A;
  const uint16_t* B;
  const uint16_t *A_low, *B_low;  // the remainders of an operand that has two bf16 a value (few tokens; tiles of up to 128), or NULL
  int64_t M, K;
  int64_t lda, ldb;  // elements between rows
  int N;             // columns of the result
  void* C;           // SWIGLU: h; SWIGLU_BWD: [dgate | dup]
  uint16_t* C_low;   // of these, what the rounding left over, or NULL
  int64_t ldc;
  int c_f32;
  const uint16_t* bias;
  const void* residual;
  int res_dtype;   // -1: none
  uint16_t* kept;  // 24-bit values: ACT: z; SWIGLU, SWIGLU_BWD: [gate | up], rows of 2 N
  int act;
  // tiles are numbered four row panels times all column tiles at a time; the first `whole` of them are made in one go, k of each of the
  // others is cut into `parts` of k_part (a multiple of 64), summed from `partial` ([tile - whole][part][rows][columns], fp32) by another kernel
  int tiles_m, tiles_n, whole, parts;
  int64_t k_part;
  float* partial;
  float* row_sums;  // of A, over k: [tile_m][tile_n][part][rows] (each column tile has every tiles_n-th k-tile), or NULL
};

struct TileAt { int m, n; };
__device__ __forceinline__ TileAt tile_at(int tile, int tiles_m, int tiles_n) {
  const int grp = tile / (4 * tiles_n), within = tile - grp * 4 * tiles_n;
  int gm = tiles_m - grp * 4;
  if (gm > 4) gm = 4;
  TileAt t;
  t.n = within / gm;
  t.m = grp * 4 + within - t.n * gm;
  return t;
}
__device__ __forceinline__ int tile_number(int m, int n, int tiles_m, int tiles_n) {
  const int grp = m / 4;
  int gm = tiles_m - grp * 4;
  if (gm > 4) gm = 4;
  return grp * 4 * tiles_n + n * gm + m - grp * 4;
}

__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
// d/dx of x sigma(x)
__device__ __forceinline__ float dsilu_f(float x, float s) { return s * fmaf(x, 1.0f - s, 1.0f); }
// d/dx of x Phi(x) = Phi(x) + x phi(x); 1 - Phi(|x|) by Abramowitz-Stegun 7.1.26 (as in gelu_erf_bf16_f), whose exponential is phi's too.
// |x| is held at 30, where phi is 0 in fp32, so that an infinite x has no infinity times zero in it; NaN is handed on.
__device__ __forceinline__ float dgelu_f(float x) {
  x = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 30.0f), -30.0f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, fabsf(x), 1.0f));
  float pol = fmaf(0.5307027145f, t, -0.7265760135f);
  pol = fmaf(pol, t, 0.7107068705f);
  pol = fmaf(pol, t, -0.142248368f);
  pol = fmaf(pol, t, 0.127414796f);
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044f);
  const float tail = pol * t * e;
  return fmaf(x * 0.3989422804014327f, e, x < 0.0f ? tail : 1.0f - tail);
}

__device__ __forceinline__ void widen8(const u32x4& w, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[2 * e] = bf16_lo(w[e]);
    o[2 * e + 1] = bf16_hi(w[e]);
  }
}
__device__ __forceinline__ u32x4 narrow8(const float (&o)[8]) {
  return u32x4{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])};
}
// what rounding to bf16 leaves over, rounded to bf16
__device__ __forceinline__ u32x4 remainder8(const float (&o)[8]) {
  const u32x4 hi = narrow8(o);
  float h[8], r[8];
  widen8(hi, h);
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = fabsf(h[e]) <= 3.3895314e38f ? o[e] - h[e] : 0.0f;  // (nothing is left over of an infinity or a NaN)
  return narrow8(r);
}
__device__ __forceinline__ void store8(void* C, int f32, int64_t at, const float (&o)[8]) {
  if (f32) {
    f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(C) + at);
    q[0] = f32x4{o[0], o[1], o[2], o[3]};
    q[1] = f32x4{o[4], o[5], o[6], o[7]};
  } else {
    *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(C) + at) = narrow8(o);
  }
}

// Values kept for the backward pass have 24 bits: sign, exponent and 15 bits of the fraction of an fp32 number, rounded to nearest, halves
// away from zero (2^-16 relative; bf16 would be one more rounding of 2^-9 in every gradient behind it, as large as that of the operand it
// ends in, and fp16 has not the range).  The upper 16 bits of all values lie in front, the lower 8 bits behind them.  Adding half a step to
// the bits is all the rounding: a NaN here has come out of bf16 numbers or of the arithmetic itself, with zeros in its lower half, and stays one.
__device__ __forceinline__ void store_kept8(uint16_t* kept, int64_t count, int64_t at, const float (&v)[8]) {
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(v[e]) + 0x80u;
  u32x4 hi;
  u32x2 lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) hi[e] = __builtin_amdgcn_perm(b[2 * e + 1], b[2 * e], 0x07060302u);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    lo[e] = __builtin_amdgcn_perm(b[4 * e + 1], b[4 * e], 0x0c0c0501u) | __builtin_amdgcn_perm(b[4 * e + 3], b[4 * e + 2], 0x05010c0cu);
  *reinterpret_cast<u32x4*>(kept + at) = hi;
  *reinterpret_cast<u32x2*>(reinterpret_cast<uint8_t*>(kept + count) + at) = lo;
}
struct Kept8 { u32x4 hi; u32x2 lo; };
__device__ __forceinline__ Kept8 load_kept8(const uint16_t* kept, int64_t count, int64_t at) {
  return Kept8{*reinterpret_cast<const u32x4*>(kept + at), *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint8_t*>(kept + count) + at)};
}
__device__ __forceinline__ void widen_kept8(const Kept8& k, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)  // byte 0: zero, 1: of lo, 2 and 3: of hi
    v[e] = __uint_as_float(__builtin_amdgcn_perm(k.hi[e >> 1], k.lo[e >> 2], ((e & 1) ? 0x0706000cu : 0x0504000cu) | (uint32_t)(e & 3) << 8));
}

// ---- operand panels in LDS

// k as rows: the 32-byte column pairs of k row k are kept at pair ^ pair_key(k).  Half a wave reads k rows k0 .. k0 + 3 and
// k0 + 8 .. k0 + 11 of one pair: 8 keys for rows of 256 B; of 128 B, where two rows lie beside each other, 4.
template <int COLS>
__device__ __forceinline__ int pair_key(int k) {
  return COLS == 128 ? (k & 3) | (((k >> 3) & 1) << 2) : ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// One operand's side of a workgroup's tile: ROWS rows (or columns, TR) of the tile, in panels
template <bool TR, int ROWS, int WAVES>
struct Panel {
  static constexpr int COLS = ROWS < 128 ? ROWS : 128;             // TR: columns of a panel
  static constexpr int BYTES = ROWS * BK * 2;
  static constexpr int LOADS = BYTES / 1024 / WAVES;               // load instructions of a wave per k-tile
  static_assert(LOADS * WAVES * 1024 == BYTES, "whole load instructions");
};

// One wave's loads of a panel, k-tile after k-tile.  What a load instruction needs is made ahead of the slot that issues it: `next` leaves a
// descriptor and offsets behind, `issue` only uses them (made at the loads, some seventy scalar instructions a k-tile stood between a memory
// slot's LDS reads and its end).
// SWIGLU weights: row 64 c + s of the tile is gate row 32 c + s, from s = 32 on up row 32 c + s - 32 (`up_rows` further on).
template <bool TR, int ROWS, int WAVES, bool SWIGLU_ROWS>
struct Loader {
  using P = Panel<TR, ROWS, WAVES>;
  static constexpr int RPI = 512 / P::COLS;  // TR: k rows of a load instruction
  static_assert(!TR || (RPI == 4 && P::LOADS % 4 == 0) || (RPI == 8 && P::LOADS % 2 == 0), "bit 3 of an instruction's k follows from its number within the wave");
  static_assert(TR || P::LOADS % 2 == 0, "the parity of 8-row blocks follows from their number within the wave");
  static_assert(!TR || ((P::COLS * BK * 2 / 1024) % P::LOADS == 0), "a wave's load instructions lie in one panel");
  lds_dma_rsrc rsrc;
  uint64_t at;             // TR: address of the k-tile's first row
  uint32_t soff[P::LOADS]; // between the load instructions
  uint32_t koff;           // otherwise: of the k-tile within a row
  uint32_t voff[2], vtail[2];
  uint32_t step, whole_bytes, tail_bytes;
  int valid;               // k-tiles from here on that hold anything
  int panel;               // TR: of this wave

  __device__ __forceinline__ void init(int64_t ld, int64_t up_rows, int lane, int wave) {
    step = TR ? (uint32_t)(BK * ld * 2) : BK * 2;
    constexpr int IPP = P::COLS * BK * 2 / 1024;  // TR: instructions of a panel
    panel = wave * P::LOADS / IPP;
#pragma unroll
    for (int j = 0; j < P::LOADS; ++j) {
      const int i = wave * P::LOADS + j;  // instruction of the tile: rows 8 i .., or of panel i / IPP
      int64_t row = TR ? (i % IPP) * RPI : 8 * i;
      if (SWIGLU_ROWS) row = (i >> 3) * 32 + (i & 3) * 8 + ((i & 4) ? up_rows : 0);
      soff[j] = (uint32_t)(row * ld * 2);
    }
#pragma unroll
    for (int par = 0; par < 2; ++par) {
      if (TR) {
        constexpr int CPR = P::COLS / 8;  // chunks of a row
        const int kr = lane / CPR, pos = lane % CPR;
        // pair_key of the instruction's k rows: with the instruction's number (par: whether k has bit 3) and the lane's
        const int key = P::COLS == 128 ? kr | (par << 2) : ((kr >> 1) & 1) | (par << 1);
        voff[par] = (uint32_t)(kr * ld * 2) + (uint32_t)((pos ^ (2 * key)) * 16);
      } else {
        const int dr = lane >> 4, pos = lane & 15;
        const int logical = pos ^ (par * 4 + dr);
        voff[par] = (uint32_t)((dr * 2 + (logical >> 3)) * ld * 2 + (logical & 7) * 16);
      }
    }
  }

  // from k = k_begin to k_end (at or before k_begin: nothing but zeros).  `base`: the tile's first row (column, TR) at k = 0; rows: how many of
  // them the matrix has from there
  __device__ __forceinline__ void start(const uint16_t* base, int64_t ld, int64_t rows, int64_t up_rows, int64_t k_begin, int64_t k_end, int lane) {
    const int64_t left = k_end > k_begin ? k_end - k_begin : 0;
    valid = (int)((left + BK - 1) / BK);
    const int64_t tail = left - (int64_t)(valid - 1) * BK;  // k of the last of them
    if (TR) {
      int64_t cols = rows - panel * P::COLS;
      if (cols < 0) cols = 0;
      at = reinterpret_cast<uint64_t>(base + k_begin * ld + panel * P::COLS);
      whole_bytes = cols ? (uint32_t)(((BK - 1) * ld + cols) * 2) : 0u;
      tail_bytes = cols ? (uint32_t)(((tail - 1) * ld + cols) * 2) : 0u;
    } else {
      at = reinterpret_cast<uint64_t>(base);
      koff = (uint32_t)(k_begin * 2);
      const int64_t all = rows <= 0 ? 0 : SWIGLU_ROWS ? up_rows + rows : rows < ROWS ? rows : ROWS;
      whole_bytes = tail_bytes = (uint32_t)(all * ld * 2);
#pragma unroll
      for (int par = 0; par < 2; ++par) {
        // (k beyond the matrix: an offset beyond any buffer's size, which arrives as zeros)
        const int chunk = ((lane & 15) ^ (par * 4 + (lane >> 4))) & 7;
        vtail[par] = chunk * 8 < tail ? voff[par] : 0x80000000u;
      }
    }
    describe();
  }
  __device__ __forceinline__ void describe() {
    rsrc = make_lds_dma_rsrc(reinterpret_cast<const void*>(at), valid > 1 ? whole_bytes : valid == 1 ? tail_bytes : 0u);
  }
  __device__ __forceinline__ void next() {
    --valid;
    if (TR) at += step;
    else koff += step;
    describe();
  }
  // into the stage at LDS address `stage` + this wave's instructions'
  __device__ __forceinline__ void issue(uint32_t stage) const {
#pragma unroll
    for (int j = 0; j < P::LOADS; ++j) {
      const int par = TR && RPI == 4 ? (j >> 1) & 1 : j & 1;
      if (TR) lds_dma_load16(rsrc, stage + (uint32_t)j * 1024u, voff[par], soff[j]);
      else lds_dma_load16(rsrc, stage + (uint32_t)j * 1024u, valid > 1 ? voff[par] : vtail[par], soff[j] + koff);
    }
  }
};

// Fragment reads of one operand: F fragments of 16 rows (columns) from row `first` of the tile on
template <bool TR, int ROWS, int WAVES, int F>
struct Fragments {
  using P = Panel<TR, ROWS, WAVES>;
  uint32_t at[TR ? F : 2];
  __device__ __forceinline__ void init(int first, int lane) {
    const int l15 = lane & 15, q = lane >> 4;
    if (TR) {
      const int e = (lane >> 2) & 3, a = lane & 3;
      const int k = 8 * q + e;  // (+ 32 per step, + 4 for the upper half: neither changes the key)
      const int panel = first / P::COLS, c0 = first % P::COLS;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int pair = c0 / 16 + f;
        at[TR ? f : 0] = (uint32_t)(panel * P::COLS * BK * 2 + k * P::COLS * 2 + ((pair ^ pair_key<P::COLS>(k)) << 5) + (a >> 1) * 16 + (a & 1) * 8);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) at[ks] = swz_off(first + l15, ks * 4 + q);
    }
  }
  template <int KS>
  __device__ __forceinline__ void request(uint32_t stage, TrFrag (&raw)[F], bf16x8 (&out)[F]) const {
    if (TR) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        raw[f].lo = lds_read_tr16_b64<KS * 32 * P::COLS * 2>(stage + at[TR ? f : 0]);
        raw[f].hi = lds_read_tr16_b64<KS * 32 * P::COLS * 2 + 4 * P::COLS * 2>(stage + at[TR ? f : 0]);
      }
    } else {
      typedef __attribute__((address_space(3))) const bf16x8* lds_frag;
#pragma unroll
      for (int f = 0; f < F; ++f) out[f] = *(lds_frag)(uintptr_t)(stage + at[KS] + f * 2048u);
    }
  }
  __device__ __forceinline__ void wait(TrFrag (&raw)[F], bf16x8 (&out)[F]) const {
    if (TR) {
      static_assert(!TR || F % 2 == 0, "pairs");
#pragma unroll
      for (int f = 0; f < F; f += 2) lds_tr_wait(raw[f], raw[f + 1]);
#pragma unroll
      for (int f = 0; f < F; ++f) out[f] = tr_frag_value(raw[f]);
    }
  }
};

// ---- epilogue of a wave's FM x FN fragments of one item; rows from row0, columns from col0 of the result, or of the item's part of
// `partial`.  16 rows at a time pass through 16 x FN x 16 floats of the wave's own LDS (16-byte chunks XOR-swizzled by the row), so that a
// lane has 8 consecutive columns of a row and memory is written and read in whole row segments of the wave's width.
template <int T, int EPI, int FM, int FN>
__device__ __forceinline__ void grad_epilogue(const GradGemm& p, const f32x4 (&acc)[FM][FN], int64_t row0, int col0, float* part, uint32_t stage, int lane_) {
  typedef __attribute__((address_space(3))) f32x4* lds4;
  int lane = lane_;
  asm volatile("" : "+v"(lane));  // what follows from the lane number is made anew here and kept out of the main loop's registers
  const int l15 = lane & 15, q = lane >> 4;
  constexpr int CH = FN * 4;                                          // chunks of a staged row
  constexpr int CHUNKS = (EPI == EPI_SWIGLU ? FN / 2 : FN) * 2;       // of 8 columns of the result
  constexpr int RPI = 64 / CHUNKS < 16 ? 64 / CHUNKS : 16, ITS = 16 / RPI;  // rows at a time
  const int rrow = lane / CHUNKS, rch = lane % CHUNKS;
  const int col = col0 + rch * 8;
  const bool col_ok = part != nullptr || col < p.N;
  // What the epilogue reads is asked for ahead of its stores (vector memory operations complete in order: a load behind a store would
  // be waited for together with it): the bias once, the other rows one row fragment ahead.  Rows and columns beyond the result: its last.
  constexpr bool LOADS = EPI == EPI_ACT || EPI == EPI_SWIGLU_BWD;
  u32x4 bias = {0u, 0u, 0u, 0u};
  u32x4 ahead[LOADS ? 2 : 1][LOADS ? ITS : 1][EPI == EPI_SWIGLU_BWD ? 3 : 2];  // residual, or upper halves of gate and up and both lower bytes
  const int64_t last_row = p.M - 1;
  const int load_col = col < p.N ? col : p.N - 8;
  auto ask = [&](int i) {
    if constexpr (LOADS) {
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        int64_t row = row0 + 16 * i + rrow + it * RPI;
        if (row > last_row) row = last_row;
        u32x4(&to)[EPI == EPI_SWIGLU_BWD ? 3 : 2] = ahead[i & 1][it];
        if constexpr (EPI == EPI_SWIGLU_BWD) {
          const int64_t at = row * (2 * (int64_t)p.N) + load_col, count = p.M * (2 * (int64_t)p.N);
          const Kept8 g = load_kept8(p.kept, count, at), u = load_kept8(p.kept, count, at + p.N);
          to[0] = g.hi;
          to[1] = u.hi;
          to[2] = u32x4{g.lo.x, g.lo.y, u.lo.x, u.lo.y};
        } else {
          const int64_t at = row * (int64_t)p.N + load_col;
          if (p.res_dtype == AERIS_F32) {
            const u32x4* src = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p.residual) + at);
            to[0] = src[0];
            to[1] = src[1];
          } else if (p.res_dtype == AERIS_BF16) {
            to[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.residual) + at);
          }
        }
      }
    }
  };
  if (EPI == EPI_ACT && p.bias) bias = *reinterpret_cast<const u32x4*>(p.bias + load_col);
  ask(0);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if (i + 1 < FM) ask(i + 1);
#pragma unroll
    for (int j = 0; j < FN; ++j) *(lds4)(uintptr_t)(stage + l15 * (CH * 16) + (((j * 4 + q) ^ (l15 & (CH - 1))) << 4)) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      const int r = rrow + it * RPI;
      auto eight = [&](int c, float (&o)[8]) {
        const f32x4 a = *(lds4)(uintptr_t)(stage + r * (CH * 16) + (((2 * c) ^ (r & (CH - 1))) << 4));
        const f32x4 b = *(lds4)(uintptr_t)(stage + r * (CH * 16) + (((2 * c + 1) ^ (r & (CH - 1))) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = a[e];
          o[4 + e] = b[e];
        }
      };
      float o[8];
      eight(rch, o);
      const int64_t row = row0 + 16 * i + r;
      if (EPI == EPI_STORE && part != nullptr) {
        store8(part, 1, row * T + col, o);
        continue;
      }
      const bool ok = col_ok && row < p.M;
      if constexpr (EPI == EPI_STORE) {
        if (ok) store8(p.C, p.c_f32, row * p.ldc + col, o);
      } else if constexpr (EPI == EPI_SWIGLU) {
        float up[8];
        eight(rch + CHUNKS, up);
        if (ok) {
          const int64_t at = row * (2 * (int64_t)p.N) + col, count = p.M * (2 * (int64_t)p.N);
          if (p.kept) {
            store_kept8(p.kept, count, at, o);
            store_kept8(p.kept, count, at + p.N, up);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = silu_f(o[e]) * up[e];
          store8(p.C, 0, row * p.ldc + col, o);
          if (T <= 128 && p.C_low) *reinterpret_cast<u32x4*>(p.C_low + row * p.ldc + col) = remainder8(o);
        }
      } else if constexpr (EPI == EPI_ACT) {
        if (ok) {
          float b[8];
          widen8(bias, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += b[e];
          const int64_t at = row * (int64_t)p.N + col;
          if (p.kept) store_kept8(p.kept, p.M * (int64_t)p.N, at, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = p.act == AERIS_ACT_SILU ? silu_f(o[e]) : p.c_f32 ? gelu_erf_f(o[e]) : gelu_erf_bf16_f(o[e]);
          if (p.res_dtype >= 0) {
            float x[8];
            const u32x4(&r)[2] = ahead[i & 1][it];
            if (p.res_dtype == AERIS_F32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                x[e] = __uint_as_float(r[0][e]);
                x[4 + e] = __uint_as_float(r[1][e]);
              }
            } else {
              widen8(r[0], x);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += x[e];
          }
          store8(p.C, p.c_f32, at, o);
        }
      } else if (ok) {  // EPI_SWIGLU_BWD
        const int64_t at = row * (2 * (int64_t)p.N) + col;
        float g[8], u[8], dg[8];
        const u32x4(&r)[3] = ahead[i & 1][it];
        widen_kept8(Kept8{r[0], u32x2{r[2].x, r[2].y}}, g);
        widen_kept8(Kept8{r[1], u32x2{r[2].z, r[2].w}}, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float s = sigmoid_f(g[e]);
          dg[e] = o[e] * u[e] * dsilu_f(g[e], s);
          o[e] *= g[e] * s;
        }
        store8(p.C, 0, at, dg);
        store8(p.C, 0, at + p.N, o);
        if (T <= 128 && p.C_low) {
          *reinterpret_cast<u32x4*>(p.C_low + at) = remainder8(dg);
          *reinterpret_cast<u32x4*>(p.C_low + at + p.N) = remainder8(o);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// the sums of A's rows over k that a wave has of its fragments (each lane's four elements are the same, so are the four lanes of a row)
template <int T, int F>
__device__ __forceinline__ void store_row_sums(const GradGemm& p, const f32x4 (&sums)[F], int tile_m, int tile_n, int part, int row, int lane) {
  if (lane >= 16) return;
  float* out = p.row_sums + (((int64_t)tile_m * p.tiles_n + tile_n) * p.parts + part) * T + row + lane;
#pragma unroll
  for (int f = 0; f < F; ++f) out[16 * f] = sums[f][0];
}

__device__ __forceinline__ bf16x8 all_ones() {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (__bf16)1.0f;
  return v;
}

// ---- tiles of T x T (128 or 64), four waves two by two.  Two stages, and two to five workgroups a CU that fill each other's waits; tiles of 64
// whose workgroups are few have four stages instead, or each k-tile would take the time of a load (300 tokens, 4096 -> 1024 with GELU 35 -> 25 us; the
// gated MLP's forward pass of 9 tokens, 1536 -> 6144: 33 -> 27 us, now 24).
template <int T, int STAGES>
constexpr int tile_lds() { return STAGES * 2 * T * BK * 2; }

// LOW: an operand has two bf16 a value, and k is gone over twice, the second time with its remainders.  Both sweeps have sums of their own, and what
// the first one's has beyond the finite numbers stays as it is: a remainder is 0 where a bf16 holds the whole value, and where the other operand is
// infinite, 0 times infinity, or a remainder of the other sign, would make NaN of an infinity (sums of their own cost no instruction in the loop; zeros for
// the infinities read in the second sweep: 33 tokens through the gated MLP of 384 -> 1088 and back 28.7 -> 31.9 us).
template <int T, int STAGES, bool A_TR, bool B_TR, int EPI, bool LOW>
__device__ __forceinline__ void grad_tile(const GradGemm& p, int item, unsigned char* smem) {
  constexpr bool SWIGLU = EPI == EPI_SWIGLU, ROW_SUMS = A_TR;
  // waves over the tile: two by two; SwiGLU tiles of 64 four by one, so that a wave has a gate column's up column too
  constexpr int WN = SWIGLU && T == 64 ? 1 : 2, WM = 4 / WN;
  constexpr int FM = T / WM / 16, FN = T / WN / 16;  // fragments of a wave
  constexpr int FS = ROW_SUMS ? FM / WN : 1;         // row fragments whose sums a wave has
  constexpr int BN_OUT = SWIGLU ? T / 2 : T;
  using PA = Panel<A_TR, T, 4>;
  using PB = Panel<B_TR, T, 4>;
  static_assert(STAGES * (PA::BYTES + PB::BYTES) == tile_lds<T, STAGES>(), "the stages");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int part = 0;
  if (item >= p.whole) {
    const int c = item - p.whole, cut_tiles = p.tiles_m * p.tiles_n - p.whole;
    part = c / cut_tiles;
    item = p.whole + c - part * cut_tiles;
  }
  const TileAt tile = tile_at(item, p.tiles_m, p.tiles_n);
  const int64_t m0 = (int64_t)tile.m * T;
  const int n0 = tile.n * BN_OUT;
  const bool cut = item >= p.whole;
  const int64_t k_begin = cut ? part * p.k_part : 0;
  int64_t k_end = cut ? k_begin + p.k_part : p.K;
  if (k_end > p.K) k_end = p.K;
  const int turns = k_end > k_begin ? (int)((k_end - k_begin + BK - 1) / BK) : 0;

  Loader<A_TR, T, 4, false> la;
  Loader<B_TR, T, 4, SWIGLU> lb;
  la.init(p.lda, 0, lane, wave);
  lb.init(p.ldb, p.N, lane, wave);
  auto start = [&](const uint16_t* A, const uint16_t* B) {
    la.start(A + (A_TR ? m0 : m0 * p.lda), p.lda, p.M - m0, 0, k_begin, k_end, lane);
    lb.start(B + (B_TR ? (int64_t)n0 : n0 * p.ldb), p.ldb, p.N - n0, p.N, k_begin, k_end, lane);
  };
  start(p.A, p.B);
  Fragments<A_TR, T, 4, FM> fa;
  Fragments<B_TR, T, 4, FN> fb;
  fa.init(wm * (T / WM), lane);
  fb.init(wn * (T / WN), lane);

  f32x4 acc[FM][FN], first[LOW ? FM : 1][LOW ? FN : 1], sums[FS];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int f = 0; f < FS; ++f) sums[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool with_sums = ROW_SUMS && p.row_sums;

  const uint32_t lds0 = lds_byte_address(smem);
  const int all_turns = LOW ? 2 * turns : turns;
  auto issue = [&](int t) {  // (past the last k-tile: loads of nothing, which keep the count of the waits the same)
    if (LOW && t == turns) start(p.A_low ? p.A_low : p.A, p.B_low ? p.B_low : p.B);
    const uint32_t stage = lds0 + (uint32_t)(t % STAGES) * (PA::BYTES + PB::BYTES);
    la.issue(stage + wave * (PA::LOADS * 1024));
    lb.issue(stage + PA::BYTES + wave * (PB::LOADS * 1024));
    la.next();
    lb.next();
  };
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) issue(t);
  int sum_turn = with_sums ? (int)((k_begin / BK) % p.tiles_n) : 0;
  for (int t = 0; t < all_turns; ++t) {
    if constexpr (LOW) {
      if (t == turns) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            first[i][j] = acc[i][j];
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
          }
      }
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * (PA::LOADS + PB::LOADS)) : "memory");
    __syncthreads();  // stage t is there; the one that is filled next has been read
    issue(t + STAGES - 1);
    const uint32_t sa = lds0 + (uint32_t)(t % STAGES) * (PA::BYTES + PB::BYTES), sb = sa + PA::BYTES;
    const bool mine = with_sums && sum_turn == tile.n;
    auto step = [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      TrFrag ra[FM], rb[FN];
      bf16x8 a[FM], b[FN];
      fa.template request<KS>(sa, ra, a);
      fb.template request<KS>(sb, rb, b);
      fa.wait(ra, a);
      fb.wait(rb, b);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
      if constexpr (ROW_SUMS) {
        if (mine) {
#pragma unroll
          for (int f = 0; f < FS; ++f) sums[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(all_ones(), wn == 0 ? a[f] : a[FM - FS + f], sums[f], 0, 0, 0);
        }
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    if (++sum_turn == p.tiles_n) sum_turn = 0;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();  // the stages are read and nothing more arrives in them: they stage the result now
  if constexpr (LOW) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fabsf(first[i][j][e]) < __builtin_inff() ? first[i][j][e] + acc[i][j][e] : first[i][j][e];
  }
  float* const at = EPI == EPI_STORE && cut ? p.partial + ((int64_t)(item - p.whole) * p.parts + part) * (T * T) : nullptr;
  const uint32_t stage = lds0 + wave * (16 * FN * 64);
  if (at) grad_epilogue<T, EPI, FM, FN>(p, acc, wm * (T / WM), wn * (T / WN), at, stage, lane);
  else grad_epilogue<T, EPI, FM, FN>(p, acc, m0 + wm * (T / WM), n0 + wn * (BN_OUT / WN), nullptr, stage, lane);
  if constexpr (ROW_SUMS) {
    if (with_sums) store_row_sums<T, FS>(p, sums, tile.m, tile.n, part, wm * (T / WM) + wn * FS * 16, lane);
  }
}

// Workgroup b runs on XCD b mod 8: neighbouring items, which share rows and columns of their operands, go to one XCD (a permutation of 0 .. n - 1),
// the whole tiles and the parts of the others each among themselves
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int xcd = b & 7, each = n >> 3, more = n & 7;
  return xcd * each + (xcd < more ? xcd : more) + (b >> 3);
}
__device__ __forceinline__ int xcd_item(const GradGemm& p, int b, int n) {
  return b < p.whole ? xcd_order(b, p.whole) : p.whole + xcd_order(b - p.whole, n - p.whole);
}

template <int T, int STAGES, bool A_TR, bool B_TR, int EPI, bool LOW>
__global__ void __launch_bounds__(256, 2) gemm_grad_tile_kernel(GradGemm p) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[tile_lds<T, STAGES>()];
  const int item = xcd_item(p, blockIdx.x, gridDim.x);
  grad_tile<T, STAGES, A_TR, B_TR, EPI, LOW>(p, item, smem);
}

// two products that do not depend on each other in one launch: the first n workgroups make dx (or dh and what follows from it), the others dw
// (LOW: dw has an operand of two bf16 a value; so has dx, which is made with its epilogue alone)
template <int T, int STAGES, int EPI, bool LOW>
__global__ void __launch_bounds__(256, 2) gemm_grad_pair_kernel(GradGemm p, GradGemm q, int n) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[tile_lds<T, STAGES>()];
  if ((int)blockIdx.x < n) grad_tile<T, STAGES, false, true, EPI, LOW && EPI == EPI_STORE>(p, xcd_item(p, blockIdx.x, n), smem);
  else grad_tile<T, STAGES, true, true, EPI_STORE, LOW>(q, xcd_item(q, blockIdx.x - n, gridDim.x - n), smem);
}

// ---- tiles of 256 x 256, eight waves (two by four, 128 x 64 each), one persistent workgroup a CU: the pipeline of the package's other
// large product (two stages of A, three of B, the two waves of a SIMD in alternating memory and compute slots, the loads' flat sequence over
// items and k-tiles running ahead through the epilogues), for operands of either layout.  An item is a tile of one part of k.
// Slots of k-tile j, numbered globally: group 0 (waves 0-3) M0 C0 M1 C1 in slots 4j .. 4j+3, group 1 one slot later.  A memory slot reads half
// a k-tile's fragments and issues 4 loads, a compute slot issues 32 MFMAs.  A: the half of a stage that a group reads is loaded by its own
// waves, A[j+1] in M0(j) over A[j-1], last read in M1(j-1).  B: B[j+2] in M1(j) (slots 4j+2, 4j+3) over B[j-1], last read in slot 4j-1.
// Waits, by counts of the loads issued since: the end of M1(j) leaves 8 outstanding (B[j+1] has arrived), the end of C1(j) 4 (A[j+1] has).
constexpr int BIG_STAGE = 256 * BK * 2;
constexpr int BIG_LDS = 5 * BIG_STAGE;

template <bool A_TR, bool B_TR, int EPI>
__global__ void __launch_bounds__(512) gemm_grad_big_kernel(GradGemm p) {
  constexpr bool SWIGLU = EPI == EPI_SWIGLU, ROW_SUMS = A_TR;
  constexpr int BN_OUT = SWIGLU ? 128 : 256;
  constexpr int FM = 8, FN = 4, FS = ROW_SUMS ? 2 : 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, wn = wave & 3;
  const uint32_t lds0 = lds_byte_address(smem), lds_b0 = lds0 + 2 * BIG_STAGE;

  // Whole tiles come in full rounds of one per CU: XCD x (workgroup number mod 8) has a contiguous eighth of them, its 32 workgroups take
  // them in turns, so that those at work together share the operands' slices in its L2.  What is left is one more round, of parts.
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int rounds = p.whole >> 8, cut_tiles = p.tiles_m * p.tiles_n - p.whole, cut_items = cut_tiles * p.parts, cut_each = (cut_items + 7) >> 3;
  const bool has_cut = slot < cut_each && xcd * cut_each + slot < cut_items;
  const int n_my = rounds + (has_cut ? 1 : 0);
  if (n_my == 0) return;
  struct Item { int64_t m0, k_begin, k_end; int n0, tile_m, tile_n, part, cut; };
  auto decode = [&](int r) {
    Item it;
    int tile;
    if (r < rounds) {
      tile = xcd * (rounds * 32) + r * 32 + slot;
      it.cut = it.part = 0;
      it.k_begin = 0;
      it.k_end = p.K;
    } else {
      const int c = xcd * cut_each + slot;  // (the tiles of one part beside each other: they read the same rows)
      it.part = c / cut_tiles;
      const int n = c - it.part * cut_tiles;
      tile = p.whole + n;
      it.cut = n * p.parts + it.part + 1;
      it.k_begin = it.part * p.k_part;
      it.k_end = it.k_begin + p.k_part < p.K ? it.k_begin + p.k_part : p.K;
    }
    const TileAt t = tile_at(tile, p.tiles_m, p.tiles_n);
    it.tile_m = t.m;
    it.tile_n = t.n;
    it.m0 = (int64_t)t.m * 256;
    it.n0 = t.n * BN_OUT;
    return it;
  };
  // k-tiles of an item (at least one: what lies beyond the end of k arrives as zeros)
  const int KT_whole = (int)((p.K + BK - 1) / BK), KT_cut = (int)(p.k_part / BK);
  auto turns_of = [&](int r) { return r < rounds ? KT_whole : KT_cut; };

  Loader<A_TR, 128, 4, false> la;
  Loader<B_TR, 256, 8, SWIGLU> lb;
  la.init(p.lda, 0, lane, wn);
  lb.init(p.ldb, p.N, lane, wave);
  int la_r = 0, la_left = 0, la_stage = 0, lb_r = 0, lb_left = 0, lb_stage = 0;  // item, its k-tiles that are left, stage
  auto la_item = [&]() {
    la_left = turns_of(la_r);
    if (la_r >= n_my) {  // past the end: loads from a descriptor without records, so that the counts of the waits stay the same
      la.start(p.A, p.lda, 0, 0, 0, 0, lane);
      return;
    }
    const Item it = decode(la_r);
    const int64_t m = it.m0 + grp * 128;
    la.start(p.A + (A_TR ? m : m * p.lda), p.lda, p.M - m, 0, it.k_begin, it.k_end, lane);
  };
  auto lb_item = [&]() {
    lb_left = turns_of(lb_r);
    if (lb_r >= n_my) {
      lb.start(p.B, p.ldb, 0, 0, 0, 0, lane);
      return;
    }
    const Item it = decode(lb_r);
    lb.start(p.B + (B_TR ? (int64_t)it.n0 : it.n0 * p.ldb), p.ldb, p.N - it.n0, p.N, it.k_begin, it.k_end, lane);
  };
  // (issue and advance apart: no branch may lie between the transposing reads of a memory slot and their wait)
  auto issue_a = [&]() { la.issue(lds0 + la_stage * BIG_STAGE + grp * (BIG_STAGE / 2) + wn * 4096); };
  auto issue_b = [&]() { lb.issue(lds_b0 + lb_stage * BIG_STAGE + wave * 4096); };
  auto step_a = [&]() {
    la_stage ^= 1;
    la.next();
  };
  auto step_b = [&]() {
    lb_stage = lb_stage == 2 ? 0 : lb_stage + 1;
    lb.next();
  };
  auto turn_a = [&]() {
    if (--la_left == 0) {
      ++la_r;
      la_item();
    }
  };
  auto turn_b = [&]() {
    if (--lb_left == 0) {
      ++lb_r;
      lb_item();
    }
  };

  Fragments<A_TR, 128, 4, FM> fa;
  Fragments<B_TR, 256, 8, FN> fb;
  fa.init(0, lane);
  fb.init(wn * 64, lane);
  f32x4 acc[FM][FN];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  clear();
  f32x4 sums[FS];
#pragma unroll
  for (int f = 0; f < FS; ++f) sums[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool with_sums = ROW_SUMS && p.row_sums;

  la_item();
  lb_item();
  issue_a();
  step_a();
  turn_a();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    issue_b();
    step_b();
    turn_b();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int sa = 0, sb = 0;
  for (int r = 0; r < n_my; ++r) {
    if (grp == 1) __builtin_amdgcn_s_barrier();  // one slot behind group 0; group 0 waits for it ahead of its epilogue
    const Item it = decode(r);
    const int KT = turns_of(r);
    int sum_turn = with_sums ? (int)((it.k_begin / BK) % p.tiles_n) : 0;
    for (int kt = 0; kt < KT; ++kt) {
      const bool mine = with_sums && sum_turn == it.tile_n;
      if (++sum_turn == p.tiles_n) sum_turn = 0;
      const uint32_t s_a = lds0 + sa * BIG_STAGE + grp * (BIG_STAGE / 2), s_b = lds_b0 + sb * BIG_STAGE;
      sa ^= 1;
      if (++sb == 3) sb = 0;
      auto half = [&](auto ks) {
        constexpr int KS = decltype(ks)::value;
        TrFrag ra[FM], rb[FN];
        bf16x8 a[FM], b[FN];
        fa.template request<KS>(s_a, ra, a);
        fb.template request<KS>(s_b, rb, b);
        __builtin_amdgcn_sched_barrier(0);
        if (KS == 0) issue_a();
        else issue_b();
        __builtin_amdgcn_sched_barrier(0);
        fa.wait(ra, a);
        fb.wait(rb, b);
        __builtin_amdgcn_s_waitcnt(KS == 0 ? 0xC07F : 0x0078);  // lgkmcnt(0); vmcnt(8) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (KS == 0) step_a();
        else step_b();
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
        if constexpr (ROW_SUMS) {
          if (mine) {
#pragma unroll
            for (int f = 0; f < FS; ++f) {
              const bf16x8 x = wn < 2 ? wn == 0 ? a[f] : a[2 + f] : wn == 2 ? a[4 + f] : a[6 + f];
              sums[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(all_ones(), x, sums[f], 0, 0, 0);
            }
          }
        }
        if (KS == 0) turn_a();
        else turn_b();
        if (KS == 1) __builtin_amdgcn_s_waitcnt(0x0F74);  // vmcnt(4)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      };
      half(std::integral_constant<int, 0>{});
      half(std::integral_constant<int, 1>{});
    }
    if (grp == 0) __builtin_amdgcn_s_barrier();
    // the A stage that is filled next is idle, and the 4 KB of it that this wave's own loads fill are written by nobody else
    const uint32_t stage = lds0 + la_stage * BIG_STAGE + grp * (BIG_STAGE / 2) + wn * 4096;
    if (EPI == EPI_STORE && it.cut && p.parts > 1) grad_epilogue<256, EPI, FM, FN>(p, acc, grp * 128, wn * 64, p.partial + (int64_t)(it.cut - 1) * 65536, stage, lane);
    else grad_epilogue<256, EPI, FM, FN>(p, acc, it.m0 + grp * 128, it.n0 + wn * (BN_OUT / 4), nullptr, stage, lane);
    clear();
    if constexpr (ROW_SUMS) {
      if (with_sums) {
        store_row_sums<256, FS>(p, sums, it.tile_m, it.tile_n, it.part, grp * 128 + wn * 32, lane);
#pragma unroll
        for (int f = 0; f < FS; ++f) sums[f] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
}

// ---- what is left when the products are made, each in a fixed order: the first n workgroups add up the parts of p's cut tiles, the next
// m those of q's (8 columns a thread), the others the bias' gradient from q's sums over k
template <int T>
__device__ __forceinline__ void part_sum(const GradGemm& p, int block) {
  constexpr int PER_TILE = T * T / 8 / 256;  // workgroups
  const int tile = block / PER_TILE, at = ((block % PER_TILE) * 256 + threadIdx.x) * 8;
  const TileAt t = tile_at(p.whole + tile, p.tiles_m, p.tiles_n);
  const int64_t row = (int64_t)t.m * T + at / T;
  const int col = t.n * T + at % T;
  if (row >= p.M || col >= p.N) return;
  const float* src = p.partial + (int64_t)tile * p.parts * (T * T) + at;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.parts; ++s) {
    const f32x4* q = reinterpret_cast<const f32x4*>(src + (int64_t)s * (T * T));
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += a[e];
      o[4 + e] += b[e];
    }
  }
  store8(p.C, p.c_f32, row * p.ldc + col, o);
}
template <int T>
__global__ void __launch_bounds__(256) grad_finish_kernel(GradGemm p, GradGemm q, int n, int m, uint16_t* bias) {
  const int block = blockIdx.x;
  if (block < n) {
    part_sum<T>(p, block);
  } else if (block < n + m) {
    part_sum<T>(q, block - n);
  } else {
    const int64_t row = (int64_t)(block - n - m) * 256 + threadIdx.x;
    if (row >= q.M) return;
    const int tm = (int)(row / T);
    float v = 0.f;
    for (int tn = 0; tn < q.tiles_n; ++tn) {
      const int parts = tile_number(tm, tn, q.tiles_m, q.tiles_n) < q.whole ? 1 : q.parts;
      const float* src = q.row_sums + ((int64_t)tm * q.tiles_n + tn) * q.parts * T + row % T;
#pragma unroll 4
      for (int s = 0; s < parts; ++s) v += src[(int64_t)s * T];
    }
    bias[row] = (uint16_t)f32_to_bf16_bits(v);
  }
}

// ---- dz = dy act'(z) (ACT_NONE: dy) rounded to bf16, and the sums of the unrounded dz over the tokens.  Bound by HBM: a wave takes 512 columns of
// one row at a time (two without activation, which it asks for before it uses the first), workgroups in turns, three a CU.  More of either in flight
// is slower: f32 dy [1036800, 1024] without activation 1145 us, 5.6 TB/s (four rows, five workgroups 1253; a cast to bf16 alone 1086), bf16 [8192, 6144]
// with GELU 65, 5.4 TB/s (76), [100000, 2048] with SiLU 260 (297).  That is for widths near a multiple of 512: narrower rows, and the last columns of others,
// leave lanes without work and a wave with few loads in flight (300000 rows with GELU: 512 columns 195 us, 5.5 TB/s, 520 271, 4.0, 136 125, 2.3, 64 128, 1.1).
struct ActGrad {
  const void* dy;
  const uint16_t* z;
  uint16_t* dz;    // NULL: not wanted (dy is bf16 and there is no activation)
  uint16_t* dz_low;  // what the rounding of dz left over, or NULL
  float* partial;  // [workgroups of a column block][N], or NULL
  int64_t M;
  int N, act;
};

template <bool DY_F32, bool ACT, bool STREAM>
__global__ void __launch_bounds__(256) act_grad_kernel(ActGrad p) {
  constexpr int ROWS = ACT ? 1 : 2;
  __shared__ f32x4 lds[4][128];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = (blockIdx.y * 64 + lane) * 8;
  const bool ok = col < p.N;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (ok) {
    for (int64_t row = ((int64_t)blockIdx.x * 4 + w) * ROWS; row < p.M; row += (int64_t)gridDim.x * 4 * ROWS) {
      u32x4 a[ROWS], b[ROWS];
      Kept8 z[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int64_t at = (row + r < p.M ? row + r : p.M - 1) * p.N + col;
        if (DY_F32) {
          const u32x4* q = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p.dy) + at);
          a[r] = __builtin_nontemporal_load(q);
          b[r] = __builtin_nontemporal_load(q + 1);
        } else {
          a[r] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.dy) + at);
        }
        if (ACT) z[r] = load_kept8(p.z, p.M * p.N, at);
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (row + r >= p.M) break;
        float d[8];
        if (DY_F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[e] = __uint_as_float(a[r][e]);
            d[4 + e] = __uint_as_float(b[r][e]);
          }
        } else {
          widen8(a[r], d);
        }
        if (ACT) {
          float v[8];
          widen_kept8(z[r], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] *= p.act == AERIS_ACT_SILU ? dsilu_f(v[e], sigmoid_f(v[e])) : dgelu_f(v[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += d[e];
        if (p.dz) {
          u32x4* const out = reinterpret_cast<u32x4*>(p.dz + (row + r) * p.N + col);
          if (STREAM) __builtin_nontemporal_store(narrow8(d), out);
          else *out = narrow8(d);
          if (!STREAM && p.dz_low) *reinterpret_cast<u32x4*>(p.dz_low + (row + r) * p.N + col) = remainder8(d);
        }
      }
    }
  }
  if (!p.partial) return;
  lds[w][lane] = f32x4{sum[0], sum[1], sum[2], sum[3]};
  lds[w][64 + lane] = f32x4{sum[4], sum[5], sum[6], sum[7]};
  __syncthreads();
  if (w == 0 && ok) {
    float* out = p.partial + (int64_t)blockIdx.x * p.N + col;
    *reinterpret_cast<f32x4*>(out) = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    *reinterpret_cast<f32x4*>(out + 4) = (lds[0][64 + lane] + lds[1][64 + lane]) + (lds[2][64 + lane] + lds[3][64 + lane]);
  }
}

// 8 columns a workgroup, 128 threads share a column's partial sums
__global__ void __launch_bounds__(1024) bias_sum_kernel(const float* partial, uint16_t* out, int parts, int N) {
  __shared__ float lds[16][8];
  const int c = threadIdx.x & 7, r = threadIdx.x >> 3, col = blockIdx.x * 8 + c;  // (N is a multiple of 8)
  float t = 0.f;
#pragma unroll 4
  for (int b = r; b < parts; b += 128) t += partial[(int64_t)b * N + col];
  t += __shfl_xor(t, 8);
  t += __shfl_xor(t, 16);
  t += __shfl_xor(t, 32);
  if ((threadIdx.x & 63) < 8) lds[threadIdx.x >> 6][c] = t;
  __syncthreads();
  if (threadIdx.x < 8) {
    t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += lds[w][c];
    out[col] = (uint16_t)f32_to_bf16_bits(t);
  }
}

// (at least two turns of a workgroup's four waves, one without activation: 300 rows of 1024 with GELU 5.6 us, with four of them 6.8)
int act_grad_parts(int64_t M, int N) {
  const int64_t n = 768 / ((N + 511) / 512), most = (M + 7) / 8;
  return n < 1 ? 1 : n < most ? (int)n : (int)most;
}

hipError_t act_grad_launch(const void* dy, int dy_f32, const void* z, void* dz, void* dz_low, float* partial, void* dbias, int64_t M, int N, int act,
                           hipStream_t stream) {
  ActGrad p;
  p.dy = dy;
  p.z = reinterpret_cast<const uint16_t*>(z);
  p.dz = reinterpret_cast<uint16_t*>(dz);
  p.dz_low = reinterpret_cast<uint16_t*>(dz_low);
  p.partial = dbias ? partial : nullptr;
  p.M = M;
  p.N = N;
  p.act = act;
  const int parts = act_grad_parts(M, N);
  const dim3 grid((unsigned)parts, (unsigned)((N + 511) / 512));
  const bool stream_out = !dz_low && M * N * 2 > (int64_t)256 << 20;  // more than the last-level cache holds until the products read it
#define GO(DY, ACT, ST) hipLaunchKernelGGL((act_grad_kernel<DY, ACT, ST>), grid, dim3(256), 0, stream, p)
  if (act != AERIS_ACT_NONE) {
    if (dy_f32) { if (stream_out) GO(true, true, true); else GO(true, true, false); }
    else { if (stream_out) GO(false, true, true); else GO(false, true, false); }
  } else if (dy_f32) {
    if (stream_out) GO(true, false, true);
    else GO(true, false, false);
  } else {
    GO(false, false, false);  // (no dz)
  }
#undef GO
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !dbias) return e;
  hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)(N / 8)), dim3(1024), 0, stream, partial, reinterpret_cast<uint16_t*>(dbias), parts, N);
  return hipGetLastError();
}

// ---- how a product is cut

struct GradPlan {
  int tile;  // 0: the result has more tiles than can be numbered
  int tiles_m, tiles_n, whole, parts;
  int64_t k_part;
  double us;  // estimate
  int64_t left() const { return (int64_t)tiles_m * tiles_n - whole; }
  int64_t items() const { return whole + left() * parts; }
  int64_t partial_bytes() const { return parts > 1 ? left() * parts * tile * tile * 4 : 0; }
  int64_t row_sum_bytes() const { return ((int64_t)tiles_m * tiles_n * parts * tile * 4 + 255) / 256 * 256; }
};

// What a product of form `epi` takes in tiles of T x T, in us.  A round of 256 tiles of 256, of 512 of 128 (two a CU) or of 1280 of 64 (five) takes
// round_k a k and tile_us beside it, a lone tile of 128 or 64 on a CU lone_k a k: fitted to products of 2048 .. 259200 rows, 128 .. 12288 columns
// and k from 64 to 64800.  Tiles beyond the last whole round may be cut along k into as many parts as fill one: 14400 tokens' dw [12288, 1536] (288
// tiles of 256 for 256 CUs) 710 -> 417 us; the parts go through memory once more, 16 to 256 KB each.
GradPlan plan_tiles(int t, int64_t M, int64_t N, int64_t K, int epi, bool low) {
  const int64_t bn = epi == EPI_SWIGLU ? t / 2 : t, tm = (M + t - 1) / t, tn = (N + bn - 1) / bn, tiles = tm * tn;
  GradPlan best = {};
  best.us = 1e30;
  if (tiles >= 1 << 24 || (low && t == 256)) return best;
  const int at_once = t == 256 ? 256 : t == 128 ? 512 : 1280, i = t == 256 ? 0 : t == 128 ? 1 : 2;
  const bool kept = epi == EPI_ACT || epi == EPI_SWIGLU;  // 3 bytes a value are written beside the result
  constexpr double K_STORE[3] = {0.0245, 0.0165, 0.018}, K_KEPT[3] = {0.0182, 0.0135, 0.0115}, K_LONE[3] = {0.0245, 0.0085, 0.005};
  constexpr double TILE_STORE[3] = {5.0, 3.0, 2.0}, TILE_KEPT[3] = {28.0, 16.0, 12.0};
  const double twice = low ? 2.0 : 1.0, round_k = twice * (kept ? K_KEPT[i] : K_STORE[i]), lone_k = twice * K_LONE[i] < round_k ? twice * K_LONE[i] : round_k;
  const double tile_us = kept || epi == EPI_SWIGLU_BWD ? TILE_KEPT[i] : TILE_STORE[i];
  const int64_t left = tiles % at_once;
  int64_t most = epi == EPI_STORE && left ? at_once / left : 1;
  if (most > K / 256) most = K / 256;
  if (most < 1) most = 1;
  for (int64_t next = 1, parts = 1; parts <= most; parts = next) {  // 1 .. 8, steps of a quarter, the most
    next = parts + (parts < 8 ? 1 : parts / 4);
    if (parts < most && next > most) next = most;
    const int64_t kp = (K + parts - 1) / parts + BK - 1, k_part = kp / BK * BK;
    const double share = (double)left * parts / at_once;  // of the last round's places
    const double last_k = lone_k + (round_k - lone_k) * share;
    double us = (double)(tiles / at_once) * (K * round_k + tile_us) + (left ? k_part * last_k + tile_us : 0.0);
    if (parts > 1) us += 5.0 + (double)left * parts * t * t * 4 * 2 / 5e6;
    if (us < best.us) {
      best.us = us;
      best.tile = t;
      best.tiles_m = (int)tm;
      best.tiles_n = (int)tn;
      best.k_part = k_part;
      best.parts = (int)((K + k_part - 1) / k_part);
      // (tiles of 256: the last round is addressed as parts, also where they are whole)
      best.whole = (int)(best.parts == 1 && t != 256 ? tiles : tiles - left);
    }
  }
  return best;
}

GradPlan plan_of(int64_t M, int64_t N, int64_t K, int epi, bool low) {
  GradPlan best = {};
  best.us = 1e30;
  for (int t : {256, 128, 64}) {
    const GradPlan g = plan_tiles(t, M, N, K, epi, low);
    if (g.us < best.us) best = g;
  }
  return best;
}

GradGemm product(const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K) {
  GradGemm p = {};
  p.A = reinterpret_cast<const uint16_t*>(A);
  p.B = reinterpret_cast<const uint16_t*>(B);
  p.lda = lda;
  p.ldb = ldb;
  p.C = C;
  p.ldc = ldc;
  p.M = M;
  p.N = (int)N;
  p.K = K;
  p.res_dtype = -1;
  return p;
}

void apply(GradGemm& p, const GradPlan& g, void* partial) {
  p.tiles_m = g.tiles_m;
  p.tiles_n = g.tiles_n;
  p.whole = g.whole;
  p.parts = g.parts;
  p.k_part = g.k_part;
  p.partial = reinterpret_cast<float*>(partial);
}

hipError_t finish(const GradGemm& p, int64_t n, const GradGemm& q, int64_t m, int tile, uint16_t* bias, hipStream_t stream) {
  const int64_t per_tile = tile * tile / 8 / 256;
  n *= per_tile;
  m *= per_tile;
  const int64_t blocks = n + m + (bias ? (q.M + 255) / 256 : 0);
  if (blocks == 0) return hipSuccess;
#define GO(T) hipLaunchKernelGGL(grad_finish_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, p, q, (int)n, (int)m, bias)
  if (tile == 256) GO(256);
  else if (tile == 128) GO(128);
  else GO(64);
#undef GO
  return hipGetLastError();
}

// up to two workgroups a CU, which tiles of 64 in four stages have room for (beyond: 1536 of them, [2048, 2048] of k = 256, 12.3 -> 15.3 us)
bool few_items(int64_t n) { return n <= 512; }

// one product; `bias`: from the sums over k of a dw
template <bool A_TR, bool B_TR, int EPI>
hipError_t launch(GradGemm& p, const GradPlan& g, void* partial, uint16_t* bias, hipStream_t stream) {
  if (g.tile == 0) return hipErrorInvalidValue;
  apply(p, g, partial);
  if (g.tile == 256) {
    const unsigned grid = g.whole ? 256 : (unsigned)((g.left() * g.parts + 7) / 8 * 8);
    hipLaunchKernelGGL((gemm_grad_big_kernel<A_TR, B_TR, EPI>), dim3(grid), dim3(512), BIG_LDS, stream, p);
  } else {
    const dim3 grid((unsigned)g.items()), block(256);
    auto go = [&](auto low) {
      constexpr bool LOW = decltype(low)::value;
      if (g.tile == 128) hipLaunchKernelGGL((gemm_grad_tile_kernel<128, 2, A_TR, B_TR, EPI, LOW>), grid, block, 0, stream, p);
      else if (few_items(g.items())) hipLaunchKernelGGL((gemm_grad_tile_kernel<64, 4, A_TR, B_TR, EPI, LOW>), grid, block, 0, stream, p);
      else hipLaunchKernelGGL((gemm_grad_tile_kernel<64, 2, A_TR, B_TR, EPI, LOW>), grid, block, 0, stream, p);
    };
    if (p.A_low || p.B_low) {
      if constexpr (EPI == EPI_STORE) go(std::true_type{});
      else return hipErrorInvalidValue;  // (no such product)
    } else {
      go(std::false_type{});
    }
  }
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : finish(p, 0, p, g.parts > 1 ? g.left() : 0, g.tile, bias, stream);
}

// A product c [M, N] = a[M, K] w[K, N] of tokens (dx, or dh with what follows from it) and the gradient dw [K2, N2] = b[M, K2]^T x[M, N2] of a
// weight, either of them or both: in one launch of tiles of one size, or one after the other where the estimates' sum is TOGETHER_US lower (each runs
// in the other's gaps, and a launch less).  Of 389 pairs, against one launch only where neither alone would have tiles of 256: 31 faster by 3 to 27 %
// (4870 tokens, 2112 x 384: 42 -> 34 us; the gated MLP's of 858 tokens, 2944 -> 1424: 99 -> 78), 10 slower by 3 to 4 %.
constexpr double TOGETHER_US = 5.0;
struct GradPair {
  bool first, second, sums;
  GradPlan g, h;
  bool together;
  int64_t partial_bytes, second_bytes, sum_bytes;
};
GradPair plan_pair(bool first, int64_t M, int64_t N, int64_t K, int epi, bool low, bool second, int64_t N2, int64_t K2, bool low2, bool sums) {
  GradPair r = {};
  r.first = first;
  r.second = second;
  r.sums = sums && second;
  if (first) r.g = plan_of(M, N, K, epi, low);
  if (second) r.h = plan_of(N2, K2, M, EPI_STORE, low2);
  if (first && second && r.g.tile && r.h.tile) {
    double us = r.g.us + r.h.us;
    for (int t : {128, 64}) {
      const GradPlan g = plan_tiles(t, M, N, K, epi, low), h = plan_tiles(t, N2, K2, M, EPI_STORE, low2);
      if (g.us + h.us - TOGETHER_US < us && g.items() + h.items() < 1 << 24) {
        us = g.us + h.us - TOGETHER_US;
        r.together = true;
        r.g = g;
        r.h = h;
      }
    }
  }
  r.partial_bytes = first ? r.g.partial_bytes() : 0;
  r.second_bytes = second ? r.h.partial_bytes() : 0;
  r.sum_bytes = r.sums ? r.h.row_sum_bytes() : 0;
  return r;
}
int64_t pair_bytes(const GradPair& r) { return r.partial_bytes + r.second_bytes + r.sum_bytes; }

template <int EPI>
hipError_t launch_pair(const GradPair& r, GradGemm p, GradGemm q, void* workspace, void* bias, hipStream_t stream) {
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  unsigned char* const ws_q = ws + r.partial_bytes;
  if (r.sums) q.row_sums = reinterpret_cast<float*>(ws_q + r.second_bytes);
  uint16_t* const b = r.sums ? reinterpret_cast<uint16_t*>(bias) : nullptr;
  if (!r.together) {
    hipError_t e = hipSuccess;
    if (r.first) e = launch<false, true, EPI>(p, r.g, ws, nullptr, stream);
    if (e == hipSuccess && r.second) e = launch<true, true, EPI_STORE>(q, r.h, ws_q, b, stream);
    return e;
  }
  apply(p, r.g, ws);
  apply(q, r.h, ws_q);
  const dim3 grid((unsigned)(r.g.items() + r.h.items())), block(256);
  const int n = (int)r.g.items();
  auto go = [&](auto low) {
    constexpr bool LOW = decltype(low)::value;
    if (r.g.tile == 128) hipLaunchKernelGGL((gemm_grad_pair_kernel<128, 2, EPI, LOW>), grid, block, 0, stream, p, q, n);
    else if (few_items(r.g.items() + r.h.items())) hipLaunchKernelGGL((gemm_grad_pair_kernel<64, 4, EPI, LOW>), grid, block, 0, stream, p, q, n);
    else hipLaunchKernelGGL((gemm_grad_pair_kernel<64, 2, EPI, LOW>), grid, block, 0, stream, p, q, n);
  };
  if (q.A_low || q.B_low) go(std::true_type{});
  else go(std::false_type{});
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : finish(p, r.g.parts > 1 ? r.g.left() : 0, q, r.h.parts > 1 ? r.h.left() : 0, r.g.tile, b, stream);
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t more(int64_t a, int64_t b) { return a > b ? a : b; }

// Few tokens: what one product rounds for the next (h; dgate and dup; dz) is kept as two bf16 a value, and the products behind it go over k
// twice.  Their errors do not average out over many tokens, and the products are bound by the weights' way through memory more than by the second sweep
// (9 tokens, 1536 -> 6144: forward 20 us with one bf16 a value, 24 with two, backward 40 and 51; 33 tokens, 384 -> 1088: 10 and 13, 13 and 16).
bool few(int64_t M) { return M <= AERIS_FEW_TOKENS; }

bool needs_dz(const aeris_linear_grad& a) { return (a.dy_dtype == AERIS_F32 || a.act != AERIS_ACT_NONE) && (a.dx || a.dw || a.dz); }
// the bias' gradient: with dz where that has to be made, otherwise with dw
bool bias_apart(const aeris_linear_grad& a) { return a.dbias && (needs_dz(a) || !a.dw || a.dy_dtype == AERIS_F32 || a.act != AERIS_ACT_NONE); }
bool low_dz(const aeris_linear_grad& a) { return needs_dz(a) && few(a.M) && (a.dx || a.dw); }
GradPair linear_pair(const aeris_linear_grad& a) {
  return plan_pair(a.dx, a.M, a.K, a.N, EPI_STORE, low_dz(a), a.dw, a.N, a.K, low_dz(a), a.dbias && !bias_apart(a));
}
GradPair hidden_pair(const aeris_feed_forward_grad& a) {  // (few tokens: no tiles of 256, whose epilogue has no remainders)
  return plan_pair(a.dx || a.dw1, a.M, a.H, a.d, EPI_SWIGLU_BWD, few(a.M), a.dw2, a.d, a.H, few(a.M), false);
}
GradPair token_pair(const aeris_feed_forward_grad& a) {
  return plan_pair(a.dx, a.M, a.d, 2 * a.H, EPI_STORE, few(a.M), a.dw1, 2 * a.H, a.d, few(a.M), false);
}

}  // namespace

hipError_t gemm_grad_configure() {
  hipError_t e = hipSuccess;
  auto one = [&](const void* f) {
    if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, BIG_LDS);
  };
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<false, false, EPI_STORE>));
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<false, false, EPI_ACT>));
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<false, false, EPI_SWIGLU>));
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<false, true, EPI_STORE>));
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<false, true, EPI_SWIGLU_BWD>));
  one(reinterpret_cast<const void*>(gemm_grad_big_kernel<true, true, EPI_STORE>));
  return e;
}

hipError_t linear_train_launch(const aeris_linear_train& a, hipStream_t stream) {
  GradGemm p = product(a.x, a.K, a.w, a.K, a.y, a.N, a.M, a.N, a.K);
  p.c_f32 = a.y_dtype == AERIS_F32;
  p.bias = reinterpret_cast<const uint16_t*>(a.bias);
  p.residual = a.residual;
  p.res_dtype = a.residual ? (int)a.res_dtype : -1;
  p.kept = reinterpret_cast<uint16_t*>(a.z);
  p.act = (int)a.act;
  return launch<false, false, EPI_ACT>(p, plan_of(a.M, a.N, a.K, EPI_ACT, false), nullptr, nullptr, stream);
}

int64_t linear_grad_workspace_bytes(const aeris_linear_grad& a) {
  int64_t n = 0;
  if (needs_dz(a) && !a.dz) n += up256(a.M * a.N * 2);
  if (low_dz(a)) n += up256(a.M * a.N * 2);
  if (bias_apart(a)) n += up256((int64_t)act_grad_parts(a.M, (int)a.N) * a.N * 4);
  return n + pair_bytes(linear_pair(a));
}

hipError_t linear_grad_launch(const aeris_linear_grad& a, void* workspace, hipStream_t stream) {
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  auto take = [&](int64_t bytes) {
    unsigned char* const at = ws;
    ws += up256(bytes);
    return at;
  };
  void* const dz = !needs_dz(a) ? nullptr : a.dz ? a.dz : take(a.M * a.N * 2);
  void* const dz_low = low_dz(a) ? take(a.M * a.N * 2) : nullptr;
  if (dz || bias_apart(a)) {
    float* const partial = bias_apart(a) ? reinterpret_cast<float*>(take((int64_t)act_grad_parts(a.M, (int)a.N) * a.N * 4)) : nullptr;
    const hipError_t e = act_grad_launch(a.dy, a.dy_dtype == AERIS_F32, a.z, dz, dz_low, partial, bias_apart(a) ? a.dbias : nullptr, a.M, (int)a.N, (int)a.act, stream);
    if (e != hipSuccess) return e;
  }
  const void* const g = dz ? dz : a.dy;
  GradGemm p = product(g, a.N, a.w, a.K, a.dx, a.K, a.M, a.K, a.N), q = product(g, a.N, a.x, a.K, a.dw, a.K, a.N, a.K, a.M);
  p.A_low = q.A_low = reinterpret_cast<const uint16_t*>(dz_low);
  return launch_pair<EPI_STORE>(linear_pair(a), p, q, ws, a.dbias, stream);
}

// The second projection has nothing to keep: it is the inference kernels' product (14400 tokens, H 6144 -> 1536: 204 us, here 240), but for few
// tokens of many hidden channels, whose k only the kernels here cut into parts (9 tokens: 22 us there, 12 here; both passes of 384 tokens 59 and 54, of
// 512 the same; H 4096: 29 and 28; H 2048 and less: 1 to 3 us shorter there), where h has remainders, and for k that is no multiple of 64.
static bool second_is_own(const aeris_feed_forward& a) { return a.H % 64 != 0 || (a.M <= 384 && a.H >= 4096) || few(a.M); }

int64_t feed_forward_train_workspace_bytes(const aeris_feed_forward& a) {
  return second_is_own(a) ? plan_of(a.M, a.d, a.H, EPI_STORE, few(a.M)).partial_bytes() : 0;
}

hipError_t feed_forward_train_launch(const aeris_feed_forward& a, void* workspace, hipStream_t stream) {
  GradGemm p = product(a.x, a.d, a.w1, a.d, a.h, a.H, a.M, a.H, a.d);
  p.kept = reinterpret_cast<uint16_t*>(a.gate_up);
  if (few(a.M)) p.C_low = reinterpret_cast<uint16_t*>(a.h) + a.M * a.H;
  const hipError_t e = launch<false, false, EPI_SWIGLU>(p, plan_of(a.M, a.H, a.d, EPI_SWIGLU, few(a.M)), nullptr, nullptr, stream);
  if (e != hipSuccess) return e;
  if (!second_is_own(a))
    return gemm_launch(a.h, a.w2, a.y, nullptr, nullptr, nullptr, a.M, (int)a.d, (int)a.H, a.d, AERIS_ACT_NONE, 0, AERIS_BF16, 0, a.M, 0, 0, 1.0f, 0, stream);
  GradGemm q = product(a.h, a.H, a.w2, a.H, a.y, a.d, a.M, a.d, a.H);
  q.A_low = p.C_low;
  return launch<false, false, EPI_STORE>(q, plan_of(a.M, a.d, a.H, EPI_STORE, few(a.M)), workspace, nullptr, stream);
}

int64_t feed_forward_grad_workspace_bytes(const aeris_feed_forward_grad& a) {
  return (a.dx || a.dw1 ? up256(a.M * a.H * (few(a.M) ? 8 : 4)) : 0) + more(pair_bytes(hidden_pair(a)), pair_bytes(token_pair(a)));
}

hipError_t feed_forward_grad_launch(const aeris_feed_forward_grad& a, void* workspace, hipStream_t stream) {
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  uint16_t* const dgu = reinterpret_cast<uint16_t*>(ws);
  uint16_t* const dgu_low = few(a.M) ? dgu + a.M * 2 * a.H : nullptr;
  if (a.dx || a.dw1) ws += up256(a.M * a.H * (few(a.M) ? 8 : 4));
  GradGemm p = product(a.dy, a.d, a.w2, a.H, dgu, 2 * a.H, a.M, a.H, a.d), q = product(a.dy, a.d, a.h, a.H, a.dw2, a.H, a.d, a.H, a.M);
  p.kept = reinterpret_cast<uint16_t*>(const_cast<void*>(a.gate_up));
  p.C_low = dgu_low;
  if (few(a.M)) q.B_low = q.B + a.M * a.H;
  const hipError_t e = launch_pair<EPI_SWIGLU_BWD>(hidden_pair(a), p, q, ws, nullptr, stream);
  if (e != hipSuccess) return e;
  p = product(dgu, 2 * a.H, a.w1, a.d, a.dx, a.d, a.M, a.d, 2 * a.H);
  q = product(dgu, 2 * a.H, a.x, a.d, a.dw1, a.d, 2 * a.H, a.d, a.M);
  p.A_low = q.A_low = dgu_low;
  return launch_pair<EPI_STORE>(token_pair(a), p, q, ws, nullptr, stream);
}

}  // namespace aeris
