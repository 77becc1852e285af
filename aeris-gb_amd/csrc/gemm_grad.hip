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
// are XOR-swizzled by the k row so that the eight k rows which half a wave reads at once lie on different banks.
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
  int64_t M, K;
  int64_t lda, ldb;  // elements between rows
  int N;             // columns of the result
  void* C;           // SWIGLU: h; SWIGLU_BWD: [dgate | dup]
  int64_t ldc;
  int c_f32;
  int64_t k_per_split, split_stride;  // columns k of one part (a multiple of 64); elements between the parts' results
  const uint16_t* bias;
  const void* residual;
  int res_dtype;  // -1: none
  uint16_t* saved;  // ACT: z; SWIGLU: [gate | up], rows of 2 N
  const uint16_t* gate_up;  // SWIGLU_BWD
  int act;
  int tiles_m, tiles_n;
};

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
__device__ __forceinline__ void store8(void* C, int f32, int64_t at, const float (&o)[8]) {
  if (f32) {
    f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(C) + at);
    q[0] = f32x4{o[0], o[1], o[2], o[3]};
    q[1] = f32x4{o[4], o[5], o[6], o[7]};
  } else {
    *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(C) + at) = narrow8(o);
  }
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

// One wave's loads of a panel.  `base`: the tile's first row (column, TR) at k = 0; rows: how many of them the matrix has from there.
// SWIGLU weights: row 64 c + s of the tile is gate row 32 c + s, from s = 32 on up row 32 c + s - 32 (`up_rows` further on).
template <bool TR, int ROWS, int WAVES, bool SWIGLU_ROWS>
struct Loader {
  using P = Panel<TR, ROWS, WAVES>;
  const uint16_t* base;
  int64_t ld, rows, k_end;
  int64_t up_rows;
  uint32_t voff[2];
  uint32_t kchunk[2];
  int wave;

  __device__ __forceinline__ void init(const uint16_t* b, int64_t ld_, int64_t rows_, int64_t k_end_, int64_t up, int lane, int wave_) {
    base = b;
    ld = ld_;
    rows = rows_;
    k_end = k_end_;
    up_rows = up;
    wave = wave_;
#pragma unroll
    for (int par = 0; par < 2; ++par) {
      if (TR) {
        constexpr int RPI = 512 / P::COLS, CPR = P::COLS / 8;  // k rows of a load instruction, chunks of a row
        const int kr = lane / CPR, pos = lane % CPR;
        // pair_key of the instruction's k rows: with the instruction's number (par: whether k has bit 3) and the lane's
        const int key = P::COLS == 128 ? kr | (par << 2) : ((kr >> 1) & 1) | (par << 1);
        static_assert(RPI == 4 || RPI == 8, "panels of 128 or 64 columns");
        voff[par] = (uint32_t)(kr * ld * 2) + (uint32_t)((pos ^ (2 * key)) * 16);
        kchunk[par] = 0;
      } else {
        const int dr = lane >> 4, pos = lane & 15;
        const int logical = pos ^ (par * 4 + dr);
        voff[par] = (uint32_t)((dr * 2 + (logical >> 3)) * ld * 2 + (logical & 7) * 16);
        kchunk[par] = (uint32_t)(logical & 7) * 8;
      }
    }
  }

  // k-tile that begins at k0, into the stage at LDS address `stage`
  __device__ __forceinline__ void issue(int64_t k0, uint32_t stage) const {
    int64_t left = k_end - k0;  // of k
    if (left < 0) left = 0;
    if (TR) {
      const int64_t kr = left < BK ? left : BK;
      constexpr int PANELS = ROWS / P::COLS, IPP = P::COLS * BK * 2 / 1024;  // instructions of a panel
      constexpr int RPI = 512 / P::COLS;
#pragma unroll
      for (int j = 0; j < P::LOADS; ++j) {
        const int i = wave * P::LOADS + j;  // instruction of the tile: panel i / IPP
        const int panel = i / IPP, ip = i % IPP;
        const int64_t cols = rows - panel * P::COLS;
        const uint32_t bytes = kr > 0 && cols > 0 ? (uint32_t)(((kr - 1) * ld + cols) * 2) : 0u;
        const lds_dma_rsrc rs = make_lds_dma_rsrc(base + k0 * ld + panel * P::COLS, bytes);
        lds_dma_load16(rs, stage + (uint32_t)i * 1024u, voff[RPI == 4 ? (j >> 1) & 1 : j & 1], (uint32_t)(ip * RPI) * (uint32_t)(ld * 2));
      }
      static_assert(PANELS == 1 || PANELS == 2, "one or two panels");
      static_assert(RPI != 4 || P::LOADS % 4 == 0, "bit 3 of k follows from the number within the wave");
      static_assert(RPI != 8 || P::LOADS % 2 == 0, "bit 3 of k follows from the number within the wave");
    } else {
      const bool tail = left < BK;
      const int64_t all = SWIGLU_ROWS ? up_rows + rows : rows < ROWS ? rows : ROWS;
      const uint32_t bytes = left > 0 ? (uint32_t)(all * ld * 2) : 0u;
      const lds_dma_rsrc rs = make_lds_dma_rsrc(base, bytes);
#pragma unroll
      for (int j = 0; j < P::LOADS; ++j) {
        const int i = wave * P::LOADS + j;  // rows 8 i ..
        int64_t row = 8 * i;
        if (SWIGLU_ROWS) row = (i >> 3) * 32 + (i & 3) * 8 + ((i & 4) ? up_rows : 0);
        static_assert(P::LOADS % 2 == 0, "the parity of 8-row blocks follows from the number within the wave");
        uint32_t vo = voff[j & 1];
        // (k beyond the matrix: an offset beyond any buffer's size, which arrives as zeros)
        if (tail && kchunk[j & 1] >= (uint32_t)left) vo = 0x80000000u;
        lds_dma_load16(rs, stage + (uint32_t)i * 1024u, vo, (uint32_t)(row * ld * 2) + (uint32_t)(k0 * 2));
      }
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

// ---- epilogue of a wave's FM x FN fragments, rows from row0, columns from col0.  A lane has 4 consecutive columns 4 q .. of row
// l15 of a fragment; a swap between lane rows of two neighbouring column fragments gives it 8 consecutive ones.
template <int FM, int FN>
__device__ __forceinline__ void eight_columns(const f32x4 (&a)[FN], int m, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[2 * m][e]), __float_as_uint(a[2 * m + 1][e]), false, false);
    o[e] = __uint_as_float(r[0]);
    o[4 + e] = __uint_as_float(r[1]);
  }
}

template <int EPI, int FM, int FN>
__device__ __forceinline__ void grad_epilogue(const GradGemm& p, const f32x4 (&acc)[FM][FN], int64_t row0, int col0, int split, int lane) {
  const int l15 = lane & 15, q = lane >> 4;
  constexpr int NP = (EPI == EPI_SWIGLU ? FN / 2 : FN) / 2;  // column pairs of the result
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t row = row0 + 16 * i + l15;
#pragma unroll
    for (int m = 0; m < NP; ++m) {
      const int col = col0 + 32 * m + 16 * (q & 1) + 8 * (q >> 1);
      float o[8];
      eight_columns<FM, FN>(acc[i], m, o);
      if constexpr (EPI == EPI_SWIGLU) {
        float up[8];
        eight_columns<FM, FN>(acc[i], m + NP, up);
        if (row >= p.M || col >= p.N) continue;
        uint16_t* s = p.saved + row * (2 * (int64_t)p.N) + col;
        *reinterpret_cast<u32x4*>(s) = narrow8(o);
        *reinterpret_cast<u32x4*>(s + p.N) = narrow8(up);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = silu_f(o[e]) * up[e];
        store8(p.C, 0, row * p.ldc + col, o);
      } else {
        if (row >= p.M || col >= p.N) continue;
        if constexpr (EPI == EPI_STORE) {
          store8(p.C, p.c_f32, split * p.split_stride + row * p.ldc + col, o);
        } else if constexpr (EPI == EPI_ACT) {
          if (p.bias) {
            float b[8];
            widen8(*reinterpret_cast<const u32x4*>(p.bias + col), b);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += b[e];
          }
          *reinterpret_cast<u32x4*>(p.saved + row * (int64_t)p.N + col) = narrow8(o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = p.act == AERIS_ACT_SILU ? silu_f(o[e]) : p.c_f32 ? gelu_erf_f(o[e]) : gelu_erf_bf16_f(o[e]);
          if (p.res_dtype >= 0) {
            const int64_t at = row * (int64_t)p.N + col;
            float r[8];
            if (p.res_dtype == AERIS_F32) {
              const float* src = reinterpret_cast<const float*>(p.residual) + at;
              const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                r[e] = a[e];
                r[4 + e] = b[e];
              }
            } else {
              widen8(*reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.residual) + at), r);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += r[e];
          }
          store8(p.C, p.c_f32, row * p.ldc + col, o);
        } else {  // EPI_SWIGLU_BWD
          const int64_t at = row * (2 * (int64_t)p.N) + col;
          float g[8], u[8], dg[8];
          widen8(*reinterpret_cast<const u32x4*>(p.gate_up + at), g);
          widen8(*reinterpret_cast<const u32x4*>(p.gate_up + at + p.N), u);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float s = sigmoid_f(g[e]);
            dg[e] = o[e] * u[e] * dsilu_f(g[e], s);
            o[e] *= g[e] * s;
          }
          store8(p.C, 0, at, dg);
          store8(p.C, 0, at + p.N, o);
        }
      }
    }
  }
}

// ---- tiles of T x T (128 or 64), four waves two by two, two stages; two or more workgroups a CU fill each other's waits
template <int T, bool A_TR, bool B_TR, int EPI>
__global__ void __launch_bounds__(256, 2) gemm_grad_tile_kernel(GradGemm p) {
  constexpr bool SWIGLU = EPI == EPI_SWIGLU;
  // waves over the tile: two by two; SwiGLU tiles of 64 four by one, so that a wave has a gate column's up column too
  constexpr int WN = SWIGLU && T == 64 ? 1 : 2, WM = 4 / WN;
  constexpr int FM = T / WM / 16, FN = T / WN / 16;  // fragments of a wave
  constexpr int BN_OUT = SWIGLU ? T / 2 : T;
  using PA = Panel<A_TR, T, 4>;
  using PB = Panel<B_TR, T, 4>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * (PA::BYTES + PB::BYTES)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles = p.tiles_m * p.tiles_n;
  const int split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles;
  const int tile_n = tile % p.tiles_n, tile_m = tile / p.tiles_n;
  const int64_t m0 = (int64_t)tile_m * T;
  const int n0 = tile_n * BN_OUT;
  const int64_t k_begin = split * p.k_per_split;
  int64_t k_end = k_begin + p.k_per_split;
  if (k_end > p.K) k_end = p.K;
  const int turns = k_end > k_begin ? (int)((k_end - k_begin + BK - 1) / BK) : 0;

  Loader<A_TR, T, 4, false> la;
  Loader<B_TR, T, 4, SWIGLU> lb;
  la.init(p.A + (A_TR ? m0 : m0 * p.lda), p.lda, p.M - m0, k_end, 0, lane, wave);
  lb.init(p.B + (B_TR ? (int64_t)n0 : n0 * p.ldb), p.ldb, p.N - n0, k_end, p.N, lane, wave);
  Fragments<A_TR, T, 4, FM> fa;
  Fragments<B_TR, T, 4, FN> fb;
  fa.init(wm * (T / WM), lane);
  fb.init(wn * (T / WN), lane);

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const uint32_t lds0 = lds_byte_address(smem);
  auto issue = [&](int t) {
    const uint32_t stage = lds0 + (uint32_t)(t & 1) * (PA::BYTES + PB::BYTES);
    la.issue(k_begin + (int64_t)t * BK, stage);
    lb.issue(k_begin + (int64_t)t * BK, stage + PA::BYTES);
  };
  if (turns > 0) issue(0);
  for (int t = 0; t < turns; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // stage t is there; the other one has been read
    if (t + 1 < turns) issue(t + 1);
    const uint32_t sa = lds0 + (uint32_t)(t & 1) * (PA::BYTES + PB::BYTES), sb = sa + PA::BYTES;
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
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
  }
  grad_epilogue<EPI, FM, FN>(p, acc, m0 + wm * (T / WM), n0 + wn * (BN_OUT / WN), split, lane);
}

// ---- sums over the parts of the tokens, in order: out[i] = sum of part[s][i]; 8 elements a thread
__global__ void __launch_bounds__(256) split_sum_kernel(const float* part, void* out, int out_f32, int64_t n, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const f32x4* q = reinterpret_cast<const f32x4*>(part + s * n + i);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += a[e];
      o[4 + e] += b[e];
    }
  }
  store8(out, out_f32, i, o);
}

// ---- dz = dy act'(z) (ACT_NONE: dy) rounded to bf16, and the sums of the unrounded dz over the tokens: a workgroup takes 512 columns
// and a share of the rows, its four waves every fourth of them; 8 columns a lane
struct ActGrad {
  const void* dy;
  const uint16_t* z;
  uint16_t* dz;    // NULL: not wanted (dy is bf16 and there is no activation)
  float* partial;  // [row shares][N], or NULL
  int64_t M, rows_per_block;
  int N, dy_f32, act;
};

__global__ void __launch_bounds__(256) act_grad_kernel(ActGrad p) {
  __shared__ f32x4 lds[4][128];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = (blockIdx.y * 64 + lane) * 8;
  const bool ok = col < p.N;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t first = (int64_t)blockIdx.x * p.rows_per_block;
  int64_t end = first + p.rows_per_block;
  if (end > p.M) end = p.M;
  if (ok) {
    for (int64_t row = first + w; row < end; row += 4) {
      const int64_t at = row * p.N + col;
      float d[8];
      if (p.dy_f32) {
        const f32x4* q = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p.dy) + at);
        const f32x4 a = q[0], b = q[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = a[e];
          d[4 + e] = b[e];
        }
      } else {
        widen8(*reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.dy) + at), d);
      }
      if (p.act != AERIS_ACT_NONE) {
        float z[8];
        widen8(*reinterpret_cast<const u32x4*>(p.z + at), z);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= p.act == AERIS_ACT_SILU ? dsilu_f(z[e], sigmoid_f(z[e])) : dgelu_f(z[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += d[e];
      if (p.dz) *reinterpret_cast<u32x4*>(p.dz + at) = narrow8(d);
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

// 32 columns a workgroup, 8 threads share a column's partial sums
__global__ void __launch_bounds__(256) bias_sum_kernel(const float* partial, uint16_t* out, int parts, int N) {
  __shared__ float lds[8][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float t = 0.f;
  if (col < N)
    for (int b = r; b < parts; b += 8) t += partial[(int64_t)b * N + col];
  lds[r][c] = t;
  __syncthreads();
  if (r == 0 && col < N) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += lds[k][c];
    out[col] = (uint16_t)f32_to_bf16_bits(v);
  }
}

int act_grad_parts(int64_t M, int N) {
  const int64_t col_blocks = (N + 511) / 512;
  int64_t n = 2048 / col_blocks;
  if (n > (M + 15) / 16) n = (M + 15) / 16;
  return n < 1 ? 1 : (int)n;
}

hipError_t act_grad_launch(const void* dy, int dy_f32, const void* z, void* dz, float* partial, void* dbias, int64_t M, int N, int act,
                           hipStream_t stream) {
  ActGrad p;
  p.dy = dy;
  p.z = reinterpret_cast<const uint16_t*>(z);
  p.dz = reinterpret_cast<uint16_t*>(dz);
  p.partial = dbias ? partial : nullptr;
  p.M = M;
  p.N = N;
  p.dy_f32 = dy_f32;
  p.act = act;
  const int parts = act_grad_parts(M, N);
  p.rows_per_block = (M + parts - 1) / parts;
  hipLaunchKernelGGL(act_grad_kernel, dim3((unsigned)parts, (unsigned)((N + 511) / 512)), dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !dbias) return e;
  hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)((N + 31) / 32)), dim3(256), 0, stream, partial, reinterpret_cast<uint16_t*>(dbias), parts, N);
  return hipGetLastError();
}

// ---- how a product is cut

struct GradPlan {
  int tile;
  int splits;
  int64_t k_per_split;
};

GradPlan plan_of(int64_t M, int N, int64_t K, bool may_split) {
  GradPlan g;
  auto tiles_of = [&](int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
  g.tile = tiles_of(128) >= 256 || (may_split && tiles_of(128) * (K / 512) >= 256) ? 128 : 64;
  g.splits = 1;
  const int64_t tiles = tiles_of(g.tile);
  if (may_split && tiles < 512) {
    int64_t s = 512 / tiles;
    if (s > K / 512) s = K / 512;
    g.splits = s < 1 ? 1 : (int)s;
  }
  g.k_per_split = ((K + g.splits - 1) / g.splits + BK - 1) / BK * BK;
  if (g.k_per_split < BK) g.k_per_split = BK;
  if (K > 0) g.splits = (int)((K + g.k_per_split - 1) / g.k_per_split);
  return g;
}

template <bool A_TR, bool B_TR, int EPI>
hipError_t launch(GradGemm p, const GradPlan& g, hipStream_t stream) {
  const int bn = EPI == EPI_SWIGLU ? g.tile / 2 : g.tile;
  const int64_t tm = (p.M + g.tile - 1) / g.tile, tn = (p.N + bn - 1) / bn;
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  p.k_per_split = g.k_per_split;
  const int64_t blocks = tm * tn * g.splits;
  if (blocks >= 1 << 24) return hipErrorInvalidValue;
  if (g.tile == 128) hipLaunchKernelGGL((gemm_grad_tile_kernel<128, A_TR, B_TR, EPI>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((gemm_grad_tile_kernel<64, A_TR, B_TR, EPI>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
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

// dw [N, K] = dz[M, N]^T x[M, K]
hipError_t weight_grad(const void* dz, const void* x, void* dw, int64_t M, int64_t N, int64_t K, float* partial, hipStream_t stream) {
  const GradPlan g = plan_of(N, (int)K, M, true);
  GradGemm p = product(dz, N, x, K, dw, K, N, K, M);
  if (g.splits > 1) {
    p.C = partial;
    p.c_f32 = 1;
    p.split_stride = N * K;
  }
  hipError_t e = launch<true, true, EPI_STORE>(p, g, stream);
  if (e != hipSuccess || g.splits == 1) return e;
  hipLaunchKernelGGL(split_sum_kernel, dim3((unsigned)((N * K / 8 + 255) / 256)), dim3(256), 0, stream, partial, dw, 0, N * K, g.splits);
  return hipGetLastError();
}
int64_t weight_grad_bytes(int64_t M, int64_t N, int64_t K) {
  const GradPlan g = plan_of(N, (int)K, M, true);
  return g.splits > 1 ? g.splits * N * K * 4 : 0;
}

// dx [M, K] = dz[M, N] w[N, K]
hipError_t input_grad(const void* dz, const void* w, void* dx, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  return launch<false, true, EPI_STORE>(product(dz, N, w, K, dx, K, M, K, N), plan_of(M, (int)K, N, false), stream);
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

bool needs_dz(const aeris_linear_grad& a) { return (a.dy_dtype == AERIS_F32 || a.act != AERIS_ACT_NONE) && (a.dx || a.dw || a.dz); }

}  // namespace

hipError_t linear_train_launch(const aeris_linear_train& a, hipStream_t stream) {
  GradGemm p = product(a.x, a.K, a.w, a.K, a.y, a.N, a.M, a.N, a.K);
  p.c_f32 = a.y_dtype == AERIS_F32;
  p.bias = reinterpret_cast<const uint16_t*>(a.bias);
  p.residual = a.residual;
  p.res_dtype = a.residual ? (int)a.res_dtype : -1;
  p.saved = reinterpret_cast<uint16_t*>(a.z);
  p.act = (int)a.act;
  return launch<false, false, EPI_ACT>(p, plan_of(a.M, (int)a.N, a.K, false), stream);
}

int64_t linear_grad_workspace_bytes(const aeris_linear_grad& a) {
  int64_t n = 0;
  if (needs_dz(a) && !a.dz) n += up256(a.M * a.N * 2);
  if (a.dbias) n += up256((int64_t)act_grad_parts(a.M, (int)a.N) * a.N * 4);
  if (a.dw) n += weight_grad_bytes(a.M, a.N, a.K);
  return n;
}

hipError_t linear_grad_launch(const aeris_linear_grad& a, void* workspace, hipStream_t stream) {
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  const void* dz = a.dy;
  void* dz_out = nullptr;
  if (needs_dz(a)) {
    dz_out = a.dz ? a.dz : ws;
    if (!a.dz) ws += up256(a.M * a.N * 2);
    dz = dz_out;
  }
  if (dz_out || a.dbias) {
    float* partial = reinterpret_cast<float*>(ws);
    if (a.dbias) ws += up256((int64_t)act_grad_parts(a.M, (int)a.N) * a.N * 4);
    const hipError_t e = act_grad_launch(a.dy, a.dy_dtype == AERIS_F32, a.z, dz_out, partial, a.dbias, a.M, (int)a.N, (int)a.act, stream);
    if (e != hipSuccess) return e;
  }
  if (a.dx) {
    const hipError_t e = input_grad(dz, a.w, a.dx, a.M, a.N, a.K, stream);
    if (e != hipSuccess) return e;
  }
  return a.dw ? weight_grad(dz, a.x, a.dw, a.M, a.N, a.K, reinterpret_cast<float*>(ws), stream) : hipSuccess;
}

hipError_t feed_forward_train_launch(const aeris_feed_forward& a, hipStream_t stream) {
  GradGemm p = product(a.x, a.d, a.w1, a.d, a.h, a.H, a.M, a.H, a.d);
  p.saved = reinterpret_cast<uint16_t*>(a.gate_up);
  hipError_t e = launch<false, false, EPI_SWIGLU>(p, plan_of(a.M, (int)a.H * 2, a.d, false), stream);
  if (e != hipSuccess) return e;
  return launch<false, false, EPI_STORE>(product(a.h, a.H, a.w2, a.H, a.y, a.d, a.M, a.d, a.H), plan_of(a.M, (int)a.d, a.H, false), stream);
}

int64_t feed_forward_grad_workspace_bytes(const aeris_feed_forward_grad& a) {
  int64_t n = a.dx || a.dw1 ? up256(a.M * a.H * 4) : 0;
  int64_t part = a.dw1 ? weight_grad_bytes(a.M, 2 * a.H, a.d) : 0;
  const int64_t part2 = a.dw2 ? weight_grad_bytes(a.M, a.d, a.H) : 0;
  return n + (part > part2 ? part : part2);
}

hipError_t feed_forward_grad_launch(const aeris_feed_forward_grad& a, void* workspace, hipStream_t stream) {
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  void* dgu = ws;
  if (a.dx || a.dw1) ws += up256(a.M * a.H * 4);
  float* partial = reinterpret_cast<float*>(ws);
  hipError_t e = hipSuccess;
  if (a.dx || a.dw1) {
    GradGemm p = product(a.dy, a.d, a.w2, a.H, dgu, 2 * a.H, a.M, a.H, a.d);
    p.gate_up = reinterpret_cast<const uint16_t*>(a.gate_up);
    e = launch<false, true, EPI_SWIGLU_BWD>(p, plan_of(a.M, (int)a.H, a.d, false), stream);
  }
  if (e == hipSuccess && a.dw2) e = weight_grad(a.dy, a.h, a.dw2, a.M, a.d, a.H, partial, stream);
  if (e == hipSuccess && a.dx) e = input_grad(dgu, a.w1, a.dx, a.M, 2 * a.H, a.d, stream);
  if (e == hipSuccess && a.dw1) e = weight_grad(dgu, a.x, a.dw1, a.M, 2 * a.H, a.d, partial, stream);
  return e;
}

}  // namespace aeris
