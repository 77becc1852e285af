// Gradients of norm_modulate (LayerNorm / RMSNorm with the noise-level modulation) in one pass over the tokens.  With u what is
// normed, n = (u - mean) r, r = (var + eps)^-1/2 (RMS: no mean), v = n gamma + beta and dv the gradient of v:
//     dn = dv gamma,  du = r (dn - mean(dn) - n mean(dn n))   (RMS: without mean(dn))
//   norm then mod (y = v (1 + s) + t):  dv = dy (1 + s), dx = du;  A = sum dy n, B = sum dy over a member's tokens give
//     ds = gamma A + beta B,  dt = B,  dgamma = sum over members of (1 + s) A,  dbeta = sum over members of (1 + s) B
//   mod then norm (u = x (1 + s) + t):  dv = dy, dx = du (1 + s);  dgamma = sum dy n,  dbeta = sum dy,  ds = sum du x,  dt = sum du
// Nothing is kept from the forward pass: mean and r are recomputed from the row, which is read anyway.
//
// Bound by HBM: x and dy are read once, dx is written once.  A wave owns a row (rows of up to 256 or 128 elements lie beside each
// other in it, rows beyond 2048 and some of bf16 belong to two or four waves of a workgroup), holds it in registers and asks for its next one before it
// sums; the sums over the tokens stay in registers while a workgroup walks down its share of a member's rows.  At the end of it the
// workgroup writes one partial sum per column, and a second kernel adds those up in a fixed order: equal calls have equal results.
// All sums are fp32: within a lane over some hundred rows, then over lanes, waves and workgroups.
// f32 x [1036800, 1024], bf16 dy: 2155 us, 4.9 TB/s; an element-wise sum of the same streams takes 2035 us here.  Rows beyond 2048: f32 x [30000, 4096]
// 268 us, 4.6 TB/s, [30000, 6144] 377, 4.9, with the modulation ahead of the norm 265 and 497.  bf16 x with the modulation ahead of the norm is bound by
// vector arithmetic (four sums a column; u and dn are formed in each of three passes over the row): [259200, 1536] 625 us, 3.8 TB/s, VALU busy 95 % of the cycles,
// against 435 us, 71 %, with the modulation behind the norm.
#include "common.h"
#include "kernels.h"

namespace aeris {

namespace {

struct NormGradParams {
  const void* x;
  const void* dy;
  void* dx;
  const void* gamma;
  const void* beta;
  const float* shift;
  const float* scale;
  float* partial;  // [segments][blocks per segment][sums][d], or NULL: no sums
  int64_t mod_stride;  // between the segments' modulation rows
  int64_t rows;        // of a segment
  int blocks_per_segment;
  int d;
  int kind;
  int param_f32;
  float eps;
};

__device__ __forceinline__ float param_at(const void* p, int f32, int c) {
  return f32 ? reinterpret_cast<const float*>(p)[c] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[c]);
}

// NV: groups of 8 columns a lane; SUB: rows beside each other in a wave; WPR: waves to a row (1, 2 or 4).
// Workgroups that a CU holds, which the registers are budgeted for (sums, the row and the next one)
template <int NV, bool PRE>
constexpr int resident() { return PRE ? (NV == 1 ? 4 : NV == 2 ? 2 : 1) : (NV == 1 ? 5 : NV == 2 ? 3 : 2); }

template <int NV, int SUB, int WPR, bool X_F32, bool DY_F32, bool PRE>
__global__ void __launch_bounds__(256, (resident<NV, PRE>())) norm_grad_kernel(NormGradParams p) {
  static_assert(SUB == 1 || (NV == 1 && WPR == 1), "rows beside each other: one column group a lane");
  constexpr int LPR = 64 * WPR / SUB;          // lanes of a row
  constexpr int SLOTS = 256 / LPR;             // rows at a time
  constexpr int GROUPS = NV * LPR;
  constexpr int SUMS = PRE ? 4 : 2;
  constexpr int COLS = GROUPS * 8;
  // the parameters, first and second four of a group's columns apart (neighbouring lanes' 16-byte reads do not share banks); the
  // sums of the row slots go over them at the end.  (Four waves to a row: a lane's columns are its own for all rows, their parameters
  // stay in its registers.)
  constexpr bool IN_LDS = WPR == 1;
  constexpr int LDS_ROWS = IN_LDS ? (SLOTS > 3 ? SLOTS : 3) : SLOTS > 1 ? SLOTS : 0;
  __shared__ __attribute__((aligned(16))) float lds[LDS_ROWS ? LDS_ROWS * COLS : 4];
  __shared__ float cross[2][4][2];
  f32x4* const sG = reinterpret_cast<f32x4*>(lds);
  f32x4* const sP1 = sG + (IN_LDS ? 2 * GROUPS : 0);
  f32x4* const sP0 = sP1 + (IN_LDS ? 2 * GROUPS : 0);
  f32x4 rG[IN_LDS ? 1 : NV][2], rP1[IN_LDS ? 1 : NV][2], rP0[IN_LDS ? 1 : NV][2];
  const int lane = threadIdx.x & (LPR - 1), slot = threadIdx.x / LPR;
  const int d = p.d;
  const float inv_d = 1.0f / (float)d;
  const int seg = blockIdx.x / p.blocks_per_segment, blk = blockIdx.x - seg * p.blocks_per_segment;
  // (rows in turns over the workgroups: those at work together read and write neighbouring rows)
  const int64_t first = (int64_t)blk * SLOTS, end = p.rows, stride = (int64_t)p.blocks_per_segment * SLOTS;
  const int64_t row_base = (int64_t)seg * p.rows;
  const float* const sh = p.shift ? p.shift + seg * p.mod_stride : nullptr;
  const float* const sc = p.scale ? p.scale + seg * p.mod_stride : nullptr;

  // 8 columns as they lie in memory, widened where they are used
  struct Raw { u32x4 x[X_F32 ? 2 : 1], y[DY_F32 ? 2 : 1]; };
  auto load_row = [&](int64_t row, Raw (&raw)[NV]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * LPR + lane) * 8;
#pragma unroll
      for (int h = 0; h < (X_F32 ? 2 : 1); ++h) raw[v].x[h] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int h = 0; h < (DY_F32 ? 2 : 1); ++h) raw[v].y[h] = u32x4{0u, 0u, 0u, 0u};
      if (col < d) {
        const int64_t at = (row_base + row) * d + col;
        const u32x4* const qx = reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned char*>(p.x) + at * (X_F32 ? 4 : 2));
        const u32x4* const qy = reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned char*>(p.dy) + at * (DY_F32 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < (X_F32 ? 2 : 1); ++h) raw[v].x[h] = __builtin_nontemporal_load(qx + h);
#pragma unroll
        for (int h = 0; h < (DY_F32 ? 2 : 1); ++h) raw[v].y[h] = __builtin_nontemporal_load(qy + h);
      }
    }
  };
  auto x_of = [](const Raw& r, int e) {
    return X_F32 ? __uint_as_float(r.x[X_F32 ? e >> 2 : 0][e & 3]) : (e & 1) ? bf16_hi(r.x[0][e >> 1]) : bf16_lo(r.x[0][e >> 1]);
  };
  auto y_of = [](const Raw& r, int e) {
    return DY_F32 ? __uint_as_float(r.y[DY_F32 ? e >> 2 : 0][e & 3]) : (e & 1) ? bf16_hi(r.y[0][e >> 1]) : bf16_lo(r.y[0][e >> 1]);
  };

  Raw cur[NV], nxt[NV];
  int64_t row = first + slot;
  if (row < end) load_row(row, cur);

#pragma unroll
  for (int v = 0; v < (IN_LDS ? (GROUPS + 255) / 256 : NV); ++v) {
    const int g = IN_LDS ? v * 256 + threadIdx.x : v * LPR + lane;
    if (IN_LDS && GROUPS % 256 && g >= GROUPS) break;
    float G[8], P1[8], P0[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = g * 8 + e;
      const float ga = c < d ? param_at(p.gamma, p.param_f32, c) : 0.f;
      const float s1 = c < d && sc ? 1.f + sc[c] : 1.f;
      G[e] = PRE ? ga : ga * s1;
      P1[e] = s1;
      P0[e] = c < d && sh ? sh[c] : 0.f;
    }
    if (!IN_LDS) {
      rG[v][0] = f32x4{G[0], G[1], G[2], G[3]};
      rG[v][1] = f32x4{G[4], G[5], G[6], G[7]};
      rP1[v][0] = f32x4{P1[0], P1[1], P1[2], P1[3]};
      rP1[v][1] = f32x4{P1[4], P1[5], P1[6], P1[7]};
      rP0[v][0] = f32x4{P0[0], P0[1], P0[2], P0[3]};
      rP0[v][1] = f32x4{P0[4], P0[5], P0[6], P0[7]};
      continue;
    }
    sG[g] = f32x4{G[0], G[1], G[2], G[3]};
    sG[GROUPS + g] = f32x4{G[4], G[5], G[6], G[7]};
    if (PRE) {
      sP1[g] = f32x4{P1[0], P1[1], P1[2], P1[3]};
      sP1[GROUPS + g] = f32x4{P1[4], P1[5], P1[6], P1[7]};
      sP0[g] = f32x4{P0[0], P0[1], P0[2], P0[3]};
      sP0[GROUPS + g] = f32x4{P0[4], P0[5], P0[6], P0[7]};
    }
  }
  __syncthreads();

  int at_lane = lane;  // (made opaque in every turn: the parameters stay in LDS, or the compiler keeps them all in registers)
  auto gain = [&](int v, int h) { return IN_LDS ? sG[h * GROUPS + v * LPR + at_lane] : rG[IN_LDS ? 0 : v][h]; };
  auto one_plus_scale = [&](int v, int h) { return IN_LDS ? sP1[h * GROUPS + v * LPR + at_lane] : rP1[IN_LDS ? 0 : v][h]; };
  auto shift_of = [&](int v, int h) { return IN_LDS ? sP0[h * GROUPS + v * LPR + at_lane] : rP0[IN_LDS ? 0 : v][h]; };

  float acc[SUMS][NV][8];
#pragma unroll
  for (int s = 0; s < SUMS; ++s)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[s][v][e] = 0.f;

  int turn = 0;
  // two sums over a row, the same value in each of its lanes
  auto row_sums = [&](float& a, float& b) {
    if (WPR == 1) {
      a = lanes_sum<SUB>(a);
      b = lanes_sum<SUB>(b);
    } else {
      a = wave_sum(a);
      b = wave_sum(b);
      const int w = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
        cross[turn][w][0] = a;
        cross[turn][w][1] = b;
      }
      __syncthreads();
      const int w0 = slot * WPR;
      a = cross[turn][w0][0] + cross[turn][w0 + 1][0];
      b = cross[turn][w0][1] + cross[turn][w0 + 1][1];
      if (WPR == 4) {
        a += cross[turn][2][0] + cross[turn][3][0];
        b += cross[turn][2][1] + cross[turn][3][1];
      }
      turn ^= 1;  // the next pair goes elsewhere: a wave may be there before another has read this one
    }
  };

  // (rows beside each other in a wave, and rows of a workgroup, take the same number of turns: the lanes of a slot without a row
  // work on zeros, whose sums are zeros and which are not stored)
  const int64_t turns = end > first ? (end - first + stride - 1) / stride : 0;
  for (int64_t it = 0; it < turns; ++it, row += stride) {
    asm volatile("" : "+v"(at_lane));
    const bool live = row < end;
    if (row + stride < end) load_row(row + stride, nxt);
    if (!live) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int h = 0; h < (X_F32 ? 2 : 1); ++h) cur[v].x[h] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int h = 0; h < (DY_F32 ? 2 : 1); ++h) cur[v].y[h] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    // u, the value that is normed (columns beyond d: 0)
    auto u_row = [&](int v, float (&u)[8]) {
      if (PRE) {
        const bool act = (v * LPR + lane) * 8 < d;
        const f32x4 p1a = one_plus_scale(v, 0), p1b = one_plus_scale(v, 1), p0a = shift_of(v, 0), p0b = shift_of(v, 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = act ? fmaf(x_of(cur[v], e), e < 4 ? p1a[e] : p1b[e - 4], e < 4 ? p0a[e] : p0b[e - 4]) : 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = x_of(cur[v], e);
      }
    };
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float u[8];
      u_row(v, u);
      const f32x4 ga = gain(v, 0), gb = gain(v, 1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float dn = y_of(cur[v], e) * (e < 4 ? ga[e] : gb[e - 4]);
        if (p.kind == AERIS_NORM_RMS) {
          s1 = fmaf(u[e], u[e], s1);
          s2 = fmaf(dn, u[e], s2);
        } else {
          s1 += u[e];
          s2 += dn;
        }
      }
    }
    row_sums(s1, s2);
    float mean = 0.f, r, c1 = 0.f, c2;  // c1 = mean(dn), c2 = mean(dn n)
    if (p.kind == AERIS_NORM_RMS) {
      r = rsqrtf(s1 * inv_d + p.eps);
      c2 = s2 * inv_d * r;
    } else {
      mean = s1 * inv_d;
      c1 = s2 * inv_d;
      float q1 = 0.f, q2 = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float u[8];
        u_row(v, u);
        const bool act = (v * LPR + lane) * 8 < d;
        const f32x4 ga = gain(v, 0), gb = gain(v, 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = act ? u[e] - mean : 0.f;
          q1 = fmaf(c, c, q1);
          q2 = fmaf(y_of(cur[v], e) * (e < 4 ? ga[e] : gb[e - 4]), c, q2);
        }
      }
      row_sums(q1, q2);
      r = rsqrtf(q1 * inv_d + p.eps);
      c2 = q2 * inv_d * r;
    }
    if (!live) r = c2 = 0.f;  // (eps 0: a row of zeros would have an infinite r)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * LPR + lane) * 8;
      float u[8];
      u_row(v, u);
      const f32x4 ga = gain(v, 0), gb = gain(v, 1);
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n = col < d ? (u[e] - mean) * r : 0.f, y = y_of(cur[v], e);
        float du = (fmaf(y, e < 4 ? ga[e] : gb[e - 4], -c1) - n * c2) * r;
        acc[0][v][e] = fmaf(y, n, acc[0][v][e]);
        acc[1][v][e] += y;
        if (PRE) {
          acc[2][v][e] = fmaf(du, x_of(cur[v], e), acc[2][v][e]);
          acc[3][v][e] += du;
          du *= one_plus_scale(v, e >> 2)[e & 3];
        }
        o[e] = du;
      }
      if (p.dx && live && col < d) {
        const int64_t at = (row_base + row) * d + col;
        if (X_F32) {
          f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.dx) + at);
          __builtin_nontemporal_store(f32x4{o[0], o[1], o[2], o[3]}, q);
          __builtin_nontemporal_store(f32x4{o[4], o[5], o[6], o[7]}, q + 1);
        } else {
          const u32x4 w = {pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])};
          __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p.dx) + at));
        }
      }
      cur[v] = nxt[v];
    }
  }
  if (!p.partial) return;

  // the row slots' sums, one quantity after the other through LDS
  float* const out = p.partial + ((int64_t)seg * p.blocks_per_segment + blk) * SUMS * d;
#pragma unroll
  for (int s = 0; s < SUMS; ++s) {
    if (SLOTS == 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = (v * LPR + lane) * 8;
        if (col < d) {
          *reinterpret_cast<f32x4*>(out + (int64_t)s * d + col) = f32x4{acc[s][v][0], acc[s][v][1], acc[s][v][2], acc[s][v][3]};
          *reinterpret_cast<f32x4*>(out + (int64_t)s * d + col + 4) = f32x4{acc[s][v][4], acc[s][v][5], acc[s][v][6], acc[s][v][7]};
        }
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        f32x4* q = reinterpret_cast<f32x4*>(lds + slot * COLS);
        const int g = v * LPR + lane;
        q[g] = f32x4{acc[s][v][0], acc[s][v][1], acc[s][v][2], acc[s][v][3]};
        q[GROUPS + g] = f32x4{acc[s][v][4], acc[s][v][5], acc[s][v][6], acc[s][v][7]};
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * GROUPS; i += 256) {
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) t += reinterpret_cast<const f32x4*>(lds + k * COLS)[i];
        const int col = (i % GROUPS) * 8 + (i / GROUPS) * 4;
        if (col < d) *reinterpret_cast<f32x4*>(out + (int64_t)s * d + col) = t;
      }
    }
  }
}

struct NormGradSums {
  const float* partial;  // [segments][blocks][sums][d]
  float* members;        // [segments][2][d]: every segment's share of dgamma and dbeta, added up by another kernel; or NULL: by this one
  const void* gamma;
  const void* beta;
  const float* scale;
  void* dgamma;
  void* dbeta;
  float* dshift;
  float* dscale;
  int64_t mod_stride;
  int segments, blocks, d, param_f32;
};

__device__ __forceinline__ void store_param_grads(const NormGradSums& p, int col, float dgamma, float dbeta) {
  if (p.param_f32) {
    if (p.dgamma) reinterpret_cast<float*>(p.dgamma)[col] = dgamma;
    if (p.dbeta) reinterpret_cast<float*>(p.dbeta)[col] = dbeta;
  } else {
    if (p.dgamma) reinterpret_cast<uint16_t*>(p.dgamma)[col] = (uint16_t)f32_to_bf16_bits(dgamma);
    if (p.dbeta) reinterpret_cast<uint16_t*>(p.dbeta)[col] = (uint16_t)f32_to_bf16_bits(dbeta);
  }
}

// 8 columns a workgroup (d is a multiple of 8); 128 threads share a column's sums over `rows` rows, q(row, sum) the address of one.
// The results are thread 0 .. 7's, whose columns they are.
template <int SUMS, class At>
__device__ __forceinline__ void column_sums(int rows, const At& q, float (*lds)[4][8], float (&t)[SUMS]) {
  const int c = threadIdx.x & 7, r = threadIdx.x >> 3;
#pragma unroll
  for (int s = 0; s < SUMS; ++s) t[s] = 0.f;
#pragma unroll 4
  for (int b = r; b < rows; b += 128)
#pragma unroll
    for (int s = 0; s < SUMS; ++s) t[s] += *q(b, s);
#pragma unroll
  for (int s = 0; s < SUMS; ++s) {  // over the 8 rows of the wave
    t[s] += __shfl_xor(t[s], 8);
    t[s] += __shfl_xor(t[s], 16);
    t[s] += __shfl_xor(t[s], 32);
  }
  __syncthreads();
  if ((threadIdx.x & 63) < 8) {
#pragma unroll
    for (int s = 0; s < SUMS; ++s) lds[threadIdx.x >> 6][s][c] = t[s];
  }
  __syncthreads();
  if (threadIdx.x < 8) {
#pragma unroll
    for (int s = 0; s < SUMS; ++s) {
      t[s] = 0.f;
#pragma unroll
      for (int w = 0; w < 16; ++w) t[s] += lds[w][s][c];
    }
  }
}

template <bool PRE>
__global__ void __launch_bounds__(1024) norm_grad_sums_kernel(NormGradSums p) {
  constexpr int SUMS = PRE ? 4 : 2;
  __shared__ float lds[16][4][8];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7);
  const float ga = param_at(p.gamma, p.param_f32, col);
  const float be = p.beta ? param_at(p.beta, p.param_f32, col) : 0.f;
  float dgamma = 0.f, dbeta = 0.f;
  const int first = p.members ? blockIdx.y : 0, last = p.members ? blockIdx.y + 1 : p.segments;
  for (int seg = first; seg < last; ++seg) {
    float t[SUMS];
    const float* const base = p.partial + (int64_t)seg * p.blocks * SUMS * p.d + col;
    column_sums<SUMS>(p.blocks, [&](int b, int s) { return base + ((int64_t)b * SUMS + s) * p.d; }, lds, t);
    if (threadIdx.x < 8) {
      float A = t[0], B = t[1], ds, dt;
      if (PRE) {
        ds = t[SUMS - 2];
        dt = t[SUMS - 1];
      } else {
        const float one = p.scale ? 1.f + p.scale[seg * p.mod_stride + col] : 1.f;
        ds = fmaf(ga, A, be * B);
        dt = B;
        A *= one;
        B *= one;
      }
      if (p.dscale) p.dscale[(int64_t)seg * p.d + col] = ds;
      if (p.dshift) p.dshift[(int64_t)seg * p.d + col] = dt;
      dgamma += A;
      dbeta += B;
    }
  }
  if (threadIdx.x < 8) {
    if (p.members) {
      p.members[((int64_t)blockIdx.y * 2) * p.d + col] = dgamma;
      p.members[((int64_t)blockIdx.y * 2 + 1) * p.d + col] = dbeta;
    } else {
      store_param_grads(p, col, dgamma, dbeta);
    }
  }
}

__global__ void __launch_bounds__(1024) norm_grad_members_kernel(NormGradSums p) {
  __shared__ float lds[16][4][8];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7);
  float t[2];
  column_sums<2>(p.segments, [&](int b, int s) { return p.members + ((int64_t)b * 2 + s) * p.d + col; }, lds, t);
  if (threadIdx.x < 8) store_param_grads(p, col, t[0], t[1]);
}

bool wants_sums(const aeris_norm_modulate_grad& a) { return a.dgamma || a.dbeta || a.dshift || a.dscale; }
bool is_pre(const aeris_norm_modulate_grad& a) { return a.order == AERIS_MOD_THEN_NORM && (a.shift || a.scale); }
int64_t segments_of(const aeris_norm_modulate_grad& a) { return (a.shift || a.scale) && a.mod_batch_stride && a.B > 1 ? a.B : 1; }

// How a call is run: column groups of a lane, rows at a time, whether a row belongs to several waves.  One wave to a row of up to 2048
// elements is the faster way (f32 x [259200, 1536] 803 against 834 us, [1036800, 1024] 2155 against 2216), but for many rows of bf16 x whose
// modulation lies ahead of the norm: four sums a column leave one wave a SIMD, whose arithmetic and memory nothing overlaps (bf16 [259200, 1536]
// 830 -> 624 us with four waves to a row, of 3.2 waves a SIMD, [1036800, 1024] 1381 -> 1330 with two, [20000, 2048] 100 -> 92; [8192, 1536] 44 -> 54).
struct Shape { int nv, slots, waves; };
Shape shape_of(const aeris_norm_modulate_grad& a) {
  if (a.d <= 512) return {1, a.d <= 128 ? 16 : a.d <= 256 ? 8 : 4, 1};
  if (a.d > 2048) return {a.d <= 4096 ? 2 : 3, 1, 4};
  if (is_pre(a) && a.x_dtype == AERIS_BF16 && a.B * a.rows_per_batch * a.d >= 30000000) return a.d <= 1024 ? Shape{1, 2, 2} : Shape{1, 1, 4};
  return {a.d <= 1024 ? 2 : a.d <= 1536 ? 3 : 4, 4, 1};
}

// Workgroups of a segment: at most one round of what the chip holds of them, and at least 32 rows each, so that the parameters' and the
// partial sums' traffic stays small beside the rows'.
int64_t blocks_of(const aeris_norm_modulate_grad& a) {
  const int64_t segments = segments_of(a), rows = a.B * a.rows_per_batch / segments;
  const Shape s = shape_of(a);
  const bool pre = is_pre(a);
  const int held = s.nv == 1 ? pre ? resident<1, true>() : resident<1, false>() : s.nv == 2 ? pre ? resident<2, true>() : resident<2, false>()
                   : s.nv == 3 ? pre ? resident<3, true>() : resident<3, false>() : pre ? resident<4, true>() : resident<4, false>();
  const int64_t least = s.slots > 8 ? 2 * s.slots : 32, n = (rows + least - 1) / least, most = 256 * held / segments;
  return n < most ? n : most > 0 ? most : 1;
}

template <int NV, int SUB, int WPR>
hipError_t launch(const NormGradParams& p, bool xf, bool yf, bool pre, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), block(256);
#define GO(XF, YF, PR) hipLaunchKernelGGL((norm_grad_kernel<NV, SUB, WPR, XF, YF, PR>), grid, block, 0, stream, p)
  if (pre) {
    if (xf) { if (yf) GO(true, true, true); else GO(true, false, true); }
    else { if (yf) GO(false, true, true); else GO(false, false, true); }
  } else {
    if (xf) { if (yf) GO(true, true, false); else GO(true, false, false); }
    else { if (yf) GO(false, true, false); else GO(false, false, false); }
  }
#undef GO
  return hipGetLastError();
}

template <int WPR>  // (bf16 x, the modulation ahead of the norm: see shape_of)
hipError_t launch_wide(const NormGradParams& p, bool yf, int64_t blocks, hipStream_t stream) {
  if (yf) hipLaunchKernelGGL((norm_grad_kernel<1, 1, WPR, false, true, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((norm_grad_kernel<1, 1, WPR, false, false, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

static int64_t norm_grad_blocks(const aeris_norm_modulate_grad& a) { return segments_of(a) * blocks_of(a); }

// many members: their sums side by side, and another kernel for what adds up over them
static bool members_apart(const aeris_norm_modulate_grad& a) { return segments_of(a) > 8; }

int64_t norm_grad_workspace_bytes(const aeris_norm_modulate_grad& a) {
  return wants_sums(a) ? (norm_grad_blocks(a) * (is_pre(a) ? 4 : 2) + (members_apart(a) ? 2 * segments_of(a) : 0)) * a.d * 4 : 0;
}

hipError_t norm_grad_launch(const aeris_norm_modulate_grad& a, void* workspace, hipStream_t stream) {
  const bool pre = is_pre(a), xf = a.x_dtype == AERIS_F32, yf = a.dy_dtype == AERIS_F32;
  const int64_t segments = segments_of(a);
  NormGradParams p;
  p.x = a.x; p.dy = a.dy; p.dx = a.dx;
  p.gamma = a.gamma; p.beta = a.beta;
  p.shift = a.shift; p.scale = a.scale;
  p.partial = wants_sums(a) ? reinterpret_cast<float*>(workspace) : nullptr;
  p.mod_stride = segments > 1 ? a.mod_batch_stride : 0;
  p.rows = a.B * a.rows_per_batch / segments;
  p.blocks_per_segment = (int)blocks_of(a);
  p.d = (int)a.d;
  p.kind = (int)a.kind;
  p.param_f32 = a.param_dtype == AERIS_F32;
  p.eps = (float)a.eps;
  const int64_t blocks = segments * p.blocks_per_segment;
  const Shape f = shape_of(a);
  hipError_t e;
  if (a.d <= 128) e = launch<1, 4, 1>(p, xf, yf, pre, blocks, stream);
  else if (a.d <= 256) e = launch<1, 2, 1>(p, xf, yf, pre, blocks, stream);
  else if (a.d <= 512) e = launch<1, 1, 1>(p, xf, yf, pre, blocks, stream);
  else if (f.waves == 2) e = launch_wide<2>(p, yf, blocks, stream);
  else if (f.waves == 4 && f.nv == 1) e = launch_wide<4>(p, yf, blocks, stream);
  else if (f.waves == 4 && f.nv == 2) e = launch<2, 1, 4>(p, xf, yf, pre, blocks, stream);
  else if (f.waves == 4) e = launch<3, 1, 4>(p, xf, yf, pre, blocks, stream);
  else if (f.nv == 2) e = launch<2, 1, 1>(p, xf, yf, pre, blocks, stream);
  else if (f.nv == 3) e = launch<3, 1, 1>(p, xf, yf, pre, blocks, stream);
  else e = launch<4, 1, 1>(p, xf, yf, pre, blocks, stream);
  if (e != hipSuccess || !p.partial) return e;
  NormGradSums s;
  s.partial = p.partial;
  s.gamma = a.gamma; s.beta = a.beta; s.scale = a.scale;
  s.dgamma = a.dgamma; s.dbeta = a.dbeta; s.dshift = a.dshift; s.dscale = a.dscale;
  s.mod_stride = p.mod_stride;
  s.segments = (int)segments;
  s.blocks = p.blocks_per_segment;
  s.d = p.d;
  s.param_f32 = p.param_f32;
  s.members = members_apart(a) ? p.partial + blocks * (pre ? 4 : 2) * p.d : nullptr;
  const dim3 grid((unsigned)(p.d / 8), s.members ? (unsigned)segments : 1u);
  if (pre) hipLaunchKernelGGL(norm_grad_sums_kernel<true>, grid, dim3(1024), 0, stream, s);
  else hipLaunchKernelGGL(norm_grad_sums_kernel<false>, grid, dim3(1024), 0, stream, s);
  e = hipGetLastError();
  if (e != hipSuccess || !s.members || !(a.dgamma || a.dbeta)) return e;
  hipLaunchKernelGGL(norm_grad_members_kernel, dim3((unsigned)(p.d / 8)), dim3(1024), 0, stream, s);
  return hipGetLastError();
}

}  // namespace aeris
