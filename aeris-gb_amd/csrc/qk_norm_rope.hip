// RMS norm of every query and key head and the position rotation in one pass over q and k, between the to_qkv projection and
// the attention:
//   n = x * rsqrt(mean(x^2) + eps) * gain          per (token, head), fp32
//   (n_a, n_b) -> (n_a cos - n_b sin, n_a sin + n_b cos)    for the pairs (a, b) of the first R elements, angles by the token's position
//   y = n * scale                                  (q: scale * log2 e, so that q is rounded to its type once, here)
// Bound by HBM: every element is read once and written once.  D / 8 lanes hold a head's row, 16 bytes of bf16 each; a thread does four heads
// of one token (one, where there are few tokens: latency), so that the token's row of the rotation table is read once for them and their loads are in
// flight together (two: 5.3 TB/s, one 4.2, eight 5.4, all sixteen heads in rounds of four with the next round's loads ahead 5.1; four 5.6).  Head
// planes: a group of heads walks through all tokens, stores that leave no line behind in the caches (1573 -> 1512 us).  Rows of heads side by
// side: the groups of a block of tokens are neighbours, so that the parts of a row are fetched together (1811 -> 1477 us), ordinary stores
// (1573 with the others).
// 720 x 1440 tokens, 16 + 16 heads of 64: planes 1512 us, rows 1477 us, 5.6 - 5.75 TB/s (an element-wise multiplication of this size: 6.26 TB/s).
#include "common.h"
#include "kernels.h"

namespace aeris {

namespace {

struct QkParams {
  aeris_qk_part part[2];
  int groups0, groups;  // groups of heads: of the first part; of both
  int blocks;           // of tokens
  int heads_first;      // the groups of a block of tokens are neighbouring workgroups (else: the blocks of a group)
  int T, n_pos, P, R, normed, interleaved, gain_f32;
  float eps;
  const float* rotation;
  const int32_t* positions;
};

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {  // over the LPR neighbouring lanes of a row, the same value in each
  v = dpp_add<0xB1, 0xF>(v);                  // quad_perm [1,0,3,2]
  v = dpp_add<0x4E, 0xF>(v);                  // quad_perm [2,3,0,1]
  if (LPR >= 8) v = dpp_add<0x141, 0xF>(v);   // row_half_mirror
  if (LPR >= 16) v = dpp_add<0x140, 0xF>(v);  // row_mirror
  return v;
}

template <int D, bool XF32, bool YF32, int HPT, bool STREAM>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkParams p) {
  constexpr int LPR = D / 8, TPB = 256 / LPR;
  const int c = threadIdx.x % LPR;
  const int group = p.heads_first ? blockIdx.x % p.groups : blockIdx.x / p.blocks;
  const int t = (int)(p.heads_first ? blockIdx.x / p.groups : blockIdx.x % p.blocks) * TPB + threadIdx.x / LPR;
  const bool ok = t < p.T;
  const int64_t tt = ok ? t : p.T - 1;
  const bool second = group >= p.groups0;
  const aeris_qk_part& part = p.part[second ? 1 : 0];
  const int h0 = (group - (second ? p.groups0 : 0)) * HPT;
  const int heads = (int)part.heads;
  const float mul = (float)part.scale;
  const int64_t xt = part.x_stride[0], xh = part.x_stride[1], yt = part.y_stride[0], yh = part.y_stride[1];  // (of one token, one head: times 0)

  u32x4 raw[HPT][XF32 ? 2 : 1];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int64_t h = h0 + i < heads ? h0 + i : heads - 1;
    if constexpr (XF32) {
      const float* x = reinterpret_cast<const float*>(part.x) + tt * xt + h * xh + c * 8;
      raw[i][0] = *reinterpret_cast<const u32x4*>(x);
      raw[i][1] = *reinterpret_cast<const u32x4*>(x + 4);
    } else {
      raw[i][0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(part.x) + tt * xt + h * xh + c * 8);
    }
  }

  // cos and sin of the lane's elements (those of an element's pair)
  const int R = p.R, half = R / 2;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  bool turns = c * 8 < R;  // whether the lane's elements are rotated: not behind the first R, not at a position outside the table
  const bool upper = !p.interleaved && c * 8 >= half;  // the lane holds the second elements of its pairs
  if (turns) {
    const uint32_t at = (uint32_t)tt % (uint32_t)p.n_pos;
    const int pos = p.positions ? p.positions[at] : (int)at;
    turns = (uint32_t)pos < (uint32_t)p.P;
    if (turns) {
      const float* row = p.rotation + (int64_t)pos * R;
      if (p.interleaved) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(row + c * 4), b = *reinterpret_cast<const f32x4*>(row + half + c * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          cs[e] = a[e / 2];
          sn[e] = b[e / 2];
        }
      } else {
        const float* r = row + (upper ? c * 8 - half : c * 8);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(r + 4 * q), b = *reinterpret_cast<const f32x4*>(r + half + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            cs[4 * q + e] = a[e];
            sn[4 * q + e] = b[e];
          }
        }
      }
    }
  }
  const int lane = threadIdx.x & 63;
  const int partner = p.interleaved || !turns ? lane : upper ? lane - half / 8 : lane + half / 8;
  const float sign = upper ? 1.f : -1.f;  // y_a = a cos - b sin, y_b = b cos + a sin

  float g[8];
  auto load_gain = [&](int64_t h) {
    const int64_t at = h * part.gain_head_stride + c * 8;
    if (p.gain_f32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(part.gain) + at);
      const f32x4 b = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(part.gain) + at + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = a[e];
        g[4 + e] = b[e];
      }
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(part.gain) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[2 * e] = bf16_lo(a[e]);
        g[2 * e + 1] = bf16_hi(a[e]);
      }
    }
  };
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = 1.f;
  const bool own_gain = part.gain && part.gain_head_stride;
  if (part.gain && !own_gain) load_gain(0);

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    if (h0 + i >= heads) break;  // (the same for the whole block)
    const int64_t h = h0 + i;
    if (own_gain) load_gain(h);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (XF32) {
        v[e] = __uint_as_float(raw[i][0][e]);
        v[4 + e] = __uint_as_float(raw[i][XF32 ? 1 : 0][e]);
      } else {
        v[2 * e] = bf16_lo(raw[i][0][e]);
        v[2 * e + 1] = bf16_hi(raw[i][0][e]);
      }
    }
    float f = 1.f;
    if (p.normed) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
      f = rsqrtf(row_sum<LPR>(s) * (1.0f / D) + p.eps);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= f * g[e];
    float y[8];
    if (R == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[e];
    } else if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        // (no product with the sine where there is no rotation: the other value may be infinite)
        y[e] = turns ? v[e] * cs[e] - v[e + 1] * sn[e] : v[e];
        y[e + 1] = turns ? v[e] * sn[e] + v[e + 1] * cs[e] : v[e + 1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = __shfl(v[e], partner, 64);
        y[e] = turns ? fmaf(sign * o, sn[e], v[e] * cs[e]) : v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= mul;
    if (!ok) continue;
    if constexpr (YF32) {
      float* o = reinterpret_cast<float*>(part.y) + tt * yt + h * yh + c * 8;
      *reinterpret_cast<f32x4*>(o) = f32x4{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{y[4], y[5], y[6], y[7]};
    } else {
      u32x4* o = reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(part.y) + tt * yt + h * yh + c * 8);
      const u32x4 w = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
      if (STREAM) __builtin_nontemporal_store(w, o);
      else *o = w;
    }
  }
}

// one head a thread up to 1600 workgroups of that kind: 4096 tokens, 4 + 4 heads of 64 4.2 us, with four 4.8; 8192 6.2, 5.7; 2048 tokens, 3 + 3 of
// 128 3.8, 4.4; 4096 5.3, 5.0
int heads_per_thread(const aeris_qk_norm_rope& a) {
  const int64_t heads = a.parts[0].heads + (a.n_parts > 1 ? a.parts[1].heads : 0);
  return a.tokens * a.head_dim / 2048 * heads >= 1600 ? 4 : 1;
}

template <int D, bool XF32, bool YF32, int HPT>
hipError_t launch(const QkParams& p0, hipStream_t stream) {
  QkParams p = p0;
  constexpr int TPB = 256 / (D / 8);
  p.groups0 = (int)((p.part[0].heads + HPT - 1) / HPT);
  p.groups = p.groups0 + (int)((p.part[1].heads + HPT - 1) / HPT);
  p.blocks = (p.T + TPB - 1) / TPB;
  p.heads_first = p.part[0].x_stride[1] < p.part[0].x_stride[0];
  const dim3 grid((unsigned)((int64_t)p.blocks * p.groups));
  if (HPT == 1 || YF32 || p.heads_first) hipLaunchKernelGGL((qk_norm_rope_kernel<D, XF32, YF32, HPT, false>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<D, XF32, YF32, HPT, (HPT > 1 && !YF32)>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D, int HPT>
hipError_t launch_types(const QkParams& p, bool x_f32, bool y_f32, hipStream_t stream) {
  if (x_f32) return y_f32 ? launch<D, true, true, HPT>(p, stream) : launch<D, true, false, HPT>(p, stream);
  return y_f32 ? launch<D, false, true, HPT>(p, stream) : launch<D, false, false, HPT>(p, stream);
}

}  // namespace

bool qk_norm_rope_supported(int64_t head_dim, int64_t rotated) {
  return (head_dim == 32 || head_dim == 64 || head_dim == 128) && rotated >= 0 && rotated <= head_dim && rotated % 16 == 0;
}

int64_t qk_norm_rope_workgroups(const aeris_qk_norm_rope& a) {
  const int64_t each = heads_per_thread(a), tokens = 2048 / a.head_dim;
  int64_t groups = 0;
  for (int i = 0; i < (int)a.n_parts; ++i) groups += (a.parts[i].heads + each - 1) / each;
  return (a.tokens + tokens - 1) / tokens * groups;
}

hipError_t qk_norm_rope_launch(const aeris_qk_norm_rope& a, hipStream_t stream) {
  QkParams p{};
  p.part[0] = a.parts[0];
  if (a.n_parts > 1) p.part[1] = a.parts[1];
  p.T = (int)a.tokens; p.P = (int)a.P; p.R = (int)a.R; p.normed = a.normed != 0; p.interleaved = a.interleaved != 0;
  p.gain_f32 = a.gain_dtype == AERIS_F32; p.eps = (float)a.eps;
  p.rotation = a.rotation; p.positions = a.R > 0 ? a.positions : nullptr;
  p.n_pos = p.positions ? (int)a.n_positions : a.P > 0 ? (int)a.P : 1;
  const bool xf = a.x_dtype == AERIS_F32, yf = a.y_dtype == AERIS_F32;
  const bool many = heads_per_thread(a) == 4;
  if (a.head_dim == 32) return many ? launch_types<32, 4>(p, xf, yf, stream) : launch_types<32, 1>(p, xf, yf, stream);
  if (a.head_dim == 64) return many ? launch_types<64, 4>(p, xf, yf, stream) : launch_types<64, 1>(p, xf, yf, stream);
  return many ? launch_types<128, 4>(p, xf, yf, stream) : launch_types<128, 1>(p, xf, yf, stream);
}

}  // namespace aeris
