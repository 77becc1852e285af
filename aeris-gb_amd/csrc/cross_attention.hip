// Attention of tokens to an encoder's states: o = softmax(scale q k^T) v over the keys that a member has (its own, up to its length and
// where its key mask lets them, behind a prefix that all members share), gfx950.
//
// A unit is one member's key head (or, where all members see the same keys, the key head with the rows of all of them); its rows are
// the queries of the heads that share the key head, 16 QN a wave.  Keys go through LDS in chunks of 64; P = exp2(logit) is formed
// without a row maximum - softmax does not depend on the subtracted constant, the maximum only guards the range -, the range of the sums is
// checked afterwards and the rows are done again with a running maximum where it was left: 2^-20 to 2^60 for the weights' (values of v from 2^-106 on do
// not vanish in theirs), up to 2^100 for the results'.  The maximum is then taken so much higher that all weights together are below 1: finite values
// of any size have finite sums.
//   K, V chunk [64][HD]  global -> LDS by the load unit (buffer_load ... lds), 16-byte pieces XOR-swizzled; a key that does not take
//                        part is not read, its row arrives as zeros (whatever it held, NaN or infinity, is multiplied by nothing)
//   S^T = K Q^T          v_mfma_f32_16x16x32_bf16; lane = one row, registers = keys; the scale, unless the producer of q has applied it (`SCALED`),
//                        multiplies the fp32 logits: q is not rounded again
//   O^T += V^T P^T       V^T by the transposing LDS read, P^T straight from the accumulators of S^T, rounded to bf16 (v's type, the matrix cores'; for
//                        16 rows as two bf16, see step()); the row sum adds the rounded values.  As two bf16 the results would be off by 0.0017 in
//                        the mean square, their own rounding, instead of 0.0023; the second product costs a quarter to a half of the time: 1 036 800
//                        queries, sixteen heads of 64, 256 keys 1181 -> 1726 us, two members of 64 800, eight heads, 1000 keys 260 -> 369, heads of
//                        128 252 -> 349, sixteen of 32, 200 keys 52 -> 76, eight members' nine queries behind a prefix of 64 800 54 -> 68
// Three ways to run that, and parts:
//   cross_attention_rows_kernel      many rows: a workgroup = a block of a unit's rows, the unit's keys streamed past its waves
//   cross_attention_keys_kernel      few rows: the waves of a workgroup divide the keys among them for the same rows
//   cross_attention_resident_kernel  few keys and many rows: a workgroup keeps the unit's keys in LDS and walks down the rows
//   PARTS of the first two           fewer rows still: the keys divided among workgroups too, each leaves its sums in the workspace in fp32 and
//                                    cross_attention_join_kernel adds them up, in their order
// plan_of() chooses, by what each would cost (its comments: what they measured).  1000 queries x 1000 keys, eight heads of 64: rows kernel 16.2 us, keys
// kernel 8.4; 4000 x 77: 5.6 and 8.0.
#include "common.h"
#include "kernels.h"
#include <cstring>
#include <type_traits>

namespace aeris {

namespace {

constexpr int KC = 64;  // keys per chunk

// What a launch does: rows of units against keys
struct Task {
  int Nk, Np;        // own and prefix keys at most (0: that part is not its task)
  int members;       // units' members: 1 where a unit holds the rows of all of them
  int rows;          // of a unit
  int qblks, splits; // workgroups of a unit: row blocks, parts of the keys
  int units;         // splits * members * key heads
  int together;      // key heads that an XCD takes at a time: one or all
  int by_rows;       // workgroups of an XCD: all units in turn, an eighth of the row blocks (else: an eighth of the units)
  int first;         // its first workgroup
  float *o, *ml;     // PARTS: [split][member][key head][row][HD], [..][2] = maximum, sum
};

// Division of n < 2^31 by a number that a launch knows: a product's upper half and a shift
struct Divisor {
  uint32_t by, factor, shift;
  __device__ __forceinline__ int of(int n) const { return by == 1 ? n : (int)(__umulhi((uint32_t)n, factor) >> shift); }
};
// (with 2^l >= by > 2^(l - 1), factor = floor(2^(31 + l) / by) + 1 is off by less than a part of 2^31)
Divisor divisor(uint32_t by) {
  uint32_t l = 1;
  while (l < 31 && (1u << l) < by) ++l;
  return {by, by == 1 ? 0 : (uint32_t)((1ull << (31 + l)) / by + 1), l - 1};
}

struct CrossParams {
  const uint16_t *q, *k, *v, *prefix_k, *prefix_v;
  uint16_t* out;
  int64_t q_batch, q_row, q_head, k_batch, k_head, v_batch, v_head, prefix_k_head, prefix_v_head, mask_batch;
  uint32_t k_row, v_row, prefix_k_row, prefix_v_row;  // bytes
  const int32_t* lengths;
  const uint8_t* mask;
  int lengths_step;  // 0: one length for all members
  int Nq, heads, kv_heads, group;
  int rows_m;        // rows of a member
  Divisor of_group, of_rows_m;
  float q_mul;
  Task task[2];
};

// 16-byte pieces of a chunk's rows.  K: the fragment reads take one piece of 16 consecutive rows; V: the 32 lanes of a pass of the transposing
// read gather two neighbouring pieces of 8 rows.  In both the 16 pieces lie on the 16 slots of a 256-byte bank period.
template <int HD>
__device__ __forceinline__ int k_swizzle(int row) { return HD == 128 ? row & 15 : HD == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }
template <int HD>
__device__ __forceinline__ int v_swizzle(int row) { return HD == 128 ? 2 * (row & 7) : HD == 64 ? 2 * ((row >> 1) & 3) : 2 * ((row >> 2) & 1); }

// The first `n` of 64 keys, n >= 0
__device__ __forceinline__ uint64_t first_keys(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// Two bf16, zeros in the place of infinities and NaN
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
  return x;
}

// A wave's 16 QN rows: queries, sums, and what a chunk in LDS does to them.
// SUM: the row sums by the matrix cores too (a product with ones), four VALU operations fewer per 8 weights and one MFMA more per 4 to 8.
template <int HD, int QN, bool SCALED, bool SUM>
struct Rows {
  static constexpr int KS = HD / 32;  // k32 steps of K Q^T
  static constexpr int KB = KC / 16;  // blocks of 16 keys per chunk
  static constexpr int DB = HD / 16;  // 16-row blocks of O^T
  typedef __attribute__((address_space(3))) const unsigned char* lds_cptr;

  bf16x8 qf[QN][KS];  // B operand: lane = row, 8 consecutive elements per k32 step
  float m[QN], l[QN];
  f32x4 lv[QN];     // SUM: the row sum so far, in each of the four
  f32x4 o[QN][DB];  // o[n][db][i] = O[row 16 n + l15][16 db + 4 q4 + i]
  lds_cptr k_lane[KS];
  uint32_t v_tr[DB];
  int q4;
  float q_mul;

  // `smem`: the first chunk of K, `v_base` bytes behind it the first of V
  __device__ __forceinline__ Rows(unsigned char* smem, uint32_t v_base, int lane, float mul) : q4(lane >> 4), q_mul(mul) {
    const int l15 = lane & 15;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      k_lane[s] = (lds_cptr)(smem + l15 * (HD * 2) + (((4 * s + q4) ^ k_swizzle<HD>(l15)) << 4));
      asm volatile("" : "+v"(k_lane[s]));
    }
    // of the 16 lanes q4, lane 4e + a reads V[key0 + 4 q4 + e][16 db + 4a ..]
    const int e = (lane >> 2) & 3, a = lane & 3, row = 4 * q4 + e;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      v_tr[db] = lds_byte_address(smem) + v_base + (uint32_t)(row * (HD * 2) + (((2 * db + (a >> 1)) ^ v_swizzle<HD>(row)) << 4) + (a & 1) * 8);
      asm volatile("" : "+v"(v_tr[db]));
    }
  }

  // the lane's rows, row0 + 16 n + lane % 16 (the last one for those behind it), of a unit: member, query and head
  __device__ __forceinline__ void row_of(const CrossParams& p, const Task& t, int hk, int row0, int n, int lane, int64_t& member, int& query, int& head) const {
    int r = row0 + n * 16 + (lane & 15);
    r = r < t.rows ? r : t.rows - 1;
    const int b = p.of_rows_m.of(r), rm = r - b * p.rows_m;
    query = p.of_group.of(rm);
    head = hk * p.group + rm - query * p.group;
    member += b;
  }
  // Whether they are neighbouring queries of one head, all there (uniform): what is then left to the lanes does not depend on the block
  __device__ __forceinline__ bool plain(const CrossParams& p, const Task& t, int row0) const {
    return p.group == 1 && t.rows == p.rows_m && row0 + 16 * QN <= t.rows;
  }
  __device__ __forceinline__ void load_q(const CrossParams& p, const Task& t, int member, int hk, int row0, int lane, bf16x8 (&f)[QN][KS]) const {
    if (plain(p, t, row0)) {
      const uint16_t* first = p.q + member * p.q_batch + row0 * p.q_row + hk * p.q_head;
      const int64_t mine = (lane & 15) * p.q_row + q4 * 8;
#pragma unroll
      for (int n = 0; n < QN; ++n)
#pragma unroll
        for (int s = 0; s < KS; ++s) f[n][s] = *reinterpret_cast<const bf16x8*>(first + n * 16 * p.q_row + mine + s * 32);
      return;
    }
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      int64_t b = member;
      int query, head;
      row_of(p, t, hk, row0, n, lane, b, query, head);
      const uint16_t* qp = p.q + b * p.q_batch + query * p.q_row + head * p.q_head + q4 * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s) f[n][s] = *reinterpret_cast<const bf16x8*>(qp + s * 32);
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      m[n] = -3.0e38f;  // (finite: a chunk all of whose logits are -infinity leaves it where it is)
      l[n] = 0.f;
      lv[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int db = 0; db < DB; ++db) o[n][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // The chunk `at` bytes behind the first; bit i of `keys`: key i takes part (at least one).  FAST: P = exp2(logit); otherwise with the running maximum
  // m, `headroom` above the logits', accumulated output and sum rescaled whenever a maximum moves.  FIRST (and FAST): the sums start here.
  template <bool FAST, bool FIRST = false>
  __device__ __forceinline__ void chunk(uint32_t at, uint64_t keys, float headroom = 0.f) {
    // PV step of 32 keys: k slots 0-3 <-> keys 32 step + 4 q4 + (0..3), slots 4-7 <-> 16 more.  The fragments of half of the row
    // blocks are read ahead of the MFMAs of the half before.
    constexpr int DH = DB / 2, PARTS = KC / 32 * 2;
    bf16x8 vfb[2][DH];
    TrFrag vtr[2][DH];
    auto load_v = [&](int part, int slot) {
#pragma unroll
      for (int d = 0; d < DH; ++d) {
        const uint32_t a0 = v_tr[(part & 1) * DH + d] + at + (part >> 1) * 32 * (HD * 2);
        vtr[slot][d].lo = lds_read_tr16_b64<0>(a0);
        vtr[slot][d].hi = lds_read_tr16_b64<16 * (HD * 2)>(a0);
      }
    };
    auto v_ready = [&](int slot) {
      if constexpr (DH == 4) lds_tr_wait(vtr[slot][0], vtr[slot][1 % DH], vtr[slot][2 % DH], vtr[slot][3 % DH]);
      else if constexpr (DH == 2) lds_tr_wait(vtr[slot][0], vtr[slot][1 % DH]);
      else lds_tr_wait(vtr[slot][0]);
#pragma unroll
      for (int d = 0; d < DH; ++d) vfb[slot][d] = tr_frag_value(vtr[slot][d]);
    };
    // (ahead of the MFMAs: behind them the reads could return into registers that the first of an accumulator's MFMAs is still writing)
    load_v(0, 0);
    __builtin_amdgcn_sched_barrier(0);

    // The wave of a SIMD that has its weights goes first: its product is the longer chain, the other's exponentials fill the gaps (1251 -> 1191 us for
    // 1 036 800 queries, sixteen heads of 64, 256 keys; first for K Q^T as well 1192, for the exponentials alone 1260; two members of 64 800, eight
    // heads, 1000 keys 273 -> 265, 269 and 270)
    __builtin_amdgcn_s_setprio(0);
    f32x4 acc[QN][KB];
    // ---- S^T: acc[n][kb][i] = logit of key 16 kb + 4 q4 + i, row 16 n + l15; K fragments are read two ahead of their MFMAs
    {
      constexpr int PF = 2, NS = KB * KS;
      const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
      bf16x8 kfr[PF + 1];
      auto read_k = [&](int t) {
        typedef __attribute__((address_space(3))) const bf16x8* frag_ptr;
        return *(frag_ptr)(k_lane[t / KB] + at + (t % KB) * 16 * (HD * 2));
      };
#pragma unroll
      for (int t = 0; t < PF; ++t) kfr[t] = read_k(t);
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        if (t + PF < NS) kfr[(t + PF) % (PF + 1)] = read_k(t + PF);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < QN; ++n)
          acc[n][t % KB] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kfr[t % (PF + 1)], qf[n][t / KB], t / KB == 0 ? zero4 : acc[n][t % KB], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // Keys that do not take part: their rows of K and V are zeros, so that FAST, where P is then 1, has them in the sum alone.  They are taken out of it
    // chunk by chunk, each lane's of its own: left in until the end they would be a sum beside which small weights are rounded away (weights of 2^-12.5,
    // a tenth of 60 000 keys masked: 2 per cent of the sum).
    if (FAST && keys != ~0ull) {
      const uint32_t lo = ~(uint32_t)keys >> (4 * q4) & 0x000f000fu, hi = ~(uint32_t)(keys >> 32) >> (4 * q4) & 0x000f000fu;
      const float ones = (float)(SUM ? KC - __builtin_popcountll(keys) : __builtin_popcount(lo) + __builtin_popcount(hi));
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        if (SUM) lv[n][0] -= ones;
        else l[n] -= ones;
      }
    }
    if (!FAST && keys != ~0ull) {
      const uint64_t mine = keys >> (4 * q4);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((mine >> (kb * 16 + i)) & 1)) {
#pragma unroll
            for (int n = 0; n < QN; ++n) acc[n][kb][i] = -INFINITY;
          }
    }

    if (!FAST) {
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        float cm = acc[n][0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; i += 2) cm = fmaxf(fmaxf(cm, acc[n][kb][i]), acc[n][kb][i + 1]);
        cm = fmaxf(cm, __shfl_xor(cm, 16, 64));
        cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
        if (SCALED) cm *= q_mul;
        const float m_new = fmaxf(m[n], cm + headroom);
        if (__builtin_amdgcn_ballot_w64(m_new > m[n]) != 0) {
          const float alpha = __builtin_amdgcn_exp2f(m[n] - m_new);
          l[n] *= alpha;
          if (SUM) lv[n] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) o[n][db] *= alpha;
          m[n] = m_new;
        }
      }
    }

    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
    uint32_t pkb[2][QN][4];
    auto p_of = [&](float a, int n) {
      return __builtin_amdgcn_exp2f(SCALED ? (FAST ? a * q_mul : fmaf(a, q_mul, -m[n])) : FAST ? a : a - m[n]);
    };
    auto exp_step = [&](int step, int n) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const f32x4& a = acc[n][2 * step + (h >> 1)];
        pkb[step & 1][n][h] = pack_bf16x2(p_of(a[2 * (h & 1)], n), p_of(a[2 * (h & 1) + 1], n));
        if (!SUM) l[n] = dot2_ones(pkb[step & 1][n][h], FIRST && step == 0 && h == 0 ? 0.f : l[n]);
      }
    };
#pragma unroll
    for (int n = 0; n < QN; ++n) exp_step(0, n);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      const int step = part >> 1;
      __builtin_amdgcn_sched_barrier(0);
      v_ready(part & 1);
      if (part + 1 < PARTS) load_v(part + 1, (part + 1) & 1);
      if (step + 1 < KC / 32) {
#pragma unroll
        for (int n = part & 1 ? QN / 2 : 0; n < (part & 1 ? QN : QN / 2); ++n) exp_step(step + 1, n);
      }
#pragma unroll
      for (int d = 0; d < DH; ++d)
#pragma unroll
        for (int n = 0; n < QN; ++n) {
          const bf16x8 pf = __builtin_bit_cast(bf16x8, u32x4{pkb[step & 1][n][0], pkb[step & 1][n][1], pkb[step & 1][n][2], pkb[step & 1][n][3]});
          f32x4& od = o[n][(part & 1) * DH + d];
          const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
          od = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vfb[part & 1][d], pf, FIRST && step == 0 ? zero4 : od, 0, 0, 0);
          if (SUM && (part & 1) && d == 0) lv[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf, FIRST && step == 0 ? zero4 : lv[n], 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // 32 keys, whose 64 or fewer rows of K and V lie `at` bytes behind the first: as chunk(), for waves that divide the keys among them.
  // EXACT, for 16 rows, where latency or reading bounds the time: the weights as two bf16 each, what the first leaves goes into a second product (error
  // 0.0024 -> 0.0017 of the result, its own rounding; nothing for one query and 64 800 keys; 32 rows would be slower by 10 to 16 per cent: five members'
  // 37 queries, 14 400 keys 25.9 -> 29.5 us, 1000 queries, eight heads of 64, 1000 keys 8.0 -> 9.3)
  template <bool FAST>
  __device__ __forceinline__ void step(uint32_t at, uint32_t keys, float headroom = 0.f) {
    constexpr bool EXACT = QN == 1;
    TrFrag vt[DB];
    f32x4 acc[QN][2];
#pragma unroll
    for (int d = 0; d < DB; ++d) {  // (ahead of the MFMAs, see chunk())
      vt[d].lo = lds_read_tr16_b64<0>(v_tr[d] + at);
      vt[d].hi = lds_read_tr16_b64<16 * (HD * 2)>(v_tr[d] + at);
    }
    __builtin_amdgcn_sched_barrier(0);
    {
      const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
      typedef __attribute__((address_space(3))) const bf16x8* frag_ptr;
      bf16x8 kf[2][KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int b = 0; b < 2; ++b) kf[b][s] = *(frag_ptr)(k_lane[s] + at + b * 16 * (HD * 2));
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int n = 0; n < QN; ++n) acc[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[b][s], qf[n][s], s == 0 ? zero4 : acc[n][b], 0, 0, 0);
    }
    if (FAST && keys != ~0u) {  // (see chunk())
      const float ones = (float)__builtin_popcount(~keys >> (4 * q4) & 0x000f000fu);
#pragma unroll
      for (int n = 0; n < QN; ++n) l[n] -= ones;
    }
    if (!FAST) {
      const uint32_t mine = keys >> (4 * q4);
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        float cm = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((mine >> (b * 16 + i)) & 1)) acc[n][b][i] = -INFINITY;
            cm = fmaxf(cm, acc[n][b][i]);
          }
        cm = fmaxf(cm, __shfl_xor(cm, 16, 64));
        cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
        if (SCALED) cm *= q_mul;
        const float m_new = fmaxf(m[n], cm + headroom), alpha = __builtin_amdgcn_exp2f(m[n] - m_new);
        l[n] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[n][db] *= alpha;
        m[n] = m_new;
      }
    }
    uint32_t pk[QN][4], rest[QN][4];
#pragma unroll
    for (int n = 0; n < QN; ++n)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const f32x4& a = acc[n][h >> 1];
        auto p_of = [&](float x) { return __builtin_amdgcn_exp2f(SCALED ? (FAST ? x * q_mul : fmaf(x, q_mul, -m[n])) : FAST ? x : x - m[n]); };
        const float p0 = p_of(a[2 * (h & 1)]), p1 = p_of(a[2 * (h & 1) + 1]);
        pk[n][h] = pack_bf16x2(p0, p1);
        l[n] = dot2_ones(pk[n][h], l[n]);
        if (EXACT) {
          rest[n][h] = pack_bf16x2(p0 - bf16_lo(pk[n][h]), p1 - bf16_hi(pk[n][h]));
          l[n] = dot2_ones(rest[n][h], l[n]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (DB == 2) {
      lds_tr_wait(vt[0], vt[1 % DB]);
    } else {
      lds_tr_wait(vt[0], vt[1 % DB], vt[2 % DB], vt[3 % DB]);
      if constexpr (DB == 8) lds_tr_wait(vt[4 % DB], vt[5 % DB], vt[6 % DB], vt[7 % DB]);
    }
    auto add = [&](const uint32_t (&p)[QN][4]) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int n = 0; n < QN; ++n)
          o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(tr_frag_value(vt[d]), __builtin_bit_cast(bf16x8, u32x4{p[n][0], p[n][1], p[n][2], p[n][3]}), o[n][d], 0, 0, 0);
    };
    add(pk);
    if (EXACT && !FAST) {
      // An infinite value times what is left of its weight, 0 or of either sign, would undo the infinity that the first product gives.  (Where no maximum is
      // taken the rows are done again: their sums are not finite.)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        vt[d].lo.x = finite_bf16x2(vt[d].lo.x);
        vt[d].lo.y = finite_bf16x2(vt[d].lo.y);
        vt[d].hi.x = finite_bf16x2(vt[d].hi.x);
        vt[d].hi.y = finite_bf16x2(vt[d].hi.y);
      }
    }
    if (EXACT) add(rest);
    __builtin_amdgcn_sched_barrier(0);
  }

  // The rows' sums.  `idle` keys of the chunks did not take part; `within`: as many of their ones are still in the sums.  Whether any row's left the range
  // in which exp2 needs no maximum (or is not a number), or is so small beside the idle keys' ones that what the two together were rounded by counts:
  // with n additions n 2^-24 2^6 of it, 2^-15 for those of a chunk's lane, 2^-13 for those of the nine chunks that may stay in LDS.  Or whether a result's
  // sum is beyond 2^100 or not a number.
  __device__ __forceinline__ bool sums(int idle, int within = 0) {
    bool bad = false;
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      if (SUM) {
        l[n] = lv[n][0];
      } else {
        l[n] += __shfl_xor(l[n], 16, 64);
        l[n] += __shfl_xor(l[n], 32, 64);
      }
      l[n] -= (float)within;
      bad = bad || !(l[n] >= 0x1p-20f && l[n] >= 0x1p-6f * (float)idle && l[n] <= 0x1p60f);
      float top = 0.f;  // (maximum, not max: NaN stays)
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, fabsf(o[n][db][i])), fabsf(o[n][db][i + 1]));
      bad = bad || !(top <= 0x1p100f);
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
  }

  // normalise (a row without any key is zeros), 8 consecutive elements a lane and store
  __device__ __forceinline__ void store(const CrossParams& p, const Task& t, int member, int hk, int row0, int lane) const {
    const int mine = 16 * (q4 & 1) + 8 * (q4 >> 1);
    auto put = [&](int n, uint16_t* op, bool there) {
      const float inv = l[n] == 0.f ? 0.f : __builtin_amdgcn_rcpf(l[n]);
#pragma unroll
      for (int m2 = 0; m2 < DB / 2; ++m2) {
        const f32x4 a = o[n][2 * m2] * inv, c = o[n][2 * m2 + 1] * inv;
        const auto rx = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[0], a[1]), pack_bf16x2(c[0], c[1]), false, false);
        const auto ry = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[2], a[3]), pack_bf16x2(c[2], c[3]), false, false);
        if (there) *reinterpret_cast<u32x4*>(op + m2 * 32) = u32x4{rx[0], ry[0], rx[1], ry[1]};
      }
    };
    if (plain(p, t, row0)) {
      uint16_t* first = p.out + (((int64_t)member * p.Nq + row0) * p.heads + hk) * HD;
      const int64_t of_lane = (lane & 15) * p.heads * HD + mine;
#pragma unroll
      for (int n = 0; n < QN; ++n) put(n, first + (int64_t)n * 16 * p.heads * HD + of_lane, true);
      return;
    }
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      int64_t b = member;
      int query, head;
      row_of(p, t, hk, row0, n, lane, b, query, head);
      put(n, p.out + ((b * p.Nq + query) * p.heads + head) * HD + mine, row0 + n * 16 + (lane & 15) < t.rows);
    }
  }
};

// How far above its logits a row's maximum is taken: weights of 2^-headroom at most, half a 1 for all keys of a task together
__device__ __forceinline__ float headroom_of(const Task& t) { return (float)(33 - __builtin_clz((uint32_t)t.Np + (uint32_t)t.Nk | 1u)); }

// A unit's keys in chunks of U: the prefix, then the member's own.
template <int U>
struct Keys {
  const unsigned char *k, *v;          // of the chunk that is loaded next
  const unsigned char *k_own, *v_own;  // of the member's first key
  uint32_t k_row, v_row;               // bytes between rows
  int left;                            // keys from that chunk to the end of the prefix, or of the member's own
  int prefix_chunks, own;
  int chunks;

  __device__ __forceinline__ Keys(const CrossParams& p, const Task& t, int member, int hk) {
    own = t.Nk;
    if (p.lengths && t.Nk > 0) {
      own = __builtin_amdgcn_readfirstlane(p.lengths[member * p.lengths_step]);
      own = own < 0 ? 0 : own < t.Nk ? own : t.Nk;
    }
    prefix_chunks = (t.Np + U - 1) / U;
    chunks = prefix_chunks + (own + U - 1) / U;
    k_own = reinterpret_cast<const unsigned char*>(p.k + member * p.k_batch + hk * p.k_head);
    v_own = reinterpret_cast<const unsigned char*>(p.v + member * p.v_batch + hk * p.v_head);
  }
  // the chunks of one part: as many for each, the same for members of any length
  __device__ __forceinline__ void part(const Task& t, int split, int& c0, int& c1) const {
    const int all = (t.Np + U - 1) / U + (t.Nk + U - 1) / U, each = (all + t.splits - 1) / t.splits;
    c0 = each * split < chunks ? each * split : chunks;
    c1 = c0 + each < chunks ? c0 + each : chunks;
  }
  __device__ __forceinline__ void seek(const CrossParams& p, const Task& t, int hk, int c) {
    if (c < prefix_chunks) {
      k_row = p.prefix_k_row;
      v_row = p.prefix_v_row;
      k = reinterpret_cast<const unsigned char*>(p.prefix_k + hk * p.prefix_k_head) + (int64_t)c * U * k_row;
      v = reinterpret_cast<const unsigned char*>(p.prefix_v + hk * p.prefix_v_head) + (int64_t)c * U * v_row;
      left = t.Np - c * U;
    } else {
      c -= prefix_chunks;
      k_row = p.k_row;
      v_row = p.v_row;
      k = k_own + (int64_t)c * U * k_row;
      v = v_own + (int64_t)c * U * v_row;
      left = own - c * U;
    }
  }
};

// Loads of a chunk of U keys into LDS by NWAVE waves: instruction i of wave w fills the rows RPI * (w + NWAVE * i) .., lane = (row, 16-byte slot).
template <int HD, int NWAVE, int U>
struct Loader {
  static constexpr int BYTES = U * HD * 2;  // of a chunk of K or of V
  static constexpr int PPR = HD / 8;        // 16-byte pieces per row
  static constexpr int RPI = 64 / PPR;      // rows that one load instruction of a wave fills
  static constexpr int LOADS = U / (RPI * NWAVE);
  static_assert(U % (RPI * NWAVE) == 0, "a chunk is a whole number of instructions of each wave");
  int row0, wave;  // the lane's row of instruction 0
  uint32_t off_k[LOADS], off_v[LOADS];

  __device__ __forceinline__ Loader(int lane, int w) : row0(RPI * w + lane / PPR), wave(w) {}
  __device__ __forceinline__ void rows(int lane, const Keys<U>& keys) {  // where the lane's pieces lie in a chunk, for the rows' present strides
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = row0 + RPI * NWAVE * i, slot = lane % PPR;
      off_k[i] = __umul24(row, keys.k_row) + (uint32_t)((slot ^ k_swizzle<HD>(row)) << 4);
      off_v[i] = __umul24(row, keys.v_row) + (uint32_t)((slot ^ v_swizzle<HD>(row)) << 4);
    }
  }
  // the chunk that `keys` stands at, into LDS at k_lds and v_lds.  Bit i of `word`: key i takes part.
  __device__ __forceinline__ void issue(const Keys<U>& keys, uint64_t word, uint32_t k_lds, uint32_t v_lds) const {
    const lds_dma_rsrc rk = make_lds_dma_rsrc(keys.k, 0x80000000u), rv = make_lds_dma_rsrc(keys.v, 0x80000000u);
    if (word == (U == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        lds_dma_load16(rk, k_lds + (uint32_t)(wave + NWAVE * i) * 1024, off_k[i], 0);
        lds_dma_load16(rv, v_lds + (uint32_t)(wave + NWAVE * i) * 1024, off_v[i], 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const bool on = (word >> (row0 + RPI * NWAVE * i)) & 1;  // (outside the descriptor: not read, zeros)
        lds_dma_load16(rk, k_lds + (uint32_t)(wave + NWAVE * i) * 1024, on ? off_k[i] : 0xFFFFF000u, 0);
        lds_dma_load16(rv, v_lds + (uint32_t)(wave + NWAVE * i) * 1024, on ? off_v[i] : 0xFFFFF000u, 0);
      }
    }
  }
  // the same, then on to the next chunk (number c + 1)
  __device__ __forceinline__ void issue_next(const CrossParams& p, const Task& t, int hk, int lane, Keys<U>& keys, int c, uint64_t word, uint32_t k_lds,
                                             uint32_t v_lds) {
    issue(keys, word, k_lds, v_lds);
    if (c + 1 == keys.prefix_chunks) {
      keys.seek(p, t, hk, c + 1);
      rows(lane, keys);
    } else {
      keys.k += (int64_t)U * keys.k_row;
      keys.v += (int64_t)U * keys.v_row;
      keys.left -= U;
    }
  }
};

// A member's key mask, as far as it has keys
struct Mask {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ Mask() : rsrc(__builtin_amdgcn_make_buffer_rsrc(nullptr, 0, 0, 0x00020000)) {}
  __device__ __forceinline__ Mask(const CrossParams& p, int member, int own)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.mask) + member * p.mask_batch, 0, own, 0x00020000)) {}
  // The byte for the lane's key of chunk c: 0 outside the member's keys (outside the descriptor, those of the prefix too, whose numbers are negative).  A
  // wave reads it a chunk ahead, beside that chunk's loads, and waits for both together: masks of any length cost no LDS and no pass of their own.
  template <int U>
  __device__ __forceinline__ uint32_t byte(const Keys<U>& keys, int c, int lane) const {
    return __builtin_amdgcn_raw_buffer_load_b8(rsrc, (uint32_t)((c - keys.prefix_chunks) * U + lane), 0, 0);
  }
};
// The mask of all of a unit's chunks of 64 as words in LDS (of the prefix: all ones), where the keys stay there and are looked at again
template <int NWAVE>
__device__ __forceinline__ void mask_words(const Mask& mask, const Keys<KC>& keys, uint64_t* words, int lane, int wave) {
  for (int c = wave; c < keys.chunks; c += NWAVE) {
    const uint64_t word = c < keys.prefix_chunks ? ~0ull : __builtin_amdgcn_ballot_w64(mask.byte(keys, c, lane) != 0);
    if (lane == 0) words[c] = word;
  }
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}

}  // namespace

// The workgroup's unit (part of the keys, member, key head) and row block, and whether there is work for it.  XCDs take units in turn, or all heads of a
// member's part at a time (`together`): rows of heads that lie side by side share lines of memory and its pages (64 members of 8000 keys, four heads of
// 32: 80 -> 41 us against heads on XCDs in turn; 256 of 500 keys, eight of 64: 42 -> 40.5).  Each turn starts one XCD further: lengths, and with them
// work, fall along members and parts, and none of them always goes to the same XCD.
__device__ __forceinline__ bool place(const CrossParams& p, const Task& t, int block, int& split, int& member, int& hk, int& qb) {
  const int at = block - t.first, xcd = at & 7, s = at >> 3;  // (a task's first workgroup is a multiple of 8)
  int unit;
  if (t.by_rows) {
    const int per = (t.qblks + 7) / 8;
    unit = s / per;
    qb = xcd * per + s % per;
  } else {
    const int i = s / t.qblks, turn = i / t.together;
    unit = (8 * turn + ((xcd + turn) & 7)) * t.together + i - turn * t.together;
    qb = s % t.qblks;
  }
  if (unit >= t.units || qb >= t.qblks) return false;
  const int bm = unit / p.kv_heads;
  hk = unit - bm * p.kv_heads;
  split = bm / t.members;
  member = bm - split * t.members;
  return true;
}

// K and V in two buffers: a chunk is loaded while the one before is worked on.  (Three and four buffers: the same times, with a row block alone on its
// CU too - a chunk takes a wave longer, 0.5 us and more, than its load.)
// PARTS: the keys are divided among workgroups, which leave their sums in the workspace.
template <int HD, int NWAVE, int QN, bool PARTS, bool SCALED, bool SUM>
__global__ void __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(2)))
cross_attention_rows_kernel(CrossParams p) {
  using Load = Loader<HD, NWAVE, KC>;
  constexpr int BYTES = Load::BYTES, V_BASE = 2 * BYTES;
  constexpr int QW = 16 * QN, QB = QW * NWAVE;  // rows per wave and workgroup
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const uint32_t smem_addr = lds_byte_address(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const Task& t = p.task[PARTS && (int)blockIdx.x >= p.task[1].first ? 1 : 0];
  int split, member, hk, qb;
  if (!place(p, t, blockIdx.x, split, member, hk, qb)) return;
  Keys<KC> keys(p, t, member, hk);
  int c0 = 0, c1 = keys.chunks;
  if (PARTS) keys.part(t, split, c0, c1);
  const int nch = c1 - c0;

  const int row0 = qb * QB + wave * QW;
  const bool wave_active = row0 < t.rows;  // wave-uniform: a wave without rows only loads and keeps the barriers
  Rows<HD, QN, SCALED, SUM> rows(smem, V_BASE, lane, p.q_mul);
  Load load(lane, wave);

  const bool masked = p.mask && t.Nk > 0;
  Mask mask;
  if (masked) mask = Mask(p, member, keys.own);
  uint32_t byte = 0;  // of the mask, for the chunk that is loaded next
  uint64_t kk[2];     // which keys of the chunks in the buffers take part
  auto issue = [&](int j, int buf) {
    const int c = c0 + j;
    kk[buf] = first_keys(keys.left);
    if (masked) {
      if (c >= keys.prefix_chunks) kk[buf] &= __builtin_amdgcn_ballot_w64(byte != 0);
      byte = mask.byte(keys, c + 1, lane);
    }
    load.issue_next(p, t, hk, lane, keys, c, kk[buf], smem_addr + buf * BYTES, smem_addr + V_BASE + buf * BYTES);
  };
  bool any = false;  // whether any key took part (uniform)
  int idle = 0;      // keys that did not, of chunks with keys that did

  auto sweep = [&](auto fast_tag) {
    constexpr bool FAST = decltype(fast_tag)::value;
    const float headroom = FAST ? 0.f : headroom_of(t);
    keys.seek(p, t, hk, c0);
    load.rows(lane, keys);
    if (masked) byte = mask.byte(keys, c0, lane);
    if (nch > 0) issue(0, 0);
    if (FAST) rows.load_q(p, t, member, hk, row0, lane, rows.qf);
    rows.reset();
    if (FAST) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the compiler knows the queries to be there (inside the loop it would wait for the chunks too)
    for (int j0 = 0; j0 < nch; j0 += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u;
        if (j >= nch) break;
        // this wave's part of chunk j has landed; behind the barrier every wave's has, and every wave is done with chunk j - 1, whose
        // buffer chunk j + 1 goes to
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (j + 1 < nch) issue(j + 1, u ^ 1);
        if (kk[u] != 0) {
          any = true;
          if (FAST) idle += KC - __builtin_popcountll(kk[u]);
          if (wave_active) rows.template chunk<FAST>(u * BYTES, kk[u], headroom);
        }
      }
    }
  };
  sweep(std::true_type{});
  bool online;
  {
    __syncthreads();  // every wave is done with the chunks: a flag in their place
    int* const redo = reinterpret_cast<int*>(smem);
    if (tid == 0) *redo = 0;
    __syncthreads();
    if (rows.sums(idle) && any && wave_active && lane == 0) *redo = 1;
    __syncthreads();
    online = __builtin_amdgcn_readfirstlane(*redo) != 0;
    if (online) {
      __syncthreads();
      sweep(std::false_type{});
      rows.sums(0);
    }
  }
  if (!PARTS) {
    rows.store(p, t, member, hk, row0, lane);
    return;
  }
#pragma unroll
  for (int n = 0; n < QN; ++n) {
    const int row = row0 + n * 16 + (lane & 15);
    if (row >= t.rows) continue;
    const int64_t at = (((int64_t)split * t.members + member) * p.kv_heads + hk) * t.rows + row;
    if (rows.q4 == 0) {
      t.ml[2 * at] = online ? rows.m[n] : 0.f;
      t.ml[2 * at + 1] = rows.l[n];
    }
#pragma unroll
    for (int db = 0; db < HD / 16; ++db)  // (not to be held in L2, which a kernel's end empties: 18.2 -> 15.2 us where the parts are 16 MB)
      __builtin_nontemporal_store(rows.o[n][db], reinterpret_cast<f32x4*>(t.o + at * HD + 16 * db + 4 * rows.q4));
  }
}

// Few rows: the waves of a workgroup divide the keys among them, 32 at a time in turn, for the same 16 QN rows; each has its own two buffers and
// keeps its own pace.  Their sums meet in LDS.  PARTS: the keys are divided among workgroups too, which leave theirs in the workspace.
template <int HD, int NWAVE, int QN, bool PARTS>
__global__ void __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 1 : 2)))
cross_attention_keys_kernel(CrossParams p) {
  constexpr int U = 32, QB = 16 * QN;
  using Load = Loader<HD, 1, U>;
  constexpr int BYTES = Load::BYTES, RING = 4 * BYTES;  // of K or V of a step; of a wave's buffers
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned char* const ring = smem + wave * RING;
  const uint32_t ring_addr = lds_byte_address(ring);

  const Task& t = p.task[PARTS && (int)blockIdx.x >= p.task[1].first ? 1 : 0];
  int split, member, hk, qb;
  if (!place(p, t, blockIdx.x, split, member, hk, qb)) return;
  Keys<U> keys(p, t, member, hk);
  int c0 = 0, c1 = keys.chunks;
  if (PARTS) keys.part(t, split, c0, c1);
  const int row0 = qb * QB;
  Rows<HD, QN, true, false> rows(ring, BYTES, lane, p.q_mul);
  Load load(lane, 0);
  const bool masked = p.mask && t.Nk > 0;
  Mask mask;
  if (masked) mask = Mask(p, member, keys.own);  // (its arguments are not waited for where there is none: 19.6 -> 19.3 us for sixteen members of one query)
  uint32_t byte = 0;  // of the mask, for the step that is loaded next
  const int steps = (c1 - c0 - wave + NWAVE - 1) / NWAVE;  // of this wave: c0 + wave, c0 + wave + NWAVE, ..
  uint32_t kk[2];
  int part_of = -1;  // whose rows' strides the loader has: 0 the prefix's, 1 the member's own
  auto issue = [&](int j, int buf) {
    const int c = c0 + wave + j * NWAVE;
    keys.seek(p, t, hk, c);
    if (part_of != (c >= keys.prefix_chunks)) {
      part_of = c >= keys.prefix_chunks;
      load.rows(lane, keys);
    }
    uint64_t w = first_keys(keys.left < U ? keys.left : U);
    if (masked) {
      if (c >= keys.prefix_chunks) w &= __builtin_amdgcn_ballot_w64(byte != 0);
      byte = mask.byte(keys, c + NWAVE, lane);
    }
    kk[buf] = (uint32_t)w;
    load.issue(keys, w & 0xffffffffull, ring_addr + buf * 2 * BYTES, ring_addr + buf * 2 * BYTES + BYTES);
  };
  bool any = false;
  int idle = 0;
  auto sweep = [&](auto fast_tag) {
    constexpr bool FAST = decltype(fast_tag)::value;
    const float headroom = FAST ? 0.f : headroom_of(t);
    if (masked) byte = mask.byte(keys, c0 + wave, lane);
    if (steps > 0) issue(0, 0);
    if (FAST) rows.load_q(p, t, member, hk, row0, lane, rows.qf);
    rows.reset();
    if (FAST) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), see the kernel above
    for (int j0 = 0; j0 < steps; j0 += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u;
        if (j >= steps) break;
        // step j's buffer is filled; then the one that step j - 1 was done with is loaded again
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (j + 1 < steps) issue(j + 1, u ^ 1);
        if (kk[u] != 0) {
          any = true;
          if (FAST) idle += U - __builtin_popcount(kk[u]);
          rows.template step<FAST>(u * 2 * BYTES, kk[u], headroom);
        }
      }
    }
  };
  sweep(std::true_type{});
  const bool online = rows.sums(idle) && any;
  if (online) {
    sweep(std::false_type{});
    rows.sums(0);
  }

  // ---- the waves' sums: [wave][row][HD] fp32, 16-byte pieces XOR-swizzled by the row, and [wave][row] maximum, sum
  __syncthreads();
  f32x4* const so = reinterpret_cast<f32x4*>(smem);
  float* const sm = reinterpret_cast<float*>(smem + NWAVE * QB * HD * 4);
  constexpr int PIECES = HD / 4, SWZ = PIECES < 16 ? PIECES - 1 : 15;
  auto piece = [](int w, int row, int c) { return (w * QB + row) * PIECES + (c ^ (row & SWZ)); };
#pragma unroll
  for (int n = 0; n < QN; ++n) {
    const int row = 16 * n + (lane & 15);
    if (rows.q4 == 0) {
      sm[2 * (wave * QB + row)] = online ? rows.m[n] : any ? 0.f : -3.0e38f;
      sm[2 * (wave * QB + row) + 1] = any ? rows.l[n] : 0.f;
    }
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) so[piece(wave, row, 4 * db + rows.q4)] = rows.o[n][db];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < (QB * PIECES + 64 * NWAVE - 1) / (64 * NWAVE); ++i) {
    const int at = i * 64 * NWAVE + tid, row = at / PIECES, c = at % PIECES;
    const int r = row0 + row;
    if (row >= QB || r >= t.rows) continue;
    float m = -3.0e38f, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) m = fmaxf(m, sm[2 * (w * QB + row)]);
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) {
      const float a = __builtin_amdgcn_exp2f(sm[2 * (w * QB + row)] - m);
      l += a * sm[2 * (w * QB + row) + 1];
      o += a * so[piece(w, row, c)];
    }
    if (PARTS) {
      const int64_t dst = (((int64_t)split * t.members + member) * p.kv_heads + hk) * t.rows + r;
      if (c == 0) {
        t.ml[2 * dst] = m;
        t.ml[2 * dst + 1] = l;
      }
      __builtin_nontemporal_store(o, reinterpret_cast<f32x4*>(t.o + dst * HD + 4 * c));
    } else {
      const int bb = p.of_rows_m.of(r), rm = r - bb * p.rows_m, query = p.of_group.of(rm), head = hk * p.group + rm - query * p.group;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      *reinterpret_cast<u32x2*>(p.out + (((int64_t)(member + bb) * p.Nq + query) * p.heads + head) * HD + 4 * c) =
          u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
    }
  }
}

// Few keys, many rows: the workgroup's unit stays in LDS, its waves walk down the row blocks, each at its own pace: no barrier behind the
// first, a block's queries are fetched while the one before is worked on.  Task::qblks is the number of workgroups of a unit.
template <int HD, int NWAVE, int QN, bool SCALED, bool SUM>
__global__ void __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(2)))
cross_attention_resident_kernel(CrossParams p, int max_chunks) {
  using Load = Loader<HD, NWAVE, KC>;
  constexpr int BYTES = Load::BYTES, QW = 16 * QN;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const uint32_t v_base = (uint32_t)max_chunks * BYTES, smem_addr = lds_byte_address(smem);
  uint64_t* const words = reinterpret_cast<uint64_t*>(smem + 2 * v_base);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Task& t = p.task[0];
  const int unit = blockIdx.x % t.units, part = blockIdx.x / t.units;
  const int member = unit / p.kv_heads, hk = unit - member * p.kv_heads;
  Keys<KC> keys(p, t, member, hk);
  const int nch = keys.chunks;
  if (p.mask && t.Nk > 0) {
    mask_words<NWAVE>(Mask(p, member, keys.own), keys, words, lane, wave);
    __syncthreads();
  }
  Rows<HD, QN, SCALED, SUM> rows(smem, v_base, lane, p.q_mul);
  Load load(lane, wave);
  const int step = t.qblks * NWAVE * QW;
  int row0 = (part * NWAVE + wave) * QW;
  bf16x8 next[QN][HD / 32];
  if (row0 < t.rows) rows.load_q(p, t, member, hk, row0, lane, next);
  keys.seek(p, t, hk, 0);
  load.rows(lane, keys);
  int idle = 0;
  auto word_of = [&](int c) {
    const int n = c < keys.prefix_chunks ? t.Np - c * KC : keys.own - (c - keys.prefix_chunks) * KC;
    uint64_t w = first_keys(n);
    if (p.mask && t.Nk > 0) w &= uniform64(words[c]);
    return w;
  };
  for (int c = 0; c < nch; ++c) {
    const uint64_t w = word_of(c);
    idle += KC - __builtin_popcountll(w);
    load.issue_next(p, t, hk, lane, keys, c, w, smem_addr + c * BYTES, smem_addr + v_base + c * BYTES);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (idle == nch * KC) {  // no keys
    rows.reset();
    for (; row0 < t.rows; row0 += step) rows.store(p, t, member, hk, row0, lane);
    return;
  }

  // Rows that need a maximum come afterwards, those of all blocks together, so that the loop that nearly all take holds no registers for them: a
  // bit for each block, or for 2, 3, .. in a row where there are more than 64
  uint64_t again = 0;
  const int start = row0, per_bit = ((t.rows - start + step - 1) / step + 63) / 64;
  for (int bit = 0, j = 0; row0 < t.rows; row0 += step) {
#pragma unroll
    for (int n = 0; n < QN; ++n)
#pragma unroll
      for (int s = 0; s < HD / 32; ++s) rows.qf[n][s] = next[n][s];
    if (row0 + step < t.rows) rows.load_q(p, t, member, hk, row0 + step, lane, next);
    int c = 0;
    if constexpr (HD == 32) {  // (its registers are few: the same time in one loop, 37.1 us and 37.5 for 64 800 x 77 keys, 52.6 and 52.2 for 200)
      rows.reset();
      do rows.template chunk<true>(c * BYTES, ~0ull);
      while (++c < nch);
    } else {  // (80 registers that need not be cleared for each block: 1216 -> 1191 us, sixteen heads of 64, 256 keys)
      rows.template chunk<true, true>(0, ~0ull);
      while (++c < nch) rows.template chunk<true>(c * BYTES, ~0ull);
    }
    if (rows.sums(idle, idle)) again |= 1ull << bit;
    else rows.store(p, t, member, hk, row0, lane);
    if (++j == per_bit) {
      j = 0;
      ++bit;
    }
  }
  for (; again != 0; again &= again - 1) {
    row0 = start + __builtin_ctzll(again) * per_bit * step;
    for (int j = 0; j < per_bit && row0 < t.rows; ++j, row0 += step) {
      rows.load_q(p, t, member, hk, row0, lane, rows.qf);
      rows.reset();
      for (int c = 0; c < nch; ++c) {
        const uint64_t w = word_of(c);
        if (w != 0) rows.template chunk<false>(c * BYTES, w, headroom_of(t));
      }
      rows.sums(0);
      rows.store(p, t, member, hk, row0, lane);
    }
  }
}

// ---------------------------------------------------------------------------------------------

namespace {

// One row's parts, up to two sets of them (of the prefix, whose rows are those of all members; of the member's own keys)
struct JoinParams {
  Task task[2];
  uint16_t* out;
  int64_t rows;  // (member, query, head)
  int Nq, heads, kv_heads, group, rows_m;
};

}  // namespace

// out[row] = sum over the parts of 2^(m - max m) o / sum of 2^(m - max m) l.  WPR waves do a row, each every WPR-th part: lane i looks at part i's
// maximum and sum, the weights then go round by lane exchange, and HD / 4 lanes read a part's row, 16 parts on the way at a time.  What it costs, 4 to 5 us,
// is the latency of two reads behind one another (a part at a time: 8 us for 16 of head size 128).
template <int HD, int WPR>
__global__ void __launch_bounds__(WPR > 4 ? 64 * WPR : 256) cross_attention_join_kernel(JoinParams p) {
  constexpr int AT_ONCE = 16;  // parts (8 and 32: half a microsecond more at 16 and at 64 parts)
  constexpr int CT = HD / 4, SUB = 64 / CT, NW = WPR > 4 ? WPR : 4;  // waves of a workgroup
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % CT, sub = lane / CT, first_part = wave % WPR;
  const int64_t row = (int64_t)blockIdx.x * (NW / WPR) + wave / WPR;
  float m = -3.0e38f, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (row < p.rows) {  // (wave-uniform)
    const int head = (int)(row % p.heads);
    const int64_t bq = row / p.heads;
    const int query = (int)(bq % p.Nq), b = (int)(bq / p.Nq);
    const int hk = head / p.group, rm = query * p.group + head - hk * p.group;
    int64_t first[2], step[2];
    float pm2[2], pl2[2];  // of the first parts of both sets: their reads are on the way together
    auto look = [&](int set, int s0, float& pm, float& pl) {
      const Task& t = p.task[set];
      pm = -3.0e38f;
      pl = 0.f;
      if (s0 + lane * WPR < t.splits) {
        const float* at = t.ml + 2 * (first[set] + (s0 + lane * WPR) * step[set]);
        pm = at[0];
        pl = at[1];
      }
    };
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      const Task& t = p.task[set];
      const bool all = t.members == 1;  // a unit's rows are those of all members
      first[set] = ((int64_t)(all ? 0 : b) * p.kv_heads + hk) * t.rows + (all ? b * p.rows_m : 0) + rm;
      step[set] = (int64_t)t.members * p.kv_heads * t.rows;
      look(set, first_part, pm2[set], pl2[set]);
    }
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      const Task& t = p.task[set];
      for (int s0 = first_part; s0 < t.splits; s0 += 64 * WPR) {
        const int n = (t.splits - s0 + WPR - 1) / WPR < 64 ? (t.splits - s0 + WPR - 1) / WPR : 64;
        float pm = pm2[set], pl = pl2[set];
        if (s0 != first_part) look(set, s0, pm, pl);
        if (pl == 0.f) pm = -3.0e38f;  // no key of this part
        float mx = pm;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        const float mn = fmaxf(m, mx), a0 = __builtin_amdgcn_exp2f(m - mn), w = pl == 0.f ? 0.f : __builtin_amdgcn_exp2f(pm - mn);
        m = mn;
        l = l * a0 + wave_sum(w * pl);
        o *= a0;
        for (int i0 = 0; i0 < n; i0 += AT_ONCE) {
          float wi[AT_ONCE / SUB];
          f32x4 po[AT_ONCE / SUB];
#pragma unroll
          for (int u = 0; u < AT_ONCE / SUB; ++u) {
            const int i = i0 + u * SUB + sub;
            wi[u] = __shfl(w, i, 64);
            const int64_t at = first[set] + (s0 + (i < n ? i : n - 1) * WPR) * step[set];
            po[u] = *reinterpret_cast<const f32x4*>(t.o + at * HD + 4 * c);
          }
#pragma unroll
          for (int u = 0; u < AT_ONCE / SUB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += wi[u] == 0.f ? 0.f : po[u][e] * wi[u];  // (a part without keys has written nothing)
        }
      }
    }
#pragma unroll
    for (int d = CT; d < 64; d *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d, 64);
  }
  if (WPR > 1) {
    __shared__ f32x4 so[NW][CT];
    __shared__ float sm[NW], sl[NW];
    if (sub == 0) so[wave][c] = o;
    if (lane == 0) {
      sm[wave] = m;
      sl[wave] = l;
    }
    __syncthreads();
    if (first_part != 0) return;
    float mx = m;
    for (int w = 1; w < WPR; ++w) mx = fmaxf(mx, sm[wave + w]);
    const float a0 = __builtin_amdgcn_exp2f(m - mx);
    o *= a0;
    l *= a0;
    for (int w = 1; w < WPR; ++w) {
      const float a = __builtin_amdgcn_exp2f(sm[wave + w] - mx);
      o += so[wave + w][c] * a;
      l += sl[wave + w] * a;
    }
  }
  if (sub == 0 && row < p.rows) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<u32x2*>(p.out + row * HD + 4 * c) = u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  }
}

// ---------------------------------------------------------------------------------------------

namespace {

constexpr int NWAVE = 4;
// Blocks of 16 rows per wave.  More of them read a K / V fragment from LDS for more rows; fewer leave registers for more waves (head size 64, 1 036 800
// queries, sixteen heads, 256 keys: 2 1286 us, 3 1222, 4 1191; 64 800, 77 keys: 52, 52, 51-56; head size 32, 200 keys: 2 53, 3 59, 4 55).
constexpr int resident_qn(int64_t head_dim) { return head_dim == 64 ? 4 : 2; }
constexpr int64_t RESIDENT_LDS = 80 * 1024;  // two workgroups per CU

// How a call is run
enum class Form { rows, keys, resident };
struct Plan {
  Task task[2];
  Form form;
  int n, qn;    // tasks; blocks of 16 rows per wave
  bool parts;   // sums go through the workspace
  int resident; // chunks that a workgroup keeps in LDS
  int64_t grid, bytes;  // workgroups; of the workspace
};

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Microseconds of a launch, fitted to measurements (1 to 64 800 queries, 77 to 4000 keys, 4 and 8 heads): a workgroup's step - a chunk of 64 keys, or 32
// keys for each of its waves - alone on its CU, and one of several there; what a round of workgroups costs besides; how many a CU holds.
struct Cost { float alone, among, round; int per_cu; };
struct Costs {
  Cost rows[3], keys[3];  // 16, 32 and 64 rows per wave; per workgroup
};
const Costs& costs_of(int64_t head_dim) {
  static const Costs c32 = {{{0.48f, 0.25f, 1.6f, 4}, {0.56f, 0.40f, 1.9f, 4}, {}}, {{0.32f, 0.27f, 1.2f, 4}, {0.41f, 0.30f, 1.6f, 4}, {0.57f, 0.45f, 2.4f, 4}}};
  static const Costs c64 = {{{0.56f, 0.40f, 1.8f, 3}, {0.75f, 0.55f, 2.2f, 3}, {1.32f, 0.95f, 5.5f, 2}}, {{0.40f, 0.30f, 1.7f, 2}, {0.48f, 0.39f, 2.4f, 2}, {0.70f, 0.65f, 3.6f, 2}}};
  static const Costs c128 = {{{0.86f, 0.65f, 1.9f, 2}, {1.12f, 0.95f, 2.3f, 2}, {}}, {{0.60f, 0.68f, 2.0f, 1}, {0.75f, 0.85f, 3.2f, 1}, {1.05f, 1.20f, 5.5f, 1}}};
  return head_dim == 32 ? c32 : head_dim == 64 ? c64 : c128;
}

// One way to run a task: kernel, rows, parts of the keys, and what it costs
struct Way {
  Form form;
  int qn, splits;
  float us;
};
int rows_of(Form form, int qn) { return 16 * qn * (form == Form::rows ? NWAVE : 1); }
int keys_of(Form form) { return form == Form::rows ? KC : 32; }
int64_t chunks_of(const Task& t, int u) { return (int64_t)div_up(t.Np, u) + div_up(t.Nk, u); }
// (parts: the sums go through the workspace in any case)
Way way_of(const Task& t, int Hk, int head_dim, Form form, int qn, int splits, bool parts) {
  const Costs& c = costs_of(head_dim);
  const Cost& one = form == Form::rows ? c.rows[qn / 2] : c.keys[qn / 2];
  const int64_t wgs = (int64_t)t.members * Hk * div_up(t.rows, rows_of(form, qn)) * splits;
  const int64_t chunks = div_up(chunks_of(t, keys_of(form)), splits), steps = form == Form::rows ? chunks : div_up(chunks, NWAVE);
  const int rounds = div_up(wgs, 256 * one.per_cu);
  const float several = one.among * div_up(wgs, 256), step = several > one.alone ? several : one.alone;
  float us = 2.4f + rounds * one.round + steps * step;
  // reading the keys, at a rate that grows with what a CU has on its way (32 KB 5.1 TB/s, 64 KB 5.7), longer where the last round leaves part of the chip idle
  const float slots = 256.f * one.per_cu;
  const float on_way = (wgs < slots ? wgs : slots) / 256.f * (form == Form::rows ? KC : 32 * NWAVE) * head_dim * 4;
  // (members after the first find the prefix in L2, at about three times memory's rate)
  const float read = 4e-6f * Hk * head_dim * ((1.f + 0.35f * (t.members - 1)) * t.Np + (float)t.members * t.Nk) / 6.4f * (1.f + 8192.f / on_way) * (rounds > 1 ? rounds * slots / wgs : 1.f);
  us = us > read ? us : read;
  // what the parts' sums cost to write and read, and the joining kernel
  if (parts || splits > 1) us += 0.55f * 4e-6f * t.members * Hk * (float)t.rows * splits * head_dim;
  if (splits > 1 && !parts) us += 6.0f;
  return {form, qn, splits, us};
}

Plan plan_of(const CrossArgs& a) {
  const int B = (int)a.B, Hk = (int)a.kv_heads, rows_m = (int)(a.Nq * (a.heads / a.kv_heads)), D = (int)a.head_dim;
  const bool own = a.Nk > 0;
  // every member sees the same keys: its rows are further rows of one unit
  const bool shared = !own || (a.k_batch_stride == 0 && a.v_batch_stride == 0 && (!a.lengths || a.lengths_stride == 0) &&
                               (!a.key_mask || a.mask_batch_stride == 0));
  Plan plan{};
  auto add = [&](Plan& plan, bool all, int64_t Nk, int64_t Np) {
    Task& t = plan.task[plan.n++];
    t.Nk = (int)Nk;
    t.Np = (int)Np;
    t.members = all ? 1 : B;
    t.rows = all ? B * rows_m : rows_m;
    t.splits = 1;
  };
  if (B == 1 || (shared && rows_m % 128 != 0)) {
    add(plan, true, a.Nk, a.Np);
  } else {
    add(plan, false, a.Nk, a.Np);
  }
  auto setup = [&](Form form, int qn) {
    plan.form = form;
    plan.qn = qn;
    plan.grid = plan.bytes = 0;
    for (int i = 0; i < plan.n; ++i) {
      Task& t = plan.task[i];
      t.qblks = div_up(t.rows, rows_of(form, qn));
      t.units = t.splits * t.members * Hk;
      // an eighth of the units per XCD, whose L2 then holds their keys for all row blocks; all units on every XCD, one after the other, an eighth of
      // the row blocks each, where the units do not divide among the XCDs and the row blocks do better.  Heads together where there are turns enough
      // to even out lengths (two members of 1000 and 600 keys on four XCDs each: 245 -> 280 us), and as many on each XCD as one by one (528 workgroups for
      // 504, where 512 fit, cost 12 per cent; lines of 128 bytes shared by heads of 32 are worth a sixteenth more)
      const int64_t eighth = div_up(t.units, 8), together = div_up(t.units / Hk, 8) * (int64_t)Hk;
      t.together = t.units / Hk >= 64 && 16 * together <= (D == 32 ? 17 : 16) * eighth ? Hk : 1;
      const int64_t by_units = (t.together > 1 ? together : eighth) * t.qblks, by_rows = div_up(t.qblks, 8) * (int64_t)t.units;
      t.by_rows = by_rows < by_units;
      t.first = (int)plan.grid;
      plan.grid += 8 * (t.by_rows ? by_rows : by_units);
      if (plan.parts) plan.bytes += ((int64_t)t.units * t.rows * (D + 2) * 4 + 255) / 256 * 256;
    }
    if (plan.n < 2) plan.task[1].first = 0x7fffffff;
  };

  // Few keys and many rows: a workgroup's keys stay (at least two row blocks for each of its waves).  As many workgroups as run at once: two per CU, four
  // of the small ones of head size 32 (64 800 queries, sixteen heads, 77 keys: 37.1 us with 1024, 38.1 with 512; of 64: 54.5 and 50.8)
  {
    Task& t = plan.task[0];
    const int64_t c = chunks_of(t, KC), lds = c * (4 * KC * D + 8), units = (int64_t)t.members * Hk;
    const int64_t per = (D == 32 && lds <= RESIDENT_LDS / 2 ? 1024 : 512) / units, blocks = div_up(t.rows, 16 * resident_qn(D) * NWAVE);
    if (c > 0 && lds <= RESIDENT_LDS && per > 0 && blocks >= 2 * per) {
      plan.form = Form::resident;
      plan.resident = (int)c;
      t.qblks = (int)per;
      t.units = (int)units;
      plan.grid = per * units;
      return plan;
    }
  }
  // Otherwise the way that costs least (eight heads of 64, 1000 keys, in us: 8000 queries, 32 rows a wave 21.8, 64 24.6; 16 000 42.3 and 35.9, whose
  // workgroups fill the chip once; 24 000 58.8 and 58.3; 64 800 150 and 140).  Parts of the keys: what fills the chip once, twice, ..
  auto choose = [&](Plan& plan) {
    Way best{Form::rows, 1, 1, 1e30f};
    int splits[2] = {1, 1};
    const bool parts = plan.parts;
    for (int f = 0; f < 6; ++f) {
      const Form form = f < 3 ? Form::rows : Form::keys;
      const int qn = 1 << (f % 3);
      if (form == Form::rows && (parts ? qn != 2 : costs_of(D).rows[qn / 2].per_cu == 0)) continue;  // (in parts 32 rows a wave)
      float us = parts ? 6.0f : 0.f;
      int s[2] = {1, 1};
      for (int i = 0; i < plan.n; ++i) {
        const Task& t = plan.task[i];
        const int64_t one = (int64_t)t.members * Hk * div_up(t.rows, rows_of(form, qn)), chunks = chunks_of(t, keys_of(form));
        Way w = way_of(t, Hk, D, form, qn, 1, parts);
        for (int slots = 256; slots <= 1024 && !(form == Form::rows && qn != 2); slots += 256) {
          const int64_t n = slots / one < div_up(chunks, NWAVE) ? slots / one : div_up(chunks, NWAVE);
          if (n <= 1) continue;
          const Way x = way_of(t, Hk, D, form, qn, (int)n, parts);
          if (x.us < w.us) w = x;
        }
        s[i] = w.splits;
        us += w.us;
      }
      if (us < best.us) {
        best = {form, qn, 1, us};
        splits[0] = s[0];
        splits[1] = s[1];
      }
    }
    for (int i = 0; i < plan.n; ++i) {
      plan.task[i].splits = splits[i];
      plan.parts = plan.parts || splits[i] > 1;
    }
    return best;
  };
  Way best = choose(plan);
  // or the prefix once for all members, behind it their own: pays from some prefix on (16 members, a query each, 12 heads of 64, 64 keys of their own:
  // prefix of 64 4.4 us in one, 11 apart; 1000 8.8, 11.5; 4000 22, 12.4)
  if (plan.task[0].members > 1 && a.Np > 0 && own && rows_m < 128) {
    Plan apart{};
    add(apart, true, 0, a.Np);
    add(apart, false, a.Nk, 0);
    apart.parts = true;
    const Way way = choose(apart);
    if (way.us < best.us) {
      plan = apart;
      best = way;
    }
  }
  setup(best.form, best.qn);
  return plan;
}

// the kernel for (sums through the workspace, scaled here, blocks of 16 rows per wave), handed to `f` with its LDS bytes
template <int HD, class F>
hipError_t with_rows_kernel(bool parts, bool scaled, int qn, const F& f) {
  constexpr int LDS = 8 * KC * HD;
  constexpr bool SUM = HD == 32;
  if (parts) return f(cross_attention_rows_kernel<HD, NWAVE, 2, true, true, false>, LDS);
  if constexpr (HD == 64)
    if (qn == 4) return scaled ? f(cross_attention_rows_kernel<HD, NWAVE, 4, false, true, true>, LDS) : f(cross_attention_rows_kernel<HD, NWAVE, 4, false, false, true>, LDS);
  if (qn == 1) return scaled ? f(cross_attention_rows_kernel<HD, NWAVE, 1, false, true, SUM>, LDS) : f(cross_attention_rows_kernel<HD, NWAVE, 1, false, false, SUM>, LDS);
  return scaled ? f(cross_attention_rows_kernel<HD, NWAVE, 2, false, true, SUM>, LDS) : f(cross_attention_rows_kernel<HD, NWAVE, 2, false, false, SUM>, LDS);
}
// the same for (sums through the workspace, blocks of 16 rows); with the bytes that the waves' sums take in the end
template <int HD, int QN, bool PARTS, class F>
hipError_t with_keys_kernel_of(const F& f) {
  return f(cross_attention_keys_kernel<HD, NWAVE, QN, PARTS>, NWAVE * 2 * 4 * 32 * HD, NWAVE * 16 * QN * (HD + 2) * 4);
}
template <int HD, class F>
hipError_t with_keys_kernel(bool parts, int qn, const F& f) {
  if (qn == 4) return parts ? with_keys_kernel_of<HD, 4, true>(f) : with_keys_kernel_of<HD, 4, false>(f);
  if (qn == 2) return parts ? with_keys_kernel_of<HD, 2, true>(f) : with_keys_kernel_of<HD, 2, false>(f);
  return parts ? with_keys_kernel_of<HD, 1, true>(f) : with_keys_kernel_of<HD, 1, false>(f);
}
template <int HD, class F>
hipError_t with_resident_kernel(bool scaled, const F& f) {
  return scaled ? f(cross_attention_resident_kernel<HD, NWAVE, resident_qn(HD), true, HD <= 64>)
                : f(cross_attention_resident_kernel<HD, NWAVE, resident_qn(HD), false, HD <= 64>);
}

template <int HD>
hipError_t launch_dim(const CrossArgs& a, Plan& plan, void* workspace, hipStream_t stream) {
  CrossParams p{};
  p.q = (const uint16_t*)a.q; p.k = (const uint16_t*)a.k; p.v = (const uint16_t*)a.v;
  p.prefix_k = (const uint16_t*)a.prefix_k; p.prefix_v = (const uint16_t*)a.prefix_v;
  p.out = (uint16_t*)a.out;
  p.q_batch = a.q_batch_stride; p.q_row = a.q_row_stride; p.q_head = a.q_head_stride;
  p.k_batch = a.k_batch_stride; p.k_head = a.k_head_stride; p.v_batch = a.v_batch_stride; p.v_head = a.v_head_stride;
  p.prefix_k_head = a.prefix_k_head_stride; p.prefix_v_head = a.prefix_v_head_stride; p.mask_batch = a.mask_batch_stride;
  p.k_row = (uint32_t)(a.k_row_stride * 2); p.v_row = (uint32_t)(a.v_row_stride * 2);
  p.prefix_k_row = (uint32_t)(a.prefix_k_row_stride * 2); p.prefix_v_row = (uint32_t)(a.prefix_v_row_stride * 2);
  p.lengths = a.lengths; p.lengths_step = (int)a.lengths_stride; p.mask = a.key_mask;
  p.Nq = (int)a.Nq; p.heads = (int)a.heads; p.kv_heads = (int)a.kv_heads; p.group = (int)(a.heads / a.kv_heads);
  p.rows_m = p.Nq * p.group;
  p.of_group = divisor((uint32_t)p.group); p.of_rows_m = divisor((uint32_t)p.rows_m);
  // (the kernels of divided keys multiply the logits in either case: they are bound by reading the keys)
  p.q_mul = a.q_prescaled ? 1.0f : (float)(a.scale * 1.4426950408889634);

  float* at = (float*)workspace;
  for (int i = 0; i < plan.n && plan.parts; ++i) {
    Task& t = plan.task[i];
    const int64_t n = (int64_t)t.units * t.rows;
    t.o = at;
    t.ml = at + n * HD;
    at += (n * (HD + 2) * 4 + 255) / 256 * 64;
  }
  p.task[0] = plan.task[0];
  p.task[1] = plan.task[1];
  auto launch = [&](auto kernel, int64_t lds) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)plan.grid), dim3(64 * NWAVE), (uint32_t)lds, stream, p);
    return hipGetLastError();
  };
  if (plan.form == Form::resident)
    return with_resident_kernel<HD>(!a.q_prescaled, [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)plan.grid), dim3(64 * NWAVE), (uint32_t)(plan.resident * (4 * KC * HD + 8)), stream, p, plan.resident);
      return hipGetLastError();
    });
  const hipError_t e = plan.form == Form::rows ? with_rows_kernel<HD>(plan.parts, !a.q_prescaled, plan.qn, [&](auto kernel, int lds) {
    return launch(kernel, lds);
  }) : with_keys_kernel<HD>(plan.parts, plan.qn, [&](auto kernel, int64_t lds, int64_t sums) {
    return launch(kernel, lds > sums ? lds : sums);
  });
  if (e != hipSuccess || !plan.parts) return e;
  JoinParams j{};
  j.task[0] = plan.task[0];
  if (plan.n > 1) j.task[1] = plan.task[1];
  j.out = p.out; j.Nq = p.Nq; j.heads = p.heads; j.kv_heads = p.kv_heads; j.group = p.group; j.rows_m = p.rows_m;
  j.rows = a.B * a.Nq * a.heads;
  const int parts = plan.task[0].splits + plan.task[1].splits;
  if (parts <= 16) hipLaunchKernelGGL((cross_attention_join_kernel<HD, 1>), dim3((unsigned)((j.rows + 3) / 4)), dim3(256), 0, stream, j);
  else if (parts <= 64) hipLaunchKernelGGL((cross_attention_join_kernel<HD, 4>), dim3((unsigned)j.rows), dim3(256), 0, stream, j);
  else hipLaunchKernelGGL((cross_attention_join_kernel<HD, 16>), dim3((unsigned)j.rows), dim3(1024), 0, stream, j);
  return hipGetLastError();
}

template <int HD>
hipError_t configure_dim() {
  hipError_t e = hipSuccess;
  auto allow = [](auto kernel, int64_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  };
  for (int i = 0; i < 6 && e == hipSuccess; ++i) {
    const int qn = i / 2 == 2 ? 4 : 1 + i / 2;
    for (int parts = 0; parts < 2 && e == hipSuccess; ++parts)
      e = with_rows_kernel<HD>(parts, i & 1, qn, [&](auto kernel, int lds) { return allow(kernel, lds); });
    if (e == hipSuccess)
      e = with_keys_kernel<HD>(i & 1, qn, [&](auto kernel, int64_t lds, int64_t sums) { return allow(kernel, lds > sums ? lds : sums); });
  }
  for (int i = 0; i < 2 && e == hipSuccess; ++i)
    e = with_resident_kernel<HD>(i, [&](auto kernel) { return allow(kernel, RESIDENT_LDS); });
  return e;
}

}  // namespace

bool cross_attention_supported(int64_t head_dim) { return head_dim == 32 || head_dim == 64 || head_dim == 128; }

hipError_t cross_attention_configure() {
  hipError_t e = configure_dim<32>();
  if (e == hipSuccess) e = configure_dim<64>();
  if (e == hipSuccess) e = configure_dim<128>();
  return e;
}

CrossPlan cross_attention_plan(const CrossArgs& a) {
  static_assert(std::is_trivially_copyable<Plan>::value && sizeof(Plan) <= sizeof(CrossPlan::inside), "the plan travels as bytes");
  const Plan plan = plan_of(a);
  int64_t units = 0;
  for (int i = 0; i < plan.n; ++i) units += (int64_t)plan.task[i].splits * plan.task[i].members * a.kv_heads;
  const int parts = plan.task[0].splits + plan.task[1].splits;
  CrossPlan c{};
  c.workspace_bytes = plan.bytes;
  // (a grid has less than 2^32 threads; up to 1024 of them join a row)
  c.fits = units < (1 << 24) && plan.grid < (1 << 24) && (!plan.parts || a.B * a.Nq * a.heads < (parts <= 16 ? 1 << 26 : parts <= 64 ? 1 << 24 : 1 << 22));
  memcpy(c.inside, &plan, sizeof(plan));
  return c;
}

hipError_t cross_attention_launch(const CrossArgs& a, const CrossPlan& c, void* workspace, hipStream_t stream) {
  Plan plan;
  memcpy(&plan, c.inside, sizeof(plan));
  if (a.head_dim == 32) return launch_dim<32>(a, plan, workspace, stream);
  if (a.head_dim == 64) return launch_dim<64>(a, plan, workspace, stream);
  return launch_dim<128>(a, plan, workspace, stream);
}

}  // namespace aeris
