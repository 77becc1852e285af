// Attention of tokens to an encoder's states: o = softmax(scale q k^T) v over the keys that a member has (its own, up to its length and
// where its key mask lets them, behind a prefix that all members share), gfx950.
//
// One workgroup = a block of rows of one (member, key head): 32 rows a wave, a row being a query of one of the heads that share the key
// head.  The keys are streamed through LDS in chunks of 64; P = exp2(logit) is formed without a row maximum, the range of the sums is
// checked afterwards and the workgroup repeats its keys with a running maximum where it was left.
//   K, V chunk [64][HD]  global -> LDS by the load unit (buffer_load ... lds), 16-byte pieces XOR-swizzled; a key that does not take
//                        part is not read, its row arrives as zeros (whatever it held, NaN or infinity, is multiplied by nothing)
//   S^T = K Q^T          v_mfma_f32_16x16x32_bf16; lane = one row, registers = keys
//   O^T += V^T P^T       V^T by the transposing LDS read, P^T straight from the accumulators of S^T, rounded to bf16; the row sum adds the
//                        rounded values
// Few rows (`SPLIT`): a row block's chunks are divided among workgroups, each leaves its sums in the workspace in fp32 and
// cross_attention_join_kernel adds them up, in their order.
#include "common.h"
#include "kernels.h"
#include <type_traits>

namespace aeris {

namespace {

constexpr int KC = 64;  // keys per chunk

struct CrossParams {
  const uint16_t *q, *k, *v, *prefix_k, *prefix_v;
  uint16_t* out;
  int64_t q_batch, q_row, q_head, k_batch, k_head, v_batch, v_head, prefix_k_head, prefix_v_head, mask_batch;
  uint32_t k_row, v_row, prefix_k_row, prefix_v_row;  // bytes
  const int32_t* lengths;
  const uint8_t* mask;
  int lengths_step;      // 0: one length for all members
  int Nk, Np;            // own and prefix keys of this launch (0: that part is not its task)
  int Nq, heads, kv_heads, group;
  int rows, rows_m;      // rows of a unit; rows of a member (fewer where a unit holds all members')
  int members;           // units' members: 1 where a unit holds all of them
  int units, qblks, splits;
  int by_rows;           // workgroups of an XCD: all units in turn, an eighth of the row blocks (else: an eighth of the units)
  float q_mul;
  float *part_o, *part_ml;  // SPLIT: [split][member][kv head][row][HD], [..][2] = maximum, sum
};

template <int HD, int NBUF>
struct CrossCfg {
  static constexpr int BYTES = KC * HD * 2;  // of a chunk of K or of V
  static constexpr int V_BASE = NBUF * BYTES;
  static constexpr int SMEM = 2 * NBUF * BYTES + 16;
};

// 16-byte pieces of a chunk's rows.  K: the fragment reads take one piece of 16 consecutive rows; V: the 32 lanes of a pass of the transposing
// read gather two neighbouring pieces of 8 rows.  In both the 16 pieces lie on the 16 slots of a 256-byte bank period.
template <int HD>
__device__ __forceinline__ int k_swizzle(int row) { return HD == 128 ? row & 15 : HD == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }
template <int HD>
__device__ __forceinline__ int v_swizzle(int row) { return HD == 128 ? 2 * (row & 7) : HD == 64 ? 2 * ((row >> 1) & 3) : 2 * ((row >> 2) & 1); }

// Rows of 64 elements: K's swizzle exchanges pieces of a row only, as the others' do (V's too).
template <int HD>
__device__ __forceinline__ uint32_t k_off(int row, int piece) { return (uint32_t)(row * (HD * 2) + ((piece ^ k_swizzle<HD>(row)) << 4)); }

}  // namespace

template <int HD, int NWAVE, int NBUF, bool MASKED, bool SPLIT>
__global__ void __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(2)))
cross_attention_kernel(CrossParams p) {
  static_assert(NBUF == 2, "a chunk is consumed while the next one is loaded");
  using Cfg = CrossCfg<HD, NBUF>;
  constexpr int QB = 32 * NWAVE;  // rows per workgroup
  constexpr int QN = 2;           // blocks of 16 rows per wave
  constexpr int KS = HD / 32;     // k32 steps of K Q^T
  constexpr int KB = KC / 16;     // blocks of 16 keys per chunk
  constexpr int DB = HD / 16;     // 16-row blocks of O^T
  constexpr int PPR = HD / 8;     // 16-byte pieces per row
  constexpr int RPI = 64 / PPR;   // rows that one load instruction of a wave fills
  static_assert(KC % (RPI * NWAVE) == 0, "a chunk is a whole number of instructions of each wave");
  constexpr int LOADS = KC / (RPI * NWAVE);

  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const uint32_t smem_addr = lds_byte_address(smem);
  int* const redo = reinterpret_cast<int*>(smem + 2 * NBUF * Cfg::BYTES);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l15 = lane & 15, q4 = lane >> 4;

  int unit, qb;
  {
    const int xcd = blockIdx.x & 7, s = blockIdx.x >> 3;
    if (p.by_rows) {
      const int per = (p.qblks + 7) / 8;
      unit = s / per;
      qb = xcd * per + s % per;
    } else {
      unit = xcd + 8 * (s / p.qblks);
      qb = s % p.qblks;
    }
    if (unit >= p.units || qb >= p.qblks) return;
  }
  const int split = unit / (p.members * p.kv_heads);
  const int bh = unit - split * (p.members * p.kv_heads);
  const int member = bh / p.kv_heads, hk = bh - member * p.kv_heads;

  // the unit's keys: chunks of the prefix, then of the member's own
  int len = p.Nk;
  if (p.lengths && p.Nk > 0) {
    len = __builtin_amdgcn_readfirstlane(p.lengths[member * p.lengths_step]);
    len = len < 0 ? 0 : len < p.Nk ? len : p.Nk;
  }
  const int cp = (p.Np + KC - 1) / KC;
  const int chunks = cp + (len + KC - 1) / KC;
  int c0 = 0, c1 = chunks;
  if (SPLIT) {
    c0 = (int)((int64_t)chunks * split / p.splits);
    c1 = (int)((int64_t)chunks * (split + 1) / p.splits);
  }
  const int nch = c1 - c0;
  const uint16_t* const k_own = p.k + member * p.k_batch + hk * p.k_head;
  const uint16_t* const v_own = p.v + member * p.v_batch + hk * p.v_head;
  const uint16_t* const k_pre = p.prefix_k + hk * p.prefix_k_head;
  const uint16_t* const v_pre = p.prefix_v + hk * p.prefix_v_head;
  const uint8_t* const mask = MASKED ? p.mask + member * p.mask_batch : nullptr;

  if (tid == 0) *redo = 0;

  // ---- Q fragments (B operand): lane = row, 8 consecutive elements per k32 step
  bool valid[QN];
  int64_t out_row[QN];
  bf16x8 qf[QN][KS];
  const int row0 = qb * QB + wave * 32;
#pragma unroll
  for (int n = 0; n < QN; ++n) {
    int r = row0 + n * 16 + l15;
    valid[n] = r < p.rows;
    if (!valid[n]) r = p.rows - 1;
    const int bb = r / p.rows_m, rm = r - bb * p.rows_m;
    const int query = rm / p.group, head = hk * p.group + rm - query * p.group;
    const int64_t b = member + bb;
    out_row[n] = (b * p.Nq + query) * p.heads + head;
    const uint16_t* qp = p.q + b * p.q_batch + query * p.q_row + head * p.q_head + q4 * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // q times scale * log2(e), rounded to bf16 once more: the accumulators are the logits in the exp2 domain.  (q_mul is 1 where the
      // producer of q has applied the factor ahead of q's only rounding.)
      const u32x4 w = *reinterpret_cast<const u32x4*>(qp + s * 32);
      u32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = pack_bf16x2(bf16_lo(w[e]) * p.q_mul, bf16_hi(w[e]) * p.q_mul);
      qf[n][s] = __builtin_bit_cast(bf16x8, x);
    }
  }
  const bool wave_active = row0 < p.rows;  // wave-uniform: a wave without rows only loads and keeps the barriers

  // ---- loads into LDS: instruction i of the wave fills the rows RPI * (wave + NWAVE * i) .., lane = (row, slot)
  uint32_t ld_row[LOADS], ld_k[LOADS], ld_v[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = RPI * (wave + NWAVE * i) + lane / PPR, slot = lane % PPR;
    ld_row[i] = row;
    ld_k[i] = (uint32_t)((slot ^ k_swizzle<HD>(row)) << 4);
    ld_v[i] = (uint32_t)((slot ^ v_swizzle<HD>(row)) << 4);
  }
  auto valid_keys = [&](int c) {  // bit i: key i of chunk c is one of the unit's (the mask aside)
    const int n = c < cp ? p.Np - c * KC : len - (c - cp) * KC;
    return n >= KC ? ~0ull : (1ull << n) - 1;
  };
  uint32_t mask_byte = 1;  // of the next chunk to be loaded, key `lane`
  auto fetch_mask = [&](int c) {
    if (MASKED) {
      mask_byte = 1;
      if (c >= cp && c < c1) {
        const int key = (c - cp) * KC + lane;
        if (key < len) mask_byte = mask[key];
      }
    }
  };
  auto issue = [&](int c, int buf, uint64_t& keys) {
    keys = valid_keys(c);
    if (MASKED) keys &= __builtin_amdgcn_ballot_w64(mask_byte != 0);
    const bool pre = c < cp;
    const int64_t key0 = (int64_t)(pre ? c : c - cp) * KC;
    const uint32_t k_row = pre ? p.prefix_k_row : p.k_row, v_row = pre ? p.prefix_v_row : p.v_row;
    const lds_dma_rsrc rk = make_lds_dma_rsrc(reinterpret_cast<const unsigned char*>(pre ? k_pre : k_own) + key0 * k_row, 0x80000000u);
    const lds_dma_rsrc rv = make_lds_dma_rsrc(reinterpret_cast<const unsigned char*>(pre ? v_pre : v_own) + key0 * v_row, 0x80000000u);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint32_t ok = __umul24(ld_row[i], k_row) + ld_k[i], ov = __umul24(ld_row[i], v_row) + ld_v[i];
      if (keys != ~0ull && !((keys >> ld_row[i]) & 1)) ok = ov = 0xFFFFF000u;  // outside the descriptor: not read, zeros
      const uint32_t at = (uint32_t)(buf * Cfg::BYTES + (wave + NWAVE * i) * 1024);
      lds_dma_load16(rk, smem_addr + at, ok, 0);
      lds_dma_load16(rv, smem_addr + Cfg::V_BASE + at, ov, 0);
    }
    fetch_mask(c + 1);
  };

  // ---- fragment addresses: per-lane part, loop-invariant; buffer, key block and step are compile-time offsets
  typedef __attribute__((address_space(3))) const unsigned char* lds_cptr;
  uint32_t v_tr[DB];  // of the 16 lanes q4, lane 4e + a reads V[key0 + 4 q4 + e][16 db + 4a ..]
  {
    const int e = (lane >> 2) & 3, a = lane & 3, row = 4 * q4 + e;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      v_tr[db] = smem_addr + (uint32_t)(Cfg::V_BASE + row * (HD * 2) + (((2 * db + (a >> 1)) ^ v_swizzle<HD>(row)) << 4) + (a & 1) * 8);
      asm volatile("" : "+v"(v_tr[db]));
    }
  }
  lds_cptr k_lane[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    k_lane[s] = (lds_cptr)(smem + k_off<HD>(l15, 4 * s + q4));
    asm volatile("" : "+v"(k_lane[s]));
  }

  float m[QN], l[QN];
  f32x4 o[QN][DB];
  bool any = false;  // whether any key took part (uniform)

  // One pass over the keys.  FAST: P = exp2(logit); otherwise with the running maximum m, accumulated output and sum rescaled whenever a
  // maximum moves.
  auto sweep = [&](auto fast_tag) {
    constexpr bool FAST = decltype(fast_tag)::value;
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      m[n] = -3.0e38f;  // (finite: a chunk all of whose logits are -infinity leaves it where it is)
      l[n] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[n][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    uint64_t keys[NBUF];
    if (nch > 0) {
      fetch_mask(c0);
      issue(c0, 0, keys[0]);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's loads into LDS have landed
    __syncthreads();

    for (int j0 = 0; j0 < nch; j0 += NBUF) {
#pragma unroll
      for (int u = 0; u < NBUF; ++u) {
        const int j = j0 + u;
        if (j >= nch) break;
        // the next chunk is requested at the start of this one and awaited at the barrier that ends it; its buffer was last read ahead of
        // the barrier that began this one
        if (j + 1 < nch) issue(c0 + j + 1, (u + 1) & 1, keys[(u + 1) & 1]);
        const uint64_t kk = keys[u];
        if (kk != 0) any = true;
        if (wave_active && kk != 0) {
          f32x4 acc[QN][KB];
          // ---- S^T: acc[n][kb][i] = logit of key 16 kb + 4 q4 + i, row 16 n + l15; K fragments are read two ahead of their MFMAs
          {
            constexpr int PF = 2, NS = KB * KS;
            const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
            bf16x8 kfr[PF + 1];
            auto read_k = [&](int t) {
              typedef __attribute__((address_space(3))) const bf16x8* frag_ptr;
              return *(frag_ptr)(k_lane[t / KB] + u * Cfg::BYTES + (t % KB) * 16 * (HD * 2));
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
          if (kk != ~0ull) {  // keys that do not take part
            const uint64_t mine = kk >> (4 * q4);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!((mine >> (kb * 16 + i)) & 1)) {
#pragma unroll
                  for (int n = 0; n < QN; ++n) acc[n][kb][i] = -INFINITY;
                }
          }

          // PV step of 32 keys: k slots 0-3 <-> keys 32 step + 4 q4 + (0..3), slots 4-7 <-> 16 more.  The fragments of half of the row
          // blocks are read ahead of the MFMAs of the half before.
          constexpr int DH = DB / 2, PARTS = KC / 32 * 2;
          bf16x8 vfb[2][DH];
          TrFrag vtr[2][DH];
          auto load_v = [&](int part, int slot) {
#pragma unroll
            for (int d = 0; d < DH; ++d) {
              const uint32_t a0 = v_tr[(part & 1) * DH + d] + u * Cfg::BYTES + (part >> 1) * 32 * (HD * 2);
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
          load_v(0, 0);

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
              const float m_new = fmaxf(m[n], cm);
              if (__builtin_amdgcn_ballot_w64(m_new > m[n]) != 0) {
                const float alpha = __builtin_amdgcn_exp2f(m[n] - m_new);
                l[n] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[n][db] *= alpha;
                m[n] = m_new;
              }
            }
          }

          uint32_t pkb[2][QN][4];
          auto exp_step = [&](int step, int n) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const float a0 = acc[n][2 * step + (h >> 1)][2 * (h & 1)], a1 = acc[n][2 * step + (h >> 1)][2 * (h & 1) + 1];
              const float e0 = __builtin_amdgcn_exp2f(FAST ? a0 : a0 - m[n]);
              const float e1 = __builtin_amdgcn_exp2f(FAST ? a1 : a1 - m[n]);
              pkb[step & 1][n][h] = pack_bf16x2(e0, e1);
              l[n] = dot2_ones(pkb[step & 1][n][h], l[n]);
            }
          };
#pragma unroll
          for (int n = 0; n < QN; ++n) exp_step(0, n);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const int step = part >> 1;
            __builtin_amdgcn_sched_barrier(0);
            v_ready(part & 1);
            if (part + 1 < PARTS) load_v(part + 1, (part + 1) & 1);
            if (step + 1 < KC / 32) exp_step(step + 1, part & 1);
#pragma unroll
            for (int d = 0; d < DH; ++d)
#pragma unroll
              for (int n = 0; n < QN; ++n) {
                const bf16x8 pf = __builtin_bit_cast(bf16x8, u32x4{pkb[step & 1][n][0], pkb[step & 1][n][1], pkb[step & 1][n][2], pkb[step & 1][n][3]});
                f32x4& od = o[n][(part & 1) * DH + d];
                od = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vfb[part & 1][d], pf, od, 0, 0, 0);
              }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next chunk, requested at the start of this one
        __syncthreads();
      }
    }
  };

  sweep(std::true_type{});
  bool online = false;
  {
    bool bad = false;
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      float lt = l[n] + __shfl_xor(l[n], 16, 64);
      lt += __shfl_xor(lt, 32, 64);
      bad = bad || !(lt >= 0x1p-40f && lt <= 0x1p100f);
    }
    if (any && wave_active && __builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) *redo = 1;
    __syncthreads();
    online = __builtin_amdgcn_readfirstlane(*redo) != 0;
    if (online) sweep(std::false_type{});
  }

#pragma unroll
  for (int n = 0; n < QN; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] += __shfl_xor(l[n], 32, 64);
    if (SPLIT) {
      const int64_t at = ((int64_t)split * p.members * p.kv_heads + bh) * p.rows + row0 + n * 16 + l15;
      if (valid[n] && q4 == 0) {
        p.part_ml[2 * at] = online ? m[n] : 0.f;
        p.part_ml[2 * at + 1] = l[n];
      }
#pragma unroll
      for (int db = 0; db < DB; ++db)
        if (valid[n]) *reinterpret_cast<f32x4*>(p.part_o + at * HD + 16 * db + 4 * q4) = o[n][db];
      continue;
    }
    // normalise; a row without any key is zeros
    const float inv = l[n] == 0.f ? 0.f : __builtin_amdgcn_rcpf(l[n]);
    uint16_t* op = p.out + out_row[n] * HD + 16 * (q4 & 1) + 8 * (q4 >> 1);
#pragma unroll
    for (int m2 = 0; m2 < DB / 2; ++m2) {  // 8 consecutive elements a lane
      const f32x4 a = o[n][2 * m2] * inv, c = o[n][2 * m2 + 1] * inv;
      const auto rx = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[0], a[1]), pack_bf16x2(c[0], c[1]), false, false);
      const auto ry = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[2], a[3]), pack_bf16x2(c[2], c[3]), false, false);
      if (valid[n]) *reinterpret_cast<u32x4*>(op + m2 * 32) = u32x4{rx[0], ry[0], rx[1], ry[1]};
    }
  }
}

// ---------------------------------------------------------------------------------------------

namespace {

// One row's parts, up to two sets of them (of the prefix, whose rows are those of all members; of the member's own keys)
struct JoinParams {
  const float *o[2], *ml[2];
  int splits[2], rows[2], members[2];
  uint16_t* out;
  int Nq, heads, kv_heads, group, rows_m;
};

}  // namespace

// out[row] = sum over the parts of 2^(m - max m) o / sum of 2^(m - max m) l.  A thread has 4 elements and every SPth part.
template <int HD>
__global__ void __launch_bounds__(256) cross_attention_join_kernel(JoinParams p) {
  constexpr int CT = HD / 4, SP = 256 / CT;
  __shared__ f32x4 so[SP][CT];
  __shared__ float sm[SP], sl[SP];
  const int c = threadIdx.x % CT, sp = threadIdx.x / CT;
  const int64_t row = blockIdx.x;  // (member, query, head)
  const int head = (int)(row % p.heads);
  const int64_t bq = row / p.heads;
  const int query = (int)(bq % p.Nq), b = (int)(bq / p.Nq);
  const int hk = head / p.group, rm = query * p.group + head - hk * p.group;
  float m = -3.0e38f, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int set = 0; set < 2; ++set) {
    const bool all = p.members[set] == 1;  // a unit's rows are those of all members
    const int64_t first = ((int64_t)(all ? 0 : b) * p.kv_heads + hk) * p.rows[set] + (all ? b * p.rows_m : 0) + rm;
    const int64_t step = (int64_t)p.members[set] * p.kv_heads * p.rows[set];
    for (int s = sp; s < p.splits[set]; s += SP) {
      const int64_t at = first + s * step;
      const float pm = p.ml[set][2 * at], pl = p.ml[set][2 * at + 1];
      if (pl == 0.f) continue;  // no key of this part: its output was never written
      const f32x4 po = *reinterpret_cast<const f32x4*>(p.o[set] + at * HD + 4 * c);
      const float mn = fmaxf(m, pm), a0 = __builtin_amdgcn_exp2f(m - mn), a1 = __builtin_amdgcn_exp2f(pm - mn);
      o = o * a0 + po * a1;
      l = l * a0 + pl * a1;
      m = mn;
    }
  }
  so[sp][c] = o;
  if (c == 0) {
    sm[sp] = m;
    sl[sp] = l;
  }
  __syncthreads();
  if (sp == 0) {
    float mx = sm[0];
    for (int s = 1; s < SP; ++s) mx = fmaxf(mx, sm[s]);
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
    for (int s = 0; s < SP; ++s) {
      const float a = __builtin_amdgcn_exp2f(sm[s] - mx);
      o += so[s][c] * a;
      l += sl[s] * a;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<u32x2*>(p.out + row * HD + 4 * c) = u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  }
}

// ---------------------------------------------------------------------------------------------

namespace {

constexpr int NWAVE = 4, NBUF = 2, QB = 32 * NWAVE;

// What one launch computes: rows of units, keys, parts
struct Task {
  bool all;      // a unit holds the rows of all members (whose keys are the same)
  int Nk, Np;    // keys of a unit at most: own, prefix
  int members, rows, qblks, splits;
  int64_t chunks() const { return (int64_t)(Np + KC - 1) / KC + (Nk + KC - 1) / KC; }
};
struct Plan {
  Task task[2];
  int n;
  bool split;
  int64_t bytes;
};

Plan plan_of(const aeris_cross_attention& a) {
  const int B = (int)a.B, rows_m = (int)(a.Nq * (a.heads / a.kv_heads));
  const bool own = a.Nk > 0;
  // every member sees the same keys: its rows are further rows of one unit
  const bool shared = !own || (a.k_batch_stride == 0 && a.v_batch_stride == 0 && (!a.lengths || a.lengths_stride == 0) &&
                               (!a.key_mask || a.mask_batch_stride == 0));
  Plan plan{};
  auto add = [&](bool all, int Nk, int Np) {
    Task& t = plan.task[plan.n++];
    t.all = all;
    t.Nk = Nk;
    t.Np = Np;
    t.members = all ? 1 : B;
    t.rows = all ? B * rows_m : rows_m;
    t.qblks = (t.rows + QB - 1) / QB;
    t.splits = 1;
  };
  if (B == 1 || (shared && rows_m % QB != 0)) {
    add(B > 1, (int)a.Nk, (int)a.Np);
  } else if (a.Np > 0 && own && rows_m < QB) {
    add(true, 0, (int)a.Np);
    add(false, (int)a.Nk, 0);
    plan.split = true;
  } else {
    add(false, (int)a.Nk, (int)a.Np);
  }
  for (int i = 0; i < plan.n; ++i) {
    Task& t = plan.task[i];
    const int64_t wgs = (int64_t)t.members * a.kv_heads * t.qblks;
    // two workgroups per CU; four chunks at least are worth a workgroup of their own
    int64_t s = 512 / wgs, most = t.chunks() / 4;
    if (s > most) s = most;
    t.splits = s < 1 ? 1 : (int)s;
    if (t.splits > 1) plan.split = true;
  }
  if (plan.split)
    for (int i = 0; i < plan.n; ++i) {
      const Task& t = plan.task[i];
      plan.bytes += (int64_t)t.splits * t.members * a.kv_heads * t.rows * (a.head_dim + 2) * 4;
      plan.bytes = (plan.bytes + 255) / 256 * 256;
    }
  return plan;
}

template <int HD, bool MASKED, bool SPLIT>
hipError_t launch_task(const CrossParams& p, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((cross_attention_kernel<HD, NWAVE, NBUF, MASKED, SPLIT>), dim3((unsigned)grid), dim3(64 * NWAVE), (CrossCfg<HD, NBUF>::SMEM),
                     stream, p);
  return hipGetLastError();
}

template <int HD>
hipError_t launch_dim(const aeris_cross_attention& a, const Plan& plan, void* workspace, hipStream_t stream) {
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
  p.q_mul = a.q_prescaled ? 1.0f : (float)(a.scale * 1.4426950408889634);

  JoinParams j{};
  float* at = (float*)workspace;
  for (int i = 0; i < plan.n; ++i) {
    const Task& t = plan.task[i];
    p.Nk = t.Nk; p.Np = t.Np; p.rows = t.rows; p.members = t.members; p.qblks = t.qblks; p.splits = t.splits;
    p.units = t.splits * t.members * p.kv_heads;
    // an eighth of the units per XCD, whose L2 then holds their keys for all row blocks; all units on every XCD, one after the other, an
    // eighth of the row blocks each, where the units do not divide among the XCDs and the row blocks do better
    const int64_t by_units = (p.units + 7) / 8 * (int64_t)p.qblks, by_rows = (p.qblks + 7) / 8 * (int64_t)p.units;
    p.by_rows = by_rows < by_units;
    const int64_t grid = 8 * (p.by_rows ? by_rows : by_units);
    if (plan.split) {
      const int64_t n = (int64_t)p.units * t.rows;
      p.part_o = at;
      p.part_ml = at + n * HD;
      at += (n * (HD + 2) * 4 + 255) / 256 * 64;
      j.o[i] = p.part_o; j.ml[i] = p.part_ml; j.splits[i] = t.splits; j.rows[i] = t.rows; j.members[i] = t.members;
    }
    const bool masked = p.mask && p.Nk > 0;
    hipError_t e = plan.split ? (masked ? launch_task<HD, true, true>(p, grid, stream) : launch_task<HD, false, true>(p, grid, stream))
                              : (masked ? launch_task<HD, true, false>(p, grid, stream) : launch_task<HD, false, false>(p, grid, stream));
    if (e != hipSuccess) return e;
  }
  if (plan.split) {
    j.out = p.out; j.Nq = p.Nq; j.heads = p.heads; j.kv_heads = p.kv_heads; j.group = p.group; j.rows_m = p.rows_m;
    hipLaunchKernelGGL((cross_attention_join_kernel<HD>), dim3((unsigned)(a.B * a.Nq * a.heads)), dim3(256), 0, stream, j);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <int HD>
hipError_t configure_dim() {
  const int n = CrossCfg<HD, NBUF>::SMEM;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(cross_attention_kernel<HD, NWAVE, NBUF, false, false>), hipFuncAttributeMaxDynamicSharedMemorySize, n);
  if (e == hipSuccess) e = hipFuncSetAttribute(reinterpret_cast<const void*>(cross_attention_kernel<HD, NWAVE, NBUF, false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, n);
  if (e == hipSuccess) e = hipFuncSetAttribute(reinterpret_cast<const void*>(cross_attention_kernel<HD, NWAVE, NBUF, true, false>), hipFuncAttributeMaxDynamicSharedMemorySize, n);
  if (e == hipSuccess) e = hipFuncSetAttribute(reinterpret_cast<const void*>(cross_attention_kernel<HD, NWAVE, NBUF, true, true>), hipFuncAttributeMaxDynamicSharedMemorySize, n);
  return e;
}

}  // namespace

bool cross_attention_supported(int head_dim) { return head_dim == 32 || head_dim == 64 || head_dim == 128; }

hipError_t cross_attention_configure() {
  hipError_t e = configure_dim<32>();
  if (e == hipSuccess) e = configure_dim<64>();
  if (e == hipSuccess) e = configure_dim<128>();
  return e;
}

int64_t cross_attention_workspace_bytes(const aeris_cross_attention& a) { return plan_of(a).bytes; }

hipError_t cross_attention_launch(const aeris_cross_attention& a, void* workspace, hipStream_t stream) {
  const Plan plan = plan_of(a);
  if (a.head_dim == 32) return launch_dim<32>(a, plan, workspace, stream);
  if (a.head_dim == 64) return launch_dim<64>(a, plan, workspace, stream);
  return launch_dim<128>(a, plan, workspace, stream);
}

}  // namespace aeris
