// Attention of tokens to an encoder's states: o = softmax(scale q k^T) v over the keys that a member has (its own, up to its length and
// where its key mask lets them, behind a prefix that all members share), gfx950.
//
// A unit is one member's key head (or, where all members see the same keys, the key head with the rows of all of them); its rows are
// the queries of the heads that share the key head, 16 QN a wave.  Keys go through LDS in chunks of 64; P = exp2(logit) is formed
// without a row maximum - softmax does not depend on the subtracted constant, the maximum only guards the range -, the range of the sums is
// checked afterwards and the rows are done again with a running maximum where it was left.
//   K, V chunk [64][HD]  global -> LDS by the load unit (buffer_load ... lds), 16-byte pieces XOR-swizzled; a key that does not take
//                        part is not read, its row arrives as zeros (whatever it held, NaN or infinity, is multiplied by nothing)
//   S^T = K Q^T          v_mfma_f32_16x16x32_bf16; lane = one row, registers = keys; the scale, unless the producer of q has applied it (`SCALED`),
//                        multiplies the fp32 logits: q is not rounded again
//   O^T += V^T P^T       V^T by the transposing LDS read, P^T straight from the accumulators of S^T, rounded to bf16; the row sum adds the
//                        rounded values
// Three ways to run that:
//   cross_attention_kernel<.., SPLIT = false>  a workgroup = a block of a unit's rows, the unit's keys streamed past it
//   cross_attention_kernel<.., SPLIT = true>   few rows: the chunks divided among workgroups, each leaves its sums in the workspace in fp32 and
//                                              cross_attention_join_kernel adds them up, in their order
//   cross_attention_resident_kernel            few keys and many rows: a workgroup keeps the unit's keys in LDS and walks down the rows
#include "common.h"
#include "kernels.h"
#include <type_traits>

namespace aeris {

namespace {

constexpr int KC = 64;           // keys per chunk
constexpr int MAX_WORDS = 1024;  // chunks of a workgroup that a key mask can cover (a word of 64 bits each, in LDS)

// What a launch does: rows of units against keys
struct Task {
  int Nk, Np;        // own and prefix keys at most (0: that part is not its task)
  int members;       // units' members: 1 where a unit holds the rows of all of them
  int rows;          // of a unit
  int qblks, splits; // workgroups of a unit: row blocks, parts of the keys
  int units;         // splits * members * key heads
  int by_rows;       // workgroups of an XCD: all units in turn, an eighth of the row blocks (else: an eighth of the units)
  int first;         // its first workgroup
  float *o, *ml;     // SPLIT: [split][member][key head][row][HD], [..][2] = maximum, sum
};

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
__device__ __forceinline__ uint64_t first_keys(int n) { return n >= KC ? ~0ull : (1ull << n) - 1; }

// A wave's 16 QN rows: queries, sums, and what a chunk in LDS does to them.
template <int HD, int QN, bool SCALED>
struct Rows {
  static constexpr int KS = HD / 32;  // k32 steps of K Q^T
  static constexpr int KB = KC / 16;  // blocks of 16 keys per chunk
  static constexpr int DB = HD / 16;  // 16-row blocks of O^T
  typedef __attribute__((address_space(3))) const unsigned char* lds_cptr;

  bf16x8 qf[QN][KS];  // B operand: lane = row, 8 consecutive elements per k32 step
  bool valid[QN];
  int64_t out_row[QN];
  float m[QN], l[QN];
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

  __device__ __forceinline__ void load_q(const CrossParams& p, int rows, int member, int hk, int row0, int lane, bf16x8 (&f)[QN][KS]) {
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      int r = row0 + n * 16 + (lane & 15);
      valid[n] = r < rows;
      if (!valid[n]) r = rows - 1;
      const int bb = r / p.rows_m, rm = r - bb * p.rows_m;
      const int query = rm / p.group, head = hk * p.group + rm - query * p.group;
      const int64_t b = member + bb;
      out_row[n] = (b * p.Nq + query) * p.heads + head;
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
#pragma unroll
      for (int db = 0; db < DB; ++db) o[n][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // The chunk `at` bytes behind the first; bit i of `keys`: key i takes part (at least one).  FAST: P = exp2(logit); otherwise with the running maximum
  // m, accumulated output and sum rescaled whenever a maximum moves.
  template <bool FAST>
  __device__ __forceinline__ void chunk(uint32_t at, uint64_t keys) {
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
    if (keys != ~0ull) {  // keys that do not take part
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
        if (SCALED) cm *= q_mul;
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
    auto p_of = [&](float a, int n) {
      return __builtin_amdgcn_exp2f(SCALED ? (FAST ? a * q_mul : fmaf(a, q_mul, -m[n])) : FAST ? a : a - m[n]);
    };
    auto exp_step = [&](int step, int n) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const f32x4& a = acc[n][2 * step + (h >> 1)];
        pkb[step & 1][n][h] = pack_bf16x2(p_of(a[2 * (h & 1)], n), p_of(a[2 * (h & 1) + 1], n));
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
          od = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vfb[part & 1][d], pf, od, 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // the sums over a row's four lanes; whether any row's left the range in which exp2 needs no maximum (or is not a number)
  __device__ __forceinline__ bool out_of_range() {
    bool bad = false;
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      l[n] += __shfl_xor(l[n], 16, 64);
      l[n] += __shfl_xor(l[n], 32, 64);
      bad = bad || !(l[n] >= 0x1p-40f && l[n] <= 0x1p100f);
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
  }

  // normalise (a row without any key is zeros), 8 consecutive elements a lane and store
  __device__ __forceinline__ void store(uint16_t* out) const {
#pragma unroll
    for (int n = 0; n < QN; ++n) {
      const float inv = l[n] == 0.f ? 0.f : __builtin_amdgcn_rcpf(l[n]);
      uint16_t* op = out + out_row[n] * HD + 16 * (q4 & 1) + 8 * (q4 >> 1);
#pragma unroll
      for (int m2 = 0; m2 < DB / 2; ++m2) {
        const f32x4 a = o[n][2 * m2] * inv, c = o[n][2 * m2 + 1] * inv;
        const auto rx = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[0], a[1]), pack_bf16x2(c[0], c[1]), false, false);
        const auto ry = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[2], a[3]), pack_bf16x2(c[2], c[3]), false, false);
        if (valid[n]) *reinterpret_cast<u32x4*>(op + m2 * 32) = u32x4{rx[0], ry[0], rx[1], ry[1]};
      }
    }
  }
};

// A unit's keys, chunk by chunk: the prefix, then the member's own.
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
    prefix_chunks = (t.Np + KC - 1) / KC;
    chunks = prefix_chunks + (own + KC - 1) / KC;
    k_own = reinterpret_cast<const unsigned char*>(p.k + member * p.k_batch + hk * p.k_head);
    v_own = reinterpret_cast<const unsigned char*>(p.v + member * p.v_batch + hk * p.v_head);
  }
  __device__ __forceinline__ void seek(const CrossParams& p, const Task& t, int hk, int c) {
    if (c < prefix_chunks) {
      k_row = p.prefix_k_row;
      v_row = p.prefix_v_row;
      k = reinterpret_cast<const unsigned char*>(p.prefix_k + hk * p.prefix_k_head) + (int64_t)c * KC * k_row;
      v = reinterpret_cast<const unsigned char*>(p.prefix_v + hk * p.prefix_v_head) + (int64_t)c * KC * v_row;
      left = t.Np - c * KC;
    } else {
      c -= prefix_chunks;
      k_row = p.k_row;
      v_row = p.v_row;
      k = k_own + (int64_t)c * KC * k_row;
      v = v_own + (int64_t)c * KC * v_row;
      left = own - c * KC;
    }
  }
};

// Loads of a chunk into LDS: instruction i of wave w fills the rows RPI * (w + NWAVE * i) .., lane = (row, 16-byte slot).
template <int HD, int NWAVE>
struct Loader {
  static constexpr int BYTES = KC * HD * 2;  // of a chunk of K or of V
  static constexpr int PPR = HD / 8;         // 16-byte pieces per row
  static constexpr int RPI = 64 / PPR;       // rows that one load instruction of a wave fills
  static constexpr int LOADS = KC / (RPI * NWAVE);
  static_assert(KC % (RPI * NWAVE) == 0, "a chunk is a whole number of instructions of each wave");
  int row0, wave;               // the lane's row of instruction 0
  uint32_t off_k[LOADS], off_v[LOADS];

  __device__ __forceinline__ Loader(int lane, int w) : row0(RPI * w + lane / PPR), wave(w) {}
  __device__ __forceinline__ void rows(int lane, const Keys& keys) {  // where the lane's pieces lie in a chunk, for the rows' present strides
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = row0 + RPI * NWAVE * i, slot = lane % PPR;
      off_k[i] = __umul24(row, keys.k_row) + (uint32_t)((slot ^ k_swizzle<HD>(row)) << 4);
      off_v[i] = __umul24(row, keys.v_row) + (uint32_t)((slot ^ v_swizzle<HD>(row)) << 4);
    }
  }
  // the chunk that `keys` stands at, into LDS at k_lds and v_lds; then on to the next one.  Bit i of `word`: key i takes part.
  __device__ __forceinline__ void issue(const CrossParams& p, const Task& t, int hk, int lane, Keys& keys, int c, uint64_t word, uint32_t k_lds,
                                        uint32_t v_lds) {
    const lds_dma_rsrc rk = make_lds_dma_rsrc(keys.k, 0x80000000u), rv = make_lds_dma_rsrc(keys.v, 0x80000000u);
    if (word == ~0ull) {
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
    if (c + 1 == keys.prefix_chunks) {
      keys.seek(p, t, hk, c + 1);
      rows(lane, keys);
    } else {
      keys.k += (int64_t)KC * keys.k_row;
      keys.v += (int64_t)KC * keys.v_row;
      keys.left -= KC;
    }
  }
};

// The key mask of a workgroup's chunks c0 .. c1 as words of 64 bits in LDS (of the prefix: all ones)
template <int NWAVE>
__device__ __forceinline__ void mask_words(const uint8_t* mask, const Keys& keys, int c0, int c1, uint64_t* words, int lane, int wave) {
  for (int c = c0 + wave; c < c1; c += NWAVE) {
    const int key = (c - keys.prefix_chunks) * KC + lane;
    const bool on = key < 0 || (key < keys.own && mask[key < keys.own ? key : 0] != 0);
    const uint64_t word = c < keys.prefix_chunks ? ~0ull : __builtin_amdgcn_ballot_w64(on);
    if (lane == 0) words[c - c0] = word;
  }
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}

template <int N>
__device__ __forceinline__ void wait_loads_and_barrier() {  // all but the wave's N youngest loads have landed, and so they have in every wave
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace

template <int HD, int NWAVE, int NBUF, int QN, bool SPLIT, bool SCALED>
__global__ void __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(2)))
cross_attention_kernel(CrossParams p) {
  using Load = Loader<HD, NWAVE>;
  constexpr int BYTES = Load::BYTES, V_BASE = NBUF * BYTES;
  constexpr int QW = 16 * QN, QB = QW * NWAVE;  // rows per wave and workgroup
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  uint64_t* const words = reinterpret_cast<uint64_t*>(smem + 2 * NBUF * BYTES);
  const uint32_t smem_addr = lds_byte_address(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const Task& t = p.task[SPLIT && (int)blockIdx.x >= p.task[1].first ? 1 : 0];
  int unit, qb;
  {
    const int at = blockIdx.x - t.first, xcd = at & 7, s = at >> 3;  // (a task's first workgroup is a multiple of 8)
    if (t.by_rows) {
      const int per = (t.qblks + 7) / 8;
      unit = s / per;
      qb = xcd * per + s % per;
    } else {
      unit = xcd + 8 * (s / t.qblks);
      qb = s % t.qblks;
    }
    if (unit >= t.units || qb >= t.qblks) return;
  }
  const int split = unit / (t.members * p.kv_heads);
  const int bh = unit - split * (t.members * p.kv_heads);
  const int member = bh / p.kv_heads, hk = bh - member * p.kv_heads;
  Keys keys(p, t, member, hk);
  int c0 = 0, c1 = keys.chunks;
  if (SPLIT) {
    c0 = (int)((int64_t)keys.chunks * split / t.splits);
    c1 = (int)((int64_t)keys.chunks * (split + 1) / t.splits);
  }
  const int nch = c1 - c0;

  const int row0 = qb * QB + wave * QW;
  const bool wave_active = row0 < t.rows;  // wave-uniform: a wave without rows only loads and keeps the barriers
  Rows<HD, QN, SCALED> rows(smem, V_BASE, lane, p.q_mul);
  Load load(lane, wave);

  const bool masked = p.mask && t.Nk > 0;
  if (masked) {
    mask_words<NWAVE>(p.mask + member * p.mask_batch, keys, c0, c1, words, lane, wave);
    __syncthreads();
  }
  auto word_of = [&](int j) {  // of chunk c0 + j, which `keys` stands at
    uint64_t w = first_keys(keys.left);
    if (masked) w &= uniform64(words[j]);
    return w;
  };
  uint64_t kk[NBUF];  // of the chunks in the buffers
  auto issue = [&](int j, int buf) {
    kk[buf] = word_of(j);
    load.issue(p, t, hk, lane, keys, c0 + j, kk[buf], smem_addr + buf * BYTES, smem_addr + V_BASE + buf * BYTES);
  };
  bool any = false;  // whether any key took part (uniform)

  auto sweep = [&](auto fast_tag) {
    constexpr bool FAST = decltype(fast_tag)::value;
    keys.seek(p, t, hk, c0);
    load.rows(lane, keys);
#pragma unroll
    for (int u = 0; u < NBUF - 1; ++u)
      if (u < nch) issue(u, u);
    if (FAST) rows.load_q(p, t.rows, member, hk, row0, lane, rows.qf);  // (behind the first chunks' loads, which take longer)
    rows.reset();
    // vmcnt(0), in a form that the compiler takes into account: a wait of its own for the queries inside the loop would be one for all chunks
    if (FAST) __builtin_amdgcn_s_waitcnt(0x0F70);
    for (int j0 = 0; j0 < nch; j0 += NBUF) {
#pragma unroll
      for (int u = 0; u < NBUF; ++u) {
        const int j = j0 + u;
        if (j >= nch) break;
        // chunk j has landed; younger ones, up to NBUF - 2 of them, may be on their way.  The barrier says so for every wave's part of it, and
        // that every wave is done with chunk j - 1, whose buffer chunk j + NBUF - 1 goes to
        if (NBUF > 2 && j + NBUF - 2 < nch) wait_loads_and_barrier<(NBUF - 2) * 2 * Load::LOADS>();
        else wait_loads_and_barrier<0>();
        if (j + NBUF - 1 < nch) issue(j + NBUF - 1, (u + NBUF - 1) % NBUF);
        if (kk[u] != 0) {
          any = true;
          if (wave_active) rows.template chunk<FAST>(u * BYTES, kk[u]);
        }
      }
    }
  };
  sweep(std::true_type{});
  bool online = false;
  {
    __syncthreads();  // every wave is done with the chunks: a flag in their place
    int* const redo = reinterpret_cast<int*>(smem);
    if (tid == 0) *redo = 0;
    __syncthreads();
    if (rows.out_of_range() && any && wave_active && lane == 0) *redo = 1;
    __syncthreads();
    online = __builtin_amdgcn_readfirstlane(*redo) != 0;
    if (online) {
      __syncthreads();
      sweep(std::false_type{});
      rows.out_of_range();
    }
  }
  if (!SPLIT) {
    rows.store(p.out);
    return;
  }
#pragma unroll
  for (int n = 0; n < QN; ++n) {
    const int64_t at = ((int64_t)split * t.members * p.kv_heads + bh) * t.rows + row0 + n * 16 + (lane & 15);
    if (!rows.valid[n]) continue;
    if (rows.q4 == 0) {
      t.ml[2 * at] = online ? rows.m[n] : 0.f;
      t.ml[2 * at + 1] = rows.l[n];
    }
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) *reinterpret_cast<f32x4*>(t.o + at * HD + 16 * db + 4 * rows.q4) = rows.o[n][db];
  }
}

// ---------------------------------------------------------------------------------------------

namespace {

// One row's parts, up to two sets of them (of the prefix, whose rows are those of all members; of the member's own keys)
struct JoinParams {
  Task task[2];
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
    const Task& t = p.task[set];
    const bool all = t.members == 1;  // a unit's rows are those of all members
    const int64_t first = ((int64_t)(all ? 0 : b) * p.kv_heads + hk) * t.rows + (all ? b * p.rows_m : 0) + rm;
    const int64_t step = (int64_t)t.members * p.kv_heads * t.rows;
    for (int s = sp; s < t.splits; s += SP) {
      const int64_t at = first + s * step;
      const float pm = t.ml[2 * at], pl = t.ml[2 * at + 1];
      const f32x4 po = *reinterpret_cast<const f32x4*>(t.o + at * HD + 4 * c);
      if (pl == 0.f) continue;  // no key of this part
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

constexpr int NWAVE = 4;
constexpr int STREAM_BUF = 2, SPLIT_BUF = 4;

struct Plan {
  Task task[2];
  int n, qn;
  bool split;
  int64_t grid, words, bytes;  // workgroups; mask words of a workgroup; of the workspace
};

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

Plan plan_of(const aeris_cross_attention& a) {
  const int B = (int)a.B, Hk = (int)a.kv_heads, rows_m = (int)(a.Nq * (a.heads / a.kv_heads));
  const bool own = a.Nk > 0, masked = a.key_mask && own;
  // every member sees the same keys: its rows are further rows of one unit
  const bool shared = !own || (a.k_batch_stride == 0 && a.v_batch_stride == 0 && (!a.lengths || a.lengths_stride == 0) &&
                               (!a.key_mask || a.mask_batch_stride == 0));
  Plan plan{};
  auto add = [&](bool all, int64_t Nk, int64_t Np) {
    Task& t = plan.task[plan.n++];
    t.Nk = (int)Nk;
    t.Np = (int)Np;
    t.members = all ? 1 : B;
    t.rows = all ? B * rows_m : rows_m;
    t.splits = 1;
  };
  if (B == 1 || (shared && rows_m % 128 != 0)) {
    add(true, a.Nk, a.Np);
  } else if (a.Np > 0 && own && rows_m < 128) {
    add(true, 0, a.Np);
    add(false, a.Nk, 0);
    plan.split = true;
  } else {
    add(false, a.Nk, a.Np);
  }
  auto chunks = [](const Task& t) { return (int64_t)div_up(t.Np, KC) + div_up(t.Nk, KC); };
  // Parts of the keys: two workgroups per CU, four chunks at least are worth a workgroup of their own; and no more than a mask's words cover
  plan.qn = 2;
  for (int i = 0; i < plan.n; ++i) {
    Task& t = plan.task[i];
    const int64_t wgs = (int64_t)t.members * Hk * div_up(t.rows, 64 * plan.qn);
    int64_t s = 512 / wgs;
    if (s > chunks(t) / 4) s = chunks(t) / 4;
    if (masked && t.Nk > 0 && s * MAX_WORDS < chunks(t)) s = div_up(chunks(t), MAX_WORDS);
    t.splits = s < 1 ? 1 : (int)s;
    if (t.splits > 1) plan.split = true;
  }
  if (plan.split) {
    plan.qn = 1;
    for (int i = 0; i < plan.n; ++i)
      if (plan.task[i].rows > 64) plan.qn = 2;
  }
  for (int i = 0; i < plan.n; ++i) {
    Task& t = plan.task[i];
    t.qblks = div_up(t.rows, 64 * plan.qn);
    t.units = t.splits * t.members * Hk;
    // an eighth of the units per XCD, whose L2 then holds their keys for all row blocks; all units on every XCD, one after the other, an
    // eighth of the row blocks each, where the units do not divide among the XCDs and the row blocks do better
    const int64_t by_units = div_up(t.units, 8) * (int64_t)t.qblks, by_rows = div_up(t.qblks, 8) * (int64_t)t.units;
    t.by_rows = by_rows < by_units;
    t.first = (int)plan.grid;
    plan.grid += 8 * (t.by_rows ? by_rows : by_units);
    if (masked && t.Nk > 0 && div_up(chunks(t), t.splits) > plan.words) plan.words = div_up(chunks(t), t.splits);
    if (plan.split) plan.bytes += ((int64_t)t.units * t.rows * (a.head_dim + 2) * 4 + 255) / 256 * 256;
  }
  if (plan.n < 2) plan.task[1].first = 0x7fffffff;
  return plan;
}

// the kernel for (parts of the keys, scaled here, blocks of 16 rows per wave), handed to `f` with its LDS bytes
template <int HD, class F>
hipError_t with_kernel(bool split, bool scaled, int qn, const F& f) {
  constexpr int CH = 2 * KC * HD * 2;
  if (split)
    return qn == 1 ? f(cross_attention_kernel<HD, NWAVE, SPLIT_BUF, 1, true, true>, SPLIT_BUF * CH)
                   : f(cross_attention_kernel<HD, NWAVE, SPLIT_BUF, 2, true, true>, SPLIT_BUF * CH);
  return scaled ? f(cross_attention_kernel<HD, NWAVE, STREAM_BUF, 2, false, true>, STREAM_BUF * CH)
                : f(cross_attention_kernel<HD, NWAVE, STREAM_BUF, 2, false, false>, STREAM_BUF * CH);
}

template <int HD>
hipError_t launch_dim(const aeris_cross_attention& a, Plan& plan, void* workspace, hipStream_t stream) {
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
  // (the kernels of divided keys multiply the logits in either case: they are bound by reading the keys)
  p.q_mul = a.q_prescaled ? 1.0f : (float)(a.scale * 1.4426950408889634);

  float* at = (float*)workspace;
  for (int i = 0; i < plan.n && plan.split; ++i) {
    Task& t = plan.task[i];
    const int64_t n = (int64_t)t.units * t.rows;
    t.o = at;
    t.ml = at + n * HD;
    at += (n * (HD + 2) * 4 + 255) / 256 * 64;
  }
  p.task[0] = plan.task[0];
  p.task[1] = plan.task[1];
  const hipError_t e = with_kernel<HD>(plan.split, !a.q_prescaled, plan.qn, [&](auto kernel, int lds) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)plan.grid), dim3(64 * NWAVE), (uint32_t)(lds + plan.words * 8), stream, p);
    return hipGetLastError();
  });
  if (e != hipSuccess || !plan.split) return e;
  JoinParams j{};
  j.task[0] = plan.task[0];
  if (plan.n > 1) j.task[1] = plan.task[1];
  j.out = p.out; j.Nq = p.Nq; j.heads = p.heads; j.kv_heads = p.kv_heads; j.group = p.group; j.rows_m = p.rows_m;
  hipLaunchKernelGGL((cross_attention_join_kernel<HD>), dim3((unsigned)(a.B * a.Nq * a.heads)), dim3(256), 0, stream, j);
  return hipGetLastError();
}

template <int HD>
hipError_t configure_dim() {
  hipError_t e = hipSuccess;
  for (int i = 0; i < 8 && e == hipSuccess; ++i)
    e = with_kernel<HD>(i & 1, i & 2, i & 4 ? 1 : 2, [](auto kernel, int lds) {
      return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds + MAX_WORDS * 8);
    });
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

int64_t cross_attention_workspace_bytes(const aeris_cross_attention& a) { return plan_of(a).bytes; }

hipError_t cross_attention_launch(const aeris_cross_attention& a, void* workspace, hipStream_t stream) {
  Plan plan = plan_of(a);
  if (a.head_dim == 32) return launch_dim<32>(a, plan, workspace, stream);
  if (a.head_dim == 64) return launch_dim<64>(a, plan, workspace, stream);
  return launch_dim<128>(a, plan, workspace, stream);
}

}  // namespace aeris
