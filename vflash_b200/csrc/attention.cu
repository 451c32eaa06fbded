// Attention over packed sequences (vfb_attention) on tcgen05.
//
// For one tile of 128 query rows (the group's heads of as many tokens as fit,
// row = token * pack + head in group) and the keys it sees, a key tile at a time:
//   S = Q K^T            tcgen05, fp32 in TMEM
//   m' = max(m, row max) P = exp2((S - m') * scale * log2 e)   registers
//   l = l * 2^(m - m') + row sum of P
//   O = O * 2^(m - m') + P V      tcgen05, P (16 bit) read from TMEM
//   out = O / l,  lse = m * scale + ln l
// S and O never leave the SM.  m only moves (and O is only multiplied) when the
// maximum grows by more than kHold binary orders, so P may reach 2^kHold (in fp16
// all of P lies 2^kLift higher); the result is the same to rounding and the pass over
// O in TMEM is rare.
//
// Roles of a block of twelve warps, one block on an SM:
//   warps 0-3, 4-7  softmax of stage 0 and stage 1, one thread per row
//   warp 8          TMA loads: Q tiles, then K and V tiles through one ring
//   warp 9          MMA issue, one thread
//   warp 10         cleans the V tiles that hold keys some row must not see
//   warp 11         works out the block's jobs and hands them to the others; whole
//                   jobs it takes, when it needs one, from the blocks of the grid that
//                   have not begun (clusterlaunchcontrol: the list needs no counter in
//                   memory, and blocks with short jobs take more of them)
// The two stages keep the tensor cores busy with one tile's products while the
// other's exponentials run.  They are
//   PAIR: two tiles of query rows against the same keys (many query rows), or
//   ALT:  one tile of query rows against even and odd key tiles, joined at the
//         end (few query rows: single tokens, short pieces).
//
// TMEM (512 columns): S of stage 0 | S of stage 1 | O0 | O1, 128 columns each; P
// overwrites the first columns of its S.  PAIR has key tiles of 128 and one
// buffer of S: the products of a stage's tile, P V and then the next S, run
// while the other stage is in its softmax.  One thread issues them, stage after
// stage: with a thread for each, their products mix, both stages get their S at
// one time and then compete for the exponentials (3900 cycles for a key tile of
// both instead of 3150).  Key tiles of 64 with two buffers of S take the
// chain S -> softmax -> P V -> S apart, but Q K^T with N = 64 takes 48 instead
// of 32 cycles a step (its operands come from shared memory at 128 bytes a
// cycle), and on long inputs the extra work costs more at the power limit
// than it gains (16.2 against 14.1 ms for 32760 tokens of 32 heads).  ALT waits
// for memory instead; there 64 keys mean shorter latencies and less padding.
//
// The exponentials (16 a cycle) take as long as the products of D = 128.  Some
// of them as a polynomial on the FMA pipe shortened neither: the chip is at its
// power limit here and the extra instructions cost clock (2 of 8: 15.1 against
// 14.6 ms at the limit, 13.2 against 12.8 ms before it is reached).
//
// Measured, repeated calls (replayed graphs in brackets, inputs that left L2):
// 32760 tokens of 32 heads, all pairs, 15.3 to 15.6 ms (13.5 while cool, then 14.9; 1130 to
// 1300 TFLOP/s, at the power limit); causal prompts of 8192 to 1 tokens, 32 on 8 heads, 754 to
// 775 us (657: 1140 TFLOP/s at a higher clock); 48 prompts of 1 to 300 tokens, heads of 64,
// 25 us (25); 17 tokens 12.5 us, bound by the host (8.5, all latency); one token of 32
// requests on 1 to 8192 cached keys 86 to 91 us (86: 4.5 TB/s), of one on 131072 keys
// 104 to 112 us (106: 5.1 TB/s).
//
// P is rounded to the operands' type because the second product takes 16 bits;
// the sum l is of the exponentials before that rounding, in fp32.
//
// Keys behind a row's limit: their scores become -inf, so P = 0; but 0 * inf
// and 0 * NaN would still spoil the second product.  Warp 10 therefore
// zeroes, in the key tiles that any row of the block sees only in part, the V
// rows behind the sequence's end and (causal) every element that is not
// finite; the latter are added back at the end to the rows that do see them.
#include <cmath>

#include "common.cuh"
#include "attention_plan.h"

namespace vfb {
namespace {

using attn::Plan;
using attn::Segment;

constexpr int kTile = 128;           // query rows in a tile
constexpr int kQPanel = kTile * 128;       // bytes of a tile's 64 elements of 16 bits, 128-byte swizzle
constexpr int kTail = 32;            // keys of a tile whose P is handed over separately
constexpr int kThreads = 384;
constexpr int kRingSlots = 16;       // at most
constexpr int kJobs = 2;             // jobs that the scheduler may be ahead
constexpr int kJobReaders = 11;      // warps that follow the schedule
// Waits for a whole job of other warps (for the next one, for room in the schedule,
// for a job's last tiles): a job of 2^31 keys takes about 30 s.  The waits inside a job
// have the usual limit, and whichever runs out first ends all of them.
constexpr uint64_t kJobTimeoutNs = 120000000000ull;
constexpr uint64_t kDrainNs = 100000000;  // for the products in flight when a block ends
constexpr float kHold = 8.0f;
// P carries a factor of 2^kLift, which cancels in O / l and comes off the
// log-sum-exp.  fp16 ends at 2^-24, and many keys that each round to 0 there may hold
// a good part of l; P is at most 2^kHold, so 2^7 more still fit below 65504, and what
// is lost of a probability is at most 2^-32 of the largest.  bf16 has fp32's range.
// The maximum times the scale is rounded before it is taken off the scores' products,
// by up to 2^-4 here and 2^-24 of it beyond, which P has no room for.  From the tile
// on in which some row's maximum goes beyond, a warp takes the maximum off those rows'
// scores first, in a loop of its own (one packed addition more for every pair: 15.97
// instead of 15.35 ms for 32760 tokens).
constexpr float kFar = 1048576.0f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr float kLn2 = 0.693147180559945309f;
// Log-sum-exp of a piece whose keys' scores are all -inf: it has no weight beside
// others, yet is no piece without keys (-inf), whose rows may be unwritten.
constexpr float kNoWeight = -3.402823466e38f;

// Rows of a workspace slot (one piece of a job): both tiles of PAIR.
constexpr int kSlotRows = 2 * kTile;

template <int DP, bool PAIR>
struct Layout {
  static constexpr int keys = PAIR ? 128 : 64;   // in a key tile
  static constexpr int buffers = 128 / keys;     // of S, for a stage
  static constexpr int panels = DP / 64;
  static constexpr int kv_panel = keys * 128;    // bytes
  static constexpr int q_tile = panels * kQPanel;
  static constexpr int kv_tile = panels * kv_panel;
  static constexpr int q_bytes = (PAIR ? 2 : 1) * q_tile;
  static constexpr int ring = DP == 128 ? (PAIR ? 5 : 11) : (PAIR ? 8 : 16);
  static constexpr int ahead = PAIR ? 1 : 4;  // key tiles whose S is issued before the first P V
  static constexpr int smem = 1024 + q_bytes + ring * kv_tile;  // tiles start on 1024 bytes
};

struct Params {
  Plan plan;
  const void *v;
  void *out;
  float *lse;
  int64_t v_token_stride, v_head_stride, out_token_stride, out_head_stride;
  int32_t pack, tokens;           // heads in a tile, tokens in a tile (pack * tokens <= 128)
  int32_t group_heads;            // query heads of one key/value head
  int32_t dim, fill_tail, split;
  float scale_log2;
  float *part_o, *part_lse;       // workspace: [slot][kSlotRows][dim], [slot][kSlotRows]
  attn::Record *records;          // workspace: [block]
  int *status;
};

// ---- small helpers -----------------------------------------------------------
__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *map, uint64_t *bar, int32_t x,
                                            int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// D (+)= A B^T, 16-bit operands from shared memory.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}

// D (+)= A B^T with A (16 bit, two elements to a column) in TMEM.
__device__ __forceinline__ void mma_f16_tmem_a(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc,
                                               uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}

// Descriptor of a V tile read with the head dimension as N: rows of 64
// contiguous N elements (128 bytes, swizzled), eight K rows to 1024 bytes, the
// next 64 N elements one panel further.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr, uint32_t panel_bytes) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  desc |= static_cast<uint64_t>(panel_bytes >> 4) << 16;  // leading offset: next 64 elements of N
  desc |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride offset: next eight rows of K
  desc |= static_cast<uint64_t>(1) << 46;
  desc |= static_cast<uint64_t>(2) << 61;
  return desc;
}

template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
  const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- two floats at a time: half the issue slots --------------------------------
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(f32x2 v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Maximum that keeps NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T>
__device__ __forceinline__ constexpr uint32_t exponent_mask() {  // both halves of a word
  return std::is_same<T, __nv_bfloat16>::value ? 0x7F807F80u : 0x7C007C00u;
}

template <typename T>
__device__ __forceinline__ constexpr uint32_t exponent_one() {  // its last bit
  return std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
}

// Lane i of four gets the i-th of u from each of them, in the order of the lanes.
__device__ __forceinline__ void transpose_in_four(uint4 (&u)[4], int lane) {
  const auto exchange = [&](uint4 &keep_low, uint4 &keep_high, int with) {
    const bool high = lane & with;
    const uint4 give = high ? keep_low : keep_high;
    uint4 got;
    got.x = __shfl_xor_sync(0xffffffffu, give.x, with);
    got.y = __shfl_xor_sync(0xffffffffu, give.y, with);
    got.z = __shfl_xor_sync(0xffffffffu, give.z, with);
    got.w = __shfl_xor_sync(0xffffffffu, give.w, with);
    if (high) keep_low = got;
    else keep_high = got;
  };
  exchange(u[0], u[1], 1);
  exchange(u[2], u[3], 1);
  exchange(u[0], u[2], 2);
  exchange(u[1], u[3], 2);
}

// ---- a job (or a piece of one) as the roles see it -----------------------------------
struct Job {
  int64_t row0, k0;     // first query row of the job in q, first key row of its sequence
  int32_t rows0, count; // index of the row in the sequence, tokens of the job (-1: no more jobs)
  int32_t nq, nk;       // of the sequence
  int32_t group;        // of heads
  int32_t t0, t1;       // key tiles
  int32_t n[2];         // key tiles of each stage
  int32_t first_masked; // key tiles from here on are seen in part by some row
  int32_t min_seen;     // keys that the job's first row sees
  int32_t slot;         // of the workspace for a piece, -1 for a whole job
  int32_t behind;       // rows behind the last sequence
  int32_t reserved;

  __device__ __forceinline__ int32_t tiles(bool pair) const { return pair ? max(n[0], n[1]) : n[0] + n[1]; }
};

template <bool PAIR>
__device__ __forceinline__ void describe(const Params &p, const Segment &s, Job &j) {
  j.rows0 = s.tile * p.plan.job_tokens;
  j.row0 = static_cast<int64_t>(s.seq.q0) + j.rows0;
  j.k0 = s.seq.k0;
  j.count = min(p.plan.job_tokens, s.seq.nq - j.rows0);
  j.nq = s.seq.nq;
  j.nk = s.seq.nk;
  j.group = s.group;
  j.t0 = s.t0;
  j.t1 = s.t1;
  j.min_seen = attn::keys_seen(p.plan, s.seq, j.rows0 + 1);
  j.first_masked = j.min_seen >> p.plan.key_shift;
  j.slot = s.slot;
  j.behind = p.plan.cu_q != nullptr && s.b == p.plan.batch;
  const int32_t tiles = max(s.t1 - s.t0, 0);
  if (PAIR) {
    // stage 0's rows may see fewer keys than the job's last row
    const uint32_t seen0 = attn::keys_seen(p.plan, s.seq, j.rows0 + min(p.tokens, j.count));
    j.n[0] = max(min(s.t1, static_cast<int32_t>((seen0 + 127) / 128)) - s.t0, 0);  // unsigned: up to 2^31 - 1 keys
    j.n[1] = j.count > p.tokens ? tiles : 0;
  } else {
    j.n[0] = (tiles + 1) / 2;
    j.n[1] = tiles / 2;
  }
}

struct Shared {
  uint64_t q_full, q_empty;
  uint64_t kv_full[kRingSlots], kv_empty[kRingSlots];
  uint64_t s_full[2][2], p_full[2][2], p_tail[2][2], pv_done[2], o_full[2], o_empty[2];
  // a V tile to be cleaned is on its way into the slot, and is clean: the MMA
  // warp waits for the latter before the slot is given back, so neither barrier
  // can run ahead of who waits for it
  uint64_t v_todo[kRingSlots], v_clean[kRingSlots];
  uint64_t stats_full, stats_empty, drain;
  uint64_t job_full[kJobs], job_empty[kJobs];
  alignas(16) uint64_t taken[2];  // the answer to take_block()
  uint64_t taken_full;
  Job jobs[kJobs];
  uint32_t tmem;
  int abort;
  int dirty;  // a non-finite element of V was taken out of a tile
};
static_assert(sizeof(Shared) + Layout<128, true>::smem <= 232448 &&
                  sizeof(Shared) + 2 * kTile * sizeof(float2) + Layout<128, false>::smem <= 232448,
              "shared memory of a block");

// Takes a block of the grid that has not begun off it: its index, or -1 if all
// have begun (then this must not be called again).  By a whole warp.
__device__ __forceinline__ int64_t take_block(Shared &sh, uint32_t phase, int *status) {
  if ((threadIdx.x & 31) == 0) {
    mbar_arrive_expect_tx(&sh.taken_full, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(sh.taken)),
                 "r"(smem_u32(&sh.taken_full))
                 : "memory");
  }
  __syncwarp();
  if (!warp_wait_quick(&sh.taken_full, phase, &sh.abort, status)) return -1;
  const volatile uint64_t *answer = sh.taken;
  uint32_t taken, block;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "mov.b128 h, {%2, %3};\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(taken), "=r"(block)
      : "l"(answer[0]), "l"(answer[1]));
  fence_proxy_async_smem();  // read before the next answer is written
  __syncwarp();
  return taken ? static_cast<int64_t>(block) : -1;
}

// A role's way through the schedule.
struct JobReader {
  Shared &sh;
  int *status;
  int slot = 0;
  uint32_t phase = 0;

  // `next` for a role of one thread.
  __device__ __forceinline__ bool next_alone(Job &j) {
    mbar_wait_through(&sh.job_full[slot], phase, &sh.abort, status, kJobTimeoutNs);
    if (*const_cast<volatile int *>(&sh.abort)) return false;
    j = sh.jobs[slot];
    mbar_arrive(&sh.job_empty[slot]);
    if (++slot == kJobs) {
      slot = 0;
      phase ^= 1;
    }
    return j.count >= 0;
  }

  // The next job in place, for a warp that reads its fields when it needs them (the
  // softmax warps have no register to spare) and gives it back with done().
  __device__ __forceinline__ bool peek() {
    return warp_wait_quick(&sh.job_full[slot], phase, &sh.abort, status, kJobTimeoutNs) && here().count >= 0;
  }
  __device__ __forceinline__ const Job &here() const { return sh.jobs[slot]; }
  __device__ __forceinline__ void done() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.job_empty[slot]);
    if (++slot == kJobs) {
      slot = 0;
      phase ^= 1;
    }
  }

  // The next job; false when there is none (or a wait ran out).
  __device__ __forceinline__ bool next(Job &j) {
    if (!warp_wait_quick(&sh.job_full[slot], phase, &sh.abort, status, kJobTimeoutNs)) return false;
    j = sh.jobs[slot];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.job_empty[slot]);
    if (++slot == kJobs) {
      slot = 0;
      phase ^= 1;
    }
    return j.count >= 0;
  }
};

// Running position in the ring of K and V tiles.
template <int RING>
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step() {
    if (++slot == RING) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// ---- softmax of one stage ----------------------------------------------------------
// Row state, and the loop over a job's key tiles.
template <typename T, int DP, bool PAIR>
struct Softmax {
  static constexpr int N = Layout<DP, PAIR>::keys, kBuffers = Layout<DP, PAIR>::buffers;
  const Params &p;
  Shared &sh;
  const uint32_t tmem_s, tmem_o;  // this warp's lanes
  const int stage;
  float m, l;            // running maximum (raw scores, as used) and sum
  uint32_t count = 0;    // key tiles of this stage so far, over all jobs

  __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t phase) {
    return warp_wait_quick(bar, phase, &sh.abort, p.status);
  }

  // `limit`: keys this row sees.  `live`: some row of the warp is a row of the job;
  // `valid`: this one is.
  __device__ __forceinline__ bool run(int32_t t0, int32_t n, int32_t stride, int32_t limit, bool live, bool valid) {
    m = -INFINITY;
    l = 0.0f;
    int32_t i = 0;
    for (; i < n; ++i, ++count) {
      if (!wait(&sh.s_full[stage][count % kBuffers], count / kBuffers & 1)) return false;
      tc_fence_after();
      if (live) {
        const int done = tile<false>((t0 + i * stride) * N, limit, i > 0, valid);
        if (done < 0) break;
        if (done == 0) return false;
      } else {
        hand_over(sh.p_full[stage]);
        hand_over(sh.p_tail[stage]);
      }
    }
    for (bool first = true; i < n; ++i, ++count, first = false) {
      if (!first && !wait(&sh.s_full[stage][count % kBuffers], count / kBuffers & 1)) return false;
      tc_fence_after();
      if (tile<true>((t0 + i * stride) * N, limit, i > 0, valid) == 0) return false;
    }
    return true;
  }

  __device__ __forceinline__ void hand_over(uint64_t (&bar)[2]) {
    tc_fence_before();
    __syncwarp();
    // by predicate: the lanes stay together for the next store to TMEM
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.u32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(&bar[count % kBuffers])),
        "r"(threadIdx.x & 31)
        : "memory");
  }

  // 1 when done, 0 after a wait that ran out, -1 (nothing done) where only tile<true> will do.
  template <bool FAR>
  __device__ __forceinline__ int tile(int32_t key0, int32_t limit, bool scale_o, bool valid) {
    const uint32_t at = tmem_s + N * (count % kBuffers);
    float s[N];
    {
      uint32_t(&r)[N / 32][32] = reinterpret_cast<uint32_t(&)[N / 32][32]>(s);
#pragma unroll
      for (int c = 0; c < N / 32; ++c) tmem_ld_32x32b_x32_issue(at + 32 * c, r[c]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < N / 32; ++c) tmem_ld_fence(r[c]);
    }
    // a row that is not part of the job is left alone: nobody reads its results
    const int32_t seen = valid ? limit - key0 : N;
    if (__any_sync(0xffffffffu, seen < N)) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= seen) s[j] = -INFINITY;
    }
    float top[4] = {m, m, m, m};
#pragma unroll
    for (int j = 0; j < N; j += 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) top[i] = max3_nan(top[i], s[j + 2 * i], s[j + 2 * i + 1]);
    }
    const float peak = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]);
    // true also for a NaN score; not while no key has been seen
    const bool move = valid && !((peak - m) * p.scale_log2 <= kHold) && peak != -INFINITY;
    if (__any_sync(0xffffffffu, move)) {
      if (!FAR && __any_sync(0xffffffffu, move && fabsf(peak * p.scale_log2) > kFar)) return -1;
      const float alpha = !move ? 1.0f : m == -INFINITY ? 0.0f : ex2((m - peak) * p.scale_log2);
      if (move) {
        m = peak;
        l *= alpha;
      }
      if (scale_o) {
        // S(count) came behind the P V that freed its buffer, so at most one phase of pv_done is open here.
        if (!wait(&sh.pv_done[stage], (count - 1) & 1)) return 0;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {  // few columns at a time: S holds the registers
          uint32_t r[16];
          tmem_ld_32x32b_x16(tmem_o + c, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
          tmem_st_32x32b_x16(tmem_o + c, r);
        }
      }
    }
    float base = m == -INFINITY ? 0.0f : m * p.scale_log2;
    if (FAR) {
      const float off = fabsf(base) > kFar ? m : 0.0f;  // the other rows' bits stay as they are
#pragma unroll
      for (int j = 0; j < N; ++j) s[j] -= off;
      if (off != 0.0f) base = 0.0f;
    }
    const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(kLift<T> - base, kLift<T> - base);
    f32x2 sum[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll
    for (int h = 0; h < N / 32; ++h) {
      uint32_t packed[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const f32x2 x = fma2(pair(s[32 * h + 2 * j], s[32 * h + 2 * j + 1]), scale2, base2);
        float a, b;
        split(x, a, b);
        a = ex2(a);
        b = ex2(b);
        sum[j & 1] = add2(sum[j & 1], pair(a, b));
        packed[j] = pack2<T>(a, b);
      }
      tmem_st_32x32b_x16(at + 16 * h, packed);
      if (32 * (h + 1) == N - kTail) {
        tmem_st_wait();
        hand_over(sh.p_full[stage]);
      }
    }
    tmem_st_wait();
    hand_over(sh.p_tail[stage]);
    float a, b, c, d;
    split(sum[0], a, b);
    split(sum[1], c, d);
    l += (a + b) + (c + d);
    return 1;
  }
};

// ---- kernel ------------------------------------------------------------------------
template <typename T, int DP, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Params p) {
  using L = Layout<DP, PAIR>;
  constexpr int kKeys = L::keys, kBuffers = L::buffers;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *s_q = smem;
  uint8_t *s_kv = smem + L::q_bytes;
  __shared__ Shared sh;
  __shared__ float2 stats[PAIR ? 1 : 2][PAIR ? 1 : kTile];  // (m, l) of each stage's rows

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (threadIdx.x < L::ring) {  // side by side: one thread takes half a microsecond for all of them
    const int i = threadIdx.x;
    mbar_init(&sh.kv_full[i], 1);
    mbar_init(&sh.kv_empty[i], 1);
    mbar_init(&sh.v_todo[i], 1);
    mbar_init(&sh.v_clean[i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 32) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(&sh.job_full[i], 1);
      mbar_init(&sh.job_empty[i], kJobReaders);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i][0], 1);
      mbar_init(&sh.s_full[i][1], 1);
      mbar_init(&sh.p_full[i][0], 4);
      mbar_init(&sh.p_full[i][1], 4);
      mbar_init(&sh.p_tail[i][0], 4);
      mbar_init(&sh.p_tail[i][1], 4);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], PAIR ? 4 : 8);  // warps that read it
    }
    mbar_init(&sh.stats_full, 8);
    mbar_init(&sh.stats_empty, 8);
    mbar_init(&sh.drain, 1);
    mbar_init(&sh.taken_full, 1);
    sh.abort = 0;
    sh.dirty = 0;
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  grid_dependency_wait();  // q, k, v and the offsets may come from the kernel before
  grid_launch_dependents();

  JobReader jobs{sh, p.status};
  Job job;

  // The block was launched with 168 registers a thread: 200 * 256 + 96 * 128 fit.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int stage = warp / 4;
    const int row = (warp % 4) * 32 + lane;  // of the tile, and TMEM lane
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    Softmax<T, DP, PAIR> sm{p, sh, lanes + 128 * stage, lanes + 256 + 128 * stage, stage};
    uint32_t o_phase[2] = {0, 0}, stats_phase = 0;
    const int token_in_tile = row / p.pack;
    const int head_in_tile = row - token_in_tile * p.pack;
    for (; jobs.peek(); jobs.done()) {
      const Job &job = jobs.here();
      const int token = token_in_tile + (PAIR ? stage * p.tokens : 0);  // of the job
      const bool valid = token_in_tile < p.tokens && token < job.count;
      int32_t limit = valid ? job.nk : 0;
      if (valid && p.plan.causal)
        limit = static_cast<int32_t>(
            min(max(static_cast<int64_t>(job.rows0) + token + 1 + job.nk - job.nq, int64_t{0}), int64_t{job.nk}));
      const bool live = __any_sync(0xffffffffu, valid);
      if (!sm.run(PAIR ? job.t0 : job.t0 + stage, job.n[stage], PAIR ? 1 : 2, limit, live, valid)) break;
      float m = sm.m, l = sm.l;
      bool have[2] = {job.n[stage] > 0, false};  // (PAIR) accumulators that hold something for this row
      float f[2] = {1.0f, 0.0f};
      if (PAIR) {
        if (have[0]) {
          if (!warp_wait_quick(&sh.o_full[stage], o_phase[stage], &sh.abort, p.status)) break;
          o_phase[stage] ^= 1;
        }
      } else {
        // The stages exchange their statistics; each joins half the columns of the accumulators.
        if (!warp_wait_quick(&sh.stats_empty, stats_phase ^ 1, &sh.abort, p.status)) break;
        stats[stage][row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.stats_full);
        if (!warp_wait_quick(&sh.stats_full, stats_phase, &sh.abort, p.status)) break;
        stats_phase ^= 1;
        const float2 s0 = stats[0][row], s1 = stats[PAIR ? 0 : 1][row];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.stats_empty);
        bool ok = true;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          have[i] = job.n[i] > 0;
          if (!have[i]) continue;
          ok = ok && warp_wait_quick(&sh.o_full[i], o_phase[i], &sh.abort, p.status);
          o_phase[i] ^= 1;
        }
        if (!ok) break;
        m = max3_nan(s0.x, s1.x, s0.x);
        const float shift = m == -INFINITY ? 0.0f : m;
        f[0] = s0.x == -INFINITY ? 0.0f : ex2((s0.x - shift) * p.scale_log2);
        f[1] = s1.x == -INFINITY ? 0.0f : ex2((s1.x - shift) * p.scale_log2);
        l = s0.y * f[0] + s1.y * f[1];
      }
      tc_fence_after();
      // A row of infinite scores is NaN however its exponentials were rounded.
      if (m == INFINITY) l = NAN;
      const int64_t piece_end = attn::min64(limit, static_cast<int64_t>(job.t1) * kKeys);
      const bool none = piece_end <= static_cast<int64_t>(job.t0) * kKeys;
      // (l == 0: all scores are -inf.  Alone that is 0 / 0; a piece leaves its sums as they are.)
      const float inv = none ? 0.0f : job.slot >= 0 && l == 0.0f ? 1.0f : 1.0f / l;
      const int64_t out_row = job.row0 + token;
      const int head = job.group * p.pack + head_in_tile;
      T *out = static_cast<T *>(p.out) + out_row * p.out_token_stride + head * p.out_head_stride;
      float *part = nullptr;
      if (job.slot >= 0) {
        const int64_t at = static_cast<int64_t>(job.slot) * kSlotRows + (PAIR ? stage * kTile : 0) + row;
        part = p.part_o + at * p.dim;
        if (valid && (PAIR || stage == 0))
          p.part_lse[at] = none ? -INFINITY : l == 0.0f ? kNoWeight : m * p.scale_log2 + (log2f(l) - kLift<T>);
      } else if (valid && (PAIR || stage == 0) && p.lse != nullptr) {
        p.lse[static_cast<int64_t>(head) * p.plan.total_q + out_row] =
            none ? -INFINITY : (m * p.scale_log2 + (log2f(l) - kLift<T>)) * kLn2;
      }
      const bool dirty = *reinterpret_cast<volatile int *>(&sh.dirty) != 0;
      if (live) {
        // Stores: four lanes exchange their rows' pieces and write 64 bytes of each row
        // together.  (Every lane its own row: 32 lines for an instruction, 1.7 us a job.)
        const unsigned valid_rows = __ballot_sync(0xffffffffu, valid) >> (lane & ~3);
        const float g0 = f[0] * inv, g1 = f[1] * inv;
        const uint32_t from = lanes + 256 + (PAIR ? 128 * stage : 0);
#pragma unroll 1
        for (int c = PAIR ? 0 : stage * (DP / 2); c < (PAIR || stage == 1 ? DP : DP / 2); c += 32) {
          if (c >= p.dim) break;
          float o[32];
          {
            uint32_t(&r)[32] = reinterpret_cast<uint32_t(&)[32]>(o);
            if (have[0]) {
              tmem_ld_32x32b_x32_issue(from + c, r);
              tmem_ld_wait();
              tmem_ld_fence(r);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = have[0] ? o[j] * g0 : 0.0f;
          if (!PAIR && have[1]) {
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              uint32_t r[16];
              tmem_ld_32x32b_x16(from + 128 + c + h, r);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[h + j] = fmaf(__uint_as_float(r[j]), g1, o[h + j]);
            }
          }
          if (valid && dirty && !none) {
            // the elements that were taken out, for the rows that see them
            const int kv_head = job.group * p.pack / p.group_heads;
            const int64_t first = static_cast<int64_t>(max(job.first_masked, job.t0)) * kKeys;
            const T *v = static_cast<const T *>(p.v) + kv_head * p.v_head_stride + job.k0 * p.v_token_stride;
            for (int64_t key = first; key < piece_end; ++key) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float x = c + j < p.dim ? static_cast<float>(v[key * p.v_token_stride + c + j]) : 0.0f;
                if (!(fabsf(x) < INFINITY)) o[j] += x;
              }
            }
          }
          const int part_of_row = lane % 4;
          uint4 u[4];
          if (job.slot >= 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float *x = o + 16 * h + 4 * j;
                u[j] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
              }
              transpose_in_four(u, lane);
              const int column = c + 16 * h + 4 * part_of_row;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if ((valid_rows >> j & 1) && column < p.dim)
                  *reinterpret_cast<uint4 *>(part + (j - part_of_row) * p.dim + column) = u[j];
            }
          } else if (!job.behind || p.fill_tail) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float *x = o + 8 * j;
              u[j] = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
            }
            transpose_in_four(u, lane);
            const int column = c + 8 * part_of_row;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              T *row_j = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), j, 4));
              if ((valid_rows >> j & 1) && column < p.dim) *reinterpret_cast<uint4 *>(row_j + column) = u[j];
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (have[0]) mbar_arrive(&sh.o_empty[PAIR ? stage : 0]);
        if (!PAIR && have[1]) mbar_arrive(&sh.o_empty[1]);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 8) {
      // ---------------- TMA producer ----------------
      RingPos<L::ring> pos;
      uint32_t q_phase = 0;
      bool ok = true;
      uint32_t issued = 0;  // slots that were ever loaded
      const bool leader = elect_one();
      const auto load = [&](const CUtensorMap *map, int32_t kv_head, int64_t key, bool masked) {
        ok = ok && warp_wait_quick(&sh.kv_empty[pos.slot], pos.phase ^ 1, &sh.abort, p.status);
        if (ok && leader) {
          mbar_arrive_expect_tx(&sh.kv_full[pos.slot], L::kv_tile);
          for (int i = 0; i < L::panels; ++i)
            tma_load_3d(s_kv + pos.slot * L::kv_tile + i * L::kv_panel, map, &sh.kv_full[pos.slot], 64 * i,
                        kv_head, static_cast<int32_t>(key));
          if (masked) mbar_arrive(&sh.v_todo[pos.slot]);
        }
        if (ok) issued |= 1u << pos.slot;
        if (ok) pos.step();
      };
      bool q_loaded = false;
      while (ok && jobs.next(job)) {
        const int32_t tiles = job.tiles(PAIR);
        if (tiles == 0) continue;
        if (!warp_wait_quick(&sh.q_empty, q_phase ^ 1, &sh.abort, p.status)) break;
        const int used = PAIR && job.count > p.tokens ? 2 : 1;
        if (leader) {
          mbar_arrive_expect_tx(&sh.q_full, used * L::panels * p.pack * p.tokens * 128);
          for (int t = 0; t < used; ++t)
            for (int i = 0; i < L::panels; ++i)
              tma_load_3d(s_q + t * L::q_tile + i * kQPanel, &map_q, &sh.q_full, 64 * i, job.group * p.pack,
                          static_cast<int32_t>(job.row0 + t * p.tokens));
        }
        q_loaded = true;
        q_phase ^= 1;
        const int32_t kv_head = job.group * p.pack / p.group_heads;
        const int64_t k0 = job.k0 + static_cast<int64_t>(job.t0) * kKeys;
        for (int32_t i = 0; i < min(tiles, L::ahead); ++i)
          load(&map_k, kv_head, k0 + static_cast<int64_t>(i) * kKeys, false);
        for (int32_t i = 0; i < tiles && ok; ++i) {
          load(&map_v, kv_head, k0 + static_cast<int64_t>(i) * kKeys, job.t0 + i >= job.first_masked);
          if (i + L::ahead < tiles)
            load(&map_k, kv_head, k0 + static_cast<int64_t>(i + L::ahead) * kKeys, false);
        }
      }
      // every load has landed before the block ends (a finished run waits for nothing here;
      // after an abort 256 tries each, far longer than a load takes)
      if (q_loaded) warp_wait_quick(&sh.q_full, q_phase ^ 1, &sh.abort, p.status);
      for (int i = 0; i < L::ring; ++i) {
        const uint32_t last = i < pos.slot ? pos.phase : pos.phase ^ 1;
        if (issued >> i & 1) warp_wait_quick(&sh.kv_full[i], last, &sh.abort, p.status);
      }
    } else if (warp == 9) {
      // ---------------- MMA issue ----------------
      // One thread: between two products it passes two or three barriers that are
      // usually ready (38 cycles each), which as a warp with an elected lane (branches,
      // votes, reconvergence) took longer than the products.  Products run over the
      // padded head dimension: TMA filled the rest with zeros.
      if (elect_one()) {
        const uint32_t idesc_s = idesc_f16<T>(kKeys, false);
        const uint32_t idesc_o = idesc_f16<T>((p.dim + 15) / 16 * 16, true);
        const uint64_t q_desc = sw128_kmajor_desc(smem_u32(s_q)), k_desc = sw128_kmajor_desc(smem_u32(s_kv));
        const uint64_t v_desc = sw128_mnmajor_desc(smem_u32(s_kv), L::kv_panel);
        RingPos<L::ring> pos;      // the item that is waited for next
        // Of the stages, in a field of 16 bits each (an array would live in local memory):
        // S and P V so far, over all jobs, modulo 4, and the phase of o_empty.
        uint32_t q_phase = 0, issued = 0, joined = 0, o_phase = 0x10001;
        uint32_t v_phase = 0;  // a bit for every slot
        const auto wait = [&](uint64_t *bar, uint32_t phase) { mbar_wait_through(bar, phase, &sh.abort, p.status); };
        const auto product_s = [&](int stage, int slot) {  // S = Q K^T
          const uint64_t a = q_desc + (PAIR ? stage * (L::q_tile >> 4) : 0);
          const uint64_t b = k_desc + slot * (L::kv_tile >> 4);
          const uint32_t buffer = issued >> 16 * stage & (kBuffers - 1);
          issued = (issued + (1u << 16 * stage)) & 0x30003u;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            mma_f16(tmem + 128 * stage + kKeys * buffer, a + ((k / 4 * kQPanel + k % 4 * 32) >> 4),
                    b + ((k / 4 * L::kv_panel + k % 4 * 32) >> 4), idesc_s, k > 0);
          tc_commit(&sh.s_full[stage][buffer]);
        };
        const auto product_o = [&](int stage, int slot, bool first, bool last) {  // O (+)= P V
          const uint32_t count = joined >> 16 * stage, buffer = count & (kBuffers - 1), phase = count / kBuffers & 1;
          joined = (joined + (1u << 16 * stage)) & 0x30003u;
          wait(&sh.p_full[stage][buffer], phase);
          if (first) {
            wait(&sh.o_empty[stage], o_phase >> 16 * stage & 1);
            o_phase ^= 1u << 16 * stage;
          }
          tc_fence_after();
          const uint64_t b = v_desc + slot * (L::kv_tile >> 4);
          const uint32_t a = tmem + 128 * stage + kKeys * buffer;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
            if (k == (kKeys - kTail) / 16) {
              wait(&sh.p_tail[stage][buffer], phase);
              tc_fence_after();
            }
            mma_f16_tmem_a(tmem + 256 + 128 * stage, a + 8 * k, b + (k * 2048 >> 4), idesc_o, k > 0 || !first);
          }
          tc_commit(&sh.pv_done[stage]);
          if (last) tc_commit(&sh.o_full[stage]);
        };
        while (jobs.next_alone(job)) {
          const int32_t tiles = job.tiles(PAIR), n0 = job.n[0], n1 = job.n[1];
          const int32_t masked = max(job.first_masked - job.t0, 0);  // tiles from here on
          if (tiles == 0) continue;
          wait(&sh.q_full, q_phase);
          q_phase ^= 1;
          // Scores of key tile i (its K is the next item); with `join`, behind the P V of
          // tile i - ahead, stage after stage.
          const auto step = [&](int32_t i, bool join, int v_slot) {
            const int32_t at = i - L::ahead;
            const int slot = pos.slot;
            const bool more = i < tiles;
            bool arrived = false;
            const auto scores = [&](int s) {
              if (!arrived) wait(&sh.kv_full[slot], pos.phase);
              arrived = true;
              product_s(s, slot);
            };
            if (PAIR) {
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const int32_t n = s == 0 ? n0 : n1;
                if (join && at < n) product_o(s, v_slot, at == 0, at == n - 1);
                if (i < n) scores(s);
              }
            } else {
              if (join) product_o(at & 1, v_slot, at < 2, at + 2 >= tiles);
              if (more) scores(i & 1);
            }
            if (join) tc_commit(&sh.kv_empty[v_slot]);
            if (more) {
              pos.step();
              tc_commit(&sh.kv_empty[slot]);
              if (i == tiles - 1) tc_commit(&sh.q_empty);
            }
          };
          for (int32_t i = 0; i < min(tiles, L::ahead); ++i) step(i, false, 0);
          for (int32_t i = 0; i < tiles; ++i) {
            const int v_slot = pos.slot;
            wait(&sh.kv_full[v_slot], pos.phase);
            pos.step();
            if (i >= masked) {
              wait(&sh.v_clean[v_slot], v_phase >> v_slot & 1);
              v_phase ^= 1u << v_slot;
            }
            step(i + L::ahead, true, v_slot);
          }
        }
        // the products issued last are over before the block ends
        tc_commit(&sh.drain);
        mbar_drain(&sh.drain, 0, kDrainNs);
      }
    } else if (warp == 11) {
      // ---------------- schedule ----------------
      Segment seg;
      int slot = 0;
      uint32_t phase = 1;
      const auto hand_out = [&](bool more) {  // by lane 0
        if (more) describe<PAIR>(p, seg, job);
        else job.count = -1;
        mbar_wait_through(&sh.job_empty[slot], phase, &sh.abort, p.status, kJobTimeoutNs);
        sh.jobs[slot] = job;
        mbar_arrive(&sh.job_full[slot]);
      };
      const auto step = [&]() {
        if (++slot == kJobs) {
          slot = 0;
          phase ^= 1;
        }
      };
      if (p.split) {
        attn::Share share;
        attn::Record record;
        share.init(p.plan, blockIdx.x, record);
        if (lane == 0) p.records[blockIdx.x] = record;
        if (__shfl_sync(0xffffffffu, share.empty(), 0))  // a share cut to nothing may be counted among a job's pieces
          for (int i = lane; i < kSlotRows; i += 32) p.part_lse[2ll * blockIdx.x * kSlotRows + i] = -INFINITY;
        if (lane == 0)
          for (bool more = true; more; step()) {
            more = share.next(p.plan, seg);
            hand_out(more);
            if (*const_cast<volatile int *>(&sh.abort)) break;
          }
      } else {
        uint32_t taken_phase = 0;
        attn::Cursor at{0, 0};
        int64_t next = blockIdx.x;
        while (next >= 0) {
          if (attn::whole_job(p.plan, static_cast<uint32_t>(next), seg, at)) {
            if (lane == 0) hand_out(true);
            __syncwarp();
            step();
            // no job is taken before there is room for it
            if (!warp_wait_quick(&sh.job_empty[slot], phase, &sh.abort, p.status, kJobTimeoutNs)) break;
          }
          next = take_block(sh, taken_phase, p.status);
          taken_phase ^= 1;
        }
        if (lane == 0) hand_out(false);
      }
    } else {
      // ---------------- cleaning of V tiles ----------------
      RingPos<L::ring> pos;
      uint32_t todo_phase = 0;  // a bit for every slot
      const auto clean = [&](int32_t t) {
        const int slot = pos.slot;
        if (!warp_wait_quick(&sh.v_todo[slot], todo_phase >> slot & 1, &sh.abort, p.status, kJobTimeoutNs)) return false;
        todo_phase ^= 1u << slot;
        if (!warp_wait_quick(&sh.kv_full[slot], pos.phase, &sh.abort, p.status)) return false;
        uint8_t *tile = s_kv + slot * L::kv_tile;
        const int32_t end = min(max(job.nk - t * kKeys, 0), kKeys);       // rows of the sequence
        const int32_t all = min(max(job.min_seen - t * kKeys, 0), kKeys);       // rows that every row sees
        const int row = lane / 8;  // lanes: eight 16-byte pieces of four rows
#pragma unroll
        for (int panel = 0; panel < L::panels; ++panel) {
          uint8_t *column = tile + panel * L::kv_panel + lane % 8 * 16;
          // Eight rows of a lane in flight; an element is not finite if adding one to its
          // exponent carries into the sign.  None is, as a rule.
#pragma unroll 1
          for (int r0 = all + row; r0 < end; r0 += 32) {
            uint32_t carry = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = r0 + 4 * i;
              uint4 x = make_uint4(0, 0, 0, 0);
              if (r < end) x = *reinterpret_cast<const uint4 *>(column + r * 128);
              const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) carry |= (word[j] & exponent_mask<T>()) + exponent_one<T>();
            }
            if (!(carry & 0x80008000u)) continue;
            *reinterpret_cast<volatile int *>(&sh.dirty) = 1;
#pragma unroll 1
            for (int r = r0; r < min(r0 + 32, end); r += 4) {
              uint32_t *word = reinterpret_cast<uint32_t *>(column + r * 128);
#pragma unroll 1
              for (int j = 0; j < 4; ++j) word[j] &= ~__vcmpeq2(word[j] & exponent_mask<T>(), exponent_mask<T>());
            }
          }
#pragma unroll 4
          for (int r = end + row; r < kKeys; r += 4)
            *reinterpret_cast<uint4 *>(column + r * 128) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __threadfence_block();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.v_clean[slot]);
        return true;
      };
      bool ok = true;
      while (ok && jobs.next(job)) {
        const int32_t tiles = job.tiles(PAIR);
        if (tiles == 0) continue;
        for (int32_t i = 0; i < min(tiles, L::ahead); ++i) pos.step();
        for (int32_t i = 0; i < tiles && ok; ++i) {
          if (job.t0 + i >= job.first_masked) ok = clean(job.t0 + i);
          pos.step();
          if (i + L::ahead < tiles) pos.step();
        }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- joining the pieces of jobs that were cut ------------------------------------------
// Block (c - 1, y): the job whose first inner cut is cut c, a part of its rows; a
// warp for a row at a time, four columns to a lane.
constexpr int kJoinWarps = 8;
constexpr int kJoinParts = 4;  // of a tile's rows

template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) attention_join_kernel(const __grid_constant__ Params p) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int c = static_cast<int>(blockIdx.x) + 1;
  const attn::Record before = p.records[c - 1], job = p.records[c];
  if (!attn::join_starts(before, job)) return;
  int pieces = 1;  // and one for every record inside the job
  for (int i0 = c;; i0 += 32) {
    const int i = i0 + lane;
    const bool same = i < p.plan.blocks && p.records[i].inside && p.records[i].start == job.start;
    const unsigned others = __ballot_sync(0xffffffffu, !same);
    pieces += others ? __ffs(others) - 1 : 32;
    if (others) break;
  }
  const int first = attn::join_first(before, job, c);
  for (int at = blockIdx.y * kJoinWarps + (threadIdx.x >> 5); at < kSlotRows; at += kJoinWarps * gridDim.y) {
    const int in_tile = at % kTile;
    const int token = in_tile / p.pack + at / kTile * p.tokens;
    if (in_tile / p.pack >= p.tokens || token >= job.count) continue;
    const auto slot_row = [&](int i) {
      return static_cast<int64_t>(i == 0 ? first : 2 * (c + i - 1)) * kSlotRows + at;
    };
    float top = -INFINITY;
    for (int i = lane; i < pieces; i += 32) top = max3_nan(top, p.part_lse[slot_row(i)], top);
    for (int o = 16; o; o >>= 1) top = max3_nan(top, __shfl_xor_sync(0xffffffffu, top, o), top);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, acc[4] = {};
    for (int i0 = 0; i0 < pieces; i0 += 32) {
      const float part = i0 + lane < pieces ? p.part_lse[slot_row(i0 + lane)] : -INFINITY;
      const float weight = ex2(part - base);
      const unsigned written = __ballot_sync(0xffffffffu, part != -INFINITY);
      sum += weight;
      const int n = min(32, pieces - i0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float w = __shfl_sync(0xffffffffu, weight, i);
        // A piece without keys may have left its rows unwritten.  One with a weight of 0 is
        // read: what it saw of infinities and NaN stays, as it does inside a job.
        if (lane * 4 < p.dim && (written >> i & 1)) {
          const float4 o = *reinterpret_cast<const float4 *>(p.part_o + slot_row(i0 + i) * p.dim + 4 * lane);
          acc[0] = fmaf(w, o.x, acc[0]);
          acc[1] = fmaf(w, o.y, acc[1]);
          acc[2] = fmaf(w, o.z, acc[2]);
          acc[3] = fmaf(w, o.w, acc[3]);
        }
      }
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = top == -INFINITY ? 0.0f : top == kNoWeight ? NAN : 1.0f / sum;
    const int head = job.group * p.pack + in_tile % p.pack;
    const int64_t row = static_cast<int64_t>(job.row0) + token;
    if (lane * 4 < p.dim) {
      uint2 t;
      t.x = pack2<T>(acc[0] * inv, acc[1] * inv);
      t.y = pack2<T>(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + row * p.out_token_stride + head * p.out_head_stride +
                                 4 * lane) = t;
    }
    if (lane == 0 && p.lse != nullptr)
      p.lse[static_cast<int64_t>(head) * p.plan.total_q + row] =
          top == -INFINITY || top == kNoWeight ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
}

// ---- host side -------------------------------------------------------------------------
constexpr int kMaxBlocks = 148;  // SMs of a B200: blocks that even shares are cut for

// Sequences of a call, below: a block passes over all of them (32 at a time, one
// by one where a share goes on behind empty ones) while its other warps wait.
constexpr int kMaxBatch = 1 << 24;

constexpr int kBandBytes = 48 << 20;  // of K and V that stay in L2 (126 MB) beside the rows read and written

struct Choice {
  int pack, tokens, groups;
  bool pair, split;
  int64_t jobs;  // whole jobs, at most
};

Choice choose(const vfb_attention_args &a) {
  Choice c;
  const int group = a.heads / a.kv_heads;
  c.pack = group;
  if (group > kTile)
    for (c.pack = kTile; group % c.pack; --c.pack) {
    }
  c.tokens = kTile / c.pack;
  c.groups = a.heads / c.pack;
  // Two tiles of rows share every key tile where a sequence has more than one on average.
  c.pair = a.total_q > static_cast<int64_t>(c.tokens) * a.batch;
  const int64_t tokens = static_cast<int64_t>(c.tokens) * (c.pair ? 2 : 1);
  const int64_t tiles = a.cu_seqlens_q == nullptr
                            ? (a.total_q + tokens - 1) / tokens
                            : attn::min64(a.total_q, a.total_q / tokens + a.batch + 1);
  c.jobs = tiles * c.groups;
  // Even shares or whole jobs?  Both estimated, in the time of a key of a job (15 ns
  // with two tiles of rows, 10 ns with one): a whole job costs a fixed time besides its
  // keys, shares cost writing and joining the pieces and going through more short
  // ones, and whole jobs leave blocks idle, all of them for the longest job where
  // there are no more jobs than blocks.  Lengths are not known here.  Prompts count
  // as equally long (the longest jobs go first).  Keys of their own are caches: half
  // equal, half with one of twice the average, which may come last; with lengths inside
  // of slots, half filled on average.  Measured, whole against even (us, 32 / 8
  // heads of 128): prompts of 1000 tokens 24 / 40, 5000 188 / 215, all tokens seen 4000
  // 245 / 247; 512 tokens after 1024, 4096, 16384 cached ones 30 / 40, 74 / 59, 247 / 135;
  // single tokens of 1 sequence on 1000 and 2000 keys 16 / 19, 26 / 20, of 64 on 500 and 1000 36 / 54,
  // 56 / 70, of 16 on 4000 50 / 61, of 32 on 1 to 8192 in slots 162 / 82.
  const double fixed = c.pair ? 350 : 600, join = c.pair ? 2000 : 1900, slope = c.pair ? 1.05 : 1.2;
  const double nk = static_cast<double>(a.total_k) / a.batch, nq = static_cast<double>(a.total_q) / a.batch;
  const double mean = a.lengths_k != nullptr ? nk / 2 : a.causal ? nk - (nq < nk ? nq : nk) / 2 : nk;
  const double rounds = static_cast<double>(c.jobs) / kMaxBlocks;
  const bool few = c.jobs <= kMaxBlocks;
  const double sorted = few ? fixed + nk : (a.causal ? rounds : std::ceil(rounds)) * (fixed + mean);
  double whole = sorted;
  if (a.lengths_k != nullptr || (a.cu_seqlens_k != nullptr && a.batch > 1)) {
    const double longest = a.lengths_k != nullptr ? nk : 2 * nk;
    const double uneven = few ? fixed + longest : rounds * (fixed + mean) + (fixed + longest) / 2;
    whole = a.lengths_k != nullptr ? uneven : (sorted + uneven) / 2;
  }
  c.split = c.jobs < 4 * kMaxBlocks && whole > join + rounds * (mean + attn::OVERHEAD) * slope;
  return c;
}

int check_args(const vfb_attention_args *a) {
  if (a == nullptr) return set_error(VFB_EINVAL, "vfb_attention: args is NULL");
  if (a->total_q < 0 || a->total_k < 0 || a->total_q >= (1ll << 31) || a->total_k >= (1ll << 31))
    return set_error(VFB_EINVAL, "vfb_attention: rows must be >= 0 and below 2^31");
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads > 65535)
    return set_error(VFB_EINVAL, "vfb_attention: heads must be a multiple of kv_heads, 1 to 65535");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return set_error(VFB_EINVAL, "vfb_attention: dim must be a multiple of 8 from 8 to 128");
  if (a->dtype != 0 && a->dtype != 1) return set_error(VFB_EINVAL, "vfb_attention: dtype must be 0 (bf16) or 1 (fp16)");
  if (a->batch < 1 || a->batch >= kMaxBatch || (a->cu_seqlens_q == nullptr && (a->batch != 1 || a->cu_seqlens_k != nullptr)))
    return set_error(VFB_EINVAL, "vfb_attention: batch must be >= 1, below 2^24, and 1 without cu_seqlens_q");
  if (a->cu_seqlens_q != nullptr && a->cu_seqlens_k == nullptr && a->total_k != a->total_q)
    return set_error(VFB_EINVAL, "vfb_attention: keys of another length need cu_seqlens_k");
  if (!(a->scale > 0.0f) || a->scale > 1.0e30f)  // times log2(e) it stays finite
    return set_error(VFB_EINVAL, "vfb_attention: scale must be positive, at most 1e30");
  const int64_t strides[] = {a->q_token_stride, a->q_head_stride, a->k_token_stride,   a->k_head_stride,
                             a->v_token_stride, a->v_head_stride, a->out_token_stride, a->out_head_stride};
  for (int64_t s : strides)
    if (s < a->dim || s % 8 || s >= (1ll << 38))
      return set_error(VFB_EINVAL, "vfb_attention: strides must be multiples of 8, at least dim");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out))
    return set_error(VFB_EINVAL, "vfb_attention: q, k, v and out must be 16-byte aligned");
  if (choose(*a).jobs >= (1ll << 31)) return set_error(VFB_EINVAL, "vfb_attention: too many rows");
  return VFB_OK;
}

// Blocks write rows while others still read theirs.
int check_overlap(const vfb_attention_args &a) {
  const auto extent = [&](const void *base, int64_t rows, int64_t heads, int64_t token_stride, int64_t head_stride) {
    return Extent{base, 2ll * a.dim, {rows, heads}, {2 * token_stride, 2 * head_stride}};
  };
  const Extent out = extent(a.out, a.total_q, a.heads, a.out_token_stride, a.out_head_stride);
  const Extent lse{a.lse, 4 * a.total_q * a.heads, {a.lse != nullptr, 1}, {}};
  const Extent operands[] = {extent(a.q, a.total_q, a.heads, a.q_token_stride, a.q_head_stride),
                             extent(a.k, a.total_k, a.kv_heads, a.k_token_stride, a.k_head_stride),
                             extent(a.v, a.total_k, a.kv_heads, a.v_token_stride, a.v_head_stride)};
  for (const Extent &t : operands)
    if (may_overlap(out, t) || may_overlap(lse, t))
      return set_error(VFB_EINVAL, "vfb_attention: out and lse may not overlap q, k or v");
  if (may_overlap(out, lse)) return set_error(VFB_EINVAL, "vfb_attention: out and lse may not overlap");
  return VFB_OK;
}

// [rows, heads, dim] as (dim, heads, rows), boxes of 64 x box_heads x box_rows.
int make_map(CUtensorMap *map, const void *base, int dtype, int64_t dim, int64_t heads, int64_t rows,
             int64_t head_stride, int64_t token_stride, int box_heads, int box_rows) {
  auto encode = tensor_map_encoder();
  if (encode == nullptr) return set_error(VFB_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                      const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(VFB_ECUDA, "vfb_attention: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return VFB_OK;
}

template <typename T, int DP, bool PAIR>
int launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const Params &p, int64_t jobs,
           cudaStream_t stream) {
  using L = Layout<DP, PAIR>;
  auto kernel = attention_kernel<T, DP, PAIR>;
  static std::atomic<uint64_t> smem_set[kMaxAttrDevices];
  int rc = ensure_smem_optin(reinterpret_cast<const void *>(kernel), L::smem, smem_set);
  if (rc != VFB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.split ? p.plan.blocks : jobs), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, q, k, v, p);
  if (err == cudaSuccess && p.split && p.plan.blocks > 1) {
    cfg.gridDim = dim3(p.plan.blocks - 1, kJoinParts * (PAIR ? 2 : 1), 1);
    cfg.blockDim = dim3(32 * kJoinWarps, 1, 1);
    cfg.dynamicSmemBytes = 0;
    err = cudaLaunchKernelEx(&cfg, attention_join_kernel<T>, p);
  }
  if (err != cudaSuccess) return set_error(VFB_ECUDA, "vfb_attention launch: %s", cudaGetErrorString(err));
  return VFB_OK;
}

int64_t slots_of(const Choice &c) { return c.split ? 2 * kMaxBlocks : 0; }

}  // namespace
}  // namespace vfb

extern "C" int64_t vfb_attention_workspace_bytes(const vfb_attention_args *args) {
  using namespace vfb;
  if (check_args(args) != VFB_OK) return -1;
  if (args->total_q == 0) return 0;
  const int64_t slots = slots_of(choose(*args));
  return slots * kSlotRows * (args->dim + 1) * static_cast<int64_t>(sizeof(float)) +
         slots / 2 * static_cast<int64_t>(sizeof(attn::Record));
}

extern "C" int vfb_attention(const vfb_attention_args *args, void *stream) {
  using namespace vfb;
  int rc = check_args(args);
  if (rc != VFB_OK) return rc;
  const vfb_attention_args &a = *args;
  if (a.total_q == 0) return VFB_OK;
  if (!a.q || !a.out || (a.total_k > 0 && (!a.k || !a.v)))
    return set_error(VFB_EINVAL, "vfb_attention: NULL pointer");
  rc = check_overlap(a);
  if (rc != VFB_OK) return rc;
  const Choice c = choose(a);
  const int64_t need = vfb_attention_workspace_bytes(args);
  if (a.workspace_bytes < need || (need > 0 && (!a.workspace || reinterpret_cast<uintptr_t>(a.workspace) % 256)))
    return set_error(VFB_EINVAL, "vfb_attention: needs %lld bytes of 256-byte aligned workspace", (long long)need);
  int sms = 0;
  rc = check_device(&sms);
  if (rc != VFB_OK) return rc;

  Params p = {};
  p.plan.cu_q = a.cu_seqlens_q;
  p.plan.cu_k = a.cu_seqlens_k;
  p.plan.len_k = a.lengths_k;
  p.plan.total_q = static_cast<int32_t>(a.total_q);
  p.plan.total_k = static_cast<int32_t>(a.total_k);
  p.plan.batch = a.batch;
  p.plan.groups = c.groups;
  attn::set_job_tokens(p.plan, c.tokens * (c.pair ? 2 : 1));
  p.plan.causal = a.causal != 0;
  p.plan.blocks = sms < kMaxBlocks ? sms : kMaxBlocks;
  p.plan.key_shift = c.pair ? 7 : 6;
  p.plan.band_keys = kBandBytes / (4 * a.dim);
  p.plan.unit_shift = c.split ? attn::unit_shift_for(c.jobs, a.total_q + a.total_k) : 0;
  p.v = a.v;
  p.out = a.out;
  p.lse = a.lse;
  p.v_token_stride = a.v_token_stride;
  p.v_head_stride = a.v_head_stride;
  p.out_token_stride = a.out_token_stride;
  p.out_head_stride = a.out_head_stride;
  p.pack = c.pack;
  p.tokens = c.tokens;
  p.group_heads = a.heads / a.kv_heads;
  p.dim = a.dim;
  p.fill_tail = a.fill_tail;
  p.split = c.split;
  p.scale_log2 = a.scale * 1.44269504088896341f;
  if (c.split) {
    p.part_o = static_cast<float *>(a.workspace);
    p.part_lse = p.part_o + slots_of(c) * kSlotRows * a.dim;
    p.records = reinterpret_cast<attn::Record *>(p.part_lse + slots_of(c) * kSlotRows);
  }
  p.status = device_status_ptr();

  CUtensorMap mq, mk, mv;
  rc = make_map(&mq, a.q, a.dtype, a.dim, a.heads, a.total_q, a.q_head_stride, a.q_token_stride, c.pack, c.tokens);
  // without keys nothing is loaded, but a map must stand for something
  const bool keys = a.total_k > 0;
  if (rc == VFB_OK)
    rc = make_map(&mk, keys ? a.k : a.q, a.dtype, a.dim, a.kv_heads, keys ? a.total_k : 1, a.k_head_stride,
                  a.k_token_stride, 1, c.pair ? 128 : 64);
  if (rc == VFB_OK)
    rc = make_map(&mv, keys ? a.v : a.q, a.dtype, a.dim, a.kv_heads, keys ? a.total_k : 1, a.v_head_stride,
                  a.v_token_stride, 1, c.pair ? 128 : 64);
  if (rc != VFB_OK) return rc;

  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto type) {
    using T = decltype(type);
    if (a.dim > 64)
      return c.pair ? launch<T, 128, true>(mq, mk, mv, p, c.jobs, s)
                    : launch<T, 128, false>(mq, mk, mv, p, c.jobs, s);
    return c.pair ? launch<T, 64, true>(mq, mk, mv, p, c.jobs, s)
                  : launch<T, 64, false>(mq, mk, mv, p, c.jobs, s);
  };
  return a.dtype == 0 ? go(__nv_bfloat16()) : go(__half());
}
