// The work order of the packed attention kernel, shared with its CPU test.
//
// A job is one tile of query rows of one sequence for one group of heads that
// read the same keys; its keys come in key tiles of 64 or 128 (Plan::key_shift).
// Two orders:
//
// * whole jobs: a list of jobs that the blocks take from its front, every job by
//   itself.  In a causal sequence the longest jobs come first, those of all head
//   groups whose keys fit into L2 together before the next shorter ones: the last jobs
//   to be taken are short, and blocks that take when they are done end within a
//   short job of one another.  (Every 148th job to a block instead: 14 to 23 % over the
//   average for lengths of 8192, 4111, 2500, 1031, 509.);
// * even shares: all jobs laid end to end, a job as long as its keys plus
//   OVERHEAD (about what loading its queries and storing its rows costs, in
//   keys), and the line cut into equal parts, one for a block.  Cuts are moved
//   to borders of key tiles.  A block's first and last job may then be pieces;
//   every piece leaves its rows and their log-sum-exp in a slot of the
//   workspace (2 * block for a block's first job, 2 * block + 1 for another),
//   and a second kernel joins them in the order of the blocks, led by a record of
//   where each block's share begins.
//
// Only totals are known on the host: lengths are device data, so the functions
// here run on the device, on one whole warp of a block with uniform arguments
// (the lanes read the sequences side by side).  On the host they run as plain
// loops.  Every block passes through them before its first load, so they are
// short: 32 bits (the line is measured in units of 2^unit_shift keys, chosen so
// that it stays below 2^31), hardly a division, both ends of a share worked out
// at once in the two halves of the warp.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define VFB_HD __host__ __device__ __forceinline__
#else
#define VFB_HD inline
#endif

namespace vfb {
namespace attn {

constexpr int64_t OVERHEAD = 256; // a job's fixed cost, in keys
constexpr int64_t SHARE = 512;    // a block's share is at least this long, unless that leaves jobs without blocks

VFB_HD int32_t min32(int32_t a, int32_t b) { return a < b ? a : b; }
VFB_HD int32_t max32(int32_t a, int32_t b) { return a > b ? a : b; }
VFB_HD int32_t clamp32(int32_t x, int32_t lo, int32_t hi) { return min32(max32(x, lo), hi); }
VFB_HD int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

struct Plan {
  const int32_t *cu_q, *cu_k, *len_k;  // device arrays, cu_q NULL: one sequence of all rows
  int32_t total_q, total_k;
  int32_t batch;
  int32_t groups;      // head groups: jobs for one tile of rows
  int32_t job_tokens;  // query tokens in a job
  int32_t causal;
  int32_t blocks;      // blocks that even shares are cut for, at most
  int32_t key_shift;   // log2 of the keys in a key tile
  int32_t band_keys;   // keys whose K and V rows of one head fit into L2
  int32_t unit_shift;  // log2 of the keys in a unit of the line
  uint32_t token_inverse, token_shift;  // n / job_tokens = high word of n * token_inverse, shifted: for n < 2^31
};

// Fills in the inverse of job_tokens.
inline void set_job_tokens(Plan &p, int32_t tokens) {
  uint32_t log = 0;
  while ((1u << log) < static_cast<uint32_t>(tokens)) ++log;
  p.job_tokens = tokens;
  // rounded up, with 31 + log bits of fraction: exact for every n < 2^31
  p.token_inverse = static_cast<uint32_t>(((1ull << (31 + log)) + tokens - 1) / tokens);
  p.token_shift = log;
}

VFB_HD uint32_t over_job_tokens(const Plan &p, uint32_t n) {
  return static_cast<uint32_t>(static_cast<uint64_t>(n) * p.token_inverse >> 31 >> p.token_shift);
}

// Unit of a line that holds at most `jobs` jobs of `keys` keys.
VFB_HD int32_t unit_shift_for(int64_t jobs, int64_t keys) {
  int32_t u = 0;
  while (jobs * (((keys + OVERHEAD) >> u) + 2) >= (1ll << 31)) ++u;
  return u;
}

// Sequence b: its rows and keys, clamped to the buffers.  b == batch stands for
// the rows behind the last sequence, which have no keys.
struct Seq {
  int32_t q0, k0;
  int32_t nq, nk;
  int32_t tiles;
};

VFB_HD int32_t num_seqs(const Plan &p) { return p.cu_q == nullptr ? 1 : p.batch + 1; }

VFB_HD Seq sequence(const Plan &p, int32_t b) {
  Seq s;
  int32_t q1, k1;
  if (p.cu_q == nullptr) {
    s.q0 = s.k0 = 0;
    q1 = p.total_q;
    k1 = p.total_k;
  } else {
    s.q0 = clamp32(p.cu_q[b], 0, p.total_q);
    if (b == p.batch) {
      q1 = p.total_q;
      s.k0 = k1 = 0;
    } else {
      q1 = clamp32(p.cu_q[b + 1], s.q0, p.total_q);
      const int32_t *cu_k = p.cu_k != nullptr ? p.cu_k : p.cu_q;
      s.k0 = clamp32(cu_k[b], 0, p.total_k);
      k1 = clamp32(cu_k[b + 1], s.k0, p.total_k);
    }
  }
  if (p.len_k != nullptr && b < p.batch) k1 = s.k0 + clamp32(p.len_k[b], 0, k1 - s.k0);
  s.nq = q1 - s.q0;
  s.nk = k1 - s.k0;
  s.tiles = s.nq > 0 ? static_cast<int32_t>(over_job_tokens(p, s.nq - 1)) + 1 : 0;
  return s;
}

// Keys that the last of `rows` leading query rows of a sequence sees.
VFB_HD int32_t keys_seen(const Plan &p, const Seq &s, int32_t rows) {
  if (!p.causal) return s.nk;
  return clamp32(rows - s.nq + s.nk, 0, s.nk);  // rows <= nq: no step leaves 32 bits
}

// Rows of the sequence up to the end of a row tile.
VFB_HD int32_t rows_to(const Plan &p, const Seq &s, int32_t tile) {
  return tile + 1 >= s.tiles ? s.nq : (tile + 1) * p.job_tokens;
}

// Key tiles of a job.
VFB_HD int32_t tiles_of(const Plan &p, const Seq &s, int32_t tile) {
  const uint32_t keys = keys_seen(p, s, rows_to(p, s, tile));
  return static_cast<int32_t>((keys + (1u << p.key_shift) - 1) >> p.key_shift);
}

// ---- even shares: lengths of jobs, in units ------------------------------------
// A causal job counts the keys its last row would see were nk >= nq: not fewer
// than it sees, and summed over the tiles in closed form.
VFB_HD uint32_t units(const Plan &p, uint32_t keys) { return (keys + (1u << p.unit_shift) - 1) >> p.unit_shift; }
VFB_HD uint32_t overhead_units(const Plan &p) { return units(p, static_cast<uint32_t>(OVERHEAD)); }
VFB_HD uint32_t units_before(const Plan &p, const Seq &s) {
  return units(p, p.causal ? max32(s.nk - s.nq, 0) : s.nk);
}

// Length of the first `tiles` jobs of one head group of the sequence.
VFB_HD uint32_t jobs_length(const Plan &p, const Seq &s, uint32_t tiles) {
  uint32_t length = tiles * (overhead_units(p) + units_before(p, s));
  if (p.causal && tiles > 0) {
    const uint32_t full = tiles < static_cast<uint32_t>(s.tiles) ? tiles : tiles - 1;
    length += (static_cast<uint32_t>(p.job_tokens) >> p.unit_shift) * (full * (full + 1) / 2);
    if (full != tiles) length += units(p, s.nq);
  }
  return length;
}

VFB_HD uint32_t line_length(const Plan &p, const Seq &s) { return jobs_length(p, s, s.tiles) * p.groups; }

// ---- scans over the sequences ----------------------------------------------------
#ifdef __CUDA_ARCH__
__device__ __forceinline__ uint32_t warp_upto(uint32_t own) {  // inclusive sum over the lanes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, own, o);
    if (lane >= o) own += t;
  }
  return own;
}
#endif

// Where a block's way through the list of whole jobs stands: the sequences from
// `b` on hold the jobs from `before` on.  The jobs that a block takes come later and later
// in the list, as a rule, so it passes over the sequences once.  (From the first
// sequence for every job: 4096 prompts of 64 tokens, 4 heads of 64, 3.0 ms instead of
// 0.26, 131072 of one token 1.4 s instead of 6.9 ms.)
struct Cursor {
  int32_t b;
  uint32_t before;
};

// Whole jobs: the sequence in which job `x` of the list lies, -1 behind the end;
// `x` becomes its place inside the sequence.
VFB_HD int32_t locate_job(const Plan &p, uint32_t &x, Cursor &at) {
  if (x < at.before) at = Cursor{0, 0};
  x -= at.before;
#ifdef __CUDA_ARCH__
  const int lane = threadIdx.x & 31;
  for (; at.b < num_seqs(p); at.b += 32) {
    const int32_t b = at.b + lane;
    const uint32_t own = b < num_seqs(p) ? static_cast<uint32_t>(sequence(p, b).tiles) * p.groups : 0u;
    const uint32_t upto = warp_upto(own);
    const unsigned hit = __ballot_sync(0xffffffffu, x < upto);
    if (hit) {
      const int first = __ffs(hit) - 1;
      x -= __shfl_sync(0xffffffffu, upto - own, first);
      return at.b + first;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
    x -= all;
    at.before += all;
  }
#else
  for (; at.b < num_seqs(p); ++at.b) {
    const uint32_t own = static_cast<uint32_t>(sequence(p, at.b).tiles) * p.groups;
    if (x < own) return at.b;
    x -= own;
    at.before += own;
  }
#endif
  return -1;
}

// ---- segments: what a block does in one go ---------------------------------------
struct Segment {
  Seq seq;
  int32_t b, group, tile;
  int32_t t0, t1;  // key tiles
  int32_t slot;    // workspace slot of a piece, -1 for a whole job
};

// Whole jobs: job `x` of the list; false behind its end.
VFB_HD bool whole_job(const Plan &p, uint32_t x, Segment &s, Cursor &at) {
  s.b = locate_job(p, x, at);
  if (s.b < 0) return false;
  s.seq = sequence(p, s.b);
  const uint32_t tiles = s.seq.tiles;
  // head groups that go side by side; jobs of one length need no order, and one
  // group after the other reads the fewest keys at a time
  const int32_t fit = p.causal ? p.band_keys / max32(s.seq.nk, 1) : 1;
  uint32_t wide = clamp32(fit, 1, p.groups);
  const uint32_t band = x / (tiles * wide);
  x -= band * tiles * wide;
  const int32_t group0 = static_cast<int32_t>(band * wide);
  wide = min32(wide, p.groups - group0);
  const int32_t i = static_cast<int32_t>(x / wide);
  s.group = group0 + static_cast<int32_t>(x - i * wide);
  s.tile = p.causal ? s.seq.tiles - 1 - i : i;
  s.t0 = 0;
  s.t1 = tiles_of(p, s.seq, s.tile);
  s.slot = -1;
  return true;
}

VFB_HD bool whole_job(const Plan &p, uint32_t x, Segment &s) {
  Cursor at{0, 0};
  return whole_job(p, x, s, at);
}

// Even shares: a job, and the key tile of it where a share begins or ends.
struct Place {
  Seq seq;
  int32_t b, group, tile;  // b == num_seqs: behind the last job
  int32_t key_tile;
  uint32_t start;          // of the job on the line
};

// To the next job on the line.
VFB_HD void advance(const Plan &p, Place &a) {
  a.start += jobs_length(p, a.seq, a.tile + 1) - jobs_length(p, a.seq, a.tile);
  a.key_tile = 0;
  if (++a.tile < a.seq.tiles) return;
  a.tile = 0;
  if (++a.group < p.groups) return;
  a.group = 0;
  do {
    if (++a.b >= num_seqs(p)) return;
    a.seq = sequence(p, a.b);
  } while (a.seq.tiles == 0);
}

// Floor of a / b for quotients below 2^20, from an fp32 estimate.
VFB_HD uint32_t quotient(uint32_t a, uint32_t b) {
  uint32_t q = static_cast<uint32_t>(static_cast<float>(a) / static_cast<float>(b));
  if (static_cast<uint64_t>(q) * b > a) --q;
  else if (static_cast<uint64_t>(q + 1) * b <= a) ++q;
  return q;
}

// The place for a cut at x, `in` units into sequence b.
VFB_HD Place place_at(const Plan &p, int32_t b, uint32_t in, uint32_t x) {
  Place a;
  a.b = b;
  a.seq = sequence(p, b);
  a.key_tile = 0;
  const uint32_t line = jobs_length(p, a.seq, a.seq.tiles);
  const uint32_t group = quotient(in, line);
  in -= group * line;
  uint32_t lo = 0, hi = a.seq.tiles;  // the last tile that starts at or before `in`
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (jobs_length(p, a.seq, mid) <= in) lo = mid;
    else hi = mid;
  }
  a.group = static_cast<int32_t>(group);
  a.tile = static_cast<int32_t>(lo);
  in -= jobs_length(p, a.seq, lo);
  a.start = x - in;
  if (in > overhead_units(p)) {  // to the nearest border of key tiles
    const uint32_t key = (in - overhead_units(p)) << p.unit_shift;
    a.key_tile = static_cast<int32_t>((key + (1u << p.key_shift) / 2) >> p.key_shift);
    if (a.key_tile > 0 && a.key_tile >= tiles_of(p, a.seq, a.tile)) advance(p, a);
  }
  return a;
}

// Length of a share: an equal part, but not below SHARE as long as every job has
// a block.
VFB_HD uint32_t share_length(const Plan &p, uint32_t length, uint32_t jobs) {
  const uint32_t equal = static_cast<uint32_t>(static_cast<float>(length) * 1.000001f / static_cast<float>(p.blocks)) + 1;
  const uint32_t job = static_cast<uint32_t>(static_cast<float>(length) / static_cast<float>(jobs > 0 ? jobs : 1));
  const uint32_t least = units(p, static_cast<uint32_t>(SHARE));
  const uint32_t want = job < least ? job : least;
  return equal > want ? equal : want;
}

// Where a block's share begins, for the join: `inside` a job (its earlier part
// belongs to blocks before), and which one.
struct Record {
  uint32_t start;    // of the job on the line
  int32_t row0;      // its first query row
  int32_t group, count, inside;
};

// The share of a block, piece by piece.
class Share {
 public:
  // The share of `block`; `record` is for the join.  On the device the answer is
  // lane 0's, which goes through the share alone.
  VFB_HD void init(const Plan &p, int32_t block, Record &record) {
    block_ = block;
    first_ = true;
    more_ = false;
    record = Record{0, 0, 0, 0, 0};
    const int32_t n = num_seqs(p);
    uint32_t length = 0, jobs = 0;
#ifdef __CUDA_ARCH__
    const int lane = threadIdx.x & 31;
    uint32_t own = 0;
    for (int32_t b = lane; b < n; b += 32) {
      const Seq s = sequence(p, b);
      own = line_length(p, s);  // stays in hand when the lanes have a sequence each
      length += own;
      jobs += s.tiles;
    }
    __syncwarp();
    length = __reduce_add_sync(0xffffffffu, length);
    jobs = __reduce_add_sync(0xffffffffu, jobs) * p.groups;
    const uint32_t share = share_length(p, length, jobs);
    // lanes 0-15 look for the share's beginning, lanes 16-31 for its end
    uint32_t x = (block + (lane >> 4)) * share, in = x;
    int32_t at = -1;
    if (static_cast<uint64_t>(block) * share >= length) return;
    for (int32_t b0 = 0; b0 < n; b0 += 32) {
      if (n > 32) own = b0 + lane < n ? line_length(p, sequence(p, b0 + lane)) : 0u;
      const uint32_t upto = warp_upto(own);
      const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
      const uint32_t in0 = __shfl_sync(0xffffffffu, in, 0), in1 = __shfl_sync(0xffffffffu, in, 16);
      const unsigned hit0 = __ballot_sync(0xffffffffu, in0 < upto), hit1 = __ballot_sync(0xffffffffu, in1 < upto);
      const unsigned hit = lane < 16 ? hit0 : hit1;
      const uint32_t before = __shfl_sync(0xffffffffu, upto - own, hit ? __ffs(hit) - 1 : 0);
      if (at < 0) {
        if (hit) at = b0 + __ffs(hit) - 1;
        in -= hit ? before : all;
      }
    }
    Place a;
    a.start = length;
    a.key_tile = 0;
    a.b = n;
    if (at >= 0) a = place_at(p, at, in, x);
    __syncwarp();
    end_start_ = __shfl_sync(0xffffffffu, a.start, 16);
    end_tile_ = __shfl_sync(0xffffffffu, a.key_tile, 16);
    at_ = a;
#else
    for (int32_t b = 0; b < n; ++b) {
      const Seq s = sequence(p, b);
      length += line_length(p, s);
      jobs += s.tiles;
    }
    const uint32_t share = share_length(p, length, jobs * p.groups);
    if (static_cast<uint64_t>(block) * share >= length) return;
    for (int end = 0; end < 2; ++end) {
      const uint32_t x = (block + end) * share;
      uint32_t in = x;
      Place a;
      a.start = length;
      a.key_tile = 0;
      a.b = n;
      for (int32_t b = 0; b < n; ++b) {
        const uint32_t own = line_length(p, sequence(p, b));
        if (in < own) {
          a = place_at(p, b, in, x);
          break;
        }
        in -= own;
      }
      if (end == 0) at_ = a;
      end_start_ = a.start;
      end_tile_ = a.key_tile;
    }
#endif
    if (at_.b >= n) return;
    more_ = before_end();
    const int32_t rows0 = at_.tile * p.job_tokens;
    record = Record{at_.start, at_.seq.q0 + rows0, at_.group, rows_to(p, at_.seq, at_.tile) - rows0, at_.key_tile > 0};
  }

  VFB_HD bool next(const Plan &p, Segment &s) {
    if (!more_) return false;
    s.seq = at_.seq;
    s.b = at_.b;
    s.group = at_.group;
    s.tile = at_.tile;
    const int32_t tiles = tiles_of(p, s.seq, s.tile);
    const bool last = at_.start == end_start_;
    s.t0 = at_.key_tile;
    s.t1 = last ? end_tile_ : tiles;
    s.slot = s.t0 == 0 && s.t1 == tiles ? -1 : 2 * block_ + (first_ ? 0 : 1);
    first_ = false;
    more_ = false;
    if (!last) {
      advance(p, at_);
      more_ = at_.b < num_seqs(p) && before_end();
    }
    return true;
  }

  // Nothing left.
  VFB_HD bool empty() const { return !more_; }

 private:
  VFB_HD bool before_end() const {
    return at_.start < end_start_ || (at_.start == end_start_ && at_.key_tile < end_tile_);
  }

  bool first_, more_;
  int32_t block_, end_tile_;
  uint32_t end_start_;
  Place at_;
};

// ---- joining the pieces ------------------------------------------------------------
// Cut c (1 <= c < blocks) is the first one inside its job when its record says
// `inside` and the one before does not lie inside the same job.  The job's
// pieces are then slot join_first() and the slots 2 * c, 2 * (c + 1), ... as long as
// the records stay inside the same job (a share cut to nothing leaves -inf in
// its slot).
VFB_HD bool join_starts(const Record &before, const Record &here) {
  return here.inside && !(before.inside && before.start == here.start);
}
VFB_HD int32_t join_first(const Record &before, const Record &here, int32_t c) {
  return 2 * (c - 1) + (before.start == here.start ? 0 : 1);
}

}  // namespace attn
}  // namespace vfb
