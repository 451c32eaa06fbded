// The work order of the packed attention kernel, shared with its CPU test.
//
// A job is one tile of query rows of one sequence for one group of heads that
// read the same keys; its keys come in key tiles of 64 or 128 (Plan::key_shift).  Two orders:
//
// * whole jobs (`split` false): job i of the list goes to block i (or is
//   strided over the blocks), every job by itself;
// * even shares (`split` true): all jobs laid end to end, a job as long as its
//   keys plus OVERHEAD (about what loading its queries and storing its rows
//   costs, in keys), and the line cut into equal parts, one for a block.  Cuts
//   are moved to whole key tiles.  A block's first and last job may then be
//   pieces; every piece leaves its rows and their log-sum-exp in a slot of the
//   workspace (2 * block for a block's first job, 2 * block + 1 for another),
//   and a second kernel joins them in the order of the blocks.
//
// Only totals are known on the host: lengths are device data, so the functions
// here run on the device, on one whole warp of a block with uniform arguments
// (the lanes read the sequences side by side).  On the host they run as plain
// loops.  Places on the line are integers below 2^53: quotients are taken in
// fp64 and corrected, several times faster than 64-bit integer division.
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

VFB_HD int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }
VFB_HD int64_t max64(int64_t a, int64_t b) { return a > b ? a : b; }

struct Plan {
  const int32_t *cu_q, *cu_k, *len_k;  // device arrays, cu_q NULL: one sequence of all rows
  int64_t total_q, total_k;
  int32_t batch;
  int32_t groups;      // head groups: jobs for one tile of rows
  int32_t job_tokens;  // query tokens in a job
  int32_t causal;
  int32_t blocks;      // blocks that even shares are cut for, at most
  int32_t key_shift;   // log2 of the keys in a key tile
};

// Sequence b: its rows and keys, clamped to the buffers.  b == batch stands for
// the rows behind the last sequence, which have no keys.
struct Seq {
  int64_t q0, k0;
  int32_t nq, nk;
  int32_t tiles;
};

VFB_HD int32_t num_seqs(const Plan &p) { return p.cu_q == nullptr ? 1 : p.batch + 1; }

VFB_HD Seq sequence(const Plan &p, int32_t b) {
  Seq s;
  int64_t q1, k1;
  if (p.cu_q == nullptr) {
    s.q0 = 0;
    q1 = p.total_q;
    s.k0 = 0;
    k1 = p.total_k;
  } else {
    s.q0 = min64(max64(p.cu_q[b], 0), p.total_q);
    if (b == p.batch) {
      q1 = p.total_q;
      s.k0 = k1 = 0;
    } else {
      q1 = min64(max64(p.cu_q[b + 1], s.q0), p.total_q);
      const int32_t *cu_k = p.cu_k != nullptr ? p.cu_k : p.cu_q;
      s.k0 = min64(max64(cu_k[b], 0), p.total_k);
      k1 = min64(max64(cu_k[b + 1], s.k0), p.total_k);
    }
  }
  if (p.len_k != nullptr && b < p.batch) k1 = s.k0 + min64(max64(p.len_k[b], 0), k1 - s.k0);
  s.nq = static_cast<int32_t>(q1 - s.q0);
  s.nk = static_cast<int32_t>(k1 - s.k0);
  s.tiles = static_cast<int32_t>((static_cast<int64_t>(s.nq) + p.job_tokens - 1) / p.job_tokens);
  return s;
}

// Keys that the last of `rows` leading query rows of a sequence sees.
VFB_HD int32_t keys_seen(const Plan &p, const Seq &s, int64_t rows) {
  if (!p.causal) return s.nk;
  return static_cast<int32_t>(min64(max64(rows + s.nk - s.nq, 0), s.nk));
}

// ---- even shares: lengths of jobs --------------------------------------------
// A causal job counts the keys its last row would see were nk >= nq: never
// fewer than it sees, and summed over the tiles in closed form.
VFB_HD int64_t job_keys(const Plan &p, const Seq &s, int64_t tile) {
  if (!p.causal) return s.nk;
  return max64(static_cast<int64_t>(s.nk) - s.nq, 0) + min64((tile + 1) * p.job_tokens, s.nq);
}

// Length of the first `tiles` jobs of one head group of the sequence.
VFB_HD int64_t jobs_length(const Plan &p, const Seq &s, int64_t tiles) {
  if (!p.causal) return tiles * (OVERHEAD + s.nk);
  if (tiles <= 0) return 0;
  const int64_t before = max64(static_cast<int64_t>(s.nk) - s.nq, 0);
  const int64_t full = tiles - 1;
  return tiles * (OVERHEAD + before) + p.job_tokens * (full * (full + 1) / 2) +
         min64(tiles * p.job_tokens, s.nq);
}

// Moves a cut at `off` inside a job of `keys` keys to a key tile's border or to
// one of the job's ends.
VFB_HD int64_t snap(const Plan &p, int64_t off, int64_t keys) {
  const int64_t at = off <= OVERHEAD ? 0 : (off - OVERHEAD + (1 << p.key_shift) / 2) >> p.key_shift << p.key_shift;
  if (at == 0) return 0;
  return OVERHEAD + min64(at, keys);
}

// ---- scans over the sequences --------------------------------------------------
// Floor of a / b for 0 <= a < 2^53, b > 0, with the fp64 inverse of b.
VFB_HD int64_t quotient(int64_t a, int64_t b, double inverse) {
  int64_t q = static_cast<int64_t>(static_cast<double>(a) * inverse);
  if (q * b > a) --q;
  else if ((q + 1) * b <= a) ++q;
  return q;
}

VFB_HD int64_t line_length(const Plan &p, const Seq &s) { return jobs_length(p, s, s.tiles) * p.groups; }

#ifdef __CUDA_ARCH__
__device__ __forceinline__ int64_t warp_inclusive(int64_t sum) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += t;
  }
  return sum;
}
#endif

struct Totals {
  int64_t length, jobs;
};

VFB_HD Totals totals(const Plan &p) {
  Totals t = {0, 0};
#ifdef __CUDA_ARCH__
  for (int32_t b = threadIdx.x & 31; b < num_seqs(p); b += 32) {
    const Seq s = sequence(p, b);
    t.length += line_length(p, s);
    t.jobs += s.tiles;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    t.length += __shfl_xor_sync(0xffffffffu, t.length, o);
    t.jobs += __shfl_xor_sync(0xffffffffu, t.jobs, o);
  }
#else
  for (int32_t b = 0; b < num_seqs(p); ++b) {
    const Seq s = sequence(p, b);
    t.length += line_length(p, s);
    t.jobs += s.tiles;
  }
#endif
  t.jobs *= p.groups;
  return t;
}

// The sequence in which position `x` lies on the line (LINE) or in the list of
// jobs; `x` becomes the position inside it.
template <bool LINE>
VFB_HD int32_t locate(const Plan &p, int64_t &x) {
#ifdef __CUDA_ARCH__
  for (int32_t b0 = 0; b0 < num_seqs(p); b0 += 32) {
    const int32_t b = b0 + (threadIdx.x & 31);
    int64_t own = 0;
    if (b < num_seqs(p)) {
      const Seq s = sequence(p, b);
      own = LINE ? line_length(p, s) : static_cast<int64_t>(s.tiles) * p.groups;
    }
    const int64_t inclusive = warp_inclusive(own);
    const unsigned hit = __ballot_sync(0xffffffffu, x < inclusive);
    if (hit) {
      const int at = __ffs(hit) - 1;
      x -= __shfl_sync(0xffffffffu, inclusive - own, at);
      return b0 + at;
    }
    x -= __shfl_sync(0xffffffffu, inclusive, 31);
  }
#else
  for (int32_t b = 0; b < num_seqs(p); ++b) {
    const Seq s = sequence(p, b);
    const int64_t own = LINE ? line_length(p, s) : static_cast<int64_t>(s.tiles) * p.groups;
    if (x < own) return b;
    x -= own;
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

// Even shares: a place on the line, moved to where it may be cut.
struct Place {
  Seq seq;
  int32_t b, group, tile;
  int64_t off;    // inside the job
  int64_t keys;   // of the job
  int64_t start;  // of the job on the line
};

VFB_HD Place place_at(const Plan &p, int64_t x) {
  Place a;
  int64_t in = x;
  a.b = locate<true>(p, in);
  a.seq = sequence(p, a.b < 0 ? 0 : a.b);
  const int64_t line = jobs_length(p, a.seq, a.seq.tiles);
  a.group = static_cast<int32_t>(quotient(in, line, 1.0 / static_cast<double>(line)));
  in -= a.group * line;
  int32_t lo = 0, hi = a.seq.tiles;  // the last tile that starts at or before `in`
  while (hi - lo > 1) {
    const int32_t mid = lo + (hi - lo) / 2;
    if (jobs_length(p, a.seq, mid) <= in) lo = mid;
    else hi = mid;
  }
  a.tile = lo;
  const int64_t raw = in - jobs_length(p, a.seq, lo);
  a.keys = job_keys(p, a.seq, lo);
  a.start = x - raw;
  a.off = snap(p, raw, a.keys);
  return a;
}

VFB_HD int32_t share_blocks(const Plan &p, int64_t length, int64_t jobs) {
  return static_cast<int32_t>(max64(1, min64(p.blocks, max64(jobs, length / SHARE))));
}

// Cut c of `blocks` on a line of `length` before it is moved.
VFB_HD int64_t cut(int64_t length, int32_t blocks, int32_t c) {
  if (c >= blocks) return length;
  return static_cast<int64_t>(static_cast<double>(length) * c / blocks);
}

// Where a block's share begins, for the join: `inside` a job (its earlier part
// belongs to blocks before), and which one.
struct Record {
  int64_t start;    // of the job on the line
  int64_t row0;     // its first query row
  int32_t group, count, inside, reserved;
};

class Order {
 public:
  // Whole jobs `block`, `block + step`, ...
  VFB_HD void init_whole(const Plan &p, int32_t block, int32_t step) {
    split_ = false;
    next_ = block;
    step_ = step;
    end_ = INT64_MAX;
  }

  // The share of `block`; `record` is for the join.
  VFB_HD void init_share(const Plan &p, int32_t block, Record &record) {
    split_ = true;
    const Totals t = totals(p);
    const int32_t blocks = share_blocks(p, t.length, t.jobs);
    next_ = end_ = 0;
    block_ = block;
    first_ = true;
    record = Record{-1, 0, 0, 0, 0, 0};
    if (t.length == 0 || block >= blocks) return;
    at_ = place_at(p, cut(t.length, blocks, block));
    next_ = at_.start + at_.off;
    end_ = t.length;
    if (block + 1 < blocks) {
      const Place e = place_at(p, cut(t.length, blocks, block + 1));
      end_ = e.start + e.off;
    }
    if (at_.off == OVERHEAD + at_.keys) advance(p);
    if (at_.b >= num_seqs(p)) return;
    const int64_t rows0 = static_cast<int64_t>(at_.tile) * p.job_tokens;
    record = Record{at_.start, at_.seq.q0 + rows0, at_.group,
                    static_cast<int32_t>(min64(p.job_tokens, at_.seq.nq - rows0)), at_.off > 0, 0};
  }

  VFB_HD bool next(const Plan &p, Segment &s) {
    if (next_ >= end_) return false;
    if (!split_) {
      int64_t in = next_;
      next_ += step_;
      s.b = locate<false>(p, in);
      if (s.b < 0) return false;
      s.seq = sequence(p, s.b);
      // jobs are fewer than 2^31
      s.group = static_cast<int32_t>(static_cast<uint32_t>(in) / static_cast<uint32_t>(s.seq.tiles));
      const int32_t i = static_cast<int32_t>(in) - s.group * s.seq.tiles;
      s.tile = p.causal ? s.seq.tiles - 1 - i : i;  // causal: the longest first
      s.t0 = 0;
      s.t1 = tiles_of(p, s.seq, s.tile);
      s.slot = -1;
      return true;
    }
    const int64_t job_end = at_.start + OVERHEAD + at_.keys;
    const int64_t stop = min64(job_end, end_);
    s.seq = at_.seq;
    s.b = at_.b;
    s.group = at_.group;
    s.tile = at_.tile;
    const int32_t tiles = tiles_of(p, s.seq, s.tile);
    s.t0 = at_.off == 0 ? 0 : static_cast<int32_t>(min64((at_.off - OVERHEAD) >> p.key_shift, tiles));
    s.t1 = stop == job_end ? tiles : static_cast<int32_t>(min64((stop - at_.start - OVERHEAD) >> p.key_shift, tiles));
    s.slot = at_.off == 0 && stop == job_end ? -1 : 2 * block_ + (first_ ? 0 : 1);
    first_ = false;
    next_ = stop;
    if (next_ < end_) advance(p);
    return true;
  }

  VFB_HD bool empty() const { return next_ >= end_; }

  static VFB_HD int32_t tiles_of(const Plan &p, const Seq &s, int32_t tile) {
    const int32_t keys = keys_seen(p, s, min64((static_cast<int64_t>(tile) + 1) * p.job_tokens, s.nq));
    return static_cast<int32_t>((static_cast<int64_t>(keys) + (1 << p.key_shift) - 1) >> p.key_shift);
  }

 private:
  VFB_HD void advance(const Plan &p) {  // to the next job on the line
    at_.start += OVERHEAD + at_.keys;
    at_.off = 0;
    if (++at_.tile == at_.seq.tiles) {
      at_.tile = 0;
      if (++at_.group == p.groups) {
        at_.group = 0;
        do {
          if (++at_.b >= num_seqs(p)) return;
          at_.seq = sequence(p, at_.b);
        } while (at_.seq.tiles == 0);
      }
    }
    at_.keys = job_keys(p, at_.seq, at_.tile);
  }

  bool split_, first_;
  int32_t block_, step_;
  int64_t next_, end_;
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
