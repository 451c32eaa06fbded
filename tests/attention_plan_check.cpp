// Walks the attention kernel's work order on the CPU: every key tile of every
// job is visited exactly once, pieces use distinct slots, and the join finds
// exactly the pieces of each job that was cut.
//
// Reads cases from standard input, one a line:
//   split blocks key_shift band_keys unit_shift grid groups job_tokens causal has_offsets batch total_q total_k  cu_q...  cu_k...  lengths_or_-1...
// and prints "ok <cases> <cut jobs>" or the first contradiction.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <tuple>
#include <vector>

#include "attention_plan.h"

using namespace vfb::attn;

static long long read_int() {
  long long x;
  if (std::scanf("%lld", &x) != 1) std::exit(3);
  return x;
}

int main() {
  long long cases = 0, cuts = 0, split;
  while (std::scanf("%lld", &split) == 1) {
    Plan p = {};
    p.blocks = static_cast<int32_t>(read_int());
    p.key_shift = static_cast<int32_t>(read_int());
    p.band_keys = static_cast<int32_t>(read_int());
    p.unit_shift = static_cast<int32_t>(read_int());
    const long long grid = read_int();
    p.groups = static_cast<int32_t>(read_int());
    set_job_tokens(p, static_cast<int32_t>(read_int()));
    p.causal = static_cast<int32_t>(read_int());
    const long long offsets = read_int();
    p.batch = static_cast<int32_t>(read_int());
    p.total_q = static_cast<int32_t>(read_int());
    p.total_k = static_cast<int32_t>(read_int());
    std::vector<int32_t> cu_q, cu_k, lengths;
    for (int i = 0; i <= p.batch; ++i) cu_q.push_back(static_cast<int32_t>(read_int()));
    for (int i = 0; i <= p.batch; ++i) cu_k.push_back(static_cast<int32_t>(read_int()));
    for (int i = 0; i < p.batch; ++i) lengths.push_back(static_cast<int32_t>(read_int()));
    if (offsets) {
      p.cu_q = cu_q.data();
      p.cu_k = cu_k.data();
    }
    if (lengths[0] >= 0) p.len_k = lengths.data();

    using Job = std::tuple<int, int, int>;  // sequence, group, tile
    std::map<Job, std::set<int>> done;
    std::map<int, std::pair<Job, std::pair<int, int>>> pieces;  // slot -> job, key tiles
    std::set<int> empty_slots;
    std::vector<Record> records;
    const int n = static_cast<int>(split ? p.blocks : grid);
    std::map<Job, bool> whole;
    for (int block = 0; block < n; ++block) {
      Share share;
      uint32_t next = block;  // of the whole jobs
      if (split) {
        Record record;
        share.init(p, block, record);
        records.push_back(record);
        if (share.empty()) empty_slots.insert(2 * block);
      }
      Segment s;
      std::map<std::pair<int, int>, int> last;  // tile of a head group in a sequence
      while (split ? share.next(p, s) : whole_job(p, next, s)) {
        next += static_cast<uint32_t>(grid);
        if (!split && p.causal && grid == 1) {  // in a head group's sequence the longest come first
          const auto at = last.emplace(std::make_pair(s.b, s.group), s.seq.tiles).first;
          if (s.tile != at->second - 1) return std::printf("order\n"), 1;
          at->second = s.tile;
        }
        const Job job{s.b, s.group, s.tile};
        if (s.seq.tiles <= s.tile || s.tile < 0 || s.group < 0 || s.group >= p.groups) return std::printf("bad job\n"), 1;
        const int tiles = tiles_of(p, s.seq, s.tile);
        if (s.t0 < 0 || s.t1 > tiles || s.t1 < s.t0) return std::printf("bad tiles %d %d of %d\n", s.t0, s.t1, tiles), 1;
        for (int t = s.t0; t < s.t1; ++t)
          if (!done[job].insert(t).second) return std::printf("tile twice\n"), 1;
        done[job];
        if (s.slot < 0) {
          if (s.t0 != 0 || s.t1 != tiles || whole.count(job)) return std::printf("whole job wrong\n"), 1;
          whole[job] = true;
        } else {
          if (!split || s.slot >= 2 * p.blocks || !pieces.emplace(s.slot, std::make_pair(job, std::make_pair(s.t0, s.t1))).second)
            return std::printf("slot %d\n", s.slot), 1;
          if (whole.count(job)) return std::printf("piece of a whole job\n"), 1;
        }
      }
    }
    for (int b = 0; b < num_seqs(p); ++b) {
      const Seq s = sequence(p, b);
      for (int g = 0; g < p.groups; ++g)
        for (int t = 0; t < s.tiles; ++t) {
          const auto it = done.find(Job{b, g, t});
          if (it == done.end() || static_cast<int>(it->second.size()) != tiles_of(p, s, t))
            return std::printf("job %d %d %d not done\n", b, g, t), 1;
        }
    }
    std::map<Job, std::set<int>> by_job;
    for (const auto &x : pieces) by_job[x.second.first].insert(x.first);
    std::set<Job> joined;
    for (int c = 1; split && c < p.blocks; ++c) {
      const Record &r = records[c], &before = records[c - 1];
      if (!join_starts(before, r)) continue;
      std::set<int> slots{join_first(before, r, c)};
      for (int i = c; i < p.blocks && records[i].inside && records[i].start == r.start; ++i) slots.insert(2 * i);
      std::set<int> real;
      std::set<Job> jobs;
      for (int x : slots) {
        const auto it = pieces.find(x);
        if (it != pieces.end()) {
          real.insert(x);
          jobs.insert(it->second.first);
        } else if (!empty_slots.count(x)) {
          return std::printf("join reads slot %d that nothing wrote\n", x), 1;
        }
      }
      if (jobs.size() != 1) return std::printf("join of several jobs\n"), 1;
      const Job job = *jobs.begin();
      if (!joined.insert(job).second) return std::printf("joined twice\n"), 1;
      if (real != by_job[job]) return std::printf("join misses pieces\n"), 1;
      const Seq s = sequence(p, std::get<0>(job));
      const int32_t rows0 = std::get<2>(job) * p.job_tokens;
      if (r.row0 != s.q0 + rows0 || r.group != std::get<1>(job) || r.count != min32(p.job_tokens, s.nq - rows0))
        return std::printf("record of another job\n"), 1;
      ++cuts;
    }
    for (const auto &x : by_job)
      if (!joined.count(x.first)) return std::printf("pieces never joined\n"), 1;
    ++cases;
  }
  std::printf("ok %lld %lld\n", cases, cuts);
  return 0;
}
