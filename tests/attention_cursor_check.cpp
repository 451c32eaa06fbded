// Walks the attention kernel's list of whole jobs on the CPU the way blocks do, from where
// each last was, and compares every job with a search from the beginning.
//
// Reads: sequences blocks groups job_tokens, and the sequences' lengths; prints "ok <jobs>
// <sequences passed over>" or the first difference.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "attention_plan.h"

using namespace vfb::attn;

static long long read_int() {
  long long x;
  if (std::scanf("%lld", &x) != 1) std::exit(3);
  return x;
}

static bool same(const Segment &a, const Segment &b) {
  return a.b == b.b && a.group == b.group && a.tile == b.tile && a.t0 == b.t0 && a.t1 == b.t1 && a.slot == b.slot &&
         a.seq.q0 == b.seq.q0 && a.seq.k0 == b.seq.k0 && a.seq.nq == b.seq.nq && a.seq.nk == b.seq.nk;
}

int main() {
  const int n = static_cast<int>(read_int()), blocks = static_cast<int>(read_int());
  Plan p = {};
  p.groups = static_cast<int32_t>(read_int());
  set_job_tokens(p, static_cast<int32_t>(read_int()));
  p.batch = n;
  p.causal = 1;
  p.key_shift = 6;
  p.band_keys = 1000;
  std::vector<int32_t> cu(n + 1, 0);
  for (int i = 0; i < n; ++i) cu[i + 1] = cu[i] + static_cast<int32_t>(read_int());
  p.cu_q = cu.data();
  p.total_q = p.total_k = cu[n] + 7;
  uint32_t jobs = 0;
  for (int b = 0; b < num_seqs(p); ++b) jobs += static_cast<uint32_t>(sequence(p, b).tiles) * p.groups;
  long long passed = 0;
  for (int block = 0; block < blocks; ++block) {
    Cursor at{0, 0};
    uint32_t x = block;
    for (int i = 0;; ++i) {
      Segment s = {}, want = {};
      const Cursor before = at;
      const bool more = whole_job(p, x, s, at);
      passed += at.b >= before.b ? at.b - before.b : at.b;
      if (more != (x < jobs)) return std::printf("job %u of %u\n", x, jobs), 1;
      if (n <= 3000 && (whole_job(p, x, want) != more || (more && !same(s, want)))) return std::printf("job %u differs\n", x), 1;
      if (!more) break;
      // now and then a job that lies before the last one: the order is not promised
      x = n <= 3000 && i % 7 == 6 && x > 40 ? x - 40 : x + blocks;
      if (i > 4 * static_cast<int>(jobs)) break;
    }
  }
  std::printf("ok %u %lld\n", jobs, passed);
  return 0;
}
