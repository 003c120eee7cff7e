// Replay of the log-probability kernel's schedule: for every CTA of a call, the
// waits and arrivals of its copying warp and of its computing warps, in order,
// until both are through or neither can go on.
#include <vector>

#include "logprobs_plan.cuh"

using namespace mtpb;

namespace {

enum Op { kMeet, kIssue, kTake };  // the floor's barrier; tile g into the ring; tile g out of it

struct Program {
  std::vector<Op> ops;
  size_t at = 0;
  bool done() const { return at == ops.size(); }
};

struct Call {
  long long rows, ld;
  int V, es, k;
  uintptr_t base;
  LpPlan plan;
  int vecs(long long t) const {  // of tile t of all rows' tiles
    const long long row = t / plan.tiles;
    return lp_tile_vecs(lp_cols(base + uintptr_t(row) * ld * es, V, es).nvec, int(t - row * plan.tiles));
  }
};

// The copying warp. `skip`: a copy passes over the tiles without vectors to the next that has some.
Program copier(const Call& c, long long t0, long long t1, int stages, bool skip) {
  Program p;
  long long t2 = t0;
  auto copy = [&] {
    while (t2 < t1) {
      const int n = c.vecs(t2++);
      if (n > 0) {
        p.ops.push_back(kIssue);
        return;
      }
      if (!skip) return;
    }
  };
  for (int i = 0; i < stages; ++i) copy();
  for (long long t = t0; t < t1;) {
    const int n = int(c.plan.tiles - t % c.plan.tiles < t1 - t ? c.plan.tiles - t % c.plan.tiles : t1 - t);
    t += n;
    for (int i = 0; i < n; ++i) {
      if (c.k && lp_refloor(c.k, i, n - 1)) p.ops.push_back(kMeet);
      copy();
    }
  }
  return p;
}

Program computer(const Call& c, long long t0, long long t1) {
  Program p;
  for (long long t = t0; t < t1;) {
    const int n = int(c.plan.tiles - t % c.plan.tiles < t1 - t ? c.plan.tiles - t % c.plan.tiles : t1 - t);
    for (int i = 0; i < n; ++i, ++t) {
      if (c.vecs(t) > 0) p.ops.push_back(kTake);
      if (c.k && lp_refloor(c.k, i, n - 1)) p.ops.push_back(kMeet);
    }
  }
  return p;
}

}  // namespace

extern "C" {

int lp_vecs_of(int nvec, int tile) { return lp_tile_vecs(nvec, tile); }

// CTAs of the call that come to a stop; *ctas_out: how many it has, *run_out: tiles a CTA.
int lp_blocked(long long rows, int V_local, int V_plan, long long ld, int base, int elem_bytes, int k, int skip, int* ctas_out,
               int* run_out) {
  const Call c{rows, ld, V_local, elem_bytes, k, uintptr_t(base), lp_plan(rows, V_plan, elem_bytes)};
  const int stages = k ? kLpStages<true> : kLpStages<false>;
  const long long total = rows * c.plan.tiles;
  int blocked = 0, ctas = 0;
  for (long long t0 = 0; t0 < total; t0 += c.plan.run, ++ctas) {
    const long long t1 = t0 + c.plan.run < total ? t0 + c.plan.run : total;
    Program a = copier(c, t0, t1, stages, skip != 0), b = computer(c, t0, t1);
    int issued = 0, taken = 0;
    for (bool moved = true; moved;) {
      moved = false;
      while (!a.done() && a.ops[a.at] == kIssue && issued - taken < stages) ++a.at, ++issued, moved = true;
      while (!b.done() && b.ops[b.at] == kTake && taken < issued) ++b.at, ++taken, moved = true;
      if (!a.done() && !b.done() && a.ops[a.at] == kMeet && b.ops[b.at] == kMeet) ++a.at, ++b.at, moved = true;
    }
    if (!a.done() || !b.done() || issued != taken) ++blocked;
  }
  *ctas_out = ctas;
  *run_out = c.plan.run;
  return blocked;
}

// 0 when the plan covers every tile of every row once with at most `parts` parts a row, or what is wrong.
int lp_plan_wrong(long long rows, int V, int elem_bytes) {
  const LpPlan p = lp_plan(rows, V, elem_bytes);
  const long long total = rows * p.tiles, ctas = (total + p.run - 1) / p.run;
  if (p.tiles < 1 || p.run < 1 || ctas > 3 * 148 || (long long)p.tiles * kLpTile * (16 / elem_bytes) < V) return 1;
  for (long long r = 0; r < rows; ++r) {
    const long long a = r * p.tiles / p.run, b = ((r + 1) * p.tiles - 1) / p.run;
    if (p.first(r) != a || p.count(r) != b - a + 1 || p.count(r) > p.parts) return 2;
  }
  return 0;
}
}
