// Every order in which the parts of the chunk kernel can meet its barriers, for a few tiles: the expansion of K and of V, the warp
// that issues products, the tensor core that completes them in order, the softmax warps (which meet in a block barrier every tile, so
// they are one here; at each tile they may or may not move their references).  Waits test a parity, as the hardware does.  A wait
// that lets its thread pass before the phase it is meant for, an operand that is not ready or still in use, and a state that
// nothing leaves are faults.
#include <cstdio>
#include <set>
#include <string>
#include <vector>

#include "kv4_chunk_order.h"

using namespace b200lm;

enum Fault { kNone, kEarly, kOperand, kEnd, kStuck };
static const char* kNames[] = {"none", "a wait passed early", "an operand not ready or in use", "the end ahead of the products", "stuck"};

struct State {
  int done[kKcBars] = {};                                  // completed phases
  int ke = 0, ve = 0;                                      // tiles expanded
  int at = 0;                                              // the issuer's step: 0 scores of tile 0, then 2 a tile
  int sx = 0, step = 0, p = 0;                             // the softmax's tile and step of it, tiles of probabilities
  bool q = false, ended = false;
  int issued = 0, finished = 0;                            // products, in order of issue
  std::string key() const {
    std::string s;
    for (int d : done) s += (char)d;
    for (int v : {ke, ve, at, sx, step, p, (int)q, (int)ended, issued, finished}) s += (char)v;
    return s;
  }
};

struct Model {
  int n;
  KcWait end;
  std::vector<int> ops;                                    // j: scores of tile j; -1 - j: O of tile j
  std::set<std::string> seen;
  Fault fault = kNone;

  Model(int n_, KcWait end_) : n(n_), end(end_) {
    ops.push_back(0);
    for (int j = 0; j < n; ++j) {
      if (j + 1 < n) ops.push_back(j + 1);
      ops.push_back(-1 - j);
    }
  }
  int scores_done(const State& s) const { int k = 0; for (int i = 0; i < s.finished; ++i) k += ops[i] >= 0; return k; }
  int o_done(const State& s) const { return s.finished - scores_done(s); }
  bool open(const State& s, KcWait w) const { return (uint32_t)(s.done[w.bar] & 1) != w.parity(); }
  bool pass(const State& s, KcWait w) {                    // true: the thread goes on
    if (!open(s, w)) return false;
    if (s.done[w.bar] <= w.phase) fault = kEarly;
    return true;
  }

  // All states that one step leads to.
  std::vector<State> next(const State& s) {
    std::vector<State> out;
    auto add = [&](const State& t) { out.push_back(t); };
    if (!s.q) { State t = s; t.q = true; ++t.done[kKcQReady]; add(t); }
    if (s.ke < n && (s.ke < 2 || pass(s, kc_empty(kKcKEmpty, s.ke)))) {
      if (s.ke >= 2 && scores_done(s) < s.ke - 1) fault = kOperand;                      // the stage is still read
      State t = s; ++t.done[kc_stage(kKcKFull, s.ke)]; ++t.ke; add(t);
    }
    if (s.ve < n && (s.ve < 2 || pass(s, kc_empty(kKcVEmpty, s.ve)))) {
      if (s.ve >= 2 && o_done(s) < s.ve - 1) fault = kOperand;
      State t = s; ++t.done[kc_stage(kKcVFull, s.ve)]; ++t.ve; add(t);
    }
    if (s.at == 0 && pass(s, {kKcQReady, 0}) && pass(s, kc_full(kKcKFull, 0))) { State t = s; t.at = 1; ++t.issued; add(t); }
    if (s.at > 0 && s.at <= 2 * n) {
      const int j = (s.at - 1) / 2;
      if (s.at % 2) {
        if (j + 1 == n) { State t = s; ++t.at; add(t); }
        else if (pass(s, kc_full(kKcKFull, j + 1)) && (j == 0 || pass(s, kc_o(j - 1)))) { State t = s; ++t.at; ++t.issued; add(t); }
      } else if (pass(s, kc_full(kKcVFull, j)) && pass(s, kc_full(kKcPFull, j))) {
        State t = s; ++t.at; ++t.issued; add(t);
      }
    }
    if (s.finished < s.issued) {
      const int op = ops[s.finished];
      State t = s;
      ++t.finished;
      if (op >= 0) {
        if (s.ke <= op || (op >= 2 && o_done(s) < op - 1)) fault = kOperand;             // over the probabilities of tile op - 2
        ++t.done[kc_stage(kKcSFull, op)];
        ++t.done[kc_stage(kKcKEmpty, op)];
      } else {
        const int j = -1 - op;
        if (s.ve <= j || s.p <= j) fault = kOperand;
        ++t.done[kKcOFull];
        ++t.done[kc_stage(kKcVEmpty, j)];
        if (j + 1 == n) ++t.done[kKcODone];
      }
      add(t);
    }
    if (s.sx < n) {
      const int j = s.sx;
      if (s.step == 0 && pass(s, kc_full(kKcSFull, j))) {
        if (scores_done(s) <= j) fault = kOperand;
        for (int moved = 0; moved <= (j > 0); ++moved) { State t = s; t.step = 1 + moved; add(t); }
      }
      if (s.step == 2 && pass(s, kc_o(j - 1))) {
        if (o_done(s) != j) fault = kOperand;                                            // O is read and written back
        State t = s; t.step = 1; add(t);
      }
      if (s.step == 1) { State t = s; t.step = 0; ++t.sx; ++t.p; ++t.done[kc_stage(kKcPFull, j)]; add(t); }
    } else if (!s.ended && s.q && open(s, end)) {
      if (s.finished < (int)ops.size()) fault = kEnd;
      else if (s.done[end.bar] <= end.phase) fault = kEarly;
      State t = s; t.ended = true; add(t);
    }
    return out;
  }
  Fault run() {
    std::vector<State> todo{State()};
    while (!todo.empty()) {
      const State s = todo.back();
      todo.pop_back();
      if (!seen.insert(s.key()).second) continue;
      const std::vector<State> to = next(s);
      if (fault != kNone) return fault;
      if (to.empty() && !(s.ended && s.finished == (int)ops.size())) return kStuck;
      todo.insert(todo.end(), to.begin(), to.end());
    }
    return kNone;
  }
};

int main() {
  for (int n = 1; n <= 9; ++n) {
    Model m(n, kc_end());
    const Fault f = m.run();
    if (f != kNone) { printf("%d tiles: %s\n", n, kNames[f]); return 1; }
  }
  // The model has to see what an end that waits for the last O by the parity of the loop's barrier would do.
  for (int n = 2; n <= 9; ++n)
    if (Model(n, kc_o(n - 1)).run() != kEnd) { printf("%d tiles: the end by parity was not found out\n", n); return 1; }
  printf("ok\n");
  return 0;
}
