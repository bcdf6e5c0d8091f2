// The factors of a segment's rows in the tree kernel with one query tile (paged_tensor.cu, SPLIT, FP16
// pages): two buffers, which the second group of softmax warps writes with the segment's q and both groups
// read, the first one up to its end.  Every order of the two groups, the MMAs' warp and the tensor
// core's arrivals is gone through, for all batches of up to four segments of up to three key tiles (K and V
// are always there: that allows more orders, not fewer).  A read must find its own segment's factors.
// "all": segments without key tiles are counted too; some order then reads another segment's.
#include <cstdio>
#include <set>
#include <string>
#include <vector>

#include "paged_ring.h"

using ib::ScaleTurn;

enum Kind { WAIT, ARRIVE, MMA, WRITE, READ };
struct Op {
    Kind kind;
    int at, n;  // barrier, and the phase waited for; buffer, and the segment
};
using Role = std::vector<Op>;

// barriers; s_full, p_full, o_full, seg_done: of the group
enum { Q_FULL, X_THERE, X_DONE, S_FULL, P_FULL = S_FULL + 2, O_FULL = P_FULL + 2, SEG_DONE = O_FULL + 2, BARS = SEG_DONE + 2 };

static std::vector<Role> build(const std::vector<int>& segs, bool all) {
    std::vector<Role> roles;
    for (int t = 0; t < 2; ++t) {
        Role r;
        ScaleTurn turn;
        int tiles = 0, firsts = 0, q_used = -1, exchanges = 0;
        for (int i = 0; i < (int)segs.size(); ++i) {
            const int n = segs[i], j0 = 1 - t;
            if (t == 1) {
                if (q_used >= 0) r.push_back({WAIT, S_FULL, q_used});
                q_used = -1;
                if (n > 0) r.push_back({WRITE, turn.buffer(), i}), r.push_back({ARRIVE, Q_FULL});
            }
            firsts += n / 2;
            if (n > 0 && !(n & 1)) q_used = firsts - 1;
            for (int j = j0;; j += 2) {
                if (j > j0) r.push_back({WAIT, O_FULL + t, tiles - 1});
                if (j >= n) break;
                r.push_back({WAIT, S_FULL + t, tiles++});
                if (j == j0) r.push_back({READ, turn.buffer(), i});
                r.push_back({ARRIVE, P_FULL + t});
            }
            if (n > j0) r.push_back({ARRIVE, SEG_DONE + t});
            if (n > 0) {
                if (t == 1) {
                    r.push_back({ARRIVE, X_THERE});
                } else {
                    r.push_back({WAIT, X_THERE, exchanges++});
                    r.push_back({READ, turn.buffer(), i});
                    r.push_back({ARRIVE, X_DONE});
                }
            }
            turn.next(all ? 1 : n);
        }
        roles.push_back(r);
    }
    Role r;  // the MMAs
    int n_q = 0, n_s[2] = {0, 0}, n_d[2] = {0, 0}, exchanges = 0;
    unsigned owed = 0;
    bool x_owed = false;
    for (int n : segs) {
        if (n == 0) continue;
        for (int j = -2; j < n; ++j) {
            const int t = ~j & 1;
            if (j >= 0) {
                if (j == 0) {
                    for (int k = 0; k < 2; ++k)
                        if (owed >> k & 1) r.push_back({WAIT, SEG_DONE + k, n_d[k]++});
                    if (x_owed) r.push_back({WAIT, X_DONE, exchanges++});
                }
                r.push_back({WAIT, P_FULL + t, n_s[t]++});
                r.push_back({MMA, O_FULL + t});
            }
            if (j + 2 < n) {
                if (j == -2) r.push_back({WAIT, Q_FULL, n_q++});
                r.push_back({MMA, S_FULL + t});
            }
        }
        owed = n > 1 ? 3 : 2;
        x_owed = true;
    }
    roles.push_back(r);
    return roles;
}

// What an order has come to: places of the roles, MMAs that are done, segments in the buffers.  Phases follow.
struct State {
    int at[3], done, held[2];
    bool operator<(const State& o) const {
        for (int i = 0; i < 3; ++i)
            if (at[i] != o.at[i]) return at[i] < o.at[i];
        if (done != o.done) return done < o.done;
        if (held[0] != o.held[0]) return held[0] < o.held[0];
        return held[1] < o.held[1];
    }
};

static int wrong = 0, stuck = 0;

static void search(const std::vector<Role>& roles) {
    // before[i][p][b]: arrivals of role i on barrier b before its place p; MMAs in their order
    std::vector<std::vector<std::vector<int>>> before(3);
    std::vector<int> mmas, issued{0};
    for (int i = 0; i < 3; ++i) {
        std::vector<int> n(BARS, 0);
        before[i].push_back(n);
        for (const Op& o : roles[i]) {
            if (o.kind == ARRIVE) ++n[o.at];
            if (o.kind == MMA) mmas.push_back(o.at);
            if (i == 2) issued.push_back((int)mmas.size());
            before[i].push_back(n);
        }
    }
    std::vector<std::vector<int>> by_mma(1, std::vector<int>(BARS, 0));
    for (int b : mmas) by_mma.push_back(by_mma.back()), ++by_mma.back()[b];
    std::set<State> seen;
    std::vector<State> open{State{{0, 0, 0}, 0, {-1, -1}}};
    seen.insert(open[0]);
    while (!open.empty()) {
        const State s = open.back();
        open.pop_back();
        bool moved = false, end = true;
        auto go = [&](const State& x) {
            moved = true;
            if (seen.insert(x).second) open.push_back(x);
        };
        for (int i = 0; i < 3; ++i) {
            if (s.at[i] == (int)roles[i].size()) continue;
            end = false;
            const Op& o = roles[i][s.at[i]];
            State x = s;
            ++x.at[i];
            if (o.kind == WAIT) {
                int phases = by_mma[s.done][o.at];
                for (int k = 0; k < 3; ++k) phases += before[k][s.at[k]][o.at];
                if (phases != o.n && phases != o.n + 1) ++wrong;  // its parity would lie
                if ((phases & 1) == (o.n & 1)) continue;
            }
            if (o.kind == WRITE) x.held[o.at] = o.n;
            if (o.kind == READ && s.held[o.at] != o.n) ++wrong;
            go(x);
        }
        if (s.done < issued[s.at[2]]) {
            end = false;
            State x = s;
            ++x.done;
            go(x);
        }
        if (!moved && !end) ++stuck;
    }
}

int main(int argc, char** argv) {
    const bool all = argc > 1 && std::string(argv[1]) == "all";
    int batches = 0;
    for (int n = 1; n <= 4; ++n)
        for (int code = 0; code < 1 << 2 * n; ++code, ++batches) {
            std::vector<int> segs;
            for (int i = 0; i < n; ++i) segs.push_back(code >> 2 * i & 3);
            search(build(segs, all));
        }
    printf("%d batches, %d faults, %d orders without an end\n", batches, wrong, stuck);
    return all ? wrong == 0 : wrong || stuck;
}
