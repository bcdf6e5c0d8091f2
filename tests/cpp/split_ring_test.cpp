// The barriers of the tree kernel with one query tile (paged_tensor.cu, SPLIT): the programs of its
// roles, made from the kernel's own order of tiles and bookkeeping of looks, run in random orders.  Every
// wait must be for a barrier's present phase or the one before (a wait goes by a phase's parity: further
// off it would pass too early or never), a tile must lie in its slot while it is used, and all roles must
// come to their ends.
#include <cstdio>
#include <cstdlib>
#include <deque>
#include <random>
#include <string>
#include <vector>

#include "paged_ring.h"

using ib::Looks;
using ib::tile_order;

struct Bar {
    int count, pending, done = 0;
};

enum Kind { WAIT, ARRIVE, ASYNC, MMA, FILL, USE, WRITE_RECENT, READ_RECENT, PARITY };
struct Op {
    Kind kind;
    int bar, n;      // barrier; the phase waited for, or a parity
    int slot, tile;  // FILL and USE: what lies in a slot; RECENT: its entry and key tile
};
struct Seg {
    int n;
    unsigned careful;  // a bit per key tile
};

static int fails = 0;
static void fail(const char* what) {
    if (fails++ < 5) printf("%s\n", what);
}

struct Model {
    int slots, recent;
    bool f32;
    std::vector<Bar> bars;
    std::vector<std::vector<Op>> roles;
    int add(int count) {
        bars.push_back(Bar{count, count});
        return (int)bars.size() - 1;
    }
};

// kv_full, kv_empty, v_there per slot; q_full, s_full, p (half, full), o_full, seg_done per group; x_there, x_done
static Model build(int slots, bool f32, const std::vector<Seg>& segs, int recent, bool forget_looks) {
    Model m;
    m.slots = slots, m.recent = recent, m.f32 = f32;
    const int fill_warps = f32 ? 6 : 3;
    std::vector<int> full(slots), empty(slots), there(slots);
    for (int i = 0; i < slots; ++i) full[i] = m.add(f32 ? fill_warps : 1), empty[i] = m.add(1), there[i] = m.add(1);
    int raw_full[2], raw_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], seg_done[2];
    const int q_full = m.add(1), x_there = m.add(1), x_done = m.add(1), done = m.add(1);
    for (int i = 0; i < 2; ++i) {
        raw_full[i] = m.add(1), raw_empty[i] = m.add(fill_warps);
        s_full[i] = m.add(1), p_half[i] = m.add(1), p_full[i] = m.add(1), o_full[i] = m.add(1), seg_done[i] = m.add(1);
    }
    // the two groups
    for (int t = 0; t < 2; ++t) {
        std::vector<Op> r;
        int tiles = 0, firsts = 0, q_used = -1, exchanges = 0, seen = 0;
        for (const Seg& g : segs) {
            const int first = seen;
            seen += g.n;
            if (t == 1) {
                if (q_used >= 0) r.push_back({WAIT, s_full[0], q_used});
                q_used = -1;
                if (g.n > 0) r.push_back({ARRIVE, q_full});
            }
            firsts += g.n / 2;
            if (g.n > 0 && !(g.n & 1)) q_used = firsts - 1;
            const int j0 = 1 - t;
            auto add_o = [&](int j) {
                r.push_back({WAIT, o_full[t], tiles - 1});
                r.push_back({READ_RECENT, 0, 0, (first + j) % recent, first + j});
            };
            for (int j = j0;; j += 2) {
                if (j > j0) add_o(j - 2);
                if (j >= g.n) break;
                r.push_back({WAIT, s_full[t], tiles++});
                r.push_back({READ_RECENT, 0, 0, (first + j) % recent, first + j});
                if (!f32) r.push_back({ARRIVE, p_half[t]});
                r.push_back({ARRIVE, p_full[t]});
            }
            if (g.n > j0) r.push_back({ARRIVE, seg_done[t]});
            if (g.n > 0) {
                if (t == 1) r.push_back({ARRIVE, x_there});
                else r.push_back({WAIT, x_there, exchanges++}), r.push_back({ARRIVE, x_done});
            }
        }
        m.roles.push_back(r);
    }
    {  // the MMAs
        std::vector<Op> r;
        int half = 0, n_q = 0, n_s[2] = {0, 0}, n_d[2] = {0, 0}, exchanges = 0, base = 0;
        unsigned owed = 0;
        bool x_owed = false;
        for (const Seg& g : segs) {
            if (g.n == 0) continue;
            for (int j = -2; j < g.n; ++j) {
                const bool s = j + 2 < g.n;
                const int t = ~j & 1, hv = half, hs = half + (j >= 0 ? 1 : 0);
                if (j >= 0) r.push_back({WAIT, full[hv % slots], hv / slots});
                if (s) r.push_back({WAIT, full[hs % slots], hs / slots});
                if (j >= 0) {
                    if (j == 0) {
                        for (int k = 0; k < 2; ++k)
                            if (owed >> k & 1) r.push_back({WAIT, seg_done[k], n_d[k]++});
                        if (x_owed) r.push_back({WAIT, x_done, exchanges++});
                    }
                    const int n = n_s[t]++;
                    if (!f32) r.push_back({WAIT, p_half[t], n});
                    r.push_back({WAIT, p_full[t], n});
                    r.push_back({USE, 0, 0, hv % slots, 2 * (base + j) + 1});
                    r.push_back({MMA, o_full[t]});
                    r.push_back({MMA, empty[hv % slots]});
                }
                if (s) {
                    if (j == -2) r.push_back({WAIT, q_full, n_q++});
                    r.push_back({USE, 0, 0, hs % slots, 2 * (base + j + 2)});
                    r.push_back({MMA, s_full[t]});
                    r.push_back({MMA, empty[hs % slots]});
                }
                half += (j >= 0) + s;
            }
            owed = g.n > 1 ? 3 : 2;
            x_owed = true;
            base += g.n;
        }
        r.push_back({MMA, done});
        r.push_back({WAIT, done, 0});
        m.roles.push_back(r);
    }
    if (!f32) {  // three warps that see to the tiles in turn
        for (int lw = 0; lw < 3; ++lw) {
            std::vector<Op> r;
            Looks looks;
            int half = 0, base = 0;
            for (const Seg& g : segs) {
                for (int e = 0; e < 2 * g.n; ++e, ++half) {
                    const int of = tile_order<true>(e, g.n), j = of >> 1, kv = of & 1, slot = half % slots;
                    const bool look = kv == 1 && (g.careful >> j & 1);
                    if (ib::tile_owner(half) != lw) {
                        if (look && !forget_looks) looks.take(slot);
                        continue;
                    }
                    if (half >= slots) r.push_back({WAIT, empty[slot], half / slots - 1});
                    if (kv == 0) r.push_back({WRITE_RECENT, 0, 0, (base + j) % recent, base + j});
                    r.push_back({FILL, 0, 0, slot, 2 * (base + j) + kv});
                    r.push_back({ASYNC, look ? there[Looks::bar(slot)] : full[slot]});
                    if (look) {
                        r.push_back({PARITY, there[Looks::bar(slot)], looks.take(slot)});
                        r.push_back({ARRIVE, full[slot]});
                    }
                }
                base += g.n;
            }
            m.roles.push_back(r);
        }
    } else {  // one warp brings in, six split
        std::vector<Op> r;
        int issued = 0;
        for (const Seg& g : segs) {
            for (int e = 0; e < 2 * g.n; ++e) {
                const int of = tile_order<true>(e, g.n), n = issued + (of >> 1), kv = of & 1;
                if (n > 0) r.push_back({WAIT, raw_empty[kv], n - 1});
                if (kv == 0) r.push_back({WRITE_RECENT, 0, 0, n % recent, n});
                r.push_back({ASYNC, raw_full[kv]});
            }
            issued += g.n;
        }
        m.roles.push_back(r);
        for (int sw = 0; sw < 6; ++sw) {
            std::vector<Op> r;
            int half = 0, base = 0;
            for (const Seg& g : segs) {
                for (int e = 0; e < 2 * g.n; ++e, ++half) {
                    const int of = tile_order<true>(e, g.n), slot = half % slots, kv = of & 1;
                    r.push_back({WAIT, raw_full[kv], base + (of >> 1)});
                    if (half >= slots) r.push_back({WAIT, empty[slot], half / slots - 1});
                    if (sw == 0) r.push_back({FILL, 0, 0, slot, 2 * base + of});
                    r.push_back({ARRIVE, full[slot]});
                    r.push_back({ARRIVE, raw_empty[kv]});
                }
                base += g.n;
            }
            m.roles.push_back(r);
        }
    }
    return m;
}

// One random order; false where some role never ends.
static bool run(Model m, std::mt19937& rng) {
    std::vector<size_t> at(m.roles.size(), 0);
    std::vector<int> in_slot(m.slots, -1), recent(m.recent, -1), read(m.recent, 0);
    std::deque<int> tensor;      // arrivals that follow the MMAs, in order
    std::vector<int> on_its_way;  // and those of copies, in any order
    auto arrive = [&](int b) {
        Bar& x = m.bars[b];
        if (--x.pending == 0) ++x.done, x.pending = x.count;
    };
    for (;;) {
        std::vector<int> can;
        bool open = !tensor.empty() || !on_its_way.empty();
        for (size_t i = 0; i < m.roles.size(); ++i) {
            if (at[i] == m.roles[i].size()) continue;
            open = true;
            const Op& o = m.roles[i][at[i]];
            if (o.kind == WAIT) {
                const int done = m.bars[o.bar].done;
                if (done != o.n && done != o.n + 1) fail("a wait for a phase that is not near");
                if ((done & 1) == (o.n & 1)) continue;
            }
            if (o.kind == PARITY && (m.bars[o.bar].done & 1) == o.n) continue;
            can.push_back((int)i);
        }
        if (!open) return true;
        const int n_can = (int)can.size() + !tensor.empty() + !on_its_way.empty();
        if (n_can == 0) return false;
        int k = (int)(rng() % n_can);
        if (k < (int)can.size()) {
            const Op& o = m.roles[can[k]][at[can[k]]++];
            switch (o.kind) {
                case ARRIVE: arrive(o.bar); break;
                case ASYNC: on_its_way.push_back(o.bar); break;
                case MMA: tensor.push_back(o.bar); break;
                case FILL: in_slot[o.slot] = o.tile; break;
                case USE:
                    if (in_slot[o.slot] != o.tile) fail("another tile in the slot");
                    break;
                case WRITE_RECENT: recent[o.slot] = o.tile; break;
                case READ_RECENT:
                    if (recent[o.slot] != o.tile) fail("another key tile's masks");
                    break;
                default: break;
            }
        } else if (k == (int)can.size() && !tensor.empty()) {
            arrive(tensor.front());
            tensor.pop_front();
        } else {
            const size_t i = rng() % on_its_way.size();
            arrive(on_its_way[i]);
            on_its_way.erase(on_its_way.begin() + i);
        }
    }
}

int main(int argc, char** argv) {
    const bool forget = argc > 1 && std::string(argv[1]) == "forget";
    std::mt19937 rng(1);
    // every K and V tile once, K before V, and in the order of the MMAs
    for (int n = 1; n < 60; ++n) {
        std::vector<int> want;
        for (int j = -2; j < n; ++j) {
            if (j >= 0) want.push_back(2 * j + 1);
            if (j + 2 < n) want.push_back(2 * (j + 2));
        }
        for (int e = 0; e < 2 * n; ++e)
            if (tile_order<true>(e, n) != want[e] || tile_order<false>(e, n) != e) fail("another order");
    }
    int stuck = 0, runs = 0;
    for (int round = 0; round < 400; ++round) {
        std::vector<Seg> segs;
        for (int i = 1 + (int)(rng() % 5); i > 0; --i) {
            const int n = (int)(rng() % (rng() % 4 ? 5 : 14));
            segs.push_back({n, (unsigned)rng() & (unsigned)rng()});
        }
        const int f32 = round & 1, slots = f32 ? (round & 2 ? 4 : 2) : (round & 2 ? 6 : 5);
        const Model m = build(slots, f32, segs, 8, forget);
        for (int k = 0; k < 20 && fails == 0; ++k, ++runs) stuck += !run(m, rng);
        if (forget && (stuck || fails)) break;
    }
    printf("%d runs, %d stuck, %d faults\n", runs, stuck, fails);
    return forget ? !(stuck || fails) : stuck || fails;
}
