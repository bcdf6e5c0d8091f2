// Every order of events in the FP16 copies of attention over pages (csrc/paged_tensor.cu, TMA
// boxes): warp 9 fills ring slots with K and V tiles in turn, V tiles of `careful` key tiles
// complete on a look barrier that the three copying warps wait for before they arrive on the slot's
// full barrier; the MMAs take full slots in order and give them back.  mbarriers are modelled as
// the hardware counts them (arrivals, bytes, phases; a wait tests a parity).  The search goes
// through all interleavings and reports a state that nothing can leave (a lost wait) or a wait that
// passes in a phase other than its own.
//
//   copy_ring_test            the kernel's assignment of barriers (csrc/paged_ring.h): 0 on success
//   copy_ring_test shared     one barrier for all slots: 0 when the search finds its lost wait
#include <cstdio>
#include <cstring>
#include <set>
#include <vector>

#include "paged_ring.h"

struct SharedLooks {
    uint32_t n = 0;
    static int bar(int) { return 0; }
    int take(int) { return (int)(n++ & 1u); }
};

constexpr int SLOTS = 3, WARPS = 3;

struct Bar {
    int8_t phase = 0, arrivals = 0, bytes = 0;  // of the phase under way; bytes: tiles still to land
};

// A phase ends with its last arrival and its last byte.
static void settle(Bar& b, int count) {
    if (b.arrivals == count && b.bytes == 0) {
        ++b.phase;
        b.arrivals = 0;
    }
}

template <typename L>
struct State {
    Bar full[SLOTS], empty[SLOTS], look[SLOTS];
    int8_t landing[2 * 8];  // of each half: 0 none, 1 under way to its full, 2 to its look barrier
    struct Warp {
        int8_t half, at;  // at: 0 wait for empty, 1 issue, 2 wait for the look, 3 arrive
        int8_t looked[SLOTS];
        L looks;
    } warp[WARPS];
    int8_t mma, in_flight;  // halves taken, given back

    std::vector<int> key() const {
        std::vector<int> k;
        auto put = [&](const Bar& b) { k.push_back((b.phase * 16 + b.arrivals) * 16 + b.bytes); };
        for (int i = 0; i < SLOTS; ++i) put(full[i]), put(empty[i]), put(look[i]);
        for (int x : landing) k.push_back(x);
        for (const Warp& w : warp) {
            k.push_back(w.half * 8 + w.at);
            for (int x : w.looked) k.push_back(x);
        }
        k.push_back(mma), k.push_back(in_flight);
        return k;
    }
};

// Warp 9 leaves wherever one of its waits runs out: every copy of its own that may still be landing
// then has to be among those that it waits for before the CTA ends.
static bool drained(const State<ib::Looks>& s) {
    const auto& me = s.warp[0];
    if (me.at != 0 && me.at != 2) return true;
    ib::Looks looks = me.looks;
    if (me.at == 2) looks.take(me.half % SLOTS);
    bool full[SLOTS] = {}, look[SLOTS] = {};  // waits that cannot pass before the bytes are there
    ib::drain_copies<SLOTS>(
        me.half, me.at == 2, looks,
        [&](int slot, int use) { full[slot] = (s.full[slot].phase & 1) == (use & 1); },
        [&](int slot, int parity) { look[slot] = (s.look[slot].phase & 1) == parity; });
    for (int h = 0; h < 2 * 8; ++h)
        if (s.landing[h] && !(s.landing[h] == 2 ? look[h % SLOTS] : full[h % SLOTS])) return false;
    return true;
}
static bool drained(const State<SharedLooks>&) { return true; }

static bool raw_drained() {
    ib::RawSent sent;
    for (int i = 0, issued = 0; i < 6; ++i) {  // K, V, K, V ...: leaving before each of them
        int k = -1, v = -1;
        sent.drain([&](int kv, int phase) { (kv ? v : k) = phase; });
        if (k != (issued + 1) / 2 - 1 || v != issued / 2 - 1) return false;
        sent.add(i & 1);
        ++issued;
    }
    return true;
}

static bool passes(const Bar& b, int parity) { return (b.phase & 1) != (parity & 1); }

template <typename L>
static int search(int tiles, unsigned careful) {
    using S = State<L>;
    const int halves = 2 * tiles;
    S start{};
    std::set<std::vector<int>> seen;
    std::vector<S> todo{start};
    seen.insert(start.key());
    int bad = 0;
    auto visit = [&](const S& s) {
        if (seen.insert(s.key()).second) todo.push_back(s);
    };
    while (!todo.empty() && !bad) {
        const S s = todo.back();
        todo.pop_back();
        bool moved = false;
        if (!drained(s)) bad = 3;
        for (int w = 0; w < WARPS; ++w) {
            const auto& me = s.warp[w];
            if (me.half == halves) continue;
            const int slot = me.half % SLOTS, use = me.half / SLOTS;
            const bool look = (me.half & 1) && (careful >> (me.half / 2) & 1);
            S n = s;
            auto& to = n.warp[w];
            if (me.at == 0) {
                if (use > 0 && !passes(s.empty[slot], use - 1)) continue;
                if (use > 0 && s.empty[slot].phase != use) bad = 1;
                to.at = w == 0 ? 1 : look ? 2 : 3;
            } else if (me.at == 1) {  // expect the bytes, one arrival, and start the copy
                Bar& b = look ? n.look[L::bar(slot)] : n.full[slot];
                ++b.arrivals, ++b.bytes;
                n.landing[me.half] = look ? 2 : 1;
                to.at = look ? 2 : 3;
            } else if (me.at == 2) {
                L after = me.looks;
                const int parity = after.take(slot), own = me.looked[L::bar(slot)];
                if (!passes(s.look[L::bar(slot)], parity)) continue;
                if (s.look[L::bar(slot)].phase != own + 1) bad = 1;
                to.looks = after;
                ++to.looked[L::bar(slot)];
                to.at = 3;
            } else {
                // warp 9's arrival went with the bytes where the tile completes on the full barrier
                if (w > 0 || look) ++n.full[slot].arrivals;
                settle(n.full[slot], WARPS);
                ++to.half;
                to.at = 0;
            }
            moved = true;
            visit(n);
        }
        for (int h = 0; h < halves; ++h)
            if (s.landing[h]) {
                S n = s;
                Bar& b = s.landing[h] == 2 ? n.look[L::bar(h % SLOTS)] : n.full[h % SLOTS];
                --b.bytes;
                settle(b, s.landing[h] == 2 ? 1 : WARPS);
                n.landing[h] = 0;
                moved = true;
                visit(n);
            }
        if (s.mma < halves && passes(s.full[s.mma % SLOTS], s.mma / SLOTS)) {
            if (s.full[s.mma % SLOTS].phase != s.mma / SLOTS + 1) bad = 1;
            S n = s;
            ++n.mma;
            moved = true;
            visit(n);
        }
        if (s.in_flight < s.mma) {  // the MMAs on a slot are done
            S n = s;
            Bar& b = n.empty[s.in_flight % SLOTS];
            ++b.arrivals;
            settle(b, 1);
            ++n.in_flight;
            moved = true;
            visit(n);
        }
        bool done = s.in_flight == halves;
        for (const auto& w : s.warp) done = done && w.half == halves;
        if (!moved && !done) bad = 2;
    }
    if (bad)
        printf("%d key tiles, careful %x: %s\n", tiles, careful,
               bad == 3   ? "a copy that nobody waits for"
               : bad == 2 ? "a wait that never ends"
                          : "a wait that passes in another phase");
    return bad;
}

int main(int argc, char** argv) {
    const bool shared = argc > 1 && !strcmp(argv[1], "shared");
    int found = !raw_drained();
    for (int tiles = 1; tiles <= 5; ++tiles)
        for (unsigned careful = 0; careful < 1u << tiles; ++careful)
            found += (shared ? search<SharedLooks>(tiles, careful)
                             : search<ib::Looks>(tiles, careful)) != 0;
    printf("%d of the patterns lose a wait\n", found);
    return shared ? found == 0 : found != 0;
}
