// A lookup that fails is tried again, one that succeeds is kept (csrc/lookup.h).
#include "lookup.h"

int main() {
    static int there, other;
    int calls = 0;
    ib::Lookup<int*> l;
    auto get = [&](int* result) {
        return l.get([&] {
            ++calls;
            return result;
        });
    };
    if (get(nullptr) || get(nullptr) || calls != 2) return 1;
    if (get(&there) != &there || calls != 3) return 2;
    if (get(&other) != &there || get(nullptr) != &there || calls != 3) return 3;
    return 0;
}
