// csrc/last_uses.h by itself (test_last_uses.py): a loop's waits and those behind it see every use of every barrier once, with its parity.
#include "last_uses.h"

#include <cstdio>
#include <vector>

#define CHECK(c) do { if (!(c)) { std::printf("failed: %s\n", #c); return 1; } } while (0)

int main() {
    for (int slots = 1; slots <= 4; slots++)
        for (int uses = 0; uses <= 40; uses++) {
            std::vector<int> seen(uses, 0);
            for (int u = slots; u < uses; u++) seen[u - slots]++;                    // what the loop itself waits for
            int last = -1;
            bool right = true;
            CHECK(ib::last_uses(uses, slots, [&](int barrier, unsigned parity) {
                int use = -1;                                                          // the barrier's phase of that parity that is not yet seen
                for (int u = barrier; u < uses; u += slots)
                    if (!seen[u]) { use = u; break; }
                right = right && use >= 0 && parity == (unsigned(use / slots) & 1u) && use > last;
                if (use >= 0) seen[use]++;
                last = use;
                return true;
            }));
            CHECK(right);
            for (int u = 0; u < uses; u++) CHECK(seen[u] == 1);
            int calls = 0;
            const bool all = ib::last_uses(uses, slots, [&](int, unsigned) { calls++; return false; });
            CHECK(uses == 0 ? all && calls == 0 : !all && calls == 1);                 // a wait that runs out ends the rest
        }
    return 0;
}
