// Compares overlap() with the bytes themselves for random operands of a small
// memory; prints how many pairs share a byte, lie in one another's gaps, and were
// answered wrongly ("yes" for operands of odd strides may also be careful).
#include <cstdio>
#include <cstring>
#include <random>
#include <set>

#include "../../arclight_amd/csrc/overlap.hpp"

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return lo + (int) (rng() % (unsigned) (hi - lo + 1)); };
    int shared = 0, gaps = 0, wrong = 0, careful = 0;
    for (int trial = 0; trial < 200000; ++trial) {
        al_tensor t[2];
        std::set<uintptr_t> bytes[2];
        bool odd = false;
        for (int k = 0; k < 2; ++k) {
            memset(&t[k], 0, sizeof(t[k]));
            t[k].data = (void *) (uintptr_t) (4096 + pick(0, 150));
            t[k].nb[0] = 4;
            uint64_t extent = 4;
            for (int i = 0; i < 4; ++i) {
                t[k].ne[i] = pick(0, 9) ? pick(1, 3) : trial % 50 ? 1 : 0;
                if (i) {
                    const int how = pick(0, 9);
                    t[k].nb[i] = how == 0 ? 0 : how == 1 ? pick(1, 40) : extent + (how < 5 ? 0 : pick(1, 30));
                    odd |= how < 2;
                }
                extent += (t[k].ne[i] > 1 ? t[k].ne[i] - 1 : 0) * t[k].nb[i];
            }
            if (pick(0, 3) == 0) std::swap(t[k].ne[1], t[k].ne[3]), std::swap(t[k].nb[1], t[k].nb[3]);
            for (int i = 0; i < t[k].ne[3]; ++i)
                for (int j = 0; j < t[k].ne[2]; ++j)
                    for (int r = 0; r < t[k].ne[1]; ++r)
                        for (int e = 0; e < 4 * t[k].ne[0]; ++e)
                            bytes[k].insert((uintptr_t) t[k].data + i * t[k].nb[3] + j * t[k].nb[2] + r * t[k].nb[1] + e);
        }
        bool want = false;
        for (uintptr_t b : bytes[0]) want |= bytes[1].count(b) > 0;
        const bool got = overlap(ByteSet(t[0], 4), ByteSet(t[1], 4));
        if (got != overlap(ByteSet(t[1], 4), ByteSet(t[0], 4))) ++wrong;
        if (got && !want && odd) ++careful;
        else wrong += got != want;
        shared += want;
        gaps += !want && !bytes[0].empty() && !bytes[1].empty() && *bytes[0].begin() <= *bytes[1].rbegin() && *bytes[1].begin() <= *bytes[0].rbegin();
    }
    printf("%d %d %d %d\n", shared, gaps, wrong, careful);
    return 0;
}
