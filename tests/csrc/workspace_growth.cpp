// Prints the size that a workspace of argv[1] bytes, beside one of argv[2], is
// given where argv[3] bytes are free, and then the sizes that were asked for.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../arclight_amd/csrc/workspace_growth.hpp"

int main(int, char ** argv) {
    const size_t bytes = strtoull(argv[1], nullptr, 0), held = strtoull(argv[2], nullptr, 0), free_bytes = strtoull(argv[3], nullptr, 0);
    std::vector<size_t> asked;
    const size_t got = grow_workspace(bytes, held, [&](size_t n) {
        asked.push_back(n);
        return n <= free_bytes;
    });
    printf("%zu", got);
    for (size_t n : asked) printf(" %zu", n);
    printf("\n");
    return 0;
}
