// Test driver for q35::PageMap (qwen3.5sharp_amd/csrc/page_map.h), built with
// g++ by tests/test_page_map.py.  First line: n_seqs max_rows n_pages
// page_rows.  Then one command per line, one answer per line (the Result's
// number, or a value):
//   map <seq> <first> <n> <page...>    unmap <seq> <first> <n>
//   len <seq> <length>                 usable <seq> <tokens>
//   page <seq> <i>
#include <cstdio>
#include <cstring>
#include <vector>

#include "page_map.h"

int main() {
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    int s, r, p, g;
    if (std::scanf("%d %d %d %d", &s, &r, &p, &g) != 4) return 2;
    q35::PageMap m(s, r, p, g);
    char cmd[32];
    while (std::scanf("%31s", cmd) == 1) {
        int a = 0, b = 0, n = 0;
        if (!std::strcmp(cmd, "map") || !std::strcmp(cmd, "unmap")) {
            if (std::scanf("%d %d %d", &a, &b, &n) != 3) return 2;
            std::vector<int> ids(n > 0 ? n : 1);
            const bool set = cmd[0] == 'm';
            for (int i = 0; set && i < n; ++i)
                if (std::scanf("%d", &ids[i]) != 1) return 2;
            std::printf("%d\n", (int)m.map(a, b, n, set ? ids.data() : nullptr));
        } else if (!std::strcmp(cmd, "len")) {
            if (std::scanf("%d %d", &a, &b) != 2) return 2;
            m.set_length(a, b);
            std::printf("%d\n", m.length(a));
        } else if (!std::strcmp(cmd, "usable")) {
            if (std::scanf("%d %d", &a, &b) != 2) return 2;
            std::printf("%d\n", (int)m.usable(a, b));
        } else if (!std::strcmp(cmd, "page")) {
            if (std::scanf("%d %d", &a, &b) != 2) return 2;
            std::printf("%d\n", m.page(a, b));
        } else {
            return 2;
        }
    }
    return 0;
}
