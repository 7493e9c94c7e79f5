// The overlap checks of csrc/overlap.h as a program: reads the addresses and
// sizes of a page plan from the command line and prints what it refuses
// ("ok" for nothing); "meet" compares regions_meet with a walk over all bytes.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>

#include "../ai-agent-framework_b200/csrc/overlap.h"

static int walk() {
    long bad = 0, n = 0;
    for (int rows = 1; rows <= 4; rows++)
        for (int width = 1; width <= 5; width++)
            for (int stride = width; stride <= 9; stride++) {
                const uintptr_t at = 40;
                std::set<uintptr_t> held;
                for (int r = 0; r < rows; r++)
                    for (int i = 0; i < width; i++) held.insert(at + r * stride + i);
                const b2::Region b{"b", (void*)at, width, rows, stride};
                for (uintptr_t p = 30; p < 90; p++)
                    for (int len = 0; len <= 6; len++) {
                        bool meets = false;
                        for (int i = 0; i < len; i++) meets |= held.count(p + i) > 0;
                        bad += b2::regions_meet(b2::Region{"a", (void*)p, len}, b) != meets;
                        n++;
                    }
            }
    std::printf("%ld of %ld wrong\n", bad, n);
    return bad != 0;
}

int main(int argc, char** argv) {
    if (argc == 2 && !std::strcmp(argv[1], "meet")) return walk();
    if (argc != 16) return 2;
    auto num = [&](int i) { return std::strtoll(argv[i], nullptr, 0); };
    auto ptr = [&](int i) { return (int32_t*)(uintptr_t)num(i); };
    b2::PagePlanArgs a{};
    a.cached = ptr(1);
    a.fresh = ptr(2);
    a.free_pages = ptr(3);
    a.n_free = ptr(4);
    a.table = ptr(5);
    a.lens = ptr(6);
    a.starts = ptr(7);
    a.slots = (int64_t*)ptr(8);
    a.positions = ptr(9);
    a.token_req = ptr(10);
    a.info = ptr(11);
    a.n_req = (int)num(12);
    a.page_size = 16;
    a.max_pages = (int)num(13);
    a.table_stride = num(14);
    a.max_tokens = (int)num(15);
    const std::string s = b2::page_plan_overlap(a);
    std::printf("%s\n", s.empty() ? "ok" : s.c_str());
    return 0;
}
