// The library's runtime record (runtime.hpp): which raster a kernel with a number of its own takes.
#include <cstdio>

#include "../../backup_1_amd/csrc/runtime.hpp"

using decx_hip::Runtime;

int main() {
    int bad = 0;
    Runtime rt;
    bad += rt.group_m != 8 || rt.group_m_or(6) != 6;
    for (const char* nothing : {(const char*)nullptr, "", "0", "-3", "many"}) {
        rt.ask_group_m(nothing);
        bad += rt.group_m != 8 || rt.group_m_or(6) != 6;
    }
    for (int v : {8, 6, 1, 40}) {                               // 8: the default, asked for
        char text[8];
        std::snprintf(text, sizeof(text), "%d", v);
        Runtime asked;
        asked.ask_group_m(text);
        bad += asked.group_m != v || asked.group_m_or(6) != v;
    }
    std::printf("%d failure(s)\n", bad);
    return bad;
}
