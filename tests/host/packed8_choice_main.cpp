// Reads lines "gemm CUS M N K" and "dw CUS ROWS IN OUT" and prints for each the kernel that om_gemm8 or om_linear_bwd_x8 takes (a
// tile's number, or "thin NW MR"), the parts that k is split into and the blocks of 128 in the longest and the last of them.
#include <cstdio>
#include <cstring>

#include "../../onemodel-csharp_amd/csrc/om_gemm8_choose.hpp"

int main() {
    char what[8];
    int cus, a, b, c;
    while (std::scanf("%7s %d %d %d %d", what, &cus, &a, &b, &c) == 5) {
        const bool gemm = !std::strcmp(what, "gemm");
        const int blocks = (int)(((int64_t)(gemm ? c : a) + 127) / 128);
        if (gemm)
            if (const om8::Thin t = om8::choose_thin(cus, a, b, blocks); t.mr) {
                std::printf("thin %d %d 1 %d %d\n", t.nw, t.mr, blocks, blocks);
                continue;
            }
        const om8::Choice ch = gemm ? om8::choose_product(cus, a, b, blocks, INT64_C(128) * blocks)
                                    : om8::choose_dw(cus, c, b, blocks, INT64_C(128) * blocks);
        int per, parts;
        om8::split_blocks(blocks, ch.splits, per, parts);
        std::printf("%s %d 0 %d %d %d\n", gemm ? "tile" : "dw", ch.tile, parts, per, blocks - (parts - 1) * per);
    }
    return 0;
}
