// Calls the entry points of the 8-bit tensors with sizes on both sides of what they take, on a context whose device does not exist:
// what a call takes goes as far as making that device current and no farther. Prints one line per call, "name status message".
#include <climits>
#include <cstdio>

#include "../../onemodel-csharp_amd/csrc/om_internal.hpp"

static om_ctx ctx;
static void say(const char *name, om_status s) { std::printf("%s %d %s\n", name, s, s ? ctx.err.c_str() : ""); }

int main() {
    alignas(16) float x[64] = {};
    alignas(16) uint8_t q[4096] = {};
    ctx.device = 1 << 20;
    ctx.num_cus = 256;

    // k, and the rows of a weight gradient
    const int k = (1 << 27) - 128;
    say("take-gemm-k", om_gemm8(&ctx, 100, 100, k, q, q, nullptr, x, 100, 0));
    say("om_gemm8-k", om_gemm8(&ctx, 100, 100, k + 1, q, q, nullptr, x, 100, 0));
    say("take-gemm-one-k", om_gemm8(&ctx, 1, 1, k, q, q, nullptr, x, 1, 0));
    say("om_gemm8-one-k", om_gemm8(&ctx, 1, 1, k + 1, q, q, nullptr, x, 1, 0));
    say("take-dw-rows", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, k, 4, 4, 0, 0, 0));
    say("om_linear_bwd_x8-rows", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, k + 1, 4, 4, 0, 0, 0));
    say("take-dw-out", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, 4, 4, (1 << 26) - 1, 0, 0, 0));
    say("om_linear_bwd_x8-out", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, 4, 4, 1 << 26, 0, 0, 0));
    // columns of a product of few rows
    say("take-gemm-n", om_gemm8(&ctx, 1, (1 << 28) - 16, 128, q, q, nullptr, x, 1 << 28, 0));
    say("om_gemm8-n", om_gemm8(&ctx, 1, (1 << 28) - 15, 128, q, q, nullptr, x, 1 << 28, 0));

    // 2^28 blocks (two of one row, or two rows of one, to a wavefront), for the transpose 2^22 squares of 128
    const int narrow = (1 << 28) - 16, wide = (1 << 24) - 1;
    say("take-pack-narrow", om_pack8(&ctx, x, 1, narrow, 1, q, nullptr));
    say("om_pack8-narrow", om_pack8(&ctx, x, 1, narrow + 1, 1, q, nullptr));
    say("take-pack-wide", om_pack8(&ctx, x, 2048, wide, 2048, q, nullptr));
    say("om_pack8-wide", om_pack8(&ctx, x, 2048, wide + 1, 2048, q, nullptr));
    say("take-pack-t", om_pack8(&ctx, x, 1, (1 << 29) - 128, 1, nullptr, q));
    say("om_pack8-t", om_pack8(&ctx, x, 1, (1 << 29) - 127, 1, nullptr, q));
    say("take-pack-both", om_pack8(&ctx, x, 1 << 18, (1 << 18) - 128, 1 << 18, q, q));
    say("om_pack8-both", om_pack8(&ctx, x, 1 << 18, (1 << 18) - 127, 1 << 18, q, q));
    say("take-unpack", om_unpack8(&ctx, q, x, 1, narrow, 1, 0));
    say("om_unpack8-unpack", om_unpack8(&ctx, q, x, 1, narrow + 1, 1, 0));
    say("take-gelu", om_gelu_fwd_x8(&ctx, x, x, q, narrow, 128));
    say("om_gelu_fwd_x8-gelu", om_gelu_fwd_x8(&ctx, x, x, q, narrow + 1, 128));
    say("take-gelu-bwd", om_gelu_bwd_x8(&ctx, x, q, x, narrow, 128, 1));
    say("om_gelu_bwd_x8-gelu", om_gelu_bwd_x8(&ctx, x, q, x, narrow + 1, 128, 1));

    // rows of LayerNorm by its kernels' widths
    const struct { int cols, rows; } norm[] = {{1, (1 << 26) - 4}, {1024, (1 << 26) - 4}, {1025, (1 << 24) - 1}, {4096, (1 << 24) - 1},
                                               {4097, (1 << 23) - 1}, {8192, (1 << 23) - 1}, {8193, (1 << 22) - 1}, {20000, (1 << 22) - 1}};
    for (const auto &n : norm) {
        say("take-norm", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, n.rows, n.cols, 1e-5f));
        say("om_layernorm_fwd_x8-norm", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, n.rows + 1, n.cols, 1e-5f));
    }
    say("take-norm-bwd", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, INT_MAX, 8192, 0, 0));
    say("take-norm-bwd-long", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, (1 << 24) - 1, 8193, 0, 0));
    say("om_layernorm_bwd_x8-long", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1 << 24, 8193, 0, 0));
    say("take-norm-bwd-wide", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1, 65535 * 1024, 0, 0));
    say("om_layernorm_bwd_x8-wide", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1, 65535 * 1024 + 1, 0, 0));

    // no rows: outputs that are kept need no device, outputs that are zeroed need the context's own
    say("ok-norm-no-rows", om_layernorm_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, nullptr, x, x, 0, 8, 0, 1));
    say("take-norm-no-rows", om_layernorm_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, nullptr, x, x, 0, 8, 0, 0));
    say("ok-linear-no-rows", om_linear_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, x, x, 0, 4, 4, 0, 1, 1));
    say("take-linear-no-rows", om_linear_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, x, x, 0, 4, 4, 0, 0, 1));
    say("take-linear-no-rows-db", om_linear_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, nullptr, x, 0, 4, 4, 0, 0, 0));
    return 0;
}
