// Calls the entry points of the 8-bit tensors with arguments they must refuse (or calls that have nothing to do), on a context
// without a device: every check runs before anything is launched or allocated. Prints one line per call, "name status
// message".
#include <climits>
#include <cstdio>

#include "../../onemodel-csharp_amd/csrc/om_internal.hpp"

static om_ctx ctx;
static void say(const char *name, om_status s) {
    std::printf("%s %d %s%s\n", name, s, s ? ctx.err.c_str() : "", ctx.scratch || ctx.scratch2 ? " DEVICE" : "");
}

int main() {
    alignas(16) float x[64] = {};
    alignas(16) uint8_t q[4096] = {};
    uint8_t *off = q + 8;  // not a multiple of 16 bytes
    ctx.device = 0;
    ctx.num_cus = 256;
    const int big = INT_MAX;

    say("pack-rows", om_pack8(&ctx, x, 8, -1, 8, q, nullptr));
    say("pack-cols", om_pack8(&ctx, x, 8, 1, -8, q, nullptr));
    say("pack-ld", om_pack8(&ctx, x, 7, 1, 8, q, nullptr));
    say("pack-none", om_pack8(&ctx, x, 8, 1, 8, nullptr, nullptr));
    say("pack-x", om_pack8(&ctx, nullptr, 8, 1, 8, q, nullptr));
    say("pack-align", om_pack8(&ctx, x, 8, 1, 8, off, nullptr));
    say("pack-align-t", om_pack8(&ctx, x, 8, 1, 8, nullptr, off));
    say("pack-many", om_pack8(&ctx, x, big, big, big, q, nullptr));
    say("pack-many-t", om_pack8(&ctx, x, big, big, big, nullptr, q));
    // one column (packed 128 bytes wide), 2^28 rows: past 2^32 threads, as is the transpose of 2^29
    say("pack-narrow", om_pack8(&ctx, x, 1, (1 << 28) + 1, 1, q, nullptr));
    say("pack-narrow-t", om_pack8(&ctx, x, 1, 1 << 29, 1, nullptr, q));
    say("ok-pack-no-rows", om_pack8(&ctx, nullptr, 8, 0, 8, q, q));
    say("ok-pack-no-cols", om_pack8(&ctx, nullptr, 8, 8, 0, q, nullptr));

    say("unpack-rows", om_unpack8(&ctx, q, x, 8, -1, 8, 0));
    say("unpack-ld", om_unpack8(&ctx, q, x, 7, 1, 8, 0));
    say("unpack-null", om_unpack8(&ctx, nullptr, x, 8, 1, 8, 0));
    say("unpack-y", om_unpack8(&ctx, q, nullptr, 8, 1, 8, 0));
    say("unpack-align", om_unpack8(&ctx, off, x, 8, 1, 8, 0));
    say("unpack-many", om_unpack8(&ctx, q, x, big, big, big, 0));
    say("unpack-narrow", om_unpack8(&ctx, q, x, 1, (1 << 28) + 1, 1, 0));
    say("ok-unpack-no-rows", om_unpack8(&ctx, nullptr, nullptr, 8, 0, 8, 1));

    say("gemm-m", om_gemm8(&ctx, -1, 4, 4, q, q, nullptr, x, 4, 0));
    say("gemm-n", om_gemm8(&ctx, 4, -1, 4, q, q, nullptr, x, 4, 0));
    say("gemm-k", om_gemm8(&ctx, 4, 4, -1, q, q, nullptr, x, 4, 0));
    say("gemm-ldc", om_gemm8(&ctx, 4, 4, 4, q, q, nullptr, x, 3, 0));
    say("gemm-a", om_gemm8(&ctx, 4, 4, 4, nullptr, q, nullptr, x, 4, 0));
    say("gemm-b", om_gemm8(&ctx, 4, 4, 4, q, nullptr, nullptr, x, 4, 0));
    say("gemm-c", om_gemm8(&ctx, 4, 4, 4, q, q, nullptr, nullptr, 4, 0));
    say("gemm-align-a", om_gemm8(&ctx, 4, 4, 4, off, q, nullptr, x, 4, 0));
    say("gemm-align-b", om_gemm8(&ctx, 4, 4, 4, q, off, nullptr, x, 4, 0));
    say("gemm-long", om_gemm8(&ctx, 40, 40, big, q, q, nullptr, x, 40, 0));
    say("gemm-wide", om_gemm8(&ctx, big, big, 1 << 20, q, q, nullptr, x, big, 0));
    say("gemm-thin", om_gemm8(&ctx, 1, 1 << 28, 128, q, q, nullptr, x, 1 << 28, 0));
    say("gemm-tiles", om_gemm8(&ctx, 20, 1 << 30, 128, q, q, nullptr, x, 1 << 30, 0));
    say("ok-gemm-no-rows", om_gemm8(&ctx, 0, 4, 4, nullptr, nullptr, nullptr, nullptr, 4, 0));
    say("ok-gemm-no-columns", om_gemm8(&ctx, 4, 0, 4, nullptr, nullptr, nullptr, nullptr, 4, 0));

    say("linear-rows", om_linear_bwd_x8(&ctx, x, q, x, x, x, x, -1, 4, 4, 0, 0, 0));
    say("linear-in", om_linear_bwd_x8(&ctx, x, q, x, x, x, x, 4, 0, 4, 0, 0, 0));
    say("linear-out", om_linear_bwd_x8(&ctx, x, q, x, x, x, x, 4, 4, 0, 0, 0, 0));
    say("linear-g", om_linear_bwd_x8(&ctx, nullptr, q, x, x, x, x, 4, 4, 4, 0, 0, 0));
    say("linear-x", om_linear_bwd_x8(&ctx, x, nullptr, x, x, x, x, 4, 4, 4, 0, 0, 0));
    say("linear-w", om_linear_bwd_x8(&ctx, x, q, nullptr, x, x, x, 4, 4, 4, 0, 0, 0));
    say("linear-align", om_linear_bwd_x8(&ctx, x, off, x, nullptr, x, x, 4, 4, 4, 0, 0, 0));
    say("linear-long", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, big, 4, 4, 0, 0, 0));
    say("linear-wide", om_linear_bwd_x8(&ctx, x, q, nullptr, nullptr, x, x, 4, 4, 1 << 26, 0, 0, 0));
    say("ok-linear-nothing", om_linear_bwd_x8(&ctx, x, nullptr, nullptr, nullptr, nullptr, nullptr, 4, 4, 4, 0, 0, 0));
    say("ok-linear-no-rows", om_linear_bwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, x, x, 0, 4, 4, 0, 1, 1));

    say("gelu-rows", om_gelu_fwd_x8(&ctx, x, x, q, -1, 8));
    say("gelu-null", om_gelu_fwd_x8(&ctx, x, x, nullptr, 1, 8));
    say("gelu-align", om_gelu_fwd_x8(&ctx, x, x, off, 1, 8));
    say("gelu-many", om_gelu_fwd_x8(&ctx, x, x, q, big, big));
    say("gelu-narrow", om_gelu_fwd_x8(&ctx, x, x, q, (1 << 28) + 1, 1));
    say("gelu-bwd-narrow", om_gelu_bwd_x8(&ctx, x, q, x, (1 << 28) + 1, 1, 0));
    say("gelu-bwd-null", om_gelu_bwd_x8(&ctx, nullptr, q, x, 1, 8, 0));
    say("gelu-bwd-align", om_gelu_bwd_x8(&ctx, x, off, x, 1, 8, 0));
    say("gelu-bwd-many", om_gelu_bwd_x8(&ctx, x, q, x, big, big, 0));
    say("ok-gelu-no-rows", om_gelu_fwd_x8(&ctx, nullptr, nullptr, nullptr, 0, 8));
    say("ok-gelu-bwd-no-cols", om_gelu_bwd_x8(&ctx, nullptr, nullptr, nullptr, 8, 0, 1));

    say("norm-rows", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, -1, 8, 1e-5f));
    say("norm-cols", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, 1, 0, 1e-5f));
    say("norm-null", om_layernorm_fwd_x8(&ctx, x, x, nullptr, x, q, x, 1, 8, 1e-5f));
    say("norm-align", om_layernorm_fwd_x8(&ctx, x, x, x, x, off, x, 1, 8, 1e-5f));
    say("norm-many", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, 1 << 26, 8, 1e-5f));
    say("norm-many-wide", om_layernorm_fwd_x8(&ctx, x, x, x, x, q, x, 1 << 24, 1025, 1e-5f));
    say("norm-bwd-many-wide", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1 << 24, 8193, 0, 0));
    say("norm-bwd-cols", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1, 0, 0, 0));
    say("norm-bwd-null", om_layernorm_bwd_x8(&ctx, x, nullptr, x, x, x, x, x, 1, 8, 0, 0));
    say("norm-bwd-align", om_layernorm_bwd_x8(&ctx, x, off, x, x, x, x, x, 1, 8, 0, 0));
    say("norm-bwd-wide", om_layernorm_bwd_x8(&ctx, x, q, x, x, x, x, x, 1, (1 << 26) + 1, 0, 0));
    say("ok-norm-no-rows", om_layernorm_fwd_x8(&ctx, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 8, 1e-5f));
    say("ok-norm-bwd-nothing", om_layernorm_bwd_x8(&ctx, x, q, x, x, nullptr, nullptr, nullptr, 1, 8, 0, 0));

    say("null-ctx", om_pack8(nullptr, x, 8, 1, 8, q, nullptr) == OM_E_ARG && om_gemm8(nullptr, 1, 1, 1, q, q, x, x, 1, 0) == OM_E_ARG &&
                            om_linear_bwd_x8(nullptr, x, q, x, x, x, x, 1, 1, 1, 0, 0, 0) == OM_E_ARG &&
                            om_layernorm_bwd_x8(nullptr, x, q, x, x, x, x, x, 1, 1, 0, 0) == OM_E_ARG
                        ? om::fail(&ctx, OM_E_ARG, "om_pack8 and the others refuse a NULL context")
                        : OM_OK);
    return 0;
}
