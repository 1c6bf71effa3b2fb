// Calls the rotary and scored-attention entry points with arguments they must refuse (or calls that have nothing to do),
// on a context without a device: every check runs before anything is launched or allocated. Prints one line per call,
// "name status message".
#include <cmath>
#include <cstdio>
#include <limits>

#include "../../onemodel-csharp_amd/csrc/om_internal.hpp"

static om_ctx ctx;
static int device_calls() { return ctx.scratch || ctx.scratch2; }

static om_rope rope() {
    om_rope r = {};
    r.rot = 8;
    r.amplitude = 1.0f;
    r.base = 10000.0;
    r.factor = 2.0;
    r.trained = 128.0;
    r.low = 1.0;
    r.high = 4.0;
    return r;
}
static om_attention_scores form() {
    om_attention_scores f = {};
    f.heads = 4;
    f.kv_heads = 2;
    return f;
}
static void say(const char *name, om_status s) { std::printf("%s %d %s%s\n", name, s, s ? ctx.err.c_str() : "", device_calls() ? " DEVICE" : ""); }

int main() {
    float x[64];
    int32_t ids[4] = {};
    ctx.device = 0;
    struct R {
        const char *name;
        void (*change)(om_rope &);
    } ropes[] = {
        {"rot-odd", [](om_rope &r) { r.rot = 7; }},
        {"rot-zero", [](om_rope &r) { r.rot = 0; }},
        {"rot-wide", [](om_rope &r) { r.rot = 10; }},
        {"layout", [](om_rope &r) { r.layout = 2; }},
        {"scaling", [](om_rope &r) { r.scaling = -1; }},
        {"base", [](om_rope &r) { r.base = 1.0; }},
        {"base-nan", [](om_rope &r) { r.base = NAN; }},
        {"amplitude", [](om_rope &r) { r.amplitude = INFINITY; }},
        {"factor", [](om_rope &r) { r.scaling = OM_ROPE_LINEAR; r.factor = 0.5; }},
        {"ntk-two", [](om_rope &r) { r.scaling = OM_ROPE_NTK; r.rot = 2; }},
        {"bands-order", [](om_rope &r) { r.scaling = OM_ROPE_BANDS; r.high = r.low; }},
        {"bands-trained", [](om_rope &r) { r.scaling = OM_ROPE_BANDS; r.trained = 0.0; }},
    };
    for (auto &c : ropes) {
        om_rope r = rope();
        c.change(r);
        say((std::string("rope-") + c.name).c_str(), om_rope_fwd(&ctx, x, 8, nullptr, 0, x, 8, 1, 1, 1, 8, &r));
    }
    om_rope r = rope();
    say("rope-null", om_rope_fwd(&ctx, x, 8, nullptr, 0, x, 8, 1, 1, 1, 8, nullptr));
    say("rope-null-x", om_rope_fwd(&ctx, nullptr, 8, nullptr, 0, x, 8, 1, 1, 1, 8, &r));
    say("rope-stride", om_rope_fwd(&ctx, x, 15, nullptr, 0, x + 16, 16, 1, 1, 2, 8, &r));
    say("rope-inplace-strides", om_rope_fwd(&ctx, x, 8, nullptr, 0, x, 9, 1, 1, 1, 8, &r));
    say("rope-inplace-acc", om_rope_bwd(&ctx, x, 8, nullptr, 0, x, 8, 1, 1, 1, 8, &r, 1));
    say("rope-seq", om_rope_fwd(&ctx, x, 8, nullptr, 0, x, 8, 1, 0, 1, 8, &r));
    say("rope-rows", om_rope_fwd(&ctx, x, 8, nullptr, 0, x, 8, -1, 1, 1, 8, &r));
    say("rope-d", om_rope_fwd(&ctx, x, 258, nullptr, 0, x, 258, 1, 1, 1, 258, &r));
    say("rope-far", om_rope_fwd(&ctx, x, 8, nullptr, INT32_MAX, x, 8, 2, 2, 1, 8, &r));
    say("ok-rope-empty", om_rope_fwd(&ctx, nullptr, 8, nullptr, 0, nullptr, 8, 0, 1, 1, 8, &r));

    struct F {
        const char *name;
        void (*change)(om_attention_scores &);
    } forms[] = {
        {"heads", [](om_attention_scores &f) { f.heads = 3; }},
        {"no-heads", [](om_attention_scores &f) { f.heads = 0; }},
        {"kv-heads", [](om_attention_scores &f) { f.kv_heads = -2; }},
        {"cap", [](om_attention_scores &f) { f.cap = -1.0f; }},
        {"cap-nan", [](om_attention_scores &f) { f.cap = NAN; }},
        {"cap-tiny", [](om_attention_scores &f) { f.cap = std::numeric_limits<float>::denorm_min(); }},
        {"scale", [](om_attention_scores &f) { f.scale = INFINITY; }},
        {"causal", [](om_attention_scores &f) { f.causal = 2; }},
        {"window", [](om_attention_scores &f) { f.window = -1; }},
    };
    auto fwd = [&](const om_attention_scores *f, int B = 1, int lq = 1, int lk = 1, int d = 4, int ldq = 16, int ldkv = 8,
                   int ldo = 16, const float *q = nullptr) {
        return om_attention_fwd_scored(&ctx, q ? q : x, ldq, x, x, ldkv, x, ldo, nullptr, B, lq, lk, d, f);
    };
    auto bwd = [&](const om_attention_scores *f, const float *st, int ldg = 16, int lddq = 16, int lddkv = 8) {
        return om_attention_bwd_scored(&ctx, x, 16, x, x, 8, x, 16, st, x, ldg, x, lddq, x, x, lddkv, 1, 1, 1, 4, f, 0);
    };
    for (auto &c : forms) {
        om_attention_scores f = form();
        c.change(f);
        say((std::string("fwd-") + c.name).c_str(), fwd(&f));
        say((std::string("bwd-") + c.name).c_str(), bwd(&f, x));
    }
    om_attention_scores f = form();
    f.q_doc = ids;
    say("fwd-one-doc", fwd(&f));
    f = form();
    say("fwd-null-form", fwd(nullptr));
    say("fwd-d-zero", fwd(&f, 1, 1, 1, 0));
    say("fwd-d-wide", fwd(&f, 1, 1, 1, 257, 2000, 2000, 2000));
    say("fwd-negative", fwd(&f, -1));
    say("fwd-rows", fwd(&f, 1 << 15, 1 << 15, 1));
    say("fwd-ldq", fwd(&f, 1, 1, 1, 4, 15));
    say("fwd-ldkv", fwd(&f, 1, 1, 1, 4, 16, 7));
    say("fwd-ldo", fwd(&f, 1, 1, 1, 4, 16, 8, 15));
    say("fwd-null-q", om_attention_fwd_scored(&ctx, nullptr, 16, x, x, 8, x, 16, nullptr, 1, 1, 1, 4, &f));
    say("fwd-null-k", om_attention_fwd_scored(&ctx, x, 16, nullptr, x, 8, x, 16, nullptr, 1, 1, 1, 4, &f));
    say("bwd-null-stats", bwd(&f, nullptr));
    say("bwd-ldg", bwd(&f, x, 15));
    say("bwd-lddq", bwd(&f, x, 16, 15));
    say("bwd-lddkv", bwd(&f, x, 16, 16, 7));
    say("ok-fwd-empty", fwd(&f, 0));
    say("ok-fwd-no-queries", fwd(&f, 1, 0));
    say("ok-bwd-nothing", om_attention_bwd_scored(&ctx, x, 16, x, x, 8, x, 16, x, x, 16, nullptr, 16, nullptr, nullptr, 8, 1, 1,
                                                  1, 4, &f, 0));
    return 0;
}
