// host_asan_layers.cpp -- test infrastructure: the host side of the fusion block's layers (workspace and
// saved-buffer carving, tile and slab plans, argument checks; csrc/otf_norm.hip, otf_ffn.hip) under
// AddressSanitizer and UndefinedBehaviorSanitizer, without a GPU: size queries, which plan and carve
// as the calls do, and calls that are refused before any HIP call (tests/test_sanitizers_layers.py).
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "otfuse.h"

static int failures = 0;
#define CHECK(cond, ...)                                         \
    do {                                                         \
        if (!(cond)) {                                           \
            fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
            fprintf(stderr, __VA_ARGS__);                        \
            fprintf(stderr, "\n");                               \
            ++failures;                                          \
        }                                                        \
    } while (0)

alignas(256) static char buffer[4096];

static otf_ffn_args ffn(int64_t rows, int64_t d, int64_t f, int32_t dtype, int skew) {
    otf_ffn_args a;
    memset(&a, 0, sizeof a);
    char* p = buffer + skew;   // never read: the queries look at alignment alone
    a.rows = rows, a.d = d, a.f = f, a.dtype = dtype, a.activation = OTF_ACT_SILU;
    a.x = p, a.ldx = d, a.w_gate = p, a.w_up = p, a.ldw_in = d, a.w_down = p, a.ldw_down = f, a.y = p, a.ldy = d;
    a.saved = buffer, a.dy = p, a.lddy = d;
    return a;
}

int main() {
    const int64_t limit = (int64_t)1 << 34;
    const int64_t rows[] = {1, 5, 8, 9, 16, 17, 64, 65, 777, 8192, 1 << 20, INT32_MAX / 8};
    const int64_t widths[] = {1, 7, 8, 63, 64, 1000, 2730, 11264, 1 << 20};
    const int32_t types[] = {OTF_F32, OTF_F16, OTF_BF16};
    long asked = 0;
    for (int64_t n : rows)
        for (int64_t d : widths)
            for (int64_t f : widths)
                for (int32_t t : types)
                    for (int skew : {0, 4}) {
                        otf_ffn_args a = ffn(n, d, f, t, skew);
                        const bool taken = d * f <= limit && n * (d > f ? d : f) <= limit;
                        const size_t es = t == OTF_F32 ? 4 : 2;
                        const size_t saved = otf_gated_ffn_saved_size(n, f, t);
                        if (n * f <= limit)
                            CHECK(saved >= (size_t)(n * f) * (8 + es), "saved %lld x %lld", (long long)n, (long long)f);
                        else
                            CHECK(saved == 0, "saved size of what is refused");
                        const size_t kept = otf_gated_ffn_workspace_size(&a);
                        a.saved = nullptr;
                        const size_t infer = otf_gated_ffn_workspace_size(&a);
                        if (taken)
                            CHECK(infer >= kept + (size_t)(n * f) * es, "inference keeps h in the workspace: %lld %lld %lld",
                                  (long long)n, (long long)d, (long long)f);
                        else
                            CHECK(infer == 0 && kept == 0, "workspace of what is refused");
                        // backward: every subset of gradients, saved named or not
                        size_t of[8];
                        for (int want = 0; want < 8; ++want) {
                            otf_ffn_args b = ffn(n, d, f, t, skew);
                            if (want & 1) b.dx = buffer, b.lddx = d;
                            if (want & 2) b.dw_gate = b.dw_up = buffer, b.lddw_in = d;
                            if (want & 4) b.dw_down = buffer, b.lddw_down = f;
                            of[want] = otf_gated_ffn_backward_workspace_size(&b);
                            b.saved = nullptr;
                            CHECK(otf_gated_ffn_backward_workspace_size(&b) == of[want], "saved is not in the workspace");
                            CHECK(taken ? of[want] >= 2 * (size_t)(n * f) * es : of[want] == 0, "dg and du: %lld %lld %lld",
                                  (long long)n, (long long)d, (long long)f);
                            ++asked;
                        }
                    }
    CHECK(asked > 40000, "sizes swept");
    // sizes that no call takes
    const int64_t huge[] = {INT64_MAX, INT64_MAX - 63, (int64_t)1 << 62, (int64_t)1 << 40, -1, 0, INT64_MIN};
    for (int64_t n : huge)
        for (int64_t m : huge) {
            CHECK(otf_gated_ffn_saved_size(n, m, OTF_F32) == 0, "saved %lld %lld", (long long)n, (long long)m);
            CHECK(otf_gated_ffn_saved_size(n, 8, OTF_BF16) == 0 && otf_gated_ffn_saved_size(8, m, OTF_BF16) == 0, "saved");
            CHECK(otf_layer_norm_backward_workspace_size(n, m) == 0, "norm %lld %lld", (long long)n, (long long)m);
            CHECK(otf_layer_norm_backward_workspace_size(n, 8) == 0 && otf_layer_norm_backward_workspace_size(8, m) == 0, "norm");
            otf_ffn_args a = ffn(n, m, m, OTF_F32, 0);
            CHECK(otf_gated_ffn_workspace_size(&a) == 0 && otf_gated_ffn_backward_workspace_size(&a) == 0, "workspace");
            CHECK(n == 0 || otf_gated_ffn(&a, buffer, sizeof buffer, nullptr) != OTF_OK, "call");
            CHECK(otf_dropout(buffer, n, nullptr, 0, buffer, n, m, n, OTF_F32, 0.5, nullptr, nullptr) != OTF_OK || n == 0 || m == 0, "dropout");
            CHECK(otf_layer_norm(buffer, n, OTF_F32, nullptr, nullptr, OTF_F32, 1e-5, m, n, buffer, n, nullptr, nullptr, nullptr) != OTF_OK || m == 0,
                  "norm call");
        }
    CHECK(otf_gated_ffn_saved_size(8, 8, 99) == 0, "saved size of no type");
    // rows and columns at the norms' limits
    for (int64_t n : {(int64_t)1, (int64_t)64, (int64_t)65, (int64_t)8191, (int64_t)1 << 24, (int64_t)INT32_MAX})
        for (int64_t c : {(int64_t)1, (int64_t)64, (int64_t)1531, (int64_t)16384, (int64_t)16385, (int64_t)INT32_MAX - 8192}) {
            const size_t ws = otf_layer_norm_backward_workspace_size(n, c);
            CHECK(n <= 64 ? ws == 0 : ws >= (size_t)c * 16, "norm workspace %lld x %lld", (long long)n, (long long)c);
            CHECK(ws % ((size_t)c * 8) == 0, "whole partials");
        }
    CHECK(otf_layer_norm_backward_workspace_size((int64_t)INT32_MAX + 1, 8) == 0, "rows past the limit");
    // refused calls
    otf_ffn_args a = ffn(20, 16, 24, OTF_BF16, 0);
    CHECK(otf_gated_ffn(nullptr, buffer, 4096, nullptr) == OTF_EINVAL && otf_gated_ffn_backward(nullptr, buffer, 4096, nullptr) == OTF_EINVAL, "null");
    CHECK(otf_gated_ffn_workspace_size(nullptr) == 0, "null");
    a.x = nullptr;
    CHECK(otf_gated_ffn(&a, buffer, 4096, nullptr) == OTF_EINVAL, "null x");
    a = ffn(20, 15, 24, OTF_BF16, 2);
    CHECK(otf_gated_ffn(&a, buffer, otf_gated_ffn_workspace_size(&a) - 1, nullptr) == OTF_EINVAL, "small workspace");
    a.dx = buffer, a.lddx = 15, a.dw_gate = a.dw_up = buffer, a.lddw_in = 15, a.dw_down = buffer, a.lddw_down = 24;
    CHECK(otf_gated_ffn_backward(&a, buffer, otf_gated_ffn_backward_workspace_size(&a) - 1, nullptr) == OTF_EINVAL, "small workspace");
    a.dw_up = nullptr;
    CHECK(otf_gated_ffn_backward(&a, buffer, 4096, nullptr) == OTF_EINVAL, "one of two gradients");
    CHECK(otf_dropout(buffer + 1, 8, nullptr, 0, buffer, 8, 2, 8, OTF_F32, 0.5, (const int64_t*)buffer, nullptr) == OTF_EINVAL, "misaligned");
    CHECK(otf_layer_norm_backward(buffer, 8, buffer, 8, OTF_F32, nullptr, OTF_F32, (float*)buffer, (float*)buffer, 1000, 8, buffer, 8, buffer,
                                  nullptr, buffer, 16, nullptr) == OTF_EINVAL, "small workspace");
    CHECK(otf_dropout_add_layer_norm_backward(buffer, 8, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, OTF_BF16, OTF_BF16, nullptr, OTF_F32,
                                              (float*)buffer, (float*)buffer, 0.0, nullptr, 2, 8, buffer, 8, buffer, 8, nullptr, nullptr, nullptr,
                                              0, nullptr) == OTF_EINVAL, "x and residual missing");
    if (failures) {
        fprintf(stderr, "%d check(s) failed\n", failures);
        return 1;
    }
    printf("host_asan_layers: host logic clean\n");
    return 0;
}
