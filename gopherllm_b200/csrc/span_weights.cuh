// What a step's attention gives cached positions, where it comes in several shares: from the parts that divide a sequence's queries,
// and from several sequences that hold a position on the same page.
#pragma once
#include "common.cuh"

struct GivenArgs {
    const float* sums;            // [parts, B, nKV, reach]: what every sequence's part gave its positions
    const int* seq_qlen;          // [B] tokens of the step
    const int* seq_ctx;           // [B] positions cached before it
    const int* pages;             // [B, max_pages]
    float* weights;               // [pages, nKV, GL_PAGE]
    int B, nKV, max_pages, n_pages, reach, parts, shared;
};

// A thread a position: blockIdx = (256 positions, key/value head, sequence).  weights[j] <- (weights[j] if it was cached before the step
// else 0) + the shares, sequence by sequence and part by part, so that no sum depends on which block comes first.  Of
// sequences that hold the page (shared) the first one adds for all.
static __global__ void __launch_bounds__(256) given_join_kernel(GivenArgs a) {
    gl_grid_wait();
    gl_grid_launch_dependents();
    const int b = blockIdx.z, g = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    const int ctx = a.seq_ctx[b], qlen = a.seq_qlen[b];
    if (qlen <= 0 || j >= min(ctx + qlen, a.reach)) return;
    const int page = a.pages[(size_t)b * a.max_pages + j / GL_PAGE];
    float given = 0.f;
    for (int o = a.shared ? 0 : b; o < (a.shared ? a.B : b + 1); ++o) {
        if (o != b) {
            const int q = a.seq_qlen[o];
            if (q <= 0 || j >= a.seq_ctx[o] + q || a.pages[(size_t)o * a.max_pages + j / GL_PAGE] != page) continue;
            if (o < b) return;
        }
        for (int p = 0; p < a.parts; ++p) given += a.sums[(((size_t)p * a.B + o) * a.nKV + g) * a.reach + j];
    }
    float* w = a.weights + ((size_t)gl_checked(page, a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
    *w = j < ctx ? *w + given : given;
}

template <typename Args>
static int launch_given_join(const Args& a, const float* sums, int parts, int shared, cudaStream_t stream) {
    if (!a.seq_qlen || a.reach <= 0 || parts < 1 || a.nKV > 65535) return GL_ERR_SHAPE;
    const GivenArgs x{sums, a.seq_qlen, a.seq_ctx, a.pages, a.weights, a.B, a.nKV, a.max_pages, a.n_pages, a.reach, parts, shared};
    return gl_launch(given_join_kernel, dim3((a.reach + 255) / 256, a.nKV, a.B), dim3(256), 0, stream, 1, x);
}
