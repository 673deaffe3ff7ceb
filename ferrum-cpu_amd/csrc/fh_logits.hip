// fh_logits.hip — edits of logits before they are sampled: penalties for repeated tokens,
// biases, grammar masks (in front of sample_with_params, slm/sampling.rs:124-210; no
// reference counterpart beyond its one penalty).
//
// out(v) = -inf where the row's mask leaves v out, else with c(v) its count in the row's list
// and on the row's path in a tree:
//   x = l(v);  c > 0: x = x > 0 ? x / rep : x rep;  x -= freq c;  c > 0: x -= pres;  x += bias(v)
// every operation rounded on its own.
#include "fh_internal.hpp"

#include <algorithm>

#pragma clang fp contract(off)

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTree = 1024;

struct EditArgs {
    const float* logits;
    float* out;
    uint32_t rows, vocab;
    fh_logits_edit e;
    uint32_t words;  // of a mask
    int segs;
};

// A workgroup takes SEG ids of a row: the counts and the biases of its own ids go to LDS
// (integer atomics: no order shows), then the logits pass through.  Bound by memory: 8 bytes
// an id and the lists once per workgroup from the caches.
template <int SEG>
__global__ void __launch_bounds__(kThreads) k_logits_edit(EditArgs a) {
    __shared__ uint32_t count[SEG], biased[SEG];
    const uint32_t row = blockIdx.x / a.segs, first = blockIdx.x % a.segs * SEG;
    const uint32_t n = min(static_cast<uint32_t>(SEG), a.vocab - first);
    const fh_logits_edit& e = a.e;
    for (uint32_t i = threadIdx.x; i < SEG; i += kThreads) {
        count[i] = 0;
        biased[i] = 0;
    }
    __syncthreads();
    const bool counted = e.d_ranges || e.d_tokens;
    if (e.d_ranges) {
        const uint32_t i0 = e.d_ranges[2 * static_cast<size_t>(row)], i1 = e.d_ranges[2 * static_cast<size_t>(row) + 1];
        for (uint64_t i = i0 + static_cast<uint64_t>(threadIdx.x); i < i1; i += kThreads) {
            const uint32_t v = e.d_recent[i] - first;
            if (v < n) atomicAdd(&count[v], 1u);
        }
    }
    if (e.d_tokens) {
        // the row's sequence begins at `begin`
        uint32_t begin;
        if (e.d_off) {
            uint32_t lo = 0, hi = static_cast<uint32_t>(e.seqs);  // the last s with off[s] <= row
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (e.d_off[mid] <= row) lo = mid;
                else hi = mid;
            }
            begin = e.d_off[lo] <= row && row < e.d_off[lo + 1] ? e.d_off[lo] : row;
        } else {
            begin = row - row % (a.rows / static_cast<uint32_t>(e.seqs));
        }
        if (threadIdx.x == 0) {
            uint32_t t = row - begin;
            for (int k = 0; k < kMaxTree; k++) {
                const uint32_t v = e.d_tokens[begin + t] - first;
                if (v < n) atomicAdd(&count[v], 1u);
                const uint32_t p = e.d_parent ? e.d_parent[begin + t] : ~0u;
                if (p >= t) break;
                t = p;
            }
        }
    }
    if (e.d_bias_off) {
        const uint32_t i0 = e.d_bias_off[row], i1 = e.d_bias_off[row + 1];
        for (uint64_t i = i0 + static_cast<uint64_t>(threadIdx.x); i < i1; i += kThreads) {
            const uint32_t v = e.d_bias_id[i] - first;
            if (v < n) atomicMax(&biased[v], static_cast<uint32_t>(i - i0 + 1));
        }
    }
    __syncthreads();
    const float rep = e.d_repetition ? e.d_repetition[row] : 1.0f, freq = e.d_frequency ? e.d_frequency[row] : 0.0f;
    const float pres = e.d_presence ? e.d_presence[row] : 0.0f;
    uint32_t m = ~0u;
    if (e.d_mask) {
        m = e.d_mask_of ? e.d_mask_of[row] : row;
        if (m >= e.masks) m = ~0u;
    }
    const float* in = a.logits + static_cast<size_t>(row) * a.vocab + first;
    float* out = a.out + static_cast<size_t>(row) * a.vocab + first;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        float x = in[i];
        if (counted && count[i]) {
            if (rep > 0.0f) x = x > 0.0f ? x / rep : x * rep;
            x -= freq * static_cast<float>(count[i]);
            x -= pres;
        }
        if (biased[i]) x += e.d_bias[e.d_bias_off[row] + static_cast<size_t>(biased[i] - 1)];
        if (m != ~0u) {
            const uint32_t v = first + i;
            if (!(e.d_mask[static_cast<size_t>(m) * a.words + (v >> 5)] >> (v & 31) & 1)) x = -INFINITY;
        }
        out[i] = x;
    }
}

}  // namespace

int fh_launch_logits_edit(fh_ctx* ctx, const float* logits, size_t rows, size_t vocab, const fh_logits_edit& e, float* out) {
    EditArgs a{logits, out, static_cast<uint32_t>(rows), static_cast<uint32_t>(vocab), e,
               static_cast<uint32_t>((vocab + 31) / 32), 0};
    constexpr int seg = 2048;
    a.segs = static_cast<int>((vocab + seg - 1) / seg);
    if (rows * a.segs > 0x7FFFFFFFu) return fh_fail(ctx, FH_ERR_LIMIT, "fh_logits_edit: more than 2^31 - 1 workgroups");
    hipLaunchKernelGGL(k_logits_edit<seg>, dim3(static_cast<unsigned>(rows * a.segs)), dim3(kThreads), 0, ctx->stream, a);
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}
