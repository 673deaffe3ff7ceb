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

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // (rows of an odd vocabulary begin anywhere)

// A workgroup takes SEG ids of a row: their logits are on their way while the counts and the biases
// of these ids gather in LDS (integer atomics: no order shows).
template <int SEG>
__global__ void __launch_bounds__(kThreads) k_logits_edit(EditArgs a) {
    constexpr int PER = SEG / (4 * kThreads);  // float4s of a thread
    __shared__ __align__(16) uint32_t count[SEG], biased[SEG];
    __shared__ uint32_t up[kMaxTree], token[kMaxTree];
    const uint32_t row = blockIdx.x / a.segs, first = blockIdx.x % a.segs * SEG;
    const uint32_t n = min(static_cast<uint32_t>(SEG), a.vocab - first);
    const fh_logits_edit& e = a.e;
    const float* in = a.logits + static_cast<size_t>(row) * a.vocab + first;
    float* out = a.out + static_cast<size_t>(row) * a.vocab + first;
    const auto place = [&](int i) { return 4 * (static_cast<uint32_t>(i) * kThreads + threadIdx.x); };
    f4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint32_t v = place(i);
        x[i] = f4{0, 0, 0, 0};
        if (v + 4 <= n) x[i] = *reinterpret_cast<const f4*>(in + v);
        else
            for (uint32_t j = 0; v + j < n; j++) x[i][j] = in[v + j];
    }
    const float rep = e.d_repetition ? e.d_repetition[row] : 1.0f, freq = e.d_frequency ? e.d_frequency[row] : 0.0f;
    const float pres = e.d_presence ? e.d_presence[row] : 0.0f;
    const bool counted = e.d_ranges || e.d_tokens;
    uint32_t mask = ~0u;
    if (e.d_mask) {
        mask = e.d_mask_of ? e.d_mask_of[row] : row;
        if (mask >= e.masks) mask = ~0u;
    }
    uint32_t words[PER];
#pragma unroll
    for (int i = 0; i < PER; i++)
        words[i] = mask != ~0u && place(i) < n ? e.d_mask[static_cast<size_t>(mask) * a.words + ((first + place(i)) >> 5)] : ~0u;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        *reinterpret_cast<uint4*>(&count[place(i)]) = make_uint4(0, 0, 0, 0);
        if (e.d_bias_off) *reinterpret_cast<uint4*>(&biased[place(i)]) = make_uint4(0, 0, 0, 0);
    }
    // the row's sequence begins at `begin`; its rows up to this one
    uint32_t begin = row;
    if (e.d_tokens) {
        if (e.d_off) {
            // the last sequence that begins at or before the row
            uint32_t last = 0;
            for (uint32_t s = threadIdx.x & 63; s < e.seqs; s += 64) last = e.d_off[s] <= row ? s + 1 : last;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) last = max(last, static_cast<uint32_t>(__shfl_xor(static_cast<int>(last), d, 64)));
            if (last && e.d_off[last - 1] <= row && row < e.d_off[last]) begin = e.d_off[last - 1];
        } else {
            begin = row - row % (a.rows / static_cast<uint32_t>(e.seqs));
        }
        if (row - begin >= kMaxTree) begin = row;  // (past the longest tree)
        for (uint32_t t = threadIdx.x; t <= row - begin; t += kThreads) {
            up[t] = e.d_parent ? e.d_parent[begin + t] : ~0u;
            token[t] = e.d_tokens[begin + t];
        }
    }
    __syncthreads();
    if (e.d_tokens && threadIdx.x == 0)
        for (uint32_t t = row - begin, next; ; t = next) {
            const uint32_t v = token[t] - first;
            next = up[t];
            if (v < n) atomicAdd(&count[v], 1u);
            if (next >= t) break;  // (a parent is a row before)
        }
    if (e.d_ranges) {
        const uint32_t i0 = e.d_ranges[2 * static_cast<size_t>(row)], i1 = e.d_ranges[2 * static_cast<size_t>(row) + 1];
        for (uint64_t i = i0 + static_cast<uint64_t>(threadIdx.x); i < i1; i += kThreads) {
            const uint32_t v = e.d_recent[i] - first;
            if (v < n) atomicAdd(&count[v], 1u);
        }
    }
    size_t b0 = 0;
    if (e.d_bias_off) {
        b0 = e.d_bias_off[row];
        const uint32_t i1 = e.d_bias_off[row + 1];
        for (uint64_t i = b0 + threadIdx.x; i < i1; i += kThreads) {
            const uint32_t v = e.d_bias_id[i] - first;
            if (v < n) atomicMax(&biased[v], static_cast<uint32_t>(i - b0 + 1));
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint32_t v = place(i);
        if (counted) {
            const uint4 c4 = *reinterpret_cast<const uint4*>(&count[v]);
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c[j]) {
                    float y = x[i][j];
                    if (rep > 0.0f) y = y > 0.0f ? y / rep : y * rep;
                    y -= freq * static_cast<float>(c[j]);
                    x[i][j] = y - pres;
                }
        }
        if (e.d_bias_off) {
            const uint4 c4 = *reinterpret_cast<const uint4*>(&biased[v]);
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c[j]) x[i][j] += e.d_bias[b0 + (c[j] - 1)];
        }
        const uint32_t stays = words[i] >> (v & 31);  // (SEG and the thread's four ids begin at multiples of 32 and 4)
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = stays >> j & 1 ? x[i][j] : -INFINITY;
        if (v + 4 <= n) *reinterpret_cast<f4*>(out + v) = x[i];
        else
            for (uint32_t j = 0; v + j < n; j++) out[v + j] = x[i][j];
    }
}

}  // namespace

int fh_launch_logits_edit(fh_ctx* ctx, const float* logits, size_t rows, size_t vocab, const fh_logits_edit& e, float* out) {
    EditArgs a{logits, out, static_cast<uint32_t>(rows), static_cast<uint32_t>(vocab), e,
               static_cast<uint32_t>((vocab + 31) / 32), 0};
    // 1024 ids a workgroup spread one row of 50257 over 50 of them, in 3.4 us (4096: 5.2); 4096 read the lists a
    // quarter as often: 256 rows of 151936 64 us (1024: 73), 64 rows either way 20.
    const auto go = [&](auto kern, size_t seg) -> int {
        const size_t segs = (vocab + seg - 1) / seg;
        if (rows > 0x7FFFFFFFu / segs) return fh_fail(ctx, FH_ERR_LIMIT, "fh_logits_edit: more than 2^31 - 1 workgroups");
        a.segs = static_cast<int>(segs);
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(rows * segs)), dim3(kThreads), 0, ctx->stream, a);
        FH_HIP(ctx, hipGetLastError());
        return FH_OK;
    };
    return rows * vocab < (size_t(1) << 24) ? go(k_logits_edit<1024>, 1024) : go(k_logits_edit<4096>, 4096);
}
