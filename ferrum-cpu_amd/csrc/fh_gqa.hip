// fh_gqa.hip — many rows of a sequence at once over its f32 key/value cache: prompts
// of different lengths packed one after the other, and trees of drafted tokens
// (Attention::forward_one, llm.rs:285-358, for rows that it feeds one by one; the trees,
// what is accepted of them and the cache made compact again have no reference
// counterpart).
//
// With K, V the cache rows of a sequence after its new rows went there, s(r, j) =
// q_r . k_j / sqrt(hd) and
//   prompt: row t at cache row c = len + t sees j <= c;
//   tree:   node t sees j < len, and len + a for itself and its ancestors a,
// out_r = sum over seen j of exp(s - max) v_j / sum of exp(s - max).
// k_gqa_append rotates and stores the new keys, stores the values, and leaves the rows' cosines and
// sines (a tree's: its nodes' paths too) and, where the keys are dealt over several workgroups,
// the plan of their shares; k_gqa_rows does the rest.  Prompts of many columns and keys have
// k_gqa_pack, k_gqa_prompt and k_gqa_rest in its place (below).
#include "fh_internal.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#pragma clang fp contract(off)

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;

typedef _Float16 h8f __attribute__((ext_vector_type(8)));
typedef _Float16 h2f __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Rows [begin, begin + count) of the call belong to sequence s, row t of them is cache
// row at + t.  What the device arrays say is cut to the call's own bounds, so no value of
// theirs leads outside its buffers.
struct Rows {
    uint32_t begin, count;
    uint64_t at;
};
__device__ __forceinline__ Rows rows_of(const uint32_t* off, const uint32_t* len, uint32_t total, uint32_t max_rows,
                                        uint32_t seqs, uint32_t s) {
    Rows r;
    if (off) {
        r.begin = min(off[s], total);
        const uint32_t fin = min(off[s + 1], total);
        r.count = fin > r.begin ? min(fin - r.begin, max_rows) : 0;
    } else {
        r.count = total / seqs;
        r.begin = r.count * s;
    }
    r.at = len ? len[s] : 0;
    return r;
}

__device__ __forceinline__ void turn_pair(float& a, float& b, float cs, float sn) {
    const float x = a, y = b;
    a = x * cs - y * sn;
    b = x * sn + y * cs;
}

// ---- rotation and storing ------------------------------------------------------------

constexpr int kMaxTree = 1024;  // nodes of a sequence's tree
constexpr int kKeys = 32;       // keys of a tile

// Division by a number of the host's: n / d = the upper half of n * (2^64 / d + 1), exact for n < 2^32.
struct Div {
    uint64_t m;
    uint32_t d;
    Div(uint32_t by = 1) : m(by > 1 ? ~uint64_t(0) / by + 1 : 0), d(by) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return m ? static_cast<uint32_t>(__umul64hi(n, m)) : n; }
};

// What a workgroup of the attention is to do where keys are dealt over several: share `split` of `shares` of
// the tiles of column block cb of a sequence (shares 0: nothing), whose first share is workgroup `first`.
struct Share {
    uint32_t s, cb, split, shares;
    uint32_t begin, count, at, first;
};
constexpr uint32_t kPlanned = 256;  // column blocks of a kv head
constexpr uint32_t kJoined = 8;      // shares of a column block that are joined at once

struct AppendArgs {
    const float* qkv;
    size_t ld;
    float *kc, *vc;
    size_t seq_stride;  // of the caches (floats)
    int n_heads, n_kv, hd;
    uint32_t seqs, total, max_rows, limit;
    const uint32_t *off, *len, *pos, *parent;
    float* q;           // [total, n_heads * hd], or NULL and
    float2* cs;         // (nullable) [total, rope_dim / 2]: cosine and sine of a row's pairs
    int first;          // the first head taken: 0, or without q n_heads
    uint32_t* seen;     // [total, words]: a node's path, bit a for node a
    int words;
    int rope_dim, neox;
    float linear;
    const float* ff;
    int heads_each, chunks;
    uint32_t* clear;  // [seqs, n_kv], 1 (NULL: nowhere): set to 0
    Share* plan;      // [places] (NULL: none): the workgroups' shares, of every kv head alike
    uint32_t places, col_blocks, cols;  // columns of a block
    Div group;
    float freq[64];
};

// Shares of nearly equal length for sequences (and for prompts, blocks) of different lengths: the least number of
// tiles q for which all blocks cut into shares of q at most are no more than the places.
template <bool TREE>
__device__ __forceinline__ void plan_shares(const AppendArgs& a) {
    constexpr int PER = kPlanned / 64;
    __shared__ uint32_t first[kPlanned + 1];
    const uint32_t units = a.seqs * a.col_blocks;
    if (threadIdx.x < 64) {
        uint32_t tiles[PER];
        int total = 0, most = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const uint32_t u = j * 64 + threadIdx.x, s = u / a.col_blocks, c0 = (u - s * a.col_blocks) * a.cols;
            tiles[j] = 0;
            if (u < units) {
                const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
                const uint32_t ncols = r.count * a.group.d;
                const uint32_t n = TREE ? r.count : a.group(min(ncols, c0 + a.cols) - 1) + 1;
                if (c0 < ncols) tiles[j] = static_cast<uint32_t>((min(r.at + n, static_cast<uint64_t>(a.limit)) + kKeys - 1) / kKeys);
            }
            total += tiles[j];
            most = max(most, static_cast<int>(tiles[j]));
        }
        for (int d = 32; d; d >>= 1) {
            total += __shfl_xor(total, d);
            most = max(most, __shfl_xor(most, d));
        }
        const auto shares = [&](uint32_t t, uint32_t q) { return (t + q - 1) / q; };
        uint32_t lo = max(2u, shares(total, a.places)), hi = max(lo, static_cast<uint32_t>(most));
        while (lo < hi) {
            const uint32_t q = (lo + hi) / 2;
            int n = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) n += shares(tiles[j], q);
            for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
            if (static_cast<uint32_t>(n) <= a.places) hi = q;
            else lo = q + 1;
        }
        uint32_t base = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            uint32_t upto = shares(tiles[j], lo);
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t x = __shfl_up(upto, d);
                if (static_cast<int>(threadIdx.x) >= d) upto += x;
            }
            first[j * 64 + threadIdx.x + 1] = base + upto;
            base += __shfl(upto, 63);
        }
        if (threadIdx.x == 0) first[0] = 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.places; i += kThreads) {
        uint32_t u = 0;  // the last block whose first share is not behind i
        for (uint32_t step = kPlanned / 2; step; step >>= 1)
            if (first[u + step] <= i) u += step;
        Share to{};
        if (u < units && i < first[u + 1]) {
            const uint32_t s = u / a.col_blocks;
            const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
            to = Share{s, u - s * a.col_blocks, i - first[u], first[u + 1] - first[u], r.begin, r.count, static_cast<uint32_t>(r.at), first[u]};
        }
        a.plan[i] = to;
    }
}

// A workgroup takes some rows of a sequence and `heads_each` of their heads: a thread
// keeps one pair of channels' sine and cosine for all of them.  (12700 rows, 2 kv heads of width 64: 8.7 us; the
// sines and cosines are half of it.  One tree of 16 rows: 4.6, three dependent loads and a launch.)
template <bool TREE>
__global__ void __launch_bounds__(kThreads) k_gqa_append(AppendArgs a) {
    const uint32_t s = blockIdx.y;
    if (s == a.seqs) {  // (one more, where there is a plan)
        if (blockIdx.x == 0) plan_shares<TREE>(a);
        return;
    }
    const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
    const int slots = a.hd / 2, each = kThreads / slots;  // rows of a workgroup
    const uint32_t t0 = blockIdx.x / a.chunks * static_cast<uint32_t>(each);
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
    if (a.clear && blockIdx.x == 0)
        for (int h = threadIdx.x; h < a.n_kv + (s + 1 == a.seqs); h += kThreads) a.clear[s * static_cast<uint32_t>(a.n_kv) + h] = 0;
    if (t0 >= r.count) return;
    __shared__ uint32_t up[TREE ? kMaxTree : 1];
    if constexpr (TREE) {
        // (a parent that is not one of the nodes before it: none)
        for (uint32_t t = threadIdx.x; t < min(r.count, t0 + each); t += kThreads) {
            const uint32_t p = a.parent[r.begin + t];
            up[t] = p < t ? p : ~0u;
        }
        __syncthreads();
    }
    const int slot = static_cast<int>(threadIdx.x) % slots;
    const uint32_t t = t0 + threadIdx.x / slots, row = r.begin + t;
    if (t >= r.count) return;
    uint32_t depth = t;
    if constexpr (TREE) {
        depth = 0;
        for (uint32_t x = up[t]; x != ~0u; x = up[x]) depth++;
        if (chunk == 0)
            for (int w = slot; w < a.words; w += slots) {
                uint32_t bits = 0;
                for (uint32_t x = t; x != ~0u; x = up[x])
                    if (static_cast<int>(x >> 5) == w) bits |= 1u << (x & 31);
                a.seen[static_cast<size_t>(row) * a.words + w] = bits;
            }
    }
    const int half = a.rope_dim / 2;
    const bool turns = slot < half;
    // the pair's two channels (past rope_dim: two that stay as they are)
    const int ia = turns ? (a.neox ? slot : 2 * slot) : 2 * slot;
    const int ib = turns ? (a.neox ? slot + half : 2 * slot + 1) : 2 * slot + 1;
    float sn = 0.0f, cs = 1.0f;
    if (turns) {
        const uint32_t p = a.pos ? a.pos[row] : static_cast<uint32_t>(r.at) + depth;
        const float f = a.ff ? a.ff[slot] : 1.0f;
        const float theta = static_cast<float>(static_cast<int>(p)) * a.freq[slot] / f * (1.0f / a.linear);
        sn = sinf(theta);
        cs = cosf(theta);
    }
    const float* x = a.qkv + row * a.ld;
    const uint64_t c = r.at + t;
    const bool fits = c < a.limit;
    const size_t kv_dim = static_cast<size_t>(a.n_kv) * a.hd;
    const size_t to = s * a.seq_stride + (fits ? c : 0) * kv_dim;
    if (a.cs && chunk == 0 && turns) a.cs[static_cast<size_t>(row) * half + slot] = make_float2(cs, sn);
    const int h0 = a.first + chunk * a.heads_each, h1 = min(a.n_heads + 2 * a.n_kv, h0 + a.heads_each);
    for (int h = h0; h < h1; h++) {
        const float* xh = x + static_cast<size_t>(h) * a.hd;
        const float u = xh[ia], w = xh[ib];
        float y = u, z = w;
        if (turns && h < a.n_heads + a.n_kv) turn_pair(y, z, cs, sn);
        float* dst;
        if (h < a.n_heads) {
            dst = a.q + (static_cast<size_t>(row) * a.n_heads + h) * a.hd;
        } else {
            if (!fits) continue;
            dst = h < a.n_heads + a.n_kv ? a.kc + to + static_cast<size_t>(h - a.n_heads) * a.hd
                                         : a.vc + to + static_cast<size_t>(h - a.n_heads - a.n_kv) * a.hd;
        }
        dst[ia] = y;
        dst[ib] = z;
    }
}

// ---- attention -------------------------------------------------------------------------

struct RowsArgs {
    const float* q;  // row r's heads at r * q_ld: rotated, or with cs to be rotated
    size_t q_ld;
    const float2* cs;  // [total, half]: cosine and sine of a row's pairs of channels
    int half, neox;
    const float *kc, *vc;
    size_t seq_stride;
    int n_heads, n_kv, hd;
    Div group, pairs, kvs;  // query heads of a kv head; (sequence, kv head) pairs; kv heads
    uint32_t seqs, total, max_rows, limit;
    const uint32_t *off, *len, *seen;
    int words;
    float scale;  // log2(e) / sqrt(hd)
    float* out;
    int col_blocks;
    const Share* plan;  // (NULL: a workgroup a block)
    uint32_t places;    // workgroups of a plan
    float2* part;
    unsigned* counters;
    const uint32_t* apart;  // [seqs, n_kv], 1: (prompt) not 0 where the blocks are k_gqa_rest's; where any are
};

__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ uint32_t mag(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
constexpr uint32_t kInf = 0x7F800000u;  // magnitudes from here on: infinity, NaN

// The largest of G consecutive lanes' values (G a power of two up to 64), in all of them.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_of(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, true));
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    if constexpr (G >= 2) v = max(v, dpp_of<0xB1>(v));
    if constexpr (G >= 4) v = max(v, dpp_of<0x4E>(v));
    if constexpr (G >= 8) v = max(v, dpp_of<0x141>(v));
    if constexpr (G >= 16) v = max(v, dpp_of<0x140>(v));
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    return v;
}
// The largest of G consecutive lanes' values of four numbers each; lane l has that of number l % 4.
template <int G>
__device__ __forceinline__ uint32_t quad_max(const uint32_t (&x)[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
    const uint32_t a = max(odd ? x[1] : x[0], dpp_of<0xB1>(odd ? x[0] : x[1]));
    const uint32_t b = max(odd ? x[3] : x[2], dpp_of<0xB1>(odd ? x[2] : x[3]));
    uint32_t v = max(high ? b : a, dpp_of<0x4E>(high ? a : b));
    v = max(v, dpp_of<0x128>(v));
    v = max(v, dpp_of<0x124>(v));
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    return v;
}
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float sum_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}

// Two f32 values as two f16 terms each: h = f16(x), l = f16(x - h), 22 bits; x - h is one instruction of
// mixed precision.  (The pair and the factor are kept from the compiler's view: it would
// convert each half there and back.)
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const h2f h = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    hi = __builtin_bit_cast(uint32_t, h);
    float minus = -1.0f;
    asm("" : "+v"(hi), "+s"(minus));
    const h2f k = __builtin_bit_cast(h2f, hi);
    const h2f l = {static_cast<_Float16>(fmaf(static_cast<float>(k.x), minus, x)),
                   static_cast<_Float16>(fmaf(static_cast<float>(k.y), minus, y))};
    lo = __builtin_bit_cast(uint32_t, l);
}
// The same where a value may be infinite (its lower term is 0 then).
__device__ __forceinline__ void split2_any(float x, float y, uint32_t& hi, uint32_t& lo) {
    const h2f h = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    const float rx = mag(x) == kInf ? 0.0f : x - static_cast<float>(h.x);
    const float ry = mag(y) == kInf ? 0.0f : y - static_cast<float>(h.y);
    const h2f l = {static_cast<_Float16>(rx), static_cast<_Float16>(ry)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// How far queries and keys are brought up, and values: 2^-e of a query times 2^-e of a key stays a
// normal number (its product with a masked score is -inf, not NaN).
constexpr int kLiftMost = 60, kValueLift = 100;
// e with x 2^e in [2^14, 2^15) for a magnitude's bits, as far as it is in range.
__device__ __forceinline__ int lift(uint32_t bits, int most) { return min(max(141 - static_cast<int>(bits >> 23), -113), most); }

__device__ __forceinline__ f32x16 mfma(h8f a, h8f b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Row of accumulator v in a lane of half `half` of a 32 x 32 product.
__device__ __forceinline__ constexpr int acc_row(int v, int half) { return (v >> 2) * 8 + half * 4 + (v & 3); }

__device__ __forceinline__ void store_part(float2* to, float2 x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_part(const float2* from) {
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float2*>(from)), __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT));
}

// What a lane has summed for its column over the keys so far: weights are 2^(score - base).
template <int OT>
struct Sums {
    static constexpr int kParts = 1 + 8 * OT;  // float2s
    float base, l;
    f32x16 o[OT];
};
template <int OT>
__device__ __forceinline__ void clear(Sums<OT>& z) {
    z.base = -FLT_MAX;
    z.l = 0.0f;
#pragma unroll
    for (int d = 0; d < OT; d++) z.o[d] = f32x16{};
}
// Weights lie at 2^10 of the largest so far, and up to 2^14 before a column's sums are brought to a
// new one (its own scores decide, not its neighbours'): their lower terms stay normal numbers of f16 far below it.
constexpr float kRaise = 14.0f;
template <int OT>
__device__ __forceinline__ void raise_base(Sums<OT>& z, float top) {
    if (__any(top > z.base + kRaise)) {
        const float m = max_halves(top), nb = m > z.base + kRaise ? m - 10.0f : z.base, f = __builtin_amdgcn_exp2f(z.base - nb);
        z.l *= f;
#pragma unroll
        for (int d = 0; d < OT; d++) z.o[d] *= f;
        z.base = nb;
    }
}
// Eight weights in two f16 terms.
__device__ __forceinline__ void split8(const float* p, h8f& hi, h8f& lo) {
    u32x4 h, l;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t x, y;
        split2(p[2 * j], p[2 * j + 1], x, y);
        h[j] = x;
        l[j] = y;
    }
    hi = __builtin_bit_cast(h8f, h);
    lo = __builtin_bit_cast(h8f, l);
}
// Eight channels times 2^e.
__device__ __forceinline__ void split8(const float* x, float up, h8f& hi, h8f& lo) {
    u32x4 h, l;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t a, b;
        split2(x[2 * j] * up, x[2 * j + 1] * up, a, b);
        h[j] = a;
        l[j] = b;
    }
    hi = __builtin_bit_cast(h8f, h);
    lo = __builtin_bit_cast(h8f, l);
}
// The same where some may be infinite (any, the same in all lanes).
__device__ __forceinline__ void split8(const float* x, float up, bool any, h8f& hi, h8f& lo) {
    u32x4 h, l;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t a, b;
        if (__builtin_expect(any, 0)) split2_any(x[2 * j] * up, x[2 * j + 1] * up, a, b);
        else split2(x[2 * j] * up, x[2 * j + 1] * up, a, b);
        h[j] = a;
        l[j] = b;
    }
    hi = __builtin_bit_cast(h8f, h);
    lo = __builtin_bit_cast(h8f, l);
}
template <int OT>
__device__ __forceinline__ void add_sums(Sums<OT>& z, const float2 (&y)[Sums<OT>::kParts]) {
    const float nb = fmaxf(z.base, y[0].x), f0 = __builtin_amdgcn_exp2f(z.base - nb), f1 = __builtin_amdgcn_exp2f(y[0].x - nb);
    z.l = z.l * f0 + y[0].y * f1;
#pragma unroll
    for (int d = 0; d < OT; d++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            z.o[d][2 * i] = z.o[d][2 * i] * f0 + y[1 + 8 * d + i].x * f1;
            z.o[d][2 * i + 1] = z.o[d][2 * i + 1] * f0 + y[1 + 8 * d + i].y * f1;
        }
    z.base = nb;
}
// The sums of the waves that shared the keys, in order, to those of kw = 0, through LDS that every wave
// is past its last read of.
template <int OT, int CW, int KW>
__device__ __forceinline__ void join_waves(Sums<OT>& z, float2* room, int cw, int kw, int lane) {
    constexpr int PL = Sums<OT>::kParts;
    if (kw > 0) {
        float2* to = room + ((kw - 1) * CW + cw) * (PL * 64) + lane;
        to[0] = make_float2(z.base, z.l);
#pragma unroll
        for (int d = 0; d < OT; d++)
#pragma unroll
            for (int i = 0; i < 8; i++) to[(1 + 8 * d + i) * 64] = make_float2(z.o[d][2 * i], z.o[d][2 * i + 1]);
    }
    __syncthreads();
    if (kw == 0)
#pragma unroll
        for (int k = 1; k < KW; k++) {
            const float2* from = room + ((k - 1) * CW + cw) * (PL * 64) + lane;
            float2 y[PL];
#pragma unroll
            for (int i = 0; i < PL; i++) y[i] = from[i * 64];
            add_sums(z, y);
        }
}

// A column's query, rotated, scaled by its own power of two, dims 16 i + 8 half + (0..7) in two f16
// terms; returns what undoes the power and brings scores to base 2.
template <int W>
__device__ __forceinline__ float load_query(const RowsArgs& a, uint32_t row, uint32_t head, int half, h8f (&qh)[W / 16], h8f (&ql)[W / 16]) {
    constexpr int KI = W / 16;
    const float* qp = a.q + row * a.q_ld + static_cast<size_t>(head) * a.hd + half * 8;
    float x[8 * KI];
#pragma unroll
    for (int i = 0; i < KI; i++) {
        const bool in = W > 32 || 16 * i + half * 8 < a.hd;
        const float4 u = in ? *reinterpret_cast<const float4*>(qp + 16 * i) : make_float4(0, 0, 0, 0);
        const float4 w = in ? *reinterpret_cast<const float4*>(qp + 16 * i + 4) : make_float4(0, 0, 0, 0);
        x[8 * i] = u.x; x[8 * i + 1] = u.y; x[8 * i + 2] = u.z; x[8 * i + 3] = u.w;
        x[8 * i + 4] = w.x; x[8 * i + 5] = w.y; x[8 * i + 6] = w.z; x[8 * i + 7] = w.w;
    }
    if (a.cs) {
        const float2* cs = a.cs + static_cast<size_t>(row) * a.half;
        if (a.neox) {  // (pairs of channels d, d + half; half a multiple of 16)
            const auto turn = [&](auto steps) {
                constexpr int S = decltype(steps)::value;
#pragma unroll
                for (int i = 0; i < S; i++)
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float4 t = *reinterpret_cast<const float4*>(cs + 16 * i + half * 8 + j);
                        turn_pair(x[8 * i + j], x[8 * (i + S) + j], t.x, t.y);
                        turn_pair(x[8 * i + j + 1], x[8 * (i + S) + j + 1], t.z, t.w);
                    }
            };
            if (W >= 128 && a.half == 64) turn(std::integral_constant<int, W >= 128 ? 4 : 1>{});
            else if (W >= 128 && a.half == 48) turn(std::integral_constant<int, W >= 128 ? 3 : 1>{});
            else if (W >= 64 && a.half == 32) turn(std::integral_constant<int, W >= 64 ? 2 : 1>{});
            else turn(std::integral_constant<int, 1>{});
        } else {
#pragma unroll
            for (int i = 0; i < KI; i++)
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    const int p = (16 * i + half * 8 + j) / 2;
                    if (p < a.half) {  // (half is even)
                        const float4 t = *reinterpret_cast<const float4*>(cs + p);
                        turn_pair(x[8 * i + j], x[8 * i + j + 1], t.x, t.y);
                        turn_pair(x[8 * i + j + 2], x[8 * i + j + 3], t.z, t.w);
                    }
                }
        }
    }
    float top = 0.0f;  // (NaN aside)
#pragma unroll
    for (int i = 0; i < 8 * KI; i++) top = fmaxf(top, fabsf(x[i]));
    top = max_halves(top);
    const bool any = __any(mag(top) == kInf);
    if (any) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8 * KI; i++) top = mag(x[i]) < kInf ? fmaxf(top, fabsf(x[i])) : top;
        top = max_halves(top);
    }
    const int e = lift(mag(top), kLiftMost);
    const float up = pow2f(e);
#pragma unroll
    for (int i = 0; i < KI; i++) split8(x + 8 * i, up, any, qh[i], ql[i]);
    return pow2f(-e) * a.scale;
}
// A workgroup's sums to memory; the last of a group of a block's workgroups joins the group's, in order, and
// the last of the groups' joins those (true: it is this one).  What a workgroup reads of others' sums comes at
// about 35 GB/s, so of n shares 2 sqrt(n) are read in turn, not n.
template <int OT, int CW>
__device__ __forceinline__ bool join_shares(Sums<OT>& z, const RowsArgs& a, uint32_t kv, uint32_t first, uint32_t split, uint32_t shares,
                                            int cw, bool mine, int lane) {
    constexpr int PL = Sums<OT>::kParts;
    __shared__ int last;
    const size_t next = static_cast<size_t>(a.kvs.d) * CW * (PL * 64);  // from share to share
    float2* part = a.part + (static_cast<size_t>(first * a.kvs.d + kv) * CW + cw) * (PL * 64) + lane;
    uint32_t group = shares;  // shares of a group
    if (shares > kJoined) {
        group = 2;
        while (group * group < shares) group++;
    }
    const uint32_t lead = split / group * group;
    unsigned* arrived = a.counters + (first + lead) * a.kvs.d + kv;
    for (uint32_t at = split, from0 = lead, step = 1, count = min(group, shares - lead);;) {
        if (mine) {
            float2* to = part + at * next;
            store_part(to, make_float2(z.base, z.l));
#pragma unroll
            for (int d = 0; d < OT; d++)
#pragma unroll
                for (int i = 0; i < 8; i++) store_part(to + (1 + 8 * d + i) * 64, make_float2(z.o[d][2 * i], z.o[d][2 * i + 1]));
        }
        // Every thread's coherent stores complete before the arrival count moves.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(arrived, 1u) == count - 1;
        __syncthreads();
        if (!last) return false;
        if (threadIdx.x == 0) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (mine) {
            clear(z);
            for (uint32_t k = 0; k < count; k++) {
                const float2* from = part + (from0 + k * step) * next;
                float2 y[PL];
#pragma unroll
                for (int i = 0; i < PL; i++) y[i] = load_part(from + i * 64);
                add_sums(z, y);
            }
        }
        if (group == shares || step == group) return true;
        at = lead;  // (read by this wave alone, and done with)
        from0 = 0;
        step = group;
        count = (shares + group - 1) / group;
        arrived = a.counters + a.places + first * a.kvs.d + kv;
    }
}
template <int W>
__device__ __forceinline__ void store_out(const Sums<W / 32>& z, const RowsArgs& a, uint32_t row, uint32_t head, int half, bool bad) {
    float* out = a.out + (static_cast<size_t>(row) * a.n_heads + head) * a.hd + half * 4;
    const float f = bad ? __builtin_nanf("") : 1.0f / z.l;
#pragma unroll
    for (int d = 0; d < W / 32; d++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            if (W == 32 && 8 * b + half * 4 >= a.hd) continue;
            *reinterpret_cast<float4*>(out + 32 * d + 8 * b) =
                make_float4(z.o[d][4 * b] * f, z.o[d][4 * b + 1] * f, z.o[d][4 * b + 2] * f, z.o[d][4 * b + 3] * f);
        }
}

// Columns are (row, query head of the kv head), heads fastest; a wave has 32 of them, a
// workgroup CW waves of columns times KW waves that deal tiles of 32 keys among them.
// A tile is read from the cache once for the workgroup and kept in LDS as MFMA
// operands: every f32 value in two f16 terms (22 bits; three products of a product's four,
// the lowest left out at 2^-22).  Each key's channels are brought to [2^14, 2^15) by a power of
// two of that key's own, undone exactly on its score; each value row's power of two goes into
// the weights (the running maximum is that of score - exponent), so that a row's accuracy
// does not hang on keys beside it that it does not see, nor on how large the values are.
// A value that is not finite would reach every column through 0 * inf: its key is staged as zeros, and
// a bit makes NaN of the columns that see it.
// S^T = K Q^T leaves a lane 16 keys of one column, which is where O^T += V^T P^T wants them.
// W: the head width brought to 32, 64 or 128.
// The vector units bound it: a tile of 32 keys of width 64 is some 300 instructions a wave (half of them for the
// staging) beside 24 products, and the two times add up.  32 trees of up to 32 nodes over up to 1023 rows, 14 and
// 2 heads: 30.1 us, about 6 until the first tile is staged, 2 a tile, 5 to join four shares.  4 trees of up to 64
// nodes over up to 16383 rows, 32 and 8 heads of width 128: 198 us a call, 2.2 TB/s of the cache and 228 TFLOP/s (three
// times that of f16 products).  Scores of tile t + 1 are multiplied while tile t's become weights (when this was added 40.7
// to 34.5 and 399 to 283 us).
template <int W, int CW, int KW>
struct Stage {
    static constexpr int KI = W / 16, OT = W / 32;
    // A half of 16 channels has 32 keys of eight channels, and room between them for the W / 8 lanes that store one
    // key's to have banks of their own.
    _Float16 k[2][KW][2][KI][2][kKeys + 128 / W][8];
    _Float16 v[2][KW][OT][2][2][64][8];  // (channel c at place of(c))
    static __device__ __forceinline__ int of(int c) { return c ^ (c >> 4 & 1); }  // (so have the lanes that store every other)
    float kdown[4][KW][kKeys];  // 2^-e of a key (step st: st % 4)
    float vexp[2][KW][kKeys];   // -e of a value row
    float vup[2][KW][kKeys];    // 2^e of it
    uint32_t poison[3][KW];     // keys with a value that is not finite (step st: st % 3)
};

// What a workgroup is to do.  Workgroups of a sequence and kv head are dealt to as few XCDs as can be,
// and the longest rows come first.  An XCD deals its workgroups to its four shader engines in turn and waits where
// one is full, so the pairs of an XCD (every eighth) come in another order for each block: with one order a long
// sequence's blocks, between others' that have none, filled one engine (16 prompts of up to 1000 rows: 228 of 512
// workgroups ran for the first 40 us).
template <int CW, bool TREE>
struct Block {
    uint32_t pair, cb, s, kv, split, shares, first;  // (first: of the block's workgroups)
    Rows r;
    uint32_t ncols, c0;
    // the wave's columns, and this lane's
    uint32_t wc, t, row, head;
    bool on, bad;
    uint32_t at, own;            // keys before the call's rows; (prompt) the keys that this column sees
    uint32_t keys, wkeys, wfull;  // of the workgroup; of the wave; those that all of its columns see
    uint32_t tile0, tile1;

    __device__ __forceinline__ bool place(const RowsArgs& a, uint32_t workgroup) {
        if (a.plan) {
            const uint32_t i = a.kvs(workgroup);
            kv = workgroup - i * a.kvs.d;
            const Share p = a.plan[i];
            s = p.s;
            pair = s * a.kvs.d + kv;
            cb = p.cb;
            split = p.split;
            shares = p.shares;
            first = p.first;
            r = Rows{p.begin, p.count, p.at};
            ncols = r.count * a.group.d;
            c0 = cb * (32 * CW);
            return shares != 0;
        }
        const uint32_t id = a.pairs(workgroup);
        pair = workgroup - id * a.pairs.d;
        if (a.pairs.d % 8 == 0) {
            const uint32_t turned = pair + 8 * id;
            pair = turned - a.pairs(turned) * a.pairs.d;
        }
        split = 0;
        shares = 1;
        cb = a.col_blocks - 1 - id;
        s = a.kvs(pair);
        kv = pair - s * a.kvs.d;
        r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
        ncols = r.count * a.group.d;
        c0 = cb * (32 * CW);
        return c0 < ncols;
    }
    __device__ __forceinline__ uint32_t upto(const RowsArgs& a, uint32_t cols) const {
        const uint32_t n = TREE ? r.count : a.group(min(ncols, cols) - 1) + 1;
        return static_cast<uint32_t>(min(r.at + n, static_cast<uint64_t>(a.limit)));
    }
    __device__ __forceinline__ void share(const RowsArgs& a, int cw) {
        at = static_cast<uint32_t>(min(r.at, static_cast<uint64_t>(a.limit)));
        keys = upto(a, c0 + 32 * CW);
        wc = c0 + cw * 32;
        wkeys = wc >= ncols ? 0 : upto(a, wc + 32);
        wfull = TREE ? at : wc >= ncols ? 0 : min(keys, at + a.group(wc) + 1);
        const uint32_t tiles = keys / kKeys + (keys % kKeys != 0);
        tile0 = 0;
        tile1 = tiles;
        if (shares > 1) {
            tile0 = tiles / shares * split + min(tiles % shares, split);
            tile1 = tile0 + tiles / shares + (split < tiles % shares ? 1 : 0);
        }
    }
    __device__ __forceinline__ void column(const RowsArgs& a, int col) {
        const uint32_t c = wc + col, cc = min(c, ncols - 1);
        t = a.group(cc);
        row = r.begin + t;
        head = kv * a.group.d + (cc - t * a.group.d);
        on = c < ncols;
        bad = r.at + t >= a.limit;
        own = on && !bad ? at + t + 1 : 0;
    }
};

template <int W, int CW, int KW, bool TREE>
__device__ __forceinline__ void rows_block(const RowsArgs& a, char* smem, Block<CW, TREE>& b) {
    constexpr int NW = CW * KW, KI = W / 16, OT = W / 32;
    constexpr int WK = KW * W / 16;            // a stage's keys in pieces of 64 threads; its values in as many
    constexpr int PER = (WK + NW - 1) / NW;    // pieces of either that a wave has; where there are more waves than pieces,
    constexpr int V0 = WK < NW ? NW - WK : 0;  // the first waves have the keys', the last the values'
    Stage<W, CW, KW>& st = *reinterpret_cast<Stage<W, CW, KW>*>(smem);
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), cw = wave % CW, kw = wave / CW;
    b.share(a, cw);
    const uint32_t keys = b.keys, at = b.at;
    // Staging.  A piece of keys: 512 / W of them, eight channels a thread; of values: 128 / W quads of keys,
    // two channels a thread.
    const size_t kv_dim = static_cast<size_t>(a.n_kv) * a.hd;
    const float* kp = a.kc + b.s * a.seq_stride + static_cast<size_t>(b.kv) * a.hd;
    const float* vp = a.vc + b.s * a.seq_stride + static_cast<size_t>(b.kv) * a.hd;
    const int kd = lane % (W / 8) * 8, vd = lane % (W / 2) * 2;  // the thread's channels
    const bool kin = W > 32 || kd < a.hd, vin = W > 32 || vd < a.hd;
    typedef float Pieces[PER][8];
    // (tile: the stage's first; past the end: its last key)
    const auto fetch_k = [&](uint32_t tile, Pieces& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int p = wave + i * NW;
            if (WK % NW != 0 && p >= WK) continue;
            const int k = p * (512 / W) + lane / (W / 8);
            const float* from = kp + static_cast<size_t>(min(tile * kKeys + k, keys - 1)) * kv_dim + kd;
            const float4 u = kin ? *reinterpret_cast<const float4*>(from) : make_float4(0, 0, 0, 0);
            const float4 w = kin ? *reinterpret_cast<const float4*>(from + 4) : make_float4(0, 0, 0, 0);
            x[i][0] = u.x; x[i][1] = u.y; x[i][2] = u.z; x[i][3] = u.w;
            x[i][4] = w.x; x[i][5] = w.y; x[i][6] = w.z; x[i][7] = w.w;
        }
    };
    const auto fetch_v = [&](uint32_t tile, Pieces& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int p = wave - V0 + i * NW;
            if (V0 && p < 0) continue;
            const int q = p * (128 / W) + lane / (W / 2);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float* from = vp + static_cast<size_t>(min(tile * kKeys + 4 * q + j, keys - 1)) * kv_dim + vd;
                const float2 u = vin ? *reinterpret_cast<const float2*>(from) : make_float2(0, 0);
                x[i][j] = u.x;
                x[i][4 + j] = u.y;
            }
        }
    };
    // (A key with an infinity has a scale that leaves its other channels nothing, and an infinity less itself as a
    // lower term: its score is NaN, as that of a key with a NaN is.)
    const auto stash_k = [&](uint32_t step, Pieces& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int p = wave + i * NW;
            if (WK % NW != 0 && p >= WK) continue;
            const int k = p * (512 / W) + lane / (W / 8), kt = k / kKeys, kk = k % kKeys;
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(x[i][j]));
            const int e = lift(group_max<W / 8>(mag(most)), kLiftMost);
            h8f hi, lo;
            split8(x[i], pow2f(e), hi, lo);
            *reinterpret_cast<h8f*>(st.k[step & 1][kt][0][kd >> 4][kd >> 3 & 1][kk]) = hi;
            *reinterpret_cast<h8f*>(st.k[step & 1][kt][1][kd >> 4][kd >> 3 & 1][kk]) = lo;
            if (kd == 0) st.kdown[step & 3][kt][kk] = pow2f(-e);
        }
    };
    const auto stash_v = [&](uint32_t step, Pieces& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int p = wave - V0 + i * NW;
            if (V0 && p < 0) continue;
            const int q = p * (128 / W) + lane / (W / 2), kt = q >> 3, qq = q & 7;
            uint32_t most[4];
#pragma unroll
            for (int j = 0; j < 4; j++) most[j] = max(mag(x[i][j]), mag(x[i][4 + j]));
            const uint32_t top = quad_max<W / 2>(most, lane);  // of key lane % 4
            const int e = lift(top, kValueLift);
            const uint32_t scale = __builtin_bit_cast(uint32_t, pow2f(e));
            const float up[4] = {__builtin_bit_cast(float, dpp_of<0x00>(scale)), __builtin_bit_cast(float, dpp_of<0x55>(scale)),
                                 __builtin_bit_cast(float, dpp_of<0xAA>(scale)), __builtin_bit_cast(float, dpp_of<0xFF>(scale))};
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = x[i][j] * up[j & 3];
            const uint64_t wrong = __ballot(top >= kInf);
            if (__builtin_expect(wrong != 0, 0)) {  // (kept out of the sums; the rows that see it are told by its bit)
                const uint32_t bad = static_cast<uint32_t>(wrong >> (lane / (W / 2) * (W / 2))) & 15;
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = bad >> (j & 3) & 1 ? 0.0f : y[j];
                if (vd == 0 && bad) atomicOr(&st.poison[step % 3][kt], bad << (4 * qq));
            }
            // keys 4 qq .. + 3 are steps 4 jq .. + 3 of lane half hq in product s2
            const int s2 = qq >> 2, jq = qq >> 1 & 1, hq = qq & 1;
#pragma unroll
            for (int ch = 0; ch < 2; ch++) {
                u32x2 hi, lo;
                uint32_t h, l;
                split2(y[4 * ch], y[4 * ch + 1], h, l);
                hi[0] = h;
                lo[0] = l;
                split2(y[4 * ch + 2], y[4 * ch + 3], h, l);
                hi[1] = h;
                lo[1] = l;
                const int dd = vd + ch;
                *reinterpret_cast<u32x2*>(&st.v[step & 1][kt][dd >> 5][s2][0][hq * 32 + st.of(dd & 31)][4 * jq]) = hi;
                *reinterpret_cast<u32x2*>(&st.v[step & 1][kt][dd >> 5][s2][1][hq * 32 + st.of(dd & 31)][4 * jq]) = lo;
            }
            if (vd < 8) {
                st.vexp[step & 1][kt][4 * qq + (lane & 3)] = static_cast<float>(-e);
                st.vup[step & 1][kt][4 * qq + (lane & 3)] = __builtin_bit_cast(float, scale);
            }
        }
    };

    Sums<OT> z;
    clear(z);
    const uint32_t steps = (b.tile1 - b.tile0 + KW - 1) / KW;
    if (threadIdx.x < 3 * KW) st.poison[threadIdx.x / KW][threadIdx.x % KW] = 0;
    Pieces kx, vx;
    h8f qh[KI], ql[KI];
    float qscale;
    {
        Pieces first;
        if (steps) {
            fetch_k(b.tile0, first);
            fetch_v(b.tile0, vx);
            fetch_k(b.tile0 + KW, kx);
        }
        b.column(a, col);
        qscale = load_query<W>(a, b.row, b.head, half, qh, ql);
        if (steps) {
            __syncthreads();  // (the poison is clear)
            stash_k(0, first);
            stash_v(0, vx);
            stash_k(1, kx);
            fetch_k(b.tile0 + 2 * KW, kx);
            fetch_v(b.tile0 + KW, vx);
        }
    }
    const uint32_t row = b.row;
    const int vplace = half * 32 + st.of(col);
    const auto scores = [&](uint32_t step) __attribute__((always_inline)) {
        f32x16 x = f32x16{};
#pragma unroll
        for (int i = 0; i < KI; i++) {
            const h8f kh = *reinterpret_cast<const h8f*>(st.k[step & 1][kw][0][i][half][col]);
            const h8f kl = *reinterpret_cast<const h8f*>(st.k[step & 1][kw][1][i][half][col]);
            x = mfma(kl, qh[i], x);
            x = mfma(kh, ql[i], x);
            x = mfma(kh, qh[i], x);
        }
        return x;
    };
    f32x16 score[2] = {f32x16{}, f32x16{}};  // of even and odd steps' tiles
    if (steps) {
        __syncthreads();
        score[0] = scores(0);
        __syncthreads();
    }
    // Step t multiplies the next tiles' scores while this one's become weights, and stages what comes after them.
    const auto work = [&](uint32_t step, f32x16& u, f32x16& next) __attribute__((always_inline)) {
        const uint32_t first = b.tile0 + step * KW, tile = first + kw, k0 = tile * kKeys;
        const int buf = step & 1;
        const uint32_t poison = __builtin_amdgcn_readfirstlane(st.poison[step % 3][kw]);
        if (threadIdx.x < KW) st.poison[(step + 2) % 3][threadIdx.x] = 0;  // (read at step - 1, written next at step + 1)
        if (tile < b.tile1 && k0 < b.wkeys) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4 down = *reinterpret_cast<const float4*>(&st.kdown[step & 3][kw][8 * g + 4 * half]);
                const float4 ve = *reinterpret_cast<const float4*>(&st.vexp[buf][kw][8 * g + 4 * half]);
                u[4 * g] = fmaf(u[4 * g] * down.x, qscale, ve.x);
                u[4 * g + 1] = fmaf(u[4 * g + 1] * down.y, qscale, ve.y);
                u[4 * g + 2] = fmaf(u[4 * g + 2] * down.z, qscale, ve.z);
                u[4 * g + 3] = fmaf(u[4 * g + 3] * down.w, qscale, ve.w);
            }
            uint32_t seen = ~0u;  // the tile's keys that this column sees
            if (k0 + kKeys > b.wfull) {
                if constexpr (TREE) {
                    const uint32_t* path = a.seen + static_cast<size_t>(row) * a.words;
                    const auto word = [&](uint32_t w) { return w < static_cast<uint32_t>(a.words) ? path[w] : 0u; };
                    if (k0 >= at) {
                        const uint32_t n = k0 - at, sh = n & 31;
                        seen = word(n >> 5) >> sh | (sh ? word((n >> 5) + 1) << (32 - sh) : 0u);
                    } else {
                        seen = at - k0 >= 32 ? ~0u : word(0) << (at - k0) | ((1u << (at - k0)) - 1);
                    }
                    seen = b.on && !b.bad ? seen : 0u;
                    if (keys - k0 < 32) seen &= (1u << (keys - k0)) - 1;
                } else {
                    seen = b.own > k0 ? (b.own - k0 >= 32 ? ~0u : (1u << (b.own - k0)) - 1) : 0u;
                }
                const uint32_t mine = seen >> (half * 4);  // (against constants: 16 shifted bits would stay in registers)
#pragma unroll
                for (int v = 0; v < 16; v++) u[v] = mine & 1u << acc_row(v, 0) ? u[v] : -INFINITY;
            }
            if (__builtin_expect(poison != 0, 0)) z.l = seen & poison ? __builtin_nanf("") : z.l;
            float top = u[0];
#pragma unroll
            for (int v = 1; v < 16; v++) top = fmaxf(top, u[v]);
            raise_base(z, top);
            next = scores(step + 1);
            float w[16];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4 vu = *reinterpret_cast<const float4*>(&st.vup[buf][kw][8 * g + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; j++) w[4 * g + j] = __builtin_amdgcn_exp2f(u[4 * g + j] - z.base);
                z.l = fmaf(w[4 * g], vu.x, z.l);
                z.l = fmaf(w[4 * g + 1], vu.y, z.l);
                z.l = fmaf(w[4 * g + 2], vu.z, z.l);
                z.l = fmaf(w[4 * g + 3], vu.w, z.l);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++) {
                h8f ph, pl;
                split8(w + 8 * s2, ph, pl);
#pragma unroll
                for (int d = 0; d < OT; d++) {
                    const h8f vh = *reinterpret_cast<const h8f*>(st.v[buf][kw][d][s2][0][vplace]);
                    const h8f vl = *reinterpret_cast<const h8f*>(st.v[buf][kw][d][s2][1][vplace]);
                    z.o[d] = mfma(vl, ph, z.o[d]);
                    z.o[d] = mfma(vh, pl, z.o[d]);
                    z.o[d] = mfma(vh, ph, z.o[d]);
                }
            }
        }
        // (past the last step: its last key's, to where nothing reads it)
        stash_k(step + 2, kx);
        stash_v(step + 1, vx);
        if (step + 2 < steps) {
            fetch_k(first + 3 * KW, kx);
            fetch_v(first + 2 * KW, vx);
        }
        __syncthreads();
    };
    for (uint32_t step = 0; step < steps; step += 2) {
        work(step, score[0], score[1]);
        if (step + 1 == steps) break;
        work(step + 1, score[1], score[0]);
    }
    z.l = sum_halves(z.l);
    if constexpr (KW > 1) {
        static_assert(sizeof(Stage<W, CW, KW>) >= (KW - 1) * CW * Sums<OT>::kParts * 64 * sizeof(float2), "the sums fit");
        join_waves<OT, CW, KW>(z, reinterpret_cast<float2*>(smem), cw, kw, lane);
    }
    if (b.shares > 1 && !join_shares<OT, CW>(z, a, b.kv, b.first, b.split, b.shares, cw, kw == 0, lane)) return;
    if (kw == 0 && b.on) store_out<W>(z, a, row, b.head, half, b.bad);
}

template <int W, int CW, int KW, bool TREE>
__global__ void __launch_bounds__(64 * CW * KW, 2) k_gqa_rows(RowsArgs a) {
    extern __shared__ __align__(16) char smem[];
    Block<CW, TREE> b;
    if (b.place(a, blockIdx.x)) rows_block<W, CW, KW, TREE>(a, smem, b);
}

// The blocks that k_gqa_prompt leaves out, if there are any: slower than if nothing had been packed, since a workgroup
// takes every num_cus-th block and a kv head's are every n_kv-th, so that one head keeps one workgroup in n_kv busy (us with no
// row apart, a row of one kv head, rows of all, and nothing packed: 1 x 8192 rows, 32 and 8 heads of width 128 1442, 3300,
// 2000 and 1655 to 1860; 16 x <= 1000, 14 and 2 heads of 64 90, 305, 260 and 107 to 114).
template <int W, int CW>
__global__ void __launch_bounds__(64 * CW, 2) k_gqa_rest(RowsArgs a, uint32_t blocks) {
    extern __shared__ __align__(16) char smem[];
    if (!a.apart[a.pairs.d]) return;
    for (uint32_t id = blockIdx.x; id < blocks; id += gridDim.x) {
        Block<CW, false> b;
        if (b.place(a, id) && a.apart[b.pair]) rows_block<W, CW, 1, false>(a, smem, b);
        __syncthreads();
    }
}

// ---- prompts ---------------------------------------------------------------------------------
//
// Many columns read the same keys, so what a key costs beside its products is done once, in
// a launch of its own: k_gqa_pack writes each tile of 32 keys as the MFMA operands that
// k_gqa_prompt loads, f16 terms under one power of two for the tile's keys and one for its
// values.  Where a tile's rows differ by more than 2^8 in their largest magnitudes, the lower terms
// of some would fall so far below f16's normal numbers that more than 2^-21 of a row were lost to
// the rows beside it.  The blocks of such a (sequence, kv head) are k_gqa_rest's, in a launch behind k_gqa_prompt's (in the
// same kernel, its registers were spilled from those of the hot loop: 16 prompts of up to 1000 rows 76 us
// and 70 without).
template <int W>
struct Packed {
    _Float16 k[W / 16][2][64][8];
    _Float16 v[W / 32][2][2][64][8];
};
struct TileInfo {
    float kdown, vexp, vup;  // 2^-e of the keys; -e and 2^e of the values
    uint32_t poison;         // keys that are not finite, or their values
};
constexpr int kApart = 8;

struct PackArgs {
    const float *kc, *vc;
    size_t seq_stride;
    int n_kv, hd, tiles;  // tiles of a (sequence, kv head)'s room
    uint32_t seqs, total, max_rows, limit;
    const uint32_t *off, *len;
    char* packed;
    TileInfo* info;
    uint32_t* apart;
};

template <int W>
__global__ void __launch_bounds__(kThreads) k_gqa_pack(PackArgs a) {
    constexpr int PER = W / 64 > 0 ? W / 64 : 1;  // pieces of 256 threads, of keys and of values each
    const uint32_t tile = blockIdx.x, kv = blockIdx.y, s = blockIdx.z;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
    const uint32_t keys = r.count ? static_cast<uint32_t>(min(r.at + r.count, static_cast<uint64_t>(a.limit))) : 0;
    if (tile * kKeys >= keys) return;
    __shared__ uint32_t top[2][kKeys];
    const size_t kv_dim = static_cast<size_t>(a.n_kv) * a.hd;
    const float* kp = a.kc + s * a.seq_stride + static_cast<size_t>(kv) * a.hd;
    const float* vp = a.vc + s * a.seq_stride + static_cast<size_t>(kv) * a.hd;
    float x[PER][8], y[PER][8];
    const auto key_of = [&](int i) { return (i * kThreads + static_cast<int>(threadIdx.x)) / (W / 8); };
    const auto quad_of = [&](int i) { return (i * kThreads + static_cast<int>(threadIdx.x)) / (W / 2); };
    const int ch = threadIdx.x % (W / 8), dv = threadIdx.x % (W / 2) * 2;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int k = key_of(i), q = quad_of(i);
        // (rows past the last key: zeros)
        const float* from = kp + static_cast<size_t>(tile * kKeys + k) * kv_dim + ch * 8;
        const bool in = k < kKeys && tile * kKeys + k < keys && (W > 32 || ch * 8 < a.hd);
        const float4 u = in ? *reinterpret_cast<const float4*>(from) : make_float4(0, 0, 0, 0);
        const float4 w = in ? *reinterpret_cast<const float4*>(from + 4) : make_float4(0, 0, 0, 0);
        x[i][0] = u.x; x[i][1] = u.y; x[i][2] = u.z; x[i][3] = u.w;
        x[i][4] = w.x; x[i][5] = w.y; x[i][6] = w.z; x[i][7] = w.w;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t key = tile * kKeys + 4 * q + j;
            const bool vin = q < 8 && key < keys && (W > 32 || dv < a.hd);
            const float2 t = vin ? *reinterpret_cast<const float2*>(vp + key * kv_dim + dv) : make_float2(0, 0);
            y[i][j] = t.x;
            y[i][4 + j] = t.y;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, mag(x[i][j]));
        m = group_max<W / 8>(m);
        if (ch == 0 && key_of(i) < kKeys) top[0][key_of(i)] = m;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t t = group_max<W / 2>(max(mag(y[i][j]), mag(y[i][4 + j])));
            if (dv == 0 && quad_of(i) < 8) top[1][4 * quad_of(i) + j] = t;
        }
    }
    __syncthreads();
    // what lane l of every wave holds of row l % 32: keys' in the lower half, values' in the upper one
    const int lane = threadIdx.x & 63, of = lane >> 5;
    const uint32_t mine = top[of][lane & 31];
    const bool used = tile * kKeys + (lane & 31) < keys && mine > 0 && mine < kInf;
    int hi = used ? static_cast<int>(mine >> 23) : 0, lo = used ? static_cast<int>(mine >> 23) : 255;
    hi = static_cast<int>(group_max<32>(static_cast<uint32_t>(hi)));
    lo = 255 - static_cast<int>(group_max<32>(static_cast<uint32_t>(255 - lo)));
    const int e = lift(static_cast<uint32_t>(hi) << 23, of ? kValueLift : kLiftMost);
    const uint32_t pair = s * static_cast<uint32_t>(a.n_kv) + kv;
    if (threadIdx.x < 64) {
        TileInfo& info = a.info[static_cast<size_t>(pair) * a.tiles + tile];
        if (lane == 0) info.kdown = pow2f(-e);
        if (lane == 32) {
            info.vexp = static_cast<float>(-e);
            info.vup = pow2f(e);
        }
        const uint64_t bad = __ballot(mine >= kInf);
        if (lane == 0) info.poison = static_cast<uint32_t>(bad >> 32 | bad);
        if (__any(hi - lo > kApart) && lane == 0) {
            atomicOr(a.apart + pair, 1u);
            atomicOr(a.apart + static_cast<uint32_t>(a.n_kv) * a.seqs, 1u);
        }
    }
    const float kup = pow2f(__builtin_amdgcn_readlane(e, 0)), vup = pow2f(__builtin_amdgcn_readlane(e, 32));
    Packed<W>& to = reinterpret_cast<Packed<W>*>(a.packed)[static_cast<size_t>(pair) * a.tiles + tile];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int k = key_of(i), q = quad_of(i);
        // (what is not finite is kept out of the products; the rows that see it are told by its bit)
        if (k < kKeys) {
            const bool bad = top[0][k] >= kInf;
            u32x4 h, l;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t b, c;
                split2(bad ? 0.0f : x[i][2 * j] * kup, bad ? 0.0f : x[i][2 * j + 1] * kup, b, c);
                h[j] = b;
                l[j] = c;
            }
            *reinterpret_cast<u32x4*>(to.k[ch >> 1][0][(ch & 1) * 32 + k]) = h;
            *reinterpret_cast<u32x4*>(to.k[ch >> 1][1][(ch & 1) * 32 + k]) = l;
        }
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = q < 8 && top[1][4 * (q & 7) + (j & 3)] >= kInf ? 0.0f : y[i][j] * vup;
        if (q < 8) {
            // keys 4 q .. + 3 are steps 4 (q / 2 % 2) .. + 3 of lane half q % 2 in product q / 4
#pragma unroll
            for (int c = 0; c < 2; c++) {
                u32x2 h, l;
                uint32_t b, d;
                split2(z[4 * c], z[4 * c + 1], b, d);
                h[0] = b;
                l[0] = d;
                split2(z[4 * c + 2], z[4 * c + 3], b, d);
                h[1] = b;
                l[1] = d;
                const int dd = dv + c;
                *reinterpret_cast<u32x2*>(&to.v[dd >> 5][q >> 2][0][(q & 1) * 32 + (dd & 31)][4 * (q >> 1 & 1)]) = h;
                *reinterpret_cast<u32x2*>(&to.v[dd >> 5][q >> 2][1][(q & 1) * 32 + (dd & 31)][4 * (q >> 1 & 1)]) = l;
            }
        }
    }
}

// NWV waves of 32 columns a workgroup.  Step t multiplies tile t + 1's scores while tile t's become
// weights, and stages tile t + 2's keys and t + 1's values, so that a wave has work for the matrix and
// for the vector units side by side.  Width 128: eight waves, near the rate of a large f16 product (1 x 8192
// rows of 32 and 8 heads 1420 us, 387 TFLOP/s or 1160 of f16 products; the clock falls as the matrix
// units fill: 2.1 GHz where they were busy 40 % of the time, 1.7 at 60 %; four waves, each tile read
// twice as often, 1557); 64: four, three to a SIMD (16 prompts of up to 1000 rows, 14 and 2 heads, 73
// us, two to a SIMD 77, eight waves 90).  64 columns a wave with a SIMD to itself: 2000 and 125.
template <int W, int NWV, int OCC>
__global__ void __launch_bounds__(64 * NWV, OCC) k_gqa_prompt(RowsArgs a, const char* packed, const TileInfo* infos,
                                                                     int room) {
    constexpr int CW = NWV, KI = W / 16, OT = W / 32, NT = 64 * NWV;
    constexpr int PIECE = W * 8 / NT;  // 16-byte loads a thread, of a tile's keys and of its values
    extern __shared__ __align__(16) char smem[];
    Block<CW, false> b;
    if (!b.place(a, blockIdx.x) || a.apart[b.pair]) return;
    struct Ring {
        u32x4 k[2][W * 8], v[2][W * 8];
    };
    Ring& ring = *reinterpret_cast<Ring*>(smem);
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    b.share(a, wave);
    const uint32_t tile0 = b.tile0, tile1 = b.tile1;
    const uint32_t mine1 = min(tile1, (b.wkeys + kKeys - 1) / kKeys);  // past the wave's last tile

    const u32x4* from = reinterpret_cast<const u32x4*>(packed) + static_cast<size_t>(b.pair) * room * (W * 16) + threadIdx.x;
    const TileInfo* info = infos + static_cast<size_t>(b.pair) * room;
    u32x4 kpiece[PIECE], vpiece[PIECE];
    const auto fetch_k = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PIECE; i++) kpiece[i] = from[static_cast<size_t>(tile) * (W * 16) + i * NT];
    };
    const auto fetch_v = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PIECE; i++) vpiece[i] = from[static_cast<size_t>(tile) * (W * 16) + W * 8 + i * NT];
    };
    const auto put_k = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PIECE; i++) ring.k[tile & 1][i * NT + threadIdx.x] = kpiece[i];
    };
    const auto put_v = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PIECE; i++) ring.v[tile & 1][i * NT + threadIdx.x] = vpiece[i];
    };
    // (the first tiles are on their way while the queries are split)
    const uint32_t second = min(tile0 + 1, max(tile1, 1u) - 1);
    u32x4 ahead[PIECE];
    if (tile0 < tile1) {
        fetch_k(second);
#pragma unroll
        for (int i = 0; i < PIECE; i++) ahead[i] = kpiece[i];
        fetch_k(tile0);
        fetch_v(tile0);
    }
    b.column(a, col);
    h8f qh[KI], ql[KI];
    const float qscale = load_query<W>(a, b.row, b.head, half, qh, ql);
    const auto scores = [&](uint32_t tile) __attribute__((always_inline)) {
        f32x16 x = f32x16{};
        const u32x4* k = ring.k[tile & 1] + lane;
#pragma unroll
        for (int i = 0; i < KI; i++) {
            const h8f kh = __builtin_bit_cast(h8f, k[(2 * i) * 64]), kl = __builtin_bit_cast(h8f, k[(2 * i + 1) * 64]);
            x = mfma(kl, qh[i], x);
            x = mfma(kh, ql[i], x);
            x = mfma(kh, qh[i], x);
        }
        return x;
    };
    Sums<OT> z;
    clear(z);
    f32x16 score[2] = {f32x16{}, f32x16{}};  // of even and odd steps' tiles
    if (tile0 < tile1) {
        put_k(tile0);
        put_v(tile0);
#pragma unroll
        for (int i = 0; i < PIECE; i++) kpiece[i] = ahead[i];
        put_k(tile0 + 1);
        __syncthreads();
        score[0] = scores(tile0);
        __syncthreads();
    }
    const auto step = [&](uint32_t tile, f32x16& now, f32x16& next) __attribute__((always_inline)) {
        const uint32_t k0 = tile * kKeys, last = tile1 - 1;
        // (past the last tile: it again, to where nothing reads it)
        fetch_k(min(tile + 2, last));
        fetch_v(min(tile + 1, last));
        if (tile < mine1) {
            const TileInfo of = info[tile];
            if (k0 + kKeys > b.wfull) {
                const uint32_t seen = b.own > k0 ? (b.own - k0 >= 32 ? ~0u : (1u << (b.own - k0)) - 1) : 0u;
                const uint32_t mine = seen >> (half * 4);
#pragma unroll
                for (int v = 0; v < 16; v++) now[v] = mine & 1u << acc_row(v, 0) ? now[v] : -INFINITY;
            }
            if (__builtin_expect(of.poison != 0, 0)) {
                const uint32_t seen = b.own > k0 ? (b.own - k0 >= 32 ? ~0u : (1u << (b.own - k0)) - 1) : 0u;
                z.l = seen & of.poison ? __builtin_nanf("") : z.l;
            }
            const float sc = of.kdown * qscale;
            float top = now[0];
#pragma unroll
            for (int v = 1; v < 16; v++) top = fmaxf(top, now[v]);
            raise_base(z, fmaf(top, sc, of.vexp));
            const float less = of.vexp - z.base;
            float u[16], sum[4] = {};
            next = scores(tile + 1);
#pragma unroll
            for (int v = 0; v < 16; v++) {
                u[v] = __builtin_amdgcn_exp2f(fmaf(now[v], sc, less));
                sum[v & 3] += u[v];
            }
            z.l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), of.vup, z.l);
            const u32x4* v = ring.v[tile & 1] + lane;
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++) {
                h8f ph, pl;
                split8(u + 8 * s2, ph, pl);
#pragma unroll
                for (int d = 0; d < OT; d++) {
                    const h8f vh = __builtin_bit_cast(h8f, v[((d * 2 + s2) * 2) * 64]);
                    const h8f vl = __builtin_bit_cast(h8f, v[((d * 2 + s2) * 2 + 1) * 64]);
                    z.o[d] = mfma(vl, ph, z.o[d]);
                    z.o[d] = mfma(vh, pl, z.o[d]);
                    z.o[d] = mfma(vh, ph, z.o[d]);
                }
            }
        }
        put_k(tile + 2);
        put_v(tile + 1);
        __syncthreads();
    };
    for (uint32_t tile = tile0; tile < tile1; tile += 2) {
        step(tile, score[0], score[1]);
        if (tile + 1 == tile1) break;
        step(tile + 1, score[1], score[0]);
    }
    z.l = sum_halves(z.l);
    if (b.shares > 1 && !join_shares<OT, CW>(z, a, b.kv, b.first, b.split, b.shares, wave, true, lane)) return;
    if (b.on) store_out<W>(z, a, b.row, b.head, half, b.bad);
}

constexpr size_t kUnits = 65536;  // counters: sequences of a tree's acceptance, or

template <int W, int CW, int KW, bool TREE>
int launch_rows(fh_ctx* ctx, const RowsArgs& a, uint32_t workgroups) {
    constexpr size_t lds = sizeof(Stage<W, CW, KW>);
    static_assert(lds <= 160 * 1024, "a stage fits the LDS");
    const auto kern = k_gqa_rows<W, CW, KW, TREE>;
    if (lds > 64 * 1024)
        FH_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    hipLaunchKernelGGL(kern, dim3(workgroups), dim3(64 * CW * KW), lds, ctx->stream, a);
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

template <int W, int NWV, int OCC>
int launch_prompt(fh_ctx* ctx, const RowsArgs& a, const PackArgs& p, uint32_t workgroups) {
    hipLaunchKernelGGL(k_gqa_pack<W>, dim3(p.tiles, a.kvs.d, a.seqs), dim3(kThreads), 0, ctx->stream, p);
    FH_HIP(ctx, hipGetLastError());
    constexpr size_t lds = 2 * W * 256;
    static_assert(lds <= 64 * 1024, "without a larger limit");
    hipLaunchKernelGGL((k_gqa_prompt<W, NWV, OCC>), dim3(workgroups), dim3(64 * NWV), lds, ctx->stream, a, p.packed, p.info, p.tiles);
    FH_HIP(ctx, hipGetLastError());
    constexpr size_t rest = sizeof(Stage<W, NWV, 1>);
    const auto kern = k_gqa_rest<W, NWV>;
    if (rest > 64 * 1024)
        FH_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(rest)));
    hipLaunchKernelGGL(kern, dim3(std::min(workgroups, static_cast<uint32_t>(ctx->num_cus))), dim3(64 * NWV), rest, ctx->stream, a, workgroups);
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

// (k_gqa_rows<128, 4, 1, ..> keeps 8 registers in scratch, 36 bytes a thread, since keys' pieces and values' groups have
// banks of their own; <128, 8, 1, ..> and the narrower ones none.)
template <int W, bool TREE>
int launch_width(fh_ctx* ctx, const RowsArgs& a, uint32_t workgroups, int cw) {
    if constexpr (W == 128) return cw == 8 ? launch_rows<W, 8, 1, TREE>(ctx, a, workgroups) : launch_rows<W, 4, 1, TREE>(ctx, a, workgroups);
    else return cw == 4 ? launch_rows<W, 4, 1, TREE>(ctx, a, workgroups) : launch_rows<W, 2, 2, TREE>(ctx, a, workgroups);
}

}  // namespace

int fh_launch_gqa_rows(fh_ctx* ctx, const fh_gqa_call& g) {
    const size_t group = g.n_heads / g.n_kv, cols = g.max_rows * group, heads = g.seqs * g.n_kv;
    const int words = g.parent ? static_cast<int>((g.max_rows + 31) / 32) : 0;
    const int w = g.hd <= 32 ? 32 : static_cast<int>(g.hd);
    const size_t tiles = (g.limit + kKeys - 1) / kKeys, pack = heads * tiles * (static_cast<size_t>(w) * 256);
    // The launches that pack the tiles and that look for blocks apart are about 15 us, won back where many column
    // blocks read the same tiles and there are enough of both (us packed and not, heads of width 64: 1 prompt of 1000
    // rows, 14 and 2 heads 41 and 32, of 2000 55 and 56; 16 of up to 1000 rows 91 and 107; 8 of up to 1000, 12 and 12
    // heads 81 and 72; of width 128, 32 and 8 heads: 1 prompt of 1000 rows 66 and 63, of 1500 106 and 112, of 2000 168
    // and 190).  Not in a room of 2 GiB and more, which would stay with the context, and be twice as large where it grows, for
    // little (ms packed and not, those heads: 24 prompts of 512 rows behind 15872, 3 GiB, 10.4 and 10.4, 32 of 1024 behind
    // 7168, 2 GiB, 12.9 and 13.8, 16 of 2048 behind 14336, 2 GiB, 23.0 and 25.6).
    const bool prompt = !g.parent && cols > 1024 && heads * cols * tiles > (size_t(3) << 19) && pack < (size_t(1) << 31);
    // Columns of a workgroup: as many as there are, while two workgroups fit a compute unit; of 64 columns and two waves that deal
    // the keys for small calls (us of 64 and of 128: one tree of 100 nodes over 4000 rows, 4 heads of width 32 24.4 and
    // 26.3, one of 16 nodes over 511, 14 and 2 heads of 64 20.6 and 20.9, 32 of up to 32 nodes over up to 1023 39.8 and
    // 36.4).  Width 128: eight waves with the keys split once for 256 columns (4 trees of up to 64 nodes over up to 16383
    // rows, 32 and 8 heads 208 us, four waves 234).
    const int cw = w == 128 ? (cols > 128 ? 8 : 4) : cols > 128 ? 4 : 2;
    const size_t blocks = (cols + 32 * cw - 1) / (32 * cw);
    if (heads * blocks > 0x7FFFFFFFu / 64) return fh_fail(ctx, FH_ERR_LIMIT, "fh_gqa_attention: more than 2^25 workgroups");
    // Keys of few columns are dealt over as many workgroups as the device holds at once, two tiles of keys each at
    // least (those 4 trees, when this was added: 215 us, 283 with equal numbers of shares for all sequences).
    const size_t cus = static_cast<size_t>(ctx->num_cus), units = g.seqs * blocks;
    // Where a compute unit has 16 tiles at most, one workgroup on each: two would meet on some while others had none (us
    // with one and with two, 14 and 2 heads of width 64: a tree of 16 nodes over 16000 rows, 8 tiles each, 34 and 39,
    // over 30000, 15 tiles, 41 and 44, over 36000, 18 tiles, 44 and 47; 8 trees of 32 nodes over up to 2000, 8 tiles, 30 and
    // 33, over up to 4000, 16 tiles, 39 and 40, over up to 5000, 20 tiles, 44 and 43; 32 and 8 heads of 128: 4 of 32 over up
    // to 3000, 12 tiles, 58 and 64, over up to 5000, 20 tiles, 72 and 74).  With as many blocks as fill half of the device
    // by themselves the two meet sooner: 32 trees of up to 32 nodes over up to 511, 8 tiles, 29 and 29, over up to 767, 12
    // tiles, 35 and 33, over up to 960, 15 tiles, 39 and 35, over up to 1023, 17 tiles, 40 and 36.
    const bool few = units * tiles * g.n_kv <= 16 * cus;
    const size_t all = cus * (cw == 8 || few ? 1 : prompt ? 3 : 2), places = all / g.n_kv;
    const bool planned = units <= std::min<size_t>(places, kPlanned) && tiles >= 4;
    const uint32_t workgroups = static_cast<uint32_t>(planned ? places * g.n_kv : heads * blocks);
    unsigned* counters = nullptr;
    if (planned) {
        void* area = nullptr;
        const int rc = fh_gqa_counters(ctx, kUnits * sizeof(unsigned), &area);
        if (rc) return rc;
        counters = static_cast<unsigned*>(area);
    }
    // Queries are rotated where they are loaded, from a table of their rows' cosines and sines; where a load
    // has not both channels of its pairs, or is not aligned, by the first launch (12700 rows of 14 and 2 heads of
    // width 64: 9.5 us of it against 21).
    const size_t half = g.rope_dim / 2;
    const bool copy = (reinterpret_cast<uintptr_t>(g.qkv) | g.ld * sizeof(float)) % 16 != 0 ||
                      (g.rope_dim && (g.rope_type == FH_ROPE_NEOX ? half % 16 != 0 : half % 2 != 0));
    const size_t q_bytes = fh_align256(copy ? g.total * g.n_heads * g.hd * sizeof(float) : g.total * half * sizeof(float2));
    const size_t seen_bytes = fh_align256(g.total * words * sizeof(uint32_t));
    const size_t part = planned ? workgroups * (cw * (1 + w / 4) * 64 * sizeof(float2)) : 0;
    const size_t plan_bytes = planned ? fh_align256(places * sizeof(Share)) : 0;
    const size_t info_bytes = prompt ? heads * tiles * sizeof(TileInfo) + (heads + 1) * sizeof(uint32_t) : 0;
    void* room = nullptr;
    const int rc = fh_kv4_room(ctx, q_bytes + seen_bytes + plan_bytes + fh_align256(part) + (prompt ? pack + info_bytes : 0), &room);
    if (rc) return rc;

    AppendArgs p{};
    p.qkv = g.qkv;
    p.ld = g.ld;
    p.kc = g.k_cache;
    p.vc = g.v_cache;
    p.seq_stride = g.capacity * g.n_kv * g.hd;
    p.n_heads = static_cast<int>(g.n_heads);
    p.n_kv = static_cast<int>(g.n_kv);
    p.hd = static_cast<int>(g.hd);
    p.seqs = static_cast<uint32_t>(g.seqs);
    p.total = static_cast<uint32_t>(g.total);
    p.max_rows = static_cast<uint32_t>(g.max_rows);
    p.limit = static_cast<uint32_t>(g.limit);
    p.off = g.off;
    p.len = g.len;
    p.pos = g.pos;
    p.parent = g.parent;
    PackArgs k{};
    if (prompt) {
        k.packed = static_cast<char*>(room) + q_bytes + seen_bytes + plan_bytes + fh_align256(part);
        k.info = reinterpret_cast<TileInfo*>(k.packed + pack);
        k.apart = reinterpret_cast<uint32_t*>(k.info + heads * tiles);
        p.clear = k.apart;
    }
    if (planned) {
        p.plan = reinterpret_cast<Share*>(static_cast<char*>(room) + q_bytes + seen_bytes);
        p.places = static_cast<uint32_t>(places);
        p.col_blocks = static_cast<uint32_t>(blocks);
        p.cols = 32 * cw;
    }
    p.group = Div(static_cast<uint32_t>(group));
    if (copy) p.q = static_cast<float*>(room);
    else if (half) p.cs = static_cast<float2*>(room);
    p.first = copy ? 0 : static_cast<int>(g.n_heads);
    p.seen = reinterpret_cast<uint32_t*>(static_cast<char*>(room) + q_bytes);
    p.words = words;
    p.rope_dim = static_cast<int>(g.rope_dim);
    p.neox = g.rope_type == FH_ROPE_NEOX;
    p.linear = g.linear_factor;
    p.ff = g.freq_factors;
    // (the frequencies as fh_rope_async forms them: in 64 bits, then rounded)
    for (size_t i = 0; i < g.rope_dim / 2; i++)
        p.freq[i] = static_cast<float>(std::pow(static_cast<double>(g.base), -2.0 * static_cast<double>(i) / static_cast<double>(g.rope_dim)));
    const size_t each = 2 * kThreads / g.hd, row_blocks = (g.max_rows + each - 1) / each, takes = (copy ? g.n_heads : 0) + 2 * g.n_kv;
    size_t chunks = 1;
    while (chunks < takes && row_blocks * g.seqs * chunks < 4 * cus) chunks *= 2;
    p.heads_each = static_cast<int>((takes + chunks - 1) / chunks);
    p.chunks = static_cast<int>((takes + p.heads_each - 1) / p.heads_each);
    const dim3 grid(static_cast<unsigned>(row_blocks * p.chunks), static_cast<unsigned>(g.seqs + planned));
    if (g.parent) hipLaunchKernelGGL(k_gqa_append<true>, grid, dim3(kThreads), 0, ctx->stream, p);
    else hipLaunchKernelGGL(k_gqa_append<false>, grid, dim3(kThreads), 0, ctx->stream, p);
    FH_HIP(ctx, hipGetLastError());

    RowsArgs a{};
    a.q = copy ? p.q : g.qkv;
    a.q_ld = copy ? g.n_heads * g.hd : g.ld;
    a.cs = p.cs;
    a.half = static_cast<int>(half);
    a.neox = p.neox;
    a.kc = g.k_cache;
    a.vc = g.v_cache;
    a.seq_stride = p.seq_stride;
    a.n_heads = p.n_heads;
    a.n_kv = p.n_kv;
    a.group = Div(static_cast<uint32_t>(group));
    a.pairs = Div(static_cast<uint32_t>(heads));
    a.kvs = Div(static_cast<uint32_t>(g.n_kv));
    a.hd = p.hd;
    a.seqs = p.seqs;
    a.total = p.total;
    a.max_rows = p.max_rows;
    a.limit = p.limit;
    a.off = g.off;
    a.len = g.len;
    a.seen = p.seen;
    a.words = words;
    a.scale = kLog2e / sqrtf(static_cast<float>(g.hd));
    a.out = g.out;
    a.col_blocks = static_cast<int>(blocks);
    a.plan = p.plan;
    a.places = workgroups;
    a.part = reinterpret_cast<float2*>(static_cast<char*>(room) + q_bytes + seen_bytes + plan_bytes);
    a.counters = counters;
    if (prompt) {
        a.apart = k.apart;
        k.kc = g.k_cache;
        k.vc = g.v_cache;
        k.seq_stride = p.seq_stride;
        k.n_kv = p.n_kv;
        k.hd = p.hd;
        k.tiles = static_cast<int>(tiles);
        k.seqs = p.seqs;
        k.total = p.total;
        k.max_rows = p.max_rows;
        k.limit = p.limit;
        k.off = g.off;
        k.len = g.len;
        return w == 32 ? launch_prompt<32, 4, 3>(ctx, a, k, workgroups) : w == 64 ? launch_prompt<64, 4, 3>(ctx, a, k, workgroups) : launch_prompt<128, 8, 2>(ctx, a, k, workgroups);
    }
    if (g.parent) return w == 32 ? launch_width<32, true>(ctx, a, workgroups, cw) : w == 64 ? launch_width<64, true>(ctx, a, workgroups, cw) : launch_width<128, true>(ctx, a, workgroups, cw);
    return w == 32 ? launch_width<32, false>(ctx, a, workgroups, cw) : w == 64 ? launch_width<64, false>(ctx, a, workgroups, cw) : launch_width<128, false>(ctx, a, workgroups, cw);
}

// ---- what is accepted of a tree ------------------------------------------------------------

namespace {

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // (the planes' addresses are not known here)

struct AcceptArgs {
    const uint32_t *parent, *tokens, *chosen, *off, *len;
    uint32_t seqs, total, max_rows;
    uint32_t *path, *count, *next, *new_len;
    const uint64_t* planes;
    size_t n_planes, kv_dim, capacity;
    uint64_t stored;  // cache rows of a sequence: nothing is accepted from there on
};

// A workgroup a sequence and cache plane (without planes, a sequence): every row finds out whether it
// continues its parent with the token chosen there, the first such is its parent's child, and one thread
// follows the children from row 0, as far as their keys and values were stored (a row that was not has scores
// that are no numbers, and rows of a path rise: none behind it was); then the plane's accepted rows move to their places, as many at a
// time as 256 threads hold.  A row moves down only, and all of a batch is read before any of it is
// written: what a write overwrites has moved or is left behind.  Latency: a chain of three loads, the
// walk and the move (one sequence of 16 rows and 48 planes 3.8 us, 32 of up to 32 rows 5.1; the walk and the move in
// launches of their own 5.9 and 6.4 and the time between).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_tree_accept(AcceptArgs a, unsigned* arrived) {
    constexpr int HOLD = 4;
    __shared__ uint32_t up[kMaxTree], child[kMaxTree], way[kMaxTree], chosen[kMaxTree];
    __shared__ uint32_t steps;
    const uint32_t s = blockIdx.x;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.seqs, s);
    const uint64_t base = a.n_planes ? a.planes[blockIdx.y] : 0;
    const uint32_t len = static_cast<uint32_t>(r.at);
    for (uint32_t t = threadIdx.x; t < r.count; t += kThreads) {
        up[t] = a.parent[r.begin + t];
        way[t] = a.tokens[r.begin + t];
        chosen[t] = a.chosen[r.begin + t];
        child[t] = ~0u;
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < r.count; t += kThreads)
        if (up[t] < t && way[t] == chosen[up[t]]) atomicMin(&child[up[t]], t);
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t n = 0;
        for (uint32_t t = 0; t < r.count && r.at + t < a.stored; t = child[t]) way[n++] = t;  // (~0 ends it)
        steps = n;
    }
    __syncthreads();
    const uint32_t n = steps;
    if (blockIdx.y == 0) {
        for (uint32_t t = threadIdx.x; t < r.count; t += kThreads) a.path[r.begin + t] = t < n ? way[t] : ~0u;
        if (threadIdx.x == 0) {
            a.count[s] = n;
            if (n) a.next[s] = chosen[way[n - 1]];
        }
    }
    // The new length goes out when every workgroup of the sequence has read the old one, which it may replace.
    if (threadIdx.x == 0) {
        const bool last = !arrived || atomicAdd(arrived + s, 1u) == gridDim.y - 1;
        if (arrived ? last : blockIdx.y == 0) {
            a.new_len[s] = len + n;
            if (arrived) __hip_atomic_store(arrived + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (!a.n_planes) return;
    const size_t width = a.kv_dim / (sizeof(T) / sizeof(float));
    T* plane = reinterpret_cast<T*>(base) + static_cast<size_t>(s) * a.capacity * width;
    for (size_t c0 = 0; c0 < width; c0 += kThreads * HOLD) {
        const uint32_t wide = static_cast<uint32_t>(min(width - c0, static_cast<size_t>(kThreads * HOLD)));
        const uint32_t rows = kThreads * HOLD / wide;  // of a batch
        for (uint32_t i0 = 1; i0 < n; i0 += rows) {
            T x[HOLD];
            size_t to[HOLD];
            bool moves[HOLD];
#pragma unroll
            for (int j = 0; j < HOLD; j++) {
                const uint32_t item = static_cast<uint32_t>(j) * kThreads + threadIdx.x, i = i0 + item / wide;
                moves[j] = item / wide < rows && i < n;
                if (!moves[j]) continue;
                const uint64_t p = way[i];
                moves[j] = p != i;
                if (!moves[j]) continue;
                to[j] = static_cast<size_t>(r.at + i) * width + c0 + item % wide;
                x[j] = plane[static_cast<size_t>(r.at + p) * width + c0 + item % wide];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < HOLD; j++)
                if (moves[j]) plane[to[j]] = x[j];
        }
    }
}

}  // namespace

int fh_launch_tree_accept(fh_ctx* ctx, const uint32_t* parent, const uint32_t* tokens, const uint32_t* chosen, size_t total,
                          const uint32_t* off, size_t seqs, size_t max_rows, const uint32_t* len, const uint64_t* planes,
                          size_t n_planes, size_t kv_dim, size_t capacity, size_t max_keys, uint32_t* path,
                          uint32_t* count, uint32_t* next, uint32_t* new_len) {
    AcceptArgs a{parent, tokens, chosen, off, len, static_cast<uint32_t>(seqs), static_cast<uint32_t>(total),
                 static_cast<uint32_t>(max_rows), path, count, next, new_len, planes, n_planes, kv_dim, capacity,
                 n_planes ? std::min(capacity, max_keys) : max_keys};
    unsigned* arrived = nullptr;
    if (new_len == len && n_planes > 1) {
        void* area = nullptr;
        const int rc = fh_gqa_counters(ctx, kUnits * sizeof(unsigned), &area);
        if (rc) return rc;
        arrived = static_cast<unsigned*>(area);
    }
    const dim3 grid(a.seqs, static_cast<unsigned>(std::max<size_t>(n_planes, 1)));
    if (kv_dim % 4 == 0) hipLaunchKernelGGL(k_tree_accept<f4>, grid, dim3(kThreads), 0, ctx->stream, a, arrived);
    else hipLaunchKernelGGL(k_tree_accept<float>, grid, dim3(kThreads), 0, ctx->stream, a, arrived);
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}
