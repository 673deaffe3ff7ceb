// fh_kv4.hip — a key/value cache held in 4 bits, and the attention over it
// (ferrum_core's KvCache and Attention::forward_one, llm.rs:285-358, whose cache
// is f32; the 4-bit form, the score options and the eviction have no reference
// counterpart).
//
// Format.  Blocks of 32 channels of one key (or value) row x: with m the first
// channel of largest magnitude, the scale d = f16(m / -8) and the levels
// q = clamp(rint(x / d), -8, 7) + 8; the block stands for d (q - 8).  Per
// (sequence, kv head) plane, positions in order:
//   k    [position][g: 4][block][4 bytes]: the 8 nibbles of word (g, block) are
//        channels 32 block + 8 g .. + 7, the eight that lane group g of an MFMA
//        holds of a row, so a lane's share of all blocks is one load;
//   v    [position / 8][n][pair of blocks][position % 8] 2-byte units: byte h,
//        nibble e is channel 2 n + e of block 2 pair + h, so that 16 bytes are
//        one lane's eight contraction steps of four output tiles (head width 32:
//        8 units, the unit's byte h is n + 8 h of the only block);
//   k_d, v_d  [position / 8][block][position % 8] f16.
#include "fh_internal.hpp"

#include <algorithm>
#include <cfloat>

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int HD>
struct Shape {
    static constexpr int NB = HD / 32;                 // blocks of a row
    static constexpr int N = HD >= 64 ? 16 : 8;        // units of v per position and pair of blocks
    static constexpr int BP = HD >= 64 ? HD / 64 : 1;  // 2-byte units of v per lane
};

struct Cache {
    uint8_t* k;
    uint16_t* kd;
    uint8_t* v;
    uint16_t* vd;
    uint32_t* pos;
    float* weight;
    int seqs, n_kv, cap;
};

struct AttnArgs {
    Cache c;
    const float* q;
    size_t ld;
    uint32_t total, max_rows, max_keys;
    int n_heads, group;
    const uint32_t *off, *len;
    float softcap, scale;
    const float* slopes;
    const uint32_t *qpos, *first, *end;
    float* out;
    float* lse;
    const float* lse_in;
    float* part;
    unsigned* counters;
    int col_tiles, splits;
};

// Rows [begin, begin + count) of the call's q / out belong to sequence s, and
// its row t is cache row at + t.  What the device arrays say is cut to the
// call's own bounds, so no value of theirs leads outside its buffers.
struct Rows {
    uint32_t begin, count;
    uint64_t at;
};
__device__ __forceinline__ Rows rows_of(const uint32_t* off, const uint32_t* len, uint32_t total, uint32_t max_rows,
                                        int seqs, int s) {
    Rows r;
    if (off) {
        r.begin = min(off[s], total);
        const uint32_t fin = min(off[s + 1], total);
        r.count = fin > r.begin ? min(fin - r.begin, max_rows) : 0;
    } else {
        r.count = total / static_cast<uint32_t>(seqs);
        r.begin = r.count * static_cast<uint32_t>(s);
    }
    r.at = len ? len[s] : 0;
    return r;
}

// One lane's share of 32 keys of a cache: lane (g, n) = (lane / 16, lane % 16)
// holds key rows 8 (n / 4) + n % 4 and + 4 as MFMA rows, and of the eight keys
// 8 g .. 8 g + 7 their scales and its output channels' value levels.
template <int HD>
struct Tile {
    uint32_t k[2][Shape<HD>::NB];
    u32x4 kd[Shape<HD>::NB];
    u32x4 v[Shape<HD>::BP];
    u32x4 vd[Shape<HD>::NB];
    uint32_t vx;  // two scales of the tile's values, for their exponent
};

struct Planes {
    const uint8_t* k;
    const uint16_t* kd;
    const uint8_t* v;
    const uint16_t* vd;
};
template <int HD>
__device__ __forceinline__ Planes planes_of(const Cache& c, int s, int kv) {
    constexpr int NB = Shape<HD>::NB;
    const size_t rows = (static_cast<size_t>(s) * c.n_kv + kv) * c.cap;
    return {c.k + rows * (HD / 2), c.kd + rows * NB, c.v + rows * (HD / 2), c.vd + rows * NB};
}

template <int HD>
__device__ __forceinline__ void load_k(const Planes& p, int cap, int tile, int lane, uint32_t (&k)[2][Shape<HD>::NB],
                                       u32x4 (&kd)[Shape<HD>::NB]) {
    constexpr int NB = Shape<HD>::NB;
    const int g = lane >> 4, n = lane & 15;
    const int key = tile * 32 + 8 * (n >> 2) + (n & 3);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        // (a tile's end past the capacity reads the last row again; the mask drops it)
        const uint8_t* a = p.k + static_cast<size_t>(min(key + 4 * h, cap - 1)) * (HD / 2) + g * (4 * NB);
        if constexpr (NB == 4) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(a);
#pragma unroll
            for (int b = 0; b < 4; b++) k[h][b] = w[b];
        } else if constexpr (NB == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(a);
            k[h][0] = w[0];
            k[h][1] = w[1];
        } else {
            k[h][0] = *reinterpret_cast<const uint32_t*>(a);
        }
    }
    const size_t o = min(tile * 4 + g, cap / 8 - 1);
#pragma unroll
    for (int b = 0; b < NB; b++) kd[b] = *reinterpret_cast<const u32x4*>(p.kd + (o * NB + b) * 8);
}

template <int HD>
__device__ __forceinline__ void load_tile(const Planes& p, int cap, int tile, int lane, Tile<HD>& t) {
    constexpr int NB = Shape<HD>::NB, N = Shape<HD>::N, BP = Shape<HD>::BP;
    load_k<HD>(p, cap, tile, lane, t.k, t.kd);
    const int g = lane >> 4, n = lane & 15, last = cap / 8 - 1;
    const size_t o = min(tile * 4 + g, last);
#pragma unroll
    for (int i = 0; i < BP; i++)
        t.v[i] = *reinterpret_cast<const u32x4*>(p.v + ((o * N + n % N) * BP + i) * 16);
#pragma unroll
    for (int b = 0; b < NB; b++) t.vd[b] = *reinterpret_cast<const u32x4*>(p.vd + (o * NB + b) * 8);
    const int i = lane % (16 * NB);
    const size_t ox = min(tile * 4 + i / (4 * NB), last);
    t.vx = *reinterpret_cast<const uint32_t*>(p.vd + ox * (NB * 8) + i % (4 * NB) * 2);
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}
__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Four levels of each 16-bit half of a word as f16 operands, level - 8 as itself:
// under the exponent of 1024 a nibble of bits 0 .. 3 is 1024 + level, one of bits 4
// .. 7 is 1024 + 16 level, and one packed add or FMA (exact) takes the 1024 and the
// 8 away.  (The matrix cores take the bare nibble too, a subnormal level * 2^-24,
// for half the instructions, but align products by the operands' exponent fields
// and cut them 23 bits below the largest: a subnormal's leading zeros come out of
// those 23 bits, 1e-5 of the result.)
template <int E>
__device__ __forceinline__ uint32_t levels2(uint32_t w) {
    const uint32_t x = ((E & 2 ? w >> 8 : w) & (E & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
    const half2v v = __builtin_bit_cast(half2v, x);
    const _Float16 sixteenth = static_cast<_Float16>(0.0625f);
    const half2v r = E & 1 ? __builtin_elementwise_fma(v, half2v{sixteenth, sixteenth}, half2v{-72, -72})
                           : v - half2v{1032, 1032};
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ half8 k_levels(uint32_t w) {
    return as_half8(levels2<0>(w), levels2<1>(w), levels2<2>(w), levels2<3>(w));
}
template <int E>  // nibble E (0 .. 3) of each 16-bit unit
__device__ __forceinline__ half8 v_levels(const u32x4& w) {
    return as_half8(levels2<E>(w[0]), levels2<E>(w[1]), levels2<E>(w[2]), levels2<E>(w[3]));
}
__device__ __forceinline__ float half_at(const u32x4& w, int i) {
    return fh_h2f(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
}
// Two f32 as a pair of f16 and what that leaves, each rounded to nearest: 22 bits in all.
// (The values are kept from the compiler's view: it would form a product's hi in one
// mixed-precision instruction, with one rounding, and lo from the twice rounded one.)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    asm("" : "+v"(a), "+v"(b));
    const half2v h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    const half2v l = {static_cast<_Float16>(a - static_cast<float>(h[0])),
                      static_cast<_Float16>(b - static_cast<float>(h[1]))};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}
__device__ __forceinline__ float across_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// c tanh(x / c).  Up to 0.6 a polynomial (least maximum error over [0, 0.36] of
// tanh(y) / y in y^2: 2.4e-9), past it 1 - 2 / (1 + e^2y), whose rounding is then
// no larger than the result's own.
__device__ __forceinline__ float capped(float x, float cap, float inv_cap) {
    const float y = x * inv_cap, a = fabsf(y), z = y * y;
    const float p = fmaf(fmaf(fmaf(fmaf(fmaf(-0.005863219499588013f, z, 0.020763587206602097f), z,
                                        -0.05377184599637985f), z, 0.13331729173660278f), z, -0.3333328366279602f), z,
                         1.0f) * y;
    const float t = copysignf(
        1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * (2.0f * kLog2e))), y);
    return cap * (a < 0.6f ? p : t);
}

// One of the 16 query columns of a wave: column c of a (sequence, kv head) is
// query row c / group, head c % group of the kv head's group.
template <int HD>
struct Column {
    half8 hi[Shape<HD>::NB], lo[Shape<HD>::NB];  // the query, scaled by a power of two, as two f16 terms
    float factor;                                // a score in scores' own unit from the MFMA's
    uint32_t row;                                // of the call
    int first, wide;                             // keys first .. first + wide - 1 are seen
    int head, qpos;
    float slope;
    bool on, bad;                                // a column of the call; one whose row has no place in the cache
};

template <int HD, bool MODS>
__device__ __forceinline__ void column_place(const AttnArgs& a, const Rows& r, int kv, uint32_t c, Column<HD>& col) {
    const uint32_t t = c / a.group, h = c - t * a.group;
    col.on = t < r.count;
    col.row = col.on ? r.begin + t : 0;
    col.head = kv * a.group + static_cast<int>(h);
    const uint64_t place = r.at + t, keys = min(static_cast<uint64_t>(min(a.max_keys, static_cast<uint32_t>(a.c.cap))),
                                                r.at + r.count);
    col.bad = col.on && place >= keys;
    uint64_t lo = 0, hi = place + 1;
    if (col.on && a.first) lo = a.first[col.row];
    if (col.on && a.end) hi = a.end[col.row];
    hi = min(hi, keys);
    if (!col.on || col.bad || lo >= hi) lo = hi = 0;
    col.first = static_cast<int>(lo);
    col.wide = static_cast<int>(hi - lo);
    if constexpr (MODS) {
        col.slope = a.slopes && col.on ? a.slopes[col.head] : 0.0f;
        col.qpos = static_cast<int>(a.qpos && col.on ? a.qpos[col.row] : static_cast<uint32_t>(place));
    }
}

// The column's query: lane group g holds channels 8 g .. 8 g + 7 of every block,
// scaled so that the largest of the row is in [2^13, 2^14) (f16 then has 2^-39
// of it as its last place).
template <int HD>
__device__ __forceinline__ void column_query(const AttnArgs& a, int lane, Column<HD>& col) {
    constexpr int NB = Shape<HD>::NB;
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const float* q = a.q + static_cast<size_t>(col.row) * a.ld + static_cast<size_t>(col.head) * HD + (lane >> 4) * 8;
    float x[NB][8];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const f32x4 u = *reinterpret_cast<const f32x4u*>(q + 32 * b), v = *reinterpret_cast<const f32x4u*>(q + 32 * b + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[b][i] = col.on ? u[i] : 0.0f;
            x[b][4 + i] = col.on ? v[i] : 0.0f;
            top = fmaxf(top, fmaxf(fabsf(x[b][i]), fabsf(x[b][4 + i])));
        }
    }
    top = across_groups_max(top);
    const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split2(ldexpf(x[b][i], 14 - e), ldexpf(x[b][4 + i], 14 - e), h[i], l[i]);
        col.hi[b] = as_half8(h[0], h[1], h[2], h[3]);
        col.lo[b] = as_half8(l[0], l[1], l[2], l[3]);
    }
    col.factor = ldexpf(a.scale, e - 14);
}

// The scores of 32 keys and 16 columns: lane (g, n) gets keys 8 g + j of column n.
template <int HD>
__device__ __forceinline__ void scores(const uint32_t (&k)[2][Shape<HD>::NB], const u32x4 (&kd)[Shape<HD>::NB],
                                       const Column<HD>& col, float (&s)[8]) {
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const half8 lv = k_levels(k[h][b]);
            const f32x4 d = mfma(lv, col.hi[b], mfma(lv, col.lo[b], f32x4{0, 0, 0, 0}));
#pragma unroll
            for (int r = 0; r < 4; r++)
                s[4 * h + r] = b == 0 ? half_at(kd[b], 4 * h + r) * d[r] : fmaf(half_at(kd[b], 4 * h + r), d[r], s[4 * h + r]);
        }
    }
}

// Scores in the exponent's unit (log2), options applied.
template <int HD, bool MODS>
__device__ __forceinline__ void finish_scores(const AttnArgs& a, const Column<HD>& col, const uint32_t* kpos, int key0,
                                              float (&s)[8]) {
    if constexpr (MODS) {
        const float inv = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x = s[j] * col.factor;
            if (a.softcap > 0.0f) x = capped(x, a.softcap, inv);
            if (a.slopes) {
                const int kp = kpos ? static_cast<int>(kpos[min(key0 + j, a.c.cap - 1)]) : key0 + j;
                x = fmaf(-col.slope, static_cast<float>(abs(col.qpos - kp)), x);
            }
            s[j] = x * kLog2e;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) s[j] *= col.factor * kLog2e;
    }
}

// What a wave has of its 16 columns: the sums of e = 2^(score - base) (l, each lane
// its own keys') and of e * value (o).
template <int HD>
struct Sums {
    f32x4 o[Shape<HD>::NB][2];
    float l, base, limit;  // base = running maximum - 10 + vexp; scores up to limit = base + 14 - vexp keep it
    int vexp;              // 2^vexp is above every value scale so far
    uint32_t vbits;        // f16 bits that such a scale may have
};

template <int HD>
__device__ __forceinline__ void clear(Sums<HD>& z) {
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++) {
        z.o[b][0] = z.o[b][1] = f32x4{0, 0, 0, 0};
    }
    z.l = 0.0f;
    z.base = z.limit = -FLT_MAX;
    z.vexp = 0;
    z.vbits = 0;
}

// One tile of 32 keys into the sums.  The weights times their block's value
// scale are the f16 operand (two terms): at most 2^14, with 2^-39 of that as
// their last place, so none of them loses bits to f16's range.
template <int HD, bool MODS, bool MASKED>
__device__ __forceinline__ void step(const AttnArgs& a, const Tile<HD>& t, int tile, int lane, const Column<HD>& col,
                                     const uint32_t* kpos, int seen_lo, int seen_hi, Sums<HD>& z) {
    constexpr int NB = Shape<HD>::NB;
    const int g = lane >> 4, n = lane & 15, key0 = tile * 32 + 8 * g;
    float s[8];
    scores<HD>(t.k, t.kd, col, s);
    finish_scores<HD, MODS>(a, col, kpos, key0, s);
    bool seen[8];
    uint32_t vx = t.vx;
    if constexpr (MASKED) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            seen[j] = static_cast<uint32_t>(key0 + j - col.first) < static_cast<uint32_t>(col.wide);
            s[j] = seen[j] ? s[j] : -INFINITY;
        }
        // (scales of keys that no column sees may hold anything)
        const int i = lane % (16 * NB), kx = tile * 32 + i / (4 * NB) * 8 + i % 4 * 2;
        if (kx < seen_lo || kx >= seen_hi) vx &= 0xFFFF0000u;
        if (kx + 1 < seen_lo || kx + 1 >= seen_hi) vx &= 0x0000FFFFu;
    }
    const float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    const uint32_t vm = max(vx & 0x7FFFu, (vx >> 16) & 0x7FFFu);
    if (__any(top > z.limit || vm > z.vbits)) {
        int v = static_cast<int>(vm);
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) v = max(v, __shfl_xor(v, m, 64));
        v = max(v, static_cast<int>(z.vbits)) >> 10;
        const int vexp = min(v, 30) - 14;
        const float m = fmaxf(z.base == -FLT_MAX ? -FLT_MAX : z.base + static_cast<float>(10 - z.vexp),
                              across_groups_max(top));
        const float base = m == -FLT_MAX ? -FLT_MAX : m + static_cast<float>(vexp - 10);
        const float f = __builtin_amdgcn_exp2f(z.base - base);
        z.l *= f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            z.o[b][0] *= f;
            z.o[b][1] *= f;
        }
        z.base = base;
        z.limit = m == -FLT_MAX ? -FLT_MAX : m + 4.0f;
        z.vexp = vexp;
        z.vbits = v >= 30 ? 0x7FFFu : static_cast<uint32_t>(v << 10 | 0x3FF);
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(s[j] - z.base);
    z.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int b = 0; b < NB; b++) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = p[2 * i] * half_at(t.vd[b], 2 * i), y = p[2 * i + 1] * half_at(t.vd[b], 2 * i + 1);
            if constexpr (MASKED) {
                x = seen[2 * i] ? x : 0.0f;
                y = seen[2 * i + 1] ? y : 0.0f;
            }
            split2(x, y, hi[i], lo[i]);
        }
        const half8 ph = as_half8(hi[0], hi[1], hi[2], hi[3]), pl = as_half8(lo[0], lo[1], lo[2], lo[3]);
        u32x4 w = t.v[HD >= 64 ? b / 2 : 0];
        if constexpr (HD == 32) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] >>= n & 8;
        }
        const half8 v0 = b & 1 ? v_levels<2>(w) : v_levels<0>(w), v1 = b & 1 ? v_levels<3>(w) : v_levels<1>(w);
        z.o[b][0] = mfma(v0, ph, mfma(v0, pl, z.o[b][0]));
        z.o[b][1] = mfma(v1, ph, mfma(v1, pl, z.o[b][1]));
    }
}

template <int HD, bool MODS>
__device__ __forceinline__ void walk(const AttnArgs& a, const Planes& p, int lane, const Column<HD>& col,
                                     const uint32_t* kpos, int t0, int t1, int stride, int full_lo, int full_hi,
                                     int seen_lo, int seen_hi, Sums<HD>& z) {
    if (t0 >= t1) return;
    Tile<HD> cur;
    load_tile<HD>(p, a.c.cap, t0, lane, cur);
    for (int t = t0; t < t1; t += stride) {
        Tile<HD> next;
        load_tile<HD>(p, a.c.cap, min(t + stride, t1 - 1), lane, next);
        if (t * 32 >= full_lo && t * 32 + 32 <= full_hi)
            step<HD, MODS, false>(a, cur, t, lane, col, kpos, seen_lo, seen_hi, z);
        else
            step<HD, MODS, true>(a, cur, t, lane, col, kpos, seen_lo, seen_hi, z);
        cur = next;
    }
}

// The keys that a wave's columns see: the union [lo, hi), and the part that every
// column of the call sees [flo, fhi).
__device__ __forceinline__ void column_range(bool on, int first, int wide, int& lo, int& hi, int& flo, int& fhi) {
    lo = wide ? first : 0x7FFFFFFF;
    hi = wide ? first + wide : 0;
    flo = on ? first : 0;
    fhi = on ? first + wide : 0x7FFFFFFF;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        lo = min(lo, __shfl_xor(lo, m, 64));
        hi = max(hi, __shfl_xor(hi, m, 64));
        flo = max(flo, __shfl_xor(flo, m, 64));
        fhi = min(fhi, __shfl_xor(fhi, m, 64));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    flo = __builtin_amdgcn_readfirstlane(flo);
    fhi = __builtin_amdgcn_readfirstlane(fhi);
}

// Channels 32 b + 8 g .. + 7 of a column, from its sums.
template <int HD>
__device__ __forceinline__ void channels(const Sums<HD>& z, int b, float factor, float (&x)[8]) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        x[2 * r] = z.o[b][0][r] * factor;
        x[2 * r + 1] = z.o[b][1][r] * factor;
    }
}

// Attention of 16 columns by one workgroup: the four waves take every fourth tile
// of the workgroup's share of the keys (KEYS), or each its own 16 columns.
template <int HD, bool MODS, bool KEYS>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_attention(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB, LD = HD + 4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    int id = static_cast<int>(blockIdx.x);
    const int split = KEYS ? id % a.splits : 0;
    if (KEYS) id /= a.splits;
    const int unit = id;  // of the arrival counters
    const int ct = KEYS ? id % a.col_tiles : id % a.col_tiles * 4 + wave;
    id /= a.col_tiles;
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    if (static_cast<uint64_t>(ct) * 16 >= static_cast<uint64_t>(r.count) * a.group) return;
    Column<HD> col;
    column_place<HD, MODS>(a, r, kv, static_cast<uint32_t>(ct) * 16 + n, col);
    int lo, hi, flo, fhi;
    column_range(col.on, col.first, col.wide, lo, hi, flo, fhi);
    column_query<HD>(a, lane, col);
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + (static_cast<size_t>(s) * a.c.n_kv + kv) * a.c.cap : nullptr;
    Sums<HD> z;
    clear<HD>(z);
    const int t_lo = lo < hi ? lo / 32 : 0, tiles = lo < hi ? (hi + 31) / 32 - t_lo : 0;
    if constexpr (!KEYS) {
        walk<HD, MODS>(a, p, lane, col, kpos, t_lo, t_lo + tiles, 1, flo, fhi, lo, hi, z);
        const float l = across_groups_sum(z.l);
        if (!col.on) return;
        float* out = a.out + (static_cast<size_t>(col.row) * a.n_heads + col.head) * HD + g * 8;
        const float f = col.bad ? __builtin_nanf("") : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float x[8];
            channels<HD>(z, b, f, x);
#pragma unroll
            for (int i = 0; i < 8; i++) out[32 * b + i] = x[i];
        }
        if (a.lse && g == 0)
            a.lse[static_cast<size_t>(col.row) * a.n_heads + col.head] =
                col.bad ? __builtin_nanf("") : (z.base + log2f(l)) * kLn2;
        return;
    } else {
        const int t0 = t_lo + static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
        const int t1 = t_lo + static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);
        walk<HD, MODS>(a, p, lane, col, kpos, t0 + wave, t1, 4, flo, fhi, lo, hi, z);
        // join the waves
        __shared__ float so[4][16][LD], sb[4][16], sl[4][16];
        __shared__ int last;
        const float l = across_groups_sum(z.l);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float x[8];
            channels<HD>(z, b, 1.0f, x);
            *reinterpret_cast<f32x4*>(&so[wave][n][32 * b + 8 * g]) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(&so[wave][n][32 * b + 8 * g + 4]) = f32x4{x[4], x[5], x[6], x[7]};
        }
        if (g == 0) {
            sb[wave][n] = z.base;
            sl[wave][n] = l;
        }
        __syncthreads();
        constexpr int PER = HD / 16;  // channels of a column that a thread joins
        const int cj = threadIdx.x >> 4, ch = (threadIdx.x & 15) * PER;
        float base = fmaxf(fmaxf(sb[0][cj], sb[1][cj]), fmaxf(sb[2][cj], sb[3][cj]));
        float sum = 0.0f, x[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(sb[w][cj] - base);
            sum = fmaf(sl[w][cj], f, sum);
#pragma unroll
            for (int i = 0; i < PER; i++) x[i] = fmaf(so[w][cj][ch + i], f, x[i]);
        }
        const uint32_t c = static_cast<uint32_t>(ct) * 16 + cj;
        Column<HD> mine;  // (its place only)
        column_place<HD, false>(a, r, kv, c, mine);
        if (a.splits > 1) {
            float* part = a.part + (static_cast<size_t>(unit) * a.splits * 16 + cj) * (HD + 2);
            float* to = part + static_cast<size_t>(split) * 16 * (HD + 2);
            if (mine.on) {
                if (ch == 0) {
                    __hip_atomic_store(to, base, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(to + 1, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
#pragma unroll
                for (int i = 0; i < PER; i++)
                    __hip_atomic_store(to + 2 + ch + i, x[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            // Every thread's coherent stores complete before the arrival count moves.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) last = atomicAdd(a.counters + unit, 1u) == static_cast<unsigned>(a.splits - 1);
            __syncthreads();
            if (!last) return;
            if (threadIdx.x == 0)
                __hip_atomic_store(a.counters + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (!mine.on) return;
            base = -FLT_MAX;
            for (int i = 0; i < a.splits; i++)
                base = fmaxf(base, __hip_atomic_load(part + static_cast<size_t>(i) * 16 * (HD + 2), __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT));
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; i++) x[i] = 0.0f;
            for (int sp = 0; sp < a.splits; sp++) {
                const float* from = part + static_cast<size_t>(sp) * 16 * (HD + 2);
                const float f = __builtin_amdgcn_exp2f(
                    __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) - base);
                sum = fmaf(__hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), f, sum);
#pragma unroll
                for (int i = 0; i < PER; i++)
                    x[i] = fmaf(__hip_atomic_load(from + 2 + ch + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), f,
                                x[i]);
            }
        }
        if (!mine.on) return;
        float* out = a.out + (static_cast<size_t>(mine.row) * a.n_heads + mine.head) * HD + ch;
        const float f = mine.bad ? __builtin_nanf("") : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < PER; i++) out[i] = x[i] * f;
        if (a.lse && ch == 0)
            a.lse[static_cast<size_t>(mine.row) * a.n_heads + mine.head] =
                mine.bad ? __builtin_nanf("") : (base + log2f(sum)) * kLn2;
    }
}

// Adds to each key's weight what every (query row, head of its group) gave it.
// A wave holds 32 keys; COLS: the workgroup's waves share one tile and take every
// fourth tile of columns, else each has a tile of its own.
template <int HD, bool MODS, bool COLS>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_weigh(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB;
    __shared__ float red[4][32];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int per = COLS ? 1 : 4, groups = (static_cast<int>((min(a.max_keys, static_cast<uint32_t>(a.c.cap)) + 31) / 32) +
                                            per - 1) / per;
    int id = static_cast<int>(blockIdx.x);
    const int tile = COLS ? id % groups : id % groups * 4 + wave;
    id /= groups;
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + (static_cast<size_t>(s) * a.c.n_kv + kv) * a.c.cap : nullptr;
    const int key0 = tile * 32 + 8 * g;
    uint32_t k[2][NB];
    u32x4 kd[NB];
    load_k<HD>(p, a.c.cap, tile, lane, k, kd);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const uint64_t cols = static_cast<uint64_t>(r.count) * a.group;
    for (uint64_t c0 = COLS ? wave * 16 : 0; c0 < cols; c0 += COLS ? 64 : 16) {
        Column<HD> col;
        column_place<HD, MODS>(a, r, kv, static_cast<uint32_t>(c0) + n, col);
        if (!__any(col.wide && col.first < tile * 32 + 32 && col.first + col.wide > tile * 32)) continue;
        column_query<HD>(a, lane, col);
        const float lse = col.on ? a.lse_in[static_cast<size_t>(col.row) * a.n_heads + col.head] * kLog2e : 0.0f;
        float x[8];
        scores<HD>(k, kd, col, x);
        finish_scores<HD, MODS>(a, col, kpos, key0, x);
#pragma unroll
        for (int j = 0; j < 8; j++)
            acc[j] += static_cast<uint32_t>(key0 + j - col.first) < static_cast<uint32_t>(col.wide)
                          ? __builtin_amdgcn_exp2f(x[j] - lse) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = fh::group_sum<16>(acc[j]);
        if (n == 0) red[wave][8 * g + j] = v;
    }
    __syncthreads();
    const int t = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (w >= per) return;
    const int key = (COLS ? tile : tile - wave + w) * 32 + t;
    const uint64_t keys = min(static_cast<uint64_t>(min(a.max_keys, static_cast<uint32_t>(a.c.cap))), r.at + r.count);
    if (static_cast<uint64_t>(key) >= keys) return;
    float* to = a.c.weight + (static_cast<size_t>(s) * a.c.n_kv + kv) * a.c.cap + key;
    *to += COLS ? (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]) : red[w][t];
}

// ---- append -------------------------------------------------------------------

struct AppendArgs {
    Cache c;
    const float* qkv;
    size_t ld;
    uint32_t total, max_rows;
    int n_heads, hd, octets, heads;  // heads: kv heads of a workgroup, with their query heads
    const uint32_t *off, *len, *pos;
    int rope_dim, neox;
    float base, linear;
    const float* ff;
    float* q;
};

// apply_rope's rotation (llm.rs:146-175, the angle of RopeScaling::angle, llm.rs:118-121, in
// 32 bits as there) with sine, cosine and products in 64 bits: a key's channel goes on to the
// border between two levels, where its last bit decides.
__device__ __forceinline__ float rope_angle(uint32_t pos, int i, const AppendArgs& a) {
#pragma clang fp contract(off)
    const float freq =
        static_cast<float>(pow(static_cast<double>(a.base), -2.0 * i / static_cast<double>(a.rope_dim)));
    const float f = a.ff ? a.ff[i] : 1.0f;
    return static_cast<float>(static_cast<int>(pos)) * freq / f * (1.0f / a.linear);
}

// One channel of a head row, rotated where it is one of the first rope_dim.
__device__ __forceinline__ float rotated(const float* x, int ch, const AppendArgs& a, const double2* turn) {
#pragma clang fp contract(off)
    const float own = x[ch];
    if (ch >= a.rope_dim) return own;
    const int half = a.rope_dim / 2;
    const bool second = a.neox ? ch >= half : ch & 1;
    const int i = a.neox ? (second ? ch - half : ch) : ch >> 1;
    const double other = x[a.neox ? (second ? ch - half : ch + half) : ch ^ 1];
    const double2 t = turn[i];  // (cosine, sine)
    return static_cast<float>(second ? other * t.y + own * t.x : own * t.x - other * t.y);
}

// The eight cache rows of one octet: rotate and store their queries, quantise
// their keys and values.  A wave's halves each take one block of 32 channels.
__global__ void __launch_bounds__(kThreads) k_kv4_append(AppendArgs a) {
    extern __shared__ char smem[];
    const int hd = a.hd, nb = hd / 32, vn = hd >= 64 ? 16 : 8, bp = hd >= 64 ? hd / 64 : 1, half = a.rope_dim / 2;
    double2* turn = reinterpret_cast<double2*>(smem);  // [8][half]
    uint8_t* kl = reinterpret_cast<uint8_t*>(turn + 8 * half);  // [heads][8][hd / 2]
    uint8_t* vl = kl + a.heads * 4 * hd;                        // [heads][vn][bp][8][2]
    uint16_t* kdl = reinterpret_cast<uint16_t*>(vl + a.heads * 4 * hd);  // [heads][nb][8]
    uint16_t* vdl = kdl + a.heads * nb * 8;
    const int h0 = static_cast<int>(blockIdx.y) * a.heads, heads = min(a.heads, a.c.n_kv - h0);
    const int group = a.n_heads / a.c.n_kv;
    const int s = static_cast<int>(blockIdx.x) / a.octets;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    const uint64_t oct = r.at / 8 + blockIdx.x % a.octets;
    // rows j0 .. j1 - 1 of the octet are new; those past the capacity are rotated only
    const int64_t at = static_cast<int64_t>(r.at) - static_cast<int64_t>(oct * 8);
    const int j0 = static_cast<int>(max(at, int64_t(0))), j1 = static_cast<int>(min(at + int64_t(r.count), int64_t(8)));
    if (j0 >= j1) return;
    const uint32_t row0 = r.begin + static_cast<uint32_t>(oct * 8 + j0 - r.at);  // the call's row of j0
    const bool store = oct < static_cast<uint64_t>(a.c.cap / 8);
    for (int i = threadIdx.x; i < (j1 - j0) * half; i += kThreads) {
        const int j = j0 + i / half;
        const uint32_t row = row0 + (j - j0);
        const uint32_t pos = a.pos ? a.pos[row] : static_cast<uint32_t>(oct * 8 + j);
        double sn, cs;
        sincos(static_cast<double>(rope_angle(pos, i % half, a)), &sn, &cs);
        turn[j * half + i % half] = make_double2(cs, sn);
    }
    __syncthreads();
    if (a.q) {
        const int wide = heads * group * hd;
        for (int i = threadIdx.x; i < (j1 - j0) * wide; i += kThreads) {
            const int jj = i / wide, c = i - jj * wide + h0 * group * hd;
            const size_t row = row0 + jj;
            a.q[row * (a.n_heads * hd) + c] =
                rotated(a.qkv + row * a.ld + c / hd * hd, c % hd, a, turn + (j0 + jj) * half);
        }
    }
    if (!store) return;
    const int side = threadIdx.x >> 5, i = threadIdx.x & 31, blocks = heads * nb;
    for (int u = side; u < (j1 - j0) * blocks * 2; u += kThreads / 32) {
        const int jj = u / (blocks * 2), v = u % 2, hb = u / 2 % blocks, h = hb / nb, b = hb % nb, j = j0 + jj;
        const size_t row = row0 + jj;
        const float* x = a.qkv + row * a.ld + static_cast<size_t>(a.n_heads + (v ? a.c.n_kv : 0) + h0 + h) * hd;
        const float y = v ? x[32 * b + i] : rotated(x, 32 * b + i, a, turn + j * half);
        float top = fabsf(y);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 32));
        const int up = threadIdx.x & 32;  // this half's place in the wave
        const uint32_t odd = static_cast<uint32_t>(__ballot(!(fabsf(y) < INFINITY)) >> up);
        const uint32_t tops = static_cast<uint32_t>(__ballot(fabsf(y) == top) >> up);
        const float m = __shfl(y, tops ? __ffs(tops) - 1 : 0, 32);
        _Float16 dh = static_cast<_Float16>(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
        if (odd) dh = __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x7E00));
        const float d = static_cast<float>(dh);
        int level = 8;
        if (!odd && d != 0.0f) {
            // the nearest level, ties to even: the quotient's own rounding can hide on which side
            // of a border the exact one lies, which the remainder (exact in one FMA) tells
            float t = rintf(y / d);
            const float rest = fmaf(-t, d, y);
            if (fabsf(rest) > 0.5f * fabsf(d)) t += (rest > 0.0f) == (d > 0.0f) ? 1.0f : -1.0f;
            level = static_cast<int>(fminf(fmaxf(t, -8.0f), 7.0f)) + 8;
        }
        const int two = level | __shfl_xor(level, 1, 32) << 4;  // (the even lane's)
        if ((i & 1) == 0) {
            if (v) vl[(((h * vn + (i >> 1) % vn) * bp + (hd >= 64 ? b >> 1 : 0)) * 8 + j) * 2 +
                      (hd >= 64 ? b & 1 : i >> 4)] = static_cast<uint8_t>(two);
            else kl[(h * 8 + j) * (hd / 2) + ((i >> 3) * nb + b) * 4 + (i & 7) / 2] = static_cast<uint8_t>(two);
        }
        if (i == 0) (v ? vdl : kdl)[(h * nb + b) * 8 + j] = __builtin_bit_cast(uint16_t, dh);
    }
    __syncthreads();
    const size_t plane = static_cast<size_t>(s) * a.c.n_kv + h0;
    // keys: words of whole rows
    const int kw = hd / 8;
    for (int u = threadIdx.x; u < heads * 8 * kw; u += kThreads) {
        const int h = u / (8 * kw), j = u / kw % 8, w = u % kw;
        if (j >= j0 && j < j1)
            reinterpret_cast<uint32_t*>(a.c.k + ((plane + h) * a.c.cap + oct * 8 + j) * (hd / 2))[w] =
                reinterpret_cast<const uint32_t*>(kl)[(h * 8 + j) * kw + w];
    }
    // values and scales: 2-byte units, eight keys side by side, at once where all eight are new
    const int vu = hd / 4;
    const bool whole = j0 == 0 && j1 == 8;
    const int rows8 = heads * (vu + 2 * nb);
    for (int u = threadIdx.x; u < rows8 * (whole ? 1 : 8); u += kThreads) {
        const int j = whole ? 0 : u % 8, q = whole ? u : u / 8, h = q / (vu + 2 * nb), w = q % (vu + 2 * nb);
        const size_t o = (plane + h) * (a.c.cap / 8) + oct;
        const uint16_t* from;
        uint16_t* to;
        if (w < vu) {
            from = reinterpret_cast<const uint16_t*>(vl) + (h * vu + w) * 8;
            to = reinterpret_cast<uint16_t*>(a.c.v) + (o * vu + w) * 8;
        } else if (w < vu + nb) {
            from = kdl + (h * nb + w - vu) * 8;
            to = a.c.kd + (o * nb + w - vu) * 8;
        } else {
            from = vdl + (h * nb + w - vu - nb) * 8;
            to = a.c.vd + (o * nb + w - vu - nb) * 8;
        }
        if (whole) *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
        else if (j >= j0 && j < j1) to[j] = from[j];
    }
    for (int u = threadIdx.x; u < heads * 8; u += kThreads) {
        const int h = u / 8, j = u % 8;
        if (j < j0 || j >= j1) continue;
        const size_t to = (plane + h) * a.c.cap + oct * 8 + j;
        if (a.c.pos) a.c.pos[to] = a.pos ? a.pos[row0 + (j - j0)] : static_cast<uint32_t>(oct * 8 + j);
        if (a.c.weight) a.c.weight[to] = 0.0f;
    }
}

// ---- read back ----------------------------------------------------------------

// Rows first[s] .. + rows - 1 of every head as f32 rows of n_kv * hd, the f32
// cache's layout.  One thread: one 4-byte word of keys (8 channels), or one
// 2-byte unit of values (4 channels).
template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_read(Cache c, const uint32_t* __restrict__ first, uint32_t rows,
                                                      float* __restrict__ ko, float* __restrict__ vo) {
    constexpr int NB = Shape<HD>::NB, BP = Shape<HD>::BP, KW = HD / 8, VU = HD / 4;
    const size_t id = blockIdx.x * static_cast<size_t>(kThreads) + threadIdx.x;
    const size_t per = static_cast<size_t>(c.n_kv) * (KW + VU);
    if (id >= per * rows * c.seqs) return;
    const int u = static_cast<int>(id % (KW + VU)), h = static_cast<int>(id / (KW + VU) % c.n_kv);
    const uint32_t t = static_cast<uint32_t>(id / per % rows);
    const int s = static_cast<int>(id / per / rows);
    const uint64_t key = static_cast<uint64_t>(first ? first[s] : 0) + t;
    const bool ok = key < static_cast<uint64_t>(c.cap);
    const size_t plane = (static_cast<size_t>(s) * c.n_kv + h) * c.cap, at = ok ? key : 0;
    const size_t row = (static_cast<size_t>(s) * rows + t) * c.n_kv + h;
    if (u < KW) {
        const int b = u >> 2, g = u & 3;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(c.k + (plane + at) * (HD / 2) + (g * NB + b) * 4);
        const float d = ok ? fh_h2f(c.kd[((plane + at) / 8 * NB + b) * 8 + at % 8]) : __builtin_nanf("");
        float* to = ko + row * HD + 32 * b + 8 * g;
#pragma unroll
        for (int i = 0; i < 8; i++) to[i] = static_cast<float>(static_cast<int>(w >> (4 * i) & 15) - 8) * d;
    } else {
        const int v = u - KW, n = v / BP, pair = v % BP;
        const uint32_t w = reinterpret_cast<const uint16_t*>(c.v)[((plane + at) / 8 * VU + n * BP + pair) * 8 + at % 8];
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int b = HD >= 64 ? 2 * pair + y : 0, ch = HD >= 64 ? 32 * b + 2 * n : 2 * (n + 8 * y);
            const float d = ok ? fh_h2f(c.vd[((plane + at) / 8 * NB + b) * 8 + at % 8]) : __builtin_nanf("");
            float* to = vo + row * HD + ch;
            to[0] = static_cast<float>(static_cast<int>(w >> (8 * y) & 15) - 8) * d;
            to[1] = static_cast<float>(static_cast<int>(w >> (8 * y + 4) & 15) - 8) * d;
        }
    }
}

// ---- eviction -----------------------------------------------------------------

// A weight as an unsigned number of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t b = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kSelect = 1024;

// Which rows of a (sequence, kv head) stay: the last `recent` and the heaviest
// of the others up to `keep`, in order; idx gets their cache rows, *count how
// many.  Four passes of an 8-bit radix select find the lightest weight that
// stays and how many of its equals do (the first ones); a last pass writes.
__global__ void __launch_bounds__(kSelect) k_kv4_select(Cache c, const uint32_t* __restrict__ len, uint32_t max_len,
                                                       uint32_t keep, uint32_t recent, uint32_t* __restrict__ idx,
                                                       uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[256], wsum[2][kSelect / 64], pick[2];
    const int s = static_cast<int>(blockIdx.x) / c.n_kv;
    const uint32_t n = min(min(len[s], max_len), static_cast<uint32_t>(c.cap));
    uint32_t* to = idx + static_cast<size_t>(blockIdx.x) * keep;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (tid == 0) counts[blockIdx.x] = min(n, keep);
    if (n <= keep) {
        for (uint32_t i = tid; i < n; i += kSelect) to[i] = i;
        return;
    }
    const uint32_t free = n - recent;
    uint32_t want = keep - recent;  // of the free rows; less than `free`
    const float* w = c.weight + static_cast<size_t>(blockIdx.x) * c.cap;
    uint32_t prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < free; i += kSelect) {
            const uint32_t o = ordered(w[i]);
            if ((o & mask) == prefix) atomicAdd(&hist[o >> shift & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // from the heaviest digit down: the one at which the count reaches `want`
            uint32_t h[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) sum += h[i] = hist[255 - (lane * 4 + i)];
            uint32_t upto = sum;
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t v = __shfl_up(upto, m, 64);
                if (lane >= m) upto += v;
            }
            uint32_t before = upto - sum;
            for (int i = 0; i < 4; i++) {
                if (before < want && before + h[i] >= want) {
                    pick[0] = 255 - (lane * 4 + i);
                    pick[1] = want - before;
                }
                before += h[i];
            }
            if (want == 0 && lane == 0) {
                pick[0] = 255;
                pick[1] = 0;
            }
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        want = pick[1];
        mask |= 255u << shift;
        __syncthreads();
    }
    // `want` of the rows that weigh exactly `prefix` stay
    uint32_t kept = 0, equal = 0;
    const bool none = keep == recent;
    for (uint32_t i0 = 0; i0 < free; i0 += kSelect) {
        const uint32_t i = i0 + tid;
        const uint32_t o = i < free ? ordered(w[i]) : 0;
        const bool eq = !none && i < free && o == prefix, gt = !none && i < free && o > prefix;
        const uint64_t below = (uint64_t(1) << lane) - 1;
        const uint64_t beq = __ballot(eq);
        if (lane == 0) wsum[0][wave] = __popcll(beq);
        __syncthreads();
        uint32_t rank = equal + __popcll(beq & below), alleq = 0;
        for (int v = 0; v < kSelect / 64; v++) {
            if (v < wave) rank += wsum[0][v];
            alleq += wsum[0][v];
        }
        const bool stay = gt || (eq && rank < want);
        const uint64_t bst = __ballot(stay);
        if (lane == 0) wsum[1][wave] = __popcll(bst);
        __syncthreads();
        uint32_t place = kept + __popcll(bst & below), all = 0;
        for (int v = 0; v < kSelect / 64; v++) {
            if (v < wave) place += wsum[1][v];
            all += wsum[1][v];
        }
        if (stay) to[place] = i;
        kept += all;
        equal += alleq;
        __syncthreads();
    }
    for (uint32_t i = tid; i < recent; i += kSelect) to[keep - recent + i] = free + i;
}

// Moves the rows that stay.  A workgroup: 64 rows of one (sequence, kv head).
template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_move(Cache c, Cache d, uint32_t keep, int chunks,
                                                      const uint32_t* __restrict__ idx,
                                                      const uint32_t* __restrict__ counts,
                                                      uint32_t* __restrict__ new_len) {
    constexpr int NB = Shape<HD>::NB, VU = HD / 4, KP = HD / 32 * 4;  // KP: words of a key row
    const int sh = static_cast<int>(blockIdx.x) / chunks, ck = static_cast<int>(blockIdx.x) % chunks;
    const uint32_t n = counts[sh], r0 = static_cast<uint32_t>(ck) * 64;
    if (ck == 0 && threadIdx.x == 0 && sh % c.n_kv == 0) new_len[sh / c.n_kv] = n;
    if (r0 >= n) return;
    __shared__ uint32_t src[64];
    const int rows = static_cast<int>(min(n - r0, 64u));
    if (threadIdx.x < 64) src[threadIdx.x] = idx[static_cast<size_t>(sh) * keep + r0 + min(static_cast<int>(threadIdx.x), rows - 1)];
    __syncthreads();
    const size_t from = static_cast<size_t>(sh) * c.cap, to = static_cast<size_t>(sh) * d.cap;
    const uint32_t* ks = reinterpret_cast<const uint32_t*>(c.k);
    uint32_t* kt = reinterpret_cast<uint32_t*>(d.k);
    for (int u = threadIdx.x; u < rows * KP; u += kThreads)
        kt[(to + r0 + u / KP) * KP + u % KP] = ks[(from + src[u / KP]) * KP + u % KP];
    // eight rows side by side: 2-byte units of the values and the scales
    for (int u = threadIdx.x; u < (VU + 2 * NB) * 64; u += kThreads) {
        const int j = u % 8, w = u / 8 % (VU + 2 * NB), o = u / (8 * (VU + 2 * NB)), row = o * 8 + j;
        if (row >= rows) continue;
        const uint32_t r = src[row];
        const size_t fo = from / 8 + r / 8, tu = to / 8 + r0 / 8 + o;
        if (w < VU)
            reinterpret_cast<uint16_t*>(d.v)[(tu * VU + w) * 8 + j] =
                reinterpret_cast<const uint16_t*>(c.v)[(fo * VU + w) * 8 + r % 8];
        else if (w < VU + NB) d.kd[(tu * NB + w - VU) * 8 + j] = c.kd[(fo * NB + w - VU) * 8 + r % 8];
        else d.vd[(tu * NB + w - VU - NB) * 8 + j] = c.vd[(fo * NB + w - VU - NB) * 8 + r % 8];
    }
    if (threadIdx.x < rows) {
        const uint32_t r = src[threadIdx.x];
        if (d.pos) d.pos[to + r0 + threadIdx.x] = c.pos ? c.pos[from + r] : r;
        if (d.weight) d.weight[to + r0 + threadIdx.x] = c.weight[from + r];
    }
}

Cache device_cache(const fh_kv4_cache& c) {
    return {c.k, c.k_d, c.v, c.v_d, c.pos, c.weight, static_cast<int>(c.seqs), static_cast<int>(c.n_kv),
            static_cast<int>(c.capacity)};
}

// The partial sums of attention whose keys are split over workgroups: at most
// kUnits of them, each 16 columns of HD + 2 floats, behind one arrival counter
// each.  One area of this size for the context's life, so a graph that was
// captured with it never loses it to a larger call.
constexpr size_t kUnits = 2048;
constexpr size_t kPartBytes = kUnits * 16 * (128 + 2) * sizeof(float);

template <int HD, bool MODS>
void launch_attention(fh_ctx* ctx, const AttnArgs& a, bool keys, size_t grid) {
    if (keys)
        hipLaunchKernelGGL((k_kv4_attention<HD, MODS, true>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                           ctx->stream, a);
    else
        hipLaunchKernelGGL((k_kv4_attention<HD, MODS, false>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                           ctx->stream, a);
}

AttnArgs attn_args(const fh_kv4_cache& c, const float* q, size_t ld, size_t total, size_t n_heads, const uint32_t* off,
                   size_t max_rows, const uint32_t* len, size_t max_keys, const fh_attn_score* sc) {
    AttnArgs a{};
    a.c = device_cache(c);
    a.q = q;
    a.ld = ld;
    a.total = static_cast<uint32_t>(total);
    a.max_rows = static_cast<uint32_t>(max_rows);
    a.max_keys = static_cast<uint32_t>(std::min(max_keys, c.capacity));
    a.n_heads = static_cast<int>(n_heads);
    a.group = static_cast<int>(n_heads / c.n_kv);
    a.off = off;
    a.len = len;
    a.scale = 1.0f / std::sqrt(static_cast<float>(c.head_dim));
    if (sc) {
        a.softcap = sc->softcap;
        a.slopes = sc->d_slopes;
        a.qpos = sc->d_pos;
        a.first = sc->d_first;
        a.end = sc->d_end;
    }
    return a;
}

}  // namespace

int fh_launch_kv4_append(fh_ctx* ctx, const fh_kv4_cache& c, const float* qkv, size_t ld, size_t total, size_t n_heads,
                         const uint32_t* off, size_t max_rows, const uint32_t* len, const uint32_t* pos,
                         size_t rope_dim, float base, int rope_type, const float* ff, float linear, float* q) {
    AppendArgs a{};
    a.c = device_cache(c);
    a.qkv = qkv;
    a.ld = ld;
    a.total = static_cast<uint32_t>(total);
    a.max_rows = static_cast<uint32_t>(max_rows);
    a.n_heads = static_cast<int>(n_heads);
    a.hd = static_cast<int>(c.head_dim);
    a.octets = static_cast<int>((max_rows + 14) / 8);  // a block of rows touches that many at most
    a.off = off;
    a.len = len;
    a.pos = pos;
    a.rope_dim = static_cast<int>(rope_dim);
    a.neox = rope_type == FH_ROPE_NEOX;
    a.base = base;
    a.linear = linear;
    a.ff = ff;
    a.q = q;
    a.heads = static_cast<int>(std::min<size_t>(c.n_kv, 8));
    const size_t lds = 8 * (rope_dim / 2) * sizeof(double2) + a.heads * (8 * c.head_dim + c.head_dim / 32 * 8 * 2 * 2);
    const dim3 grid(static_cast<unsigned>(c.seqs * a.octets), static_cast<unsigned>((c.n_kv + a.heads - 1) / a.heads));
    hipLaunchKernelGGL(k_kv4_append, grid, dim3(kThreads), lds, ctx->stream, a);
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

int fh_launch_kv4_attention(fh_ctx* ctx, const fh_kv4_cache& c, const float* q, size_t ld, size_t total, size_t n_heads,
                            const uint32_t* off, size_t max_rows, const uint32_t* len, size_t max_keys,
                            const fh_attn_score* sc, float* out, float* lse) {
    AttnArgs a = attn_args(c, q, ld, total, n_heads, off, max_rows, len, max_keys, sc);
    a.out = out;
    a.lse = lse;
    const size_t cols = max_rows * a.group, tiles16 = (cols + 15) / 16, key_tiles = (a.max_keys + 31) / 32;
    const size_t units = c.seqs * c.n_kv * tiles16;
    const bool keys = units < 4 * static_cast<size_t>(ctx->num_cus);
    size_t grid;
    if (keys) {
        a.col_tiles = static_cast<int>(tiles16);
        size_t splits = std::max<size_t>(1, 2 * ctx->num_cus / units);
        splits = std::min(splits, std::max<size_t>(1, key_tiles / 8));
        if (units * splits > kUnits) splits = 1;
        a.splits = static_cast<int>(splits);
        grid = units * splits;
        if (splits > 1) {
            void* area = nullptr;
            const int rc = fh_kv4_area(ctx, kUnits * sizeof(unsigned) + kPartBytes, &area);
            if (rc) return rc;
            a.counters = static_cast<unsigned*>(area);
            a.part = reinterpret_cast<float*>(a.counters + kUnits);
        }
    } else {
        a.col_tiles = static_cast<int>((tiles16 + 3) / 4);
        a.splits = 1;
        grid = c.seqs * c.n_kv * a.col_tiles;
    }
    if (grid > 0x7FFFFFFF) return fh_fail(ctx, FH_ERR_LIMIT, "fh_kv4_attention: more than 2^31 - 1 workgroups");
    const bool mods = a.softcap > 0.0f || a.slopes;
    switch (c.head_dim) {
        case 32: mods ? launch_attention<32, true>(ctx, a, keys, grid) : launch_attention<32, false>(ctx, a, keys, grid); break;
        case 64: mods ? launch_attention<64, true>(ctx, a, keys, grid) : launch_attention<64, false>(ctx, a, keys, grid); break;
        default: mods ? launch_attention<128, true>(ctx, a, keys, grid) : launch_attention<128, false>(ctx, a, keys, grid); break;
    }
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

template <int HD, bool MODS>
static void launch_weigh(fh_ctx* ctx, const AttnArgs& a, bool cols, size_t grid) {
    if (cols)
        hipLaunchKernelGGL((k_kv4_weigh<HD, MODS, true>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                           ctx->stream, a);
    else
        hipLaunchKernelGGL((k_kv4_weigh<HD, MODS, false>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                           ctx->stream, a);
}

int fh_launch_kv4_weigh(fh_ctx* ctx, const fh_kv4_cache& c, const float* q, size_t ld, size_t total, size_t n_heads,
                        const uint32_t* off, size_t max_rows, const uint32_t* len, size_t max_keys,
                        const fh_attn_score* sc, const float* lse) {
    AttnArgs a = attn_args(c, q, ld, total, n_heads, off, max_rows, len, max_keys, sc);
    a.lse_in = lse;
    const bool cols = max_rows * a.group > 16;
    const size_t tiles = (a.max_keys + 31) / 32, groups = cols ? tiles : (tiles + 3) / 4;
    const size_t grid = c.seqs * c.n_kv * groups;
    if (grid > 0x7FFFFFFF) return fh_fail(ctx, FH_ERR_LIMIT, "fh_kv4_weigh: more than 2^31 - 1 workgroups");
    const bool mods = a.softcap > 0.0f || a.slopes;
    switch (c.head_dim) {
        case 32: mods ? launch_weigh<32, true>(ctx, a, cols, grid) : launch_weigh<32, false>(ctx, a, cols, grid); break;
        case 64: mods ? launch_weigh<64, true>(ctx, a, cols, grid) : launch_weigh<64, false>(ctx, a, cols, grid); break;
        default: mods ? launch_weigh<128, true>(ctx, a, cols, grid) : launch_weigh<128, false>(ctx, a, cols, grid); break;
    }
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

int fh_launch_kv4_read(fh_ctx* ctx, const fh_kv4_cache& c, const uint32_t* first, size_t rows, float* k, float* v) {
    const Cache d = device_cache(c);
    const size_t n = c.seqs * rows * c.n_kv * (c.head_dim / 8 + c.head_dim / 4);
    const dim3 grid(static_cast<unsigned>((n + kThreads - 1) / kThreads));
    const uint32_t r = static_cast<uint32_t>(rows);
    switch (c.head_dim) {
        case 32: hipLaunchKernelGGL((k_kv4_read<32>), grid, dim3(kThreads), 0, ctx->stream, d, first, r, k, v); break;
        case 64: hipLaunchKernelGGL((k_kv4_read<64>), grid, dim3(kThreads), 0, ctx->stream, d, first, r, k, v); break;
        default: hipLaunchKernelGGL((k_kv4_read<128>), grid, dim3(kThreads), 0, ctx->stream, d, first, r, k, v); break;
    }
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

int fh_launch_kv4_evict(fh_ctx* ctx, const fh_kv4_cache& src, const fh_kv4_cache& dst, const uint32_t* len,
                        size_t max_len, size_t keep, size_t recent, uint32_t* new_len) {
    const Cache c = device_cache(src), d = device_cache(dst);
    const size_t heads = src.seqs * src.n_kv, idx_bytes = fh_align256(heads * keep * sizeof(uint32_t));
    void* ws = nullptr;
    const int rc = fh_workspace(ctx, idx_bytes + heads * sizeof(uint32_t), &ws);
    if (rc) return rc;
    uint32_t* idx = static_cast<uint32_t*>(ws);
    uint32_t* counts = reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + idx_bytes);
    hipLaunchKernelGGL(k_kv4_select, dim3(static_cast<unsigned>(heads)), dim3(kSelect), 0, ctx->stream, c, len,
                       static_cast<uint32_t>(std::min(max_len, src.capacity)), static_cast<uint32_t>(keep),
                       static_cast<uint32_t>(recent), idx, counts);
    FH_HIP(ctx, hipGetLastError());
    const int chunks = static_cast<int>((keep + 63) / 64);
    const dim3 grid(static_cast<unsigned>(heads * chunks));
    const uint32_t kp = static_cast<uint32_t>(keep);
    switch (src.head_dim) {
        case 32: hipLaunchKernelGGL((k_kv4_move<32>), grid, dim3(kThreads), 0, ctx->stream, c, d, kp, chunks, idx, counts, new_len); break;
        case 64: hipLaunchKernelGGL((k_kv4_move<64>), grid, dim3(kThreads), 0, ctx->stream, c, d, kp, chunks, idx, counts, new_len); break;
        default: hipLaunchKernelGGL((k_kv4_move<128>), grid, dim3(kThreads), 0, ctx->stream, c, d, kp, chunks, idx, counts, new_len); break;
    }
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}
