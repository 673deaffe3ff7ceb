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
#include <cmath>
#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
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
    int weigh_cols;  // tiles of columns a batch
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

// One lane's share of 32 keys of a cache on its way: lane (g, n) = (lane / 16, lane %
// 16) holds key rows 8 (n / 4) + n % 4 and + 4 as MFMA rows and its output channels'
// value levels of the eight keys 8 g .. 8 g + 7; and one 64th of the tile's scales
// (lanes 0 .. 31 the keys', 32 .. 63 the values'), which go through LDS to the
// lanes that want them: loaded as wanted, each would come 16 times over.
template <int HD>
struct Tile {
    uint32_t k[2][Shape<HD>::NB];
    u32x4 v[Shape<HD>::BP];
    uint32_t sc[HD == 128 ? 2 : 1];
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
__device__ __forceinline__ void load_k(const Planes& p, int cap, int tile, int lane, uint32_t (&k)[2][Shape<HD>::NB]) {
    constexpr int NB = Shape<HD>::NB;
    const int g = lane >> 4, n = lane & 15;
    const int key = tile * 32 + 8 * (n >> 2) + (n & 3);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        // (a tile's end past the capacity reads the last row again; the mask drops it)
        const uint8_t* a = p.k + (static_cast<uint32_t>(min(key + 4 * h, cap - 1)) * (HD / 2) + g * (4 * NB));
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
}
template <int HD>
__device__ __forceinline__ void load_kd(const Planes& p, int cap, int tile, int lane, u32x4 (&kd)[Shape<HD>::NB]) {
    const uint32_t o = min(tile * 4 + (lane >> 4), cap / 8 - 1);
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++)
        kd[b] = *reinterpret_cast<const u32x4*>(p.kd + o * (Shape<HD>::NB * 8) + b * 8);
}

template <int HD>
__device__ __forceinline__ void load_v(const Planes& p, int cap, int tile, int lane, Tile<HD>& t) {
    constexpr int N = Shape<HD>::N, BP = Shape<HD>::BP;
    const int g = lane >> 4, n = lane & 15;
    const uint32_t vo = min(tile * 4 + g, cap / 8 - 1) * (N * BP * 16) + n % N * (BP * 16);
#pragma unroll
    for (int i = 0; i < BP; i++) t.v[i] = *reinterpret_cast<const u32x4*>(p.v + vo + i * 16);
}
// (scales: of keys for lanes 0 .. 31, of values for the others; eight lanes an octet, NB each, as they lie)
template <int HD>
__device__ __forceinline__ void load_scales(const uint16_t* scales, int cap, int tile, int lane, Tile<HD>& t) {
    constexpr int NB = Shape<HD>::NB;
    const uint16_t* a = scales + (min(tile * 4 + (lane >> 3 & 3), cap / 8 - 1) * (8 * NB) + (lane & 7) * NB);
    if constexpr (NB == 4) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(a);
        t.sc[0] = w[0];
        t.sc[1] = w[1];
    } else if constexpr (NB == 2) {
        t.sc[0] = *reinterpret_cast<const uint32_t*>(a);
    } else {
        t.sc[0] = *a;
    }
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}
__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// A constant that the compiler does not know: it then keeps a product or a mask with it in
// the one instruction that takes it (v_fma_mix_f32, v_and_or_b32).
__device__ __forceinline__ float hidden(float c) {
    asm("" : "+v"(c));
    return c;
}
__device__ __forceinline__ uint32_t hidden(uint32_t c) {
    asm("" : "+v"(c));
    return c;
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
    const uint32_t x = ((E & 2 ? w >> 8 : w) & (E & 1 ? 0x00F000F0u : 0x000F000Fu)) | hidden(0x64006400u);
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
// Two f32 as a pair of f16 and what that leaves, each rounded to nearest: 22 bits in all, for
// queries and weights alike.  A third term would make every product half as long again for
// less than the roundings of the sums behind it (check_attention's count of a score: 2^-21).
// (The values and the pair are kept from the compiler's view: it would form a product's
// hi in one mixed-precision instruction, with one rounding, and lo from the twice rounded
// one, or the pair twice over.)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    asm("" : "+v"(a), "+v"(b));
    const half2v h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    hi = __builtin_bit_cast(uint32_t, h);
    asm("" : "+v"(hi));
    const half2v k = __builtin_bit_cast(half2v, hi);
    const float minus = hidden(-1.0f);
    const half2v l = {static_cast<_Float16>(fmaf(static_cast<float>(k[0]), minus, a)),
                      static_cast<_Float16>(fmaf(static_cast<float>(k[1]), minus, b))};
    lo = __builtin_bit_cast(uint32_t, l);
}
// A lane's value with those of the other three lane groups (its column's other keys).
struct Pair {
    float a, b;
};
__device__ __forceinline__ Pair halves(float v) {  // of the wave, each in every lane
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const uint32_t a = r[0], b = r[1];
    return {__uint_as_float(a), __uint_as_float(b)};
}
__device__ __forceinline__ Pair rows16(float v) {  // of each half
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const uint32_t a = r[0], b = r[1];
    return {__uint_as_float(a), __uint_as_float(b)};
}
__device__ __forceinline__ float across_groups_max(float v) {
    Pair p = halves(v);
    p = rows16(fmaxf(p.a, p.b));
    return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float across_groups_sum(float v) {
    Pair p = halves(v);
    p = rows16(p.a + p.b);
    return p.a + p.b;
}
// Over the 16 lanes of a group.
__device__ __forceinline__ int group_min(int v) {
    v = min(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false));
    return min(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, false));
}

// Eight scores x, in units of `unit`, capped: cap tanh(x unit / cap), in the same units.
// Up to 0.6 a polynomial (least maximum error over [0, 0.36] of tanh(y) / y in y^2:
// 2.4e-9), past it, where a wave has such scores, 1 - 2 / (1 + e^2y), whose rounding
// is then no larger than the result's own.
__device__ __forceinline__ void cap_scores(float (&x)[8], float cap, float unit) {
    const float in = fminf(unit / cap, FLT_MAX);  // (0 times it stays 0)
    float y[8], top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        y[j] = x[j] * in;
        top = fmaxf(top, fabsf(y[j]));
        const float z = y[j] * y[j];
        x[j] *= fmaf(fmaf(fmaf(fmaf(fmaf(-0.005863219499588013f, z, 0.020763587206602097f), z, -0.05377184599637985f), z,
                               0.13331729173660278f), z, -0.3333328366279602f), z, 1.0f);
    }
    if (__any(top > 0.6f)) {
        const float out = cap / unit;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float a = fabsf(y[j]);
            const float t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * (2.0f * kLog2e)));
            x[j] = a > 0.6f ? copysignf(out * t, y[j]) : x[j];
        }
    }
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
    if (col.on && a.first) lo = static_cast<uint32_t>(max(static_cast<int>(a.first[col.row]), 0));  // (a window's may be below 0)
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
// (a column that is not the call's: row 0's, whose result goes nowhere)
// scaled so that the largest of the row is in [2^13, 2^14) (f16 then has 2^-39
// of it as its last place; below 2^-96 by 2^110 only, so that factor stays normal:
// such a row's scores are nothing beside 1).
template <int HD>
__device__ __forceinline__ void load_query(const AttnArgs& a, int lane, const Column<HD>& col,
                                           float (&x)[Shape<HD>::NB][8]) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const float* q = a.q + static_cast<size_t>(col.row) * a.ld + static_cast<size_t>(col.head) * HD + (lane >> 4) * 8;
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++) {
        const f32x4 u = *reinterpret_cast<const f32x4u*>(q + 32 * b), v = *reinterpret_cast<const f32x4u*>(q + 32 * b + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[b][i] = u[i];
            x[b][4 + i] = v[i];
        }
    }
}
template <int HD>
__device__ __forceinline__ void split_query(const AttnArgs& a, const float (&x)[Shape<HD>::NB][8], Column<HD>& col) {
    constexpr int NB = Shape<HD>::NB;
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[b][i]));
    top = across_groups_max(top);
    const int e = top > 0.0f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -96) : 0;
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
template <int HD>
__device__ __forceinline__ void column_query(const AttnArgs& a, int lane, Column<HD>& col) {
    float x[Shape<HD>::NB][8];
    load_query<HD>(a, lane, col, x);
    split_query<HD>(a, x, col);
}

// A wave's queries: of 16 columns, or (T = 2) of at most eight, twice: lanes n < 8 have
// them for the first tile of a pair of tiles, zeros for the second, lanes n >= 8 the other
// way around.  The products of both tiles then add up to each lane's own, and what
// follows them is done once for both tiles.
template <int HD, int T>
struct Queries {
    half8 hi[T][Shape<HD>::NB], lo[T][Shape<HD>::NB];
};
template <int HD, int T>
__device__ __forceinline__ Queries<HD, T> queries_of(const Column<HD>& col, int n) {
    Queries<HD, T> q;
    const half8 none = as_half8(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < T; i++)
#pragma unroll
        for (int b = 0; b < Shape<HD>::NB; b++) {
            const bool mine = T == 1 || n >> 3 == i;
            q.hi[i][b] = mine ? col.hi[b] : none;
            q.lo[i][b] = mine ? col.lo[b] : none;
        }
    return q;
}

// The scores of 32 keys and 16 columns (of two tiles' and eight): lane (g, n) gets keys
// 8 g + j of its tile and column.
template <int HD, int T>
__device__ __forceinline__ void scores(const Tile<HD> (&t)[T], const u32x4 (&kd)[Shape<HD>::NB],
                                       const Queries<HD, T>& q, float (&s)[8]) {
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4 d = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < T; i++) {
                const half8 lv = k_levels(t[i].k[h][b]);
                d = mfma(lv, q.hi[i][b], mfma(lv, q.lo[i][b], d));
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
                s[4 * h + r] = b == 0 ? half_at(kd[b], 4 * h + r) * d[r] : fmaf(half_at(kd[b], 4 * h + r), d[r], s[4 * h + r]);
        }
    }
}

// Less slope * distance, of the octet of keys at key0.
__device__ __forceinline__ void less_distance(const AttnArgs& a, float slope, int qpos, const uint32_t* kpos, int key0,
                                              float (&x)[8]) {
    float d[8];
    if (kpos) {
        typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
        const u32x4u* from = reinterpret_cast<const u32x4u*>(kpos + min(key0, a.c.cap - 8));
        const u32x4u u = from[0], v = from[1];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            d[j] = static_cast<float>(qpos - static_cast<int>(u[j]));
            d[4 + j] = static_cast<float>(qpos - static_cast<int>(v[j]));
        }
    } else {
        const float d0 = static_cast<float>(qpos - key0);
#pragma unroll
        for (int j = 0; j < 8; j++) d[j] = d0 - static_cast<float>(j);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = fmaf(-slope, fabsf(d[j]), x[j]);
}

// Options applied: scores then in the exponent's unit (log2), as they were without any.
template <int HD, bool MODS>
__device__ __forceinline__ void finish_scores(const AttnArgs& a, const Column<HD>& col, const uint32_t* kpos, int key0,
                                              float (&s)[8]) {
    if constexpr (MODS) {
        if (a.softcap > 0.0f) cap_scores(s, a.softcap, col.factor);
        const float unit = col.factor * kLog2e;
#pragma unroll
        for (int j = 0; j < 8; j++) s[j] *= unit;
        if (a.slopes) less_distance(a, col.slope * kLog2e, col.qpos, kpos, key0, s);
    }
}

// What a wave has of its 16 columns: the sums of e = 2^(score - base) (l, each lane
// its own keys') and of e * value (o).  base is 10 below the largest of score + E so
// far, 2^E being above the key's value scales: what counts is not how large a weight
// is but how large its product, so that a row whose keys have small values is as
// exact beside a row, or a key of no weight, with large ones.
template <int HD, int T>
struct Sums {
    f32x4 o[T][Shape<HD>::NB][2];  // (of each tile of a pair: the other tile's columns mean nothing)
    float l, base;
};

template <int HD, int T>
__device__ __forceinline__ void clear(Sums<HD, T>& z) {
#pragma unroll
    for (int i = 0; i < T; i++)
#pragma unroll
        for (int b = 0; b < Shape<HD>::NB; b++) z.o[i][b][0] = z.o[i][b][1] = f32x4{0, 0, 0, 0};
    z.l = 0.0f;
    z.base = -FLT_MAX;
}

// 1024 + the exponent field, as f16, of the largest scale of each key: a word of two
// keys of one block in, the same keys' of all blocks out.  Of the eight lanes of an
// octet, lanes j and j ^ 4 (two blocks) or j, j ^ 2, j ^ 4 and j ^ 6 (four) have one
// key's blocks.
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t lanes(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
template <int NB>
__device__ __forceinline__ uint32_t key_exponents(uint32_t scales) {
    uint32_t x = scales & 0x7C007C00u;
    if constexpr (NB == 4) {
        x = larger(x, lanes<0x4E>(x));                // j ^ 2
        x = larger(x, lanes<0x141>(lanes<0xB1>(x)));  // (j ^ 7) ^ 1, which has what j ^ 4 has
    } else if constexpr (NB == 2) {
        x = larger(x, lanes<0x141>(lanes<0x1B>(x)));  // (j ^ 7) ^ 3
    }
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, x) >> 10) | 0x64006400u;
}

// T tiles of 32 keys, at `tile` and behind, into the sums.  next(0), (1) and (2): the tiles'
// scales, keys and values are used up.  The weights times their
// block's value scale are the f16 operand (two terms): at most 2^14, with 2^-39 of that
// as their last place, which is 2^-35 of the row's largest.  swap: the wave's LDS
// room for the tiles' scales.
constexpr int kSwap = 64;  // 2-byte words of it: 64 scales a block, 64 exponents
template <int HD, bool MODS, bool MASKED, int T, typename Next>
__device__ __forceinline__ void step(const AttnArgs& a, const Tile<HD> (&t)[T], int tile, int t1, int lane,
                                     const Column<HD>& col, const Queries<HD, T>& q, const uint32_t* kpos,
                                     uint16_t* swap, Sums<HD, T>& z, Next next) {
    constexpr int NB = Shape<HD>::NB, SW = kSwap * (NB + 1);
    const int g = lane >> 4, n = lane & 15, mine = T == 2 ? n >> 3 : 0, key0 = (tile + mine) * 32 + 8 * g;
    // (a wave's LDS instructions run in order: only the compiler has to be held)
#pragma unroll
    for (int i = 0; i < T; i++) {
        uint16_t* to = swap + i * SW;
        // the scales, and their keys' largest exponents behind them (those of the keys' own go unread)
        uint16_t* large = to + 64 * NB + (lane >> 3) * 8;
        const auto& sc = t[i].sc;
        if constexpr (NB == 4) {
            *reinterpret_cast<u32x2*>(to + lane * 4) = u32x2{sc[0], sc[1]};
            *reinterpret_cast<u32x2*>(large + lane % 2 * 4) = u32x2{key_exponents<NB>(sc[0]), key_exponents<NB>(sc[1])};
        } else if constexpr (NB == 2) {
            *reinterpret_cast<uint32_t*>(to + lane * 2) = sc[0];
            *reinterpret_cast<uint32_t*>(large + lane % 4 * 2) = key_exponents<NB>(sc[0]);
        } else {
            to[lane] = static_cast<uint16_t>(sc[0]);
            large[lane % 8] = static_cast<uint16_t>(key_exponents<NB>(sc[0]));
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    u32x4 kd[NB], vd[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        kd[b] = *reinterpret_cast<const u32x4*>(swap + mine * SW + (g * NB + b) * 8);
        vd[b] = *reinterpret_cast<const u32x4*>(swap + mine * SW + ((4 + g) * NB + b) * 8);
    }
    const u32x4 e = *reinterpret_cast<const u32x4*>(swap + mine * SW + 64 * NB + (4 + g) * 8);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float s[8];
    next(0);
    scores<HD, T>(t, kd, q, s);
    next(1);
    finish_scores<HD, MODS>(a, col, kpos, key0, s);
    bool seen[8];
    if constexpr (MASKED) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            seen[j] = static_cast<uint32_t>(key0 + j - col.first) < static_cast<uint32_t>(col.wide) &&
                      (T == 1 || tile + mine < t1);
            s[j] = seen[j] ? s[j] : -INFINITY;
        }
    }
    const float f = MODS ? 1.0f : col.factor * kLog2e;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; j++) top = fmaxf(top, fmaf(s[j], f, half_at(e, j)));
    top -= 1024.0f + 14.0f;  // (the scale is below 2^(field - 14))
    if (__any(top > z.base + 14.0f)) {
        const float m = fmaxf(z.base == -FLT_MAX ? -FLT_MAX : z.base + 10.0f, across_groups_max(top));
        const float base = m == -FLT_MAX ? -FLT_MAX : m - 10.0f;
        const float k = __builtin_amdgcn_exp2f(z.base - base);
        z.l *= k;
#pragma unroll
        for (int i = 0; i < T; i++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                z.o[i][b][0] *= k;
                z.o[i][b][1] *= k;
            }
        z.base = base;
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], f, -z.base));
    z.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    const float zero = hidden(0.0f);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = fmaf(p[2 * i], half_at(vd[b], 2 * i), zero), y = fmaf(p[2 * i + 1], half_at(vd[b], 2 * i + 1), zero);
            if constexpr (MASKED) {
                x = seen[2 * i] ? x : 0.0f;
                y = seen[2 * i + 1] ? y : 0.0f;
            }
            split2(x, y, hi[i], lo[i]);
        }
        const half8 ph = as_half8(hi[0], hi[1], hi[2], hi[3]), pl = as_half8(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
        for (int i = 0; i < T; i++) {
            u32x4 w = t[i].v[HD >= 64 ? b / 2 : 0];
            if constexpr (HD == 32) {
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] >>= n & 8;
            }
            const half8 v0 = b & 1 ? v_levels<2>(w) : v_levels<0>(w), v1 = b & 1 ? v_levels<3>(w) : v_levels<1>(w);
            z.o[i][b][0] = mfma(v0, ph, mfma(v0, pl, z.o[i][b][0]));
            z.o[i][b][1] = mfma(v1, ph, mfma(v1, pl, z.o[i][b][1]));
        }
    }
    next(2);
}

// The columns' queries against T tiles at t0, t0 + stride, .. below t1.  Two steps' tiles are
// at hand; what comes after them is loaded part by part as soon as a step has used
// up what lies in its place (8 x <= 32767 keys of 32 and 8 heads of width 128 63.6 us, with the
// loads behind the step 65.4, with one place 66).
template <int HD, bool MODS, int T>
__device__ __forceinline__ void walk(const AttnArgs& a, const Planes& p, int lane, Column<HD>& col,
                                     const uint32_t* kpos, int t0, int t1, int stride, int full_lo, int full_hi,
                                     uint16_t* swap, Sums<HD, T>& z) {
    if (t0 >= t1) return;
    const uint16_t* scales = lane < 32 ? p.kd : p.vd;
    Tile<HD> tiles[2][T];
    const auto load = [&](int d, int t, int part) {
#pragma unroll
        for (int i = 0; i < T; i++) {
            const int at = min(t + i, t1 - 1);
            if (part == 0) load_scales<HD>(scales, a.c.cap, at, lane, tiles[d][i]);
            if (part == 1) load_k<HD>(p, a.c.cap, at, lane, tiles[d][i].k);
            if (part == 2) load_v<HD>(p, a.c.cap, at, lane, tiles[d][i]);
        }
    };
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
        for (int part = 0; part < 3; part++) load(d, t0 + d * stride, part);
    column_query<HD>(a, lane, col);  // (its loads wait beside the tiles')
    const Queries<HD, T> q = queries_of<HD, T>(col, lane & 15);
    const auto work = [&](auto place, int t) {
        constexpr int d = decltype(place)::value;
        const auto next = [&](int part) { load(d, t + 2 * stride, part); };
        if (t * 32 >= full_lo && (t + T) * 32 <= full_hi && t + T <= t1)
            step<HD, MODS, false, T>(a, tiles[d], t, t1, lane, col, q, kpos, swap, z, next);
        else
            step<HD, MODS, true, T>(a, tiles[d], t, t1, lane, col, q, kpos, swap, z, next);
    };
    for (int t = t0; t < t1; t += 2 * stride) {
        work(std::integral_constant<int, 0>{}, t);
        if (t + stride >= t1) break;
        work(std::integral_constant<int, 1>{}, t + stride);
    }
}

// The keys that a wave's columns see: the union [lo, hi), and the part that every
// column of the call sees [flo, fhi).
__device__ __forceinline__ void column_range(bool on, int first, int wide, int& lo, int& hi, int& flo, int& fhi) {
    lo = wide ? first : 0x7FFFFFFF;
    hi = wide ? first + wide : 0;
    flo = on ? first : 0;
    fhi = on ? first + wide : 0x7FFFFFFF;
    lo = __builtin_amdgcn_readfirstlane(group_min(lo));
    hi = -__builtin_amdgcn_readfirstlane(group_min(-hi));
    flo = -__builtin_amdgcn_readfirstlane(group_min(-flo));
    fhi = __builtin_amdgcn_readfirstlane(group_min(fhi));
}

// Channels 32 b + 8 g .. + 7 of a column, from its sums.
template <int HD, int T>
__device__ __forceinline__ void channels(const Sums<HD, T>& z, int b, int n, float (&x)[8]) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        x[2 * r] = T == 2 && n >= 8 ? z.o[T - 1][b][0][r] : z.o[0][b][0][r];
        x[2 * r + 1] = T == 2 && n >= 8 ? z.o[T - 1][b][1][r] : z.o[0][b][1][r];
    }
}

// Two floats of memory that other workgroups read and write, 8-byte aligned.
__device__ __forceinline__ void store2(float* to, float a, float b) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, make_float2(a, b)), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load2(const float* from) {
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(from)),
                                                        __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Attention of 16 columns (T = 2: of at most eight, two tiles at a time) by one workgroup: the
// four waves take every fourth tile, or pair, of the workgroup's share of the keys.
// Waves share no keys, so none waits for another before the join.  Bound by
// VALU issue (a tile of width 64 is 200 instructions beside 16 MFMAs, most of them per
// column, in use or not): 8 x <= 32767 keys of 32 and 8 heads of width 128 64 us, 3.7 TB/s
// of cache, VALU busy 79 %; 64 x <= 8000 keys of 12 heads of width 64 82 us, 4.1 TB/s.
// Short calls are latency: 1 x 511 keys of 14 and 2 heads 6 us.
template <int HD, bool MODS, int T>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_attention(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB, LD = HD + 4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    int id = static_cast<int>(blockIdx.x);
    const int split = id % a.splits;
    id /= a.splits;
    const int unit = id, heads = a.c.seqs * a.c.n_kv;
    const int ct = a.col_tiles - 1 - id / heads;  // (the longest rows first)
    id %= heads;
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    if (static_cast<uint64_t>(ct) * 16 >= static_cast<uint64_t>(r.count) * a.group) return;
    Column<HD> col;
    column_place<HD, MODS>(a, r, kv, static_cast<uint32_t>(ct) * 16 + (T == 2 ? n & 7 : n), col);
    int lo, hi, flo, fhi;
    column_range(col.on, col.first, col.wide, lo, hi, flo, fhi);
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + (static_cast<size_t>(s) * a.c.n_kv + kv) * a.c.cap : nullptr;
    Sums<HD, T> z;
    clear<HD, T>(z);
    const int t_lo = lo < hi ? lo / 32 : 0, tiles = lo < hi ? (hi + 31) / 32 - t_lo : 0;
    // (at most 2^20 tiles and 2^10 splits)
    const uint32_t each = static_cast<uint32_t>(tiles), of = static_cast<uint32_t>(a.splits);
    const int t0 = t_lo + static_cast<int>(each * split / of), t1 = t_lo + static_cast<int>(each * (split + 1) / of);
    __shared__ __align__(16) float so[4][16][LD];
    __shared__ float sb[4][16], sl[4][16];
    // (a wave's room for scales is in its own part of the sums')
    walk<HD, MODS, T>(a, p, lane, col, kpos, t0 + T * wave, t1, 4 * T, flo, fhi, reinterpret_cast<uint16_t*>(so[wave]), z);
    // join the waves
    __shared__ int last;
    const float l = across_groups_sum(z.l);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float x[8];
        channels<HD, T>(z, b, n, x);
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
    float base = -FLT_MAX, sum = 0.0f, x[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4 * T; w++) base = fmaxf(base, sb[w / T][(cj + w % T * 8) & 15]);
#pragma unroll
    for (int w = 0; w < 4 * T; w++) {
        const int from = (cj + w % T * 8) & 15;
        const float f = __builtin_amdgcn_exp2f(sb[w / T][from] - base);
        sum = fmaf(sl[w / T][from], f, sum);
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = fmaf(so[w / T][from][ch + i], f, x[i]);
    }
    const uint32_t c = static_cast<uint32_t>(ct) * 16 + cj;
    Column<HD> mine;  // (its place only)
    column_place<HD, false>(a, r, kv, c, mine);
    if (a.splits > 1) {
        constexpr int PL = HD + 2;
        float* part = a.part + static_cast<size_t>(unit) * a.splits * 16 * PL;
        if (mine.on) {
            float* to = part + (static_cast<size_t>(split) * 16 + cj) * PL;
            if (ch == 0) store2(to, base, sum);
#pragma unroll
            for (int i = 0; i < PER; i += 2) store2(to + 2 + ch + i, x[i], x[i + 1]);
        }
        // Every thread's coherent stores complete before the arrival count moves.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(a.counters + unit, 1u) == static_cast<unsigned>(a.splits - 1);
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0)
            __hip_atomic_store(a.counters + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // Sixteen threads a column; with fewer than 16 columns they also share out the
        // splits (each eight at a time, their loads in flight together), and join in LDS.
        const int cols = min(16, static_cast<int>(r.count * a.group - static_cast<uint32_t>(ct) * 16));
        const int lanes = cols > 8 ? 16 : cols > 4 ? 8 : cols > 2 ? 4 : cols, sets = 16 / lanes;
        const int jc = cj % lanes, set = cj / lanes;
        base = -FLT_MAX;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = 0.0f;
        if (jc < cols) {
            constexpr int R = 8;
            for (int s0 = set; s0 < a.splits; s0 += R * sets) {
                float2 st[R], v[R][PER / 2];
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const float* from = part + (static_cast<size_t>(min(s0 + i * sets, a.splits - 1)) * 16 + jc) * PL;
                    st[i] = load2(from);
#pragma unroll
                    for (int k = 0; k < PER / 2; k++) v[i][k] = load2(from + 2 + ch + 2 * k);
                }
                float m = base;
#pragma unroll
                for (int i = 0; i < R; i++) m = fmaxf(m, st[i].x);  // (repeats of the last change nothing)
                const float k0 = __builtin_amdgcn_exp2f(base - m);
                base = m;
                sum *= k0;
#pragma unroll
                for (int k = 0; k < PER; k++) x[k] *= k0;
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const float f = s0 + i * sets < a.splits ? __builtin_amdgcn_exp2f(st[i].x - m) : 0.0f;
                    sum = fmaf(st[i].y, f, sum);
#pragma unroll
                    for (int k = 0; k < PER / 2; k++) {
                        x[2 * k] = fmaf(v[i][k].x, f, x[2 * k]);
                        x[2 * k + 1] = fmaf(v[i][k].y, f, x[2 * k + 1]);
                    }
                }
            }
        }
        if (sets > 1) {
            float(*sx)[LD] = so[0];
#pragma unroll
            for (int i = 0; i < PER; i++) sx[cj][ch + i] = x[i];
            if (ch == 0) {
                sb[0][cj] = base;
                sl[0][cj] = sum;
            }
            __syncthreads();
            if (cj < cols) {
                base = -FLT_MAX;
                for (int i = 0; i < sets; i++) base = fmaxf(base, sb[0][cj + i * lanes]);
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < PER; i++) x[i] = 0.0f;
                for (int q = 0; q < sets; q++) {
                    const float f = __builtin_amdgcn_exp2f(sb[0][cj + q * lanes] - base);
                    sum = fmaf(sl[0][cj + q * lanes], f, sum);
#pragma unroll
                    for (int i = 0; i < PER; i++) x[i] = fmaf(sx[cj + q * lanes][ch + i], f, x[i]);
                }
            }
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

// ---- attention of many columns --------------------------------------------------

// What is staged of 32 keys, as the matrix cores take it: fragments [lane][8 f16].
template <int HD>
struct Stage {
    uint32_t k[2][Shape<HD>::NB][2][64][4];  // keys as MFMA rows 0 .. 15 and 16 .. 31, by block and f16 term
    uint32_t v[Shape<HD>::NB][2][2][64][4];  // values, by block, channel parity and f16 term
};
// What a column keeps here rather than in registers (which would be spilled).
struct Place {
    float unit, factor, slope;  // unit: log2 units of a score, distance off
    int qpos, first, wide;
    uint32_t row;   // all ones: not a column of the call
    uint32_t head;  // the top bit: its row has no place in the cache
};

// Staged scales are 2^kLift above their key's exponent: a level times a scale is below 2^15
// then, and a block's scale exact in f16 as far as 2^25 below the key's largest (below 1 it
// would be to 2^13 only), or at any distance where that is under 2^12: an f16 scale's last
// place is 2^-24 at least.
constexpr int kLift = 12;

// Of four tiles' keys: the block scales under 2^(e - kLift) (0 of a key that nobody sees or
// that holds a NaN), e being the largest exponent of a key's own; as 2^(e - kLift) of keys
// (NaN where they hold one), as e and 2^-e of values.
template <int HD>
struct Room {
    Stage<HD> stage[2];
    Place place[128];
    float kup[4][32], ve[4][32], vdown[4][32];
    uint16_t d[2][4][Shape<HD>::NB][32];  // of values, of keys
    uint32_t nan[4];                      // a bit a key whose values hold one
    int range[2];
};

// One thread's share of a tile on its way to LDS.
template <int HD>
struct Load {
    static constexpr int W = HD == 128 ? 2 : 1;  // words of keys
    uint32_t k[W];
    u32x4 v;
    uint16_t d[Shape<HD>::NB];  // a key's scales, two tiles ahead (lanes 0 .. 31 of one wave values', the others keys')
};

// A thread stages the levels of one key (MFMA row n of half h), channels 8 g .. + 7 of
// blocks kb .. kb + W - 1; and of octet g the nibbles at ve (head width 128: both) of
// the 2-byte units of lane n in block vb.
template <int HD>
struct Part {
    static constexpr int BP = Shape<HD>::BP, W = Load<HD>::W;
    int n, g, h, kb, vb, ve;
    __device__ __forceinline__ explicit Part(int tid) {
        n = tid & 15;
        g = tid >> 4 & 3;
        h = tid >> 6 & 1;
        kb = (tid >> 7) * W;
        vb = HD == 128 ? tid >> 6 : tid >> 6 & 1;
        ve = HD == 128 ? 0 : tid >> 7;
    }
    __device__ __forceinline__ int key() const { return 8 * (n >> 2) + (n & 3) + 4 * h; }
    __device__ __forceinline__ int unit() const { return n * BP + vb / 2; }
    __device__ __forceinline__ int shift() const { return vb % 2 * 8; }
};

template <int HD>
__device__ __forceinline__ void load_part(const Planes& p, int cap, int tile, const Part<HD>& w, Load<HD>& t) {
    constexpr int NB = Shape<HD>::NB, VU = HD / 4;
    // (a tile's end past the capacity reads the last rows again; they weigh nothing)
    const uint32_t key = min(tile * 32 + w.key(), cap - 1), o = min(tile * 4 + w.g, cap / 8 - 1);
    const uint8_t* a = p.k + static_cast<size_t>(key * (HD / 2) + (w.g * NB + w.kb) * 4);
    if constexpr (HD == 128) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(a);
        t.k[0] = x[0];
        t.k[1] = x[1];
    } else {
        t.k[0] = *reinterpret_cast<const uint32_t*>(a);
    }
    t.v = *reinterpret_cast<const u32x4*>(p.v + (o * VU + w.unit()) * 16);
}

__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ uint32_t bits(half2v x) { return __builtin_bit_cast(uint32_t, x); }

// level * scale in f16 and what that leaves, both exact: 15 bits.
__device__ __forceinline__ void times_scale(uint32_t level, half2v scale, uint32_t& hi, uint32_t& lo) {
    const half2v x = as_half2(level), h = x * scale;
    hi = bits(h);
    lo = bits(__builtin_elementwise_fma(x, scale, -h));
}
template <int HD, int I>
__device__ __forceinline__ void store_values(const Part<HD>& w, const u32x4& v, const u32x4& d, Stage<HD>& st) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) times_scale(levels2<I>(v[i] >> w.shift()), as_half2(d[i]), hi[i], lo[i]);
    const int lane = w.g * 16 + w.n;
    *reinterpret_cast<u32x4*>(st.v[w.vb][I][0][lane]) = u32x4{hi[0], hi[1], hi[2], hi[3]};
    *reinterpret_cast<u32x4*>(st.v[w.vb][I][1][lane]) = u32x4{lo[0], lo[1], lo[2], lo[3]};
}

template <int HD>
__device__ __forceinline__ void store_part(int tile, const Part<HD>& w, const Load<HD>& t, Room<HD>& room) {
    const int lane = w.g * 16 + w.n, f = tile & 3;
    Stage<HD>& st = room.stage[tile & 1];
#pragma unroll
    for (int i = 0; i < Load<HD>::W; i++) {
        const _Float16 x = __builtin_bit_cast(_Float16, room.d[1][f][w.kb + i][w.key()]);
        const half2v sc = {x, x};
        uint32_t hi[4], lo[4];
        times_scale(levels2<0>(t.k[i]), sc, hi[0], lo[0]);
        times_scale(levels2<1>(t.k[i]), sc, hi[1], lo[1]);
        times_scale(levels2<2>(t.k[i]), sc, hi[2], lo[2]);
        times_scale(levels2<3>(t.k[i]), sc, hi[3], lo[3]);
        *reinterpret_cast<u32x4*>(st.k[w.h][w.kb + i][0][lane]) = u32x4{hi[0], hi[1], hi[2], hi[3]};
        *reinterpret_cast<u32x4*>(st.k[w.h][w.kb + i][1][lane]) = u32x4{lo[0], lo[1], lo[2], lo[3]};
    }
    const u32x4 d = *reinterpret_cast<const u32x4*>(&room.d[0][f][w.vb][8 * w.g]);
    if constexpr (HD == 128) {
        store_values<HD, 0>(w, t.v, d, st);
        store_values<HD, 1>(w, t.v, d, st);
    } else {
        if (w.ve) store_values<HD, 1>(w, t.v, d, st);
        else store_values<HD, 0>(w, t.v, d, st);
    }
}

constexpr int kPromptTiles = 2;  // tiles of 16 columns of a wave

// Attention of 128 columns of one (sequence, kv head): four waves with 32
// columns each walk the same keys, 32 at a time, expanded once into LDS for all
// of them: keys and values as level * scale in two exact f16 terms, so that
// neither a score nor a weight takes its scale block by block, and every product
// of an f32 operand (two terms as well) is three matrix products, the lowest left
// out (2^-22).  The range of f16 is each key's own: 2^-e here, 2^e on its score or
// weight, e being the key's largest block's exponent and nothing of any other key's, so that
// a row has the bits of what it sees whatever the other 127 columns see.  The running maximum
// is that of score + e.  A block of values counts, as in k_kv4_attention, down to 2^-34 of the
// row's largest weight times scale; one of keys down to 2^-36 of its key's largest.
// At two waves a SIMD every register counts: what a column or a tile keeps is in LDS
// (spilled, 4 x 2048 rows of documents, 32 and 8 heads of width 128, take 265 us; 220 so).
// 16 columns a wave instead of 32: 312.  4 x 2000 causal rows of the same heads 366 us, 358
// TFLOP/s or 1,075 of f16 products, near a large f16 product's rate (MFMA 46 % busy, VALU 52 %);
// short documents: VALU 58 %, MFMA 33 %.
template <int HD, bool MODS>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_prompt(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB, CT = kPromptTiles;
    extern __shared__ __align__(16) char smem[];
    Room<HD>& room = *reinterpret_cast<Room<HD>*>(smem);
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int heads = a.c.seqs * a.c.n_kv;
    const int id = static_cast<int>(blockIdx.x) % heads;
    const int ct0 = (a.col_tiles - 1 - static_cast<int>(blockIdx.x) / heads) * 4 * CT;  // (the longest rows first)
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    if (static_cast<uint64_t>(ct0) * 16 >= static_cast<uint64_t>(r.count) * a.group) return;
    Column<HD> col[CT];  // (their queries alone stay)
    int lo = 0x7FFFFFFF, hi = 0, flo = 0, fhi = 0x7FFFFFFF;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        column_place<HD, MODS>(a, r, kv, static_cast<uint32_t>(ct0 + wave * CT + c) * 16 + n, col[c]);
        int x, y, fx, fy;
        column_range(col[c].on, col[c].first, col[c].wide, x, y, fx, fy);
        lo = min(lo, x);
        hi = max(hi, y);
        flo = max(flo, fx);
        fhi = min(fhi, fy);
    }
    if (tid == 0) {
        room.range[0] = 0x7FFFFFFF;
        room.range[1] = 0;
    }
    __syncthreads();
    if (lane == 0) {
        atomicMin(&room.range[0], lo);
        atomicMax(&room.range[1], hi);
    }
    __syncthreads();
    const int glo = room.range[0], ghi = room.range[1];
    const int t0 = glo < ghi ? glo / 32 : 0, t1 = glo < ghi ? (ghi + 31) / 32 : 0;
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + (static_cast<size_t>(s) * a.c.n_kv + kv) * a.c.cap : nullptr;
    const Part<HD> part(tid);
    Load<HD> ld;
    const auto load_scales = [&](int tile) {
        const uint32_t key = min(tile * 32 + (lane & 31), a.c.cap - 1);
        const uint16_t* from = (lane < 32 ? p.vd : p.kd) + key / 8 * (NB * 8) + key % 8;
#pragma unroll
        for (int b = 0; b < NB; b++) ld.d[b] = from[b * 8];
    };
    if (t0 < t1) load_part<HD>(p, a.c.cap, t0, part, ld);
#pragma unroll
    for (int c = 0; c < CT; c++) {
        column_query<HD>(a, lane, col[c]);
        if (g == 0) {
            const float unit = MODS && a.slopes ? kLog2e : col[c].factor * kLog2e;
            Place& to = room.place[(wave * CT + c) * 16 + n];
            to = Place{unit, col[c].factor, MODS ? col[c].slope : 0.0f, MODS ? col[c].qpos : 0, col[c].first, col[c].wide,
                       col[c].on ? col[c].row : ~0u, static_cast<uint32_t>(col[c].head) | (col[c].bad ? 0x80000000u : 0u)};
        }
    }
    __syncthreads();
    const auto key_factors = [&](int tile) {  // of key lane % 32, from ld.d
        const int i = tile & 3, j = lane & 31, key = tile * 32 + j;
        int e = -14;
        bool fine = true;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int x = ld.d[b] >> 10 & 31;
            fine = fine && x < 31;
            e = max(e, x - 14);
        }
        const bool seen = key >= glo && key < ghi, use = fine && seen;
        e = use ? e : 0;
        const uint64_t nans = __ballot(seen && !fine);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const float x = ldexpf(fh_h2f(ld.d[b]), kLift - e);
            room.d[lane >> 5][i][b][j] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(use ? x : 0.0f));
        }
        if (lane < 32) {
            room.ve[i][j] = static_cast<float>(e);
            room.vdown[i][j] = ldexpf(1.0f, -e);
            if (lane == 0) room.nan[i] = static_cast<uint32_t>(nans);
        } else {
            room.kup[i][j] = fine || !seen ? ldexpf(1.0f, e - kLift) : __builtin_nanf("");
        }
    };
    f32x4 o[CT][NB][2];
    float l[CT], base[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        l[c] = 0.0f;
        base[c] = -FLT_MAX;
#pragma unroll
        for (int b = 0; b < NB; b++) o[c][b][0] = o[c][b][1] = f32x4{0, 0, 0, 0};
    }
    if (t0 < t1) {
        if (wave < 2) {
            load_scales(t0 + wave);
            key_factors(t0 + wave);
        }
        __syncthreads();
        store_part<HD>(t0, part, ld, room);
    }
    for (int t = t0; t < t1; t++) {
        __syncthreads();
        if (t + 1 < t1) load_part<HD>(p, a.c.cap, t + 1, part, ld);
        if (wave == (t & 3)) load_scales(t + 2);
        const Stage<HD>& st = room.stage[t & 1];
        if (t * 32 < hi && t * 32 + 32 > lo) {
            f32x4 d[CT][2];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8 kh = *reinterpret_cast<const half8*>(st.k[h][b][0][lane]);
                    const half8 kl = *reinterpret_cast<const half8*>(st.k[h][b][1][lane]);
#pragma unroll
                    for (int c = 0; c < CT; c++)
                        d[c][h] = mfma(kh, col[c].hi[b], mfma(kh, col[c].lo[b], mfma(kl, col[c].hi[b],
                                       b == 0 ? f32x4{0, 0, 0, 0} : d[c][h])));
                }
            const bool full = t * 32 >= flo && t * 32 + 32 <= fhi;
            const int key0 = t * 32 + 8 * g;
            half8 ph[CT], pl[CT];
            const uint32_t nan = __builtin_amdgcn_readfirstlane(room.nan[t & 3]);
            const float *kup = room.kup[t & 3] + 8 * g, *ve = room.ve[t & 3] + 8 * g, *vdown = room.vdown[t & 3] + 8 * g;
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const Place& at = room.place[(wave * CT + c) * 16 + n];
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = d[c][j >> 2][j & 3] * kup[j];
                if constexpr (MODS) {
                    if (a.softcap > 0.0f) cap_scores(x, a.softcap, at.factor);
                    if (a.slopes) {
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] *= at.factor;
                        less_distance(a, at.slope, at.qpos, kpos, key0, x);
                    }
                }
                if (!full) {
                    const int before = key0 - at.first, wide = at.wide;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        x[j] = static_cast<uint32_t>(before + j) < static_cast<uint32_t>(wide) ? x[j] : -INFINITY;
                }
                const float f = at.unit;
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[j] = fmaf(x[j], f, ve[j]);
                    top = fmaxf(top, x[j]);
                }
                if (__any(top > base[c] + 14.0f)) {
                    const float m = fmaxf(base[c] == -FLT_MAX ? -FLT_MAX : base[c] + 10.0f, across_groups_max(top));
                    const float nb = m == -FLT_MAX ? -FLT_MAX : m - 10.0f, k = __builtin_amdgcn_exp2f(base[c] - nb);
                    l[c] *= k;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        o[c][b][0] *= k;
                        o[c][b][1] *= k;
                    }
                    base[c] = nb;
                }
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; j++) e[j] = __builtin_amdgcn_exp2f(x[j] - base[c]);
#pragma unroll
                for (int j = 0; j < 8; j++) l[c] = fmaf(e[j], vdown[j], l[c]);
                if (nan) {  // (that of a key that this row does not see stays out)
#pragma unroll
                    for (int j = 0; j < 8; j++) e[j] = (nan >> (8 * g + j) & 1) && x[j] != -INFINITY ? __builtin_nanf("") : e[j];
                }
                uint32_t hw[4], lw[4];
#pragma unroll
                for (int j = 0; j < 4; j++) split2(e[2 * j], e[2 * j + 1], hw[j], lw[j]);
                ph[c] = as_half8(hw[0], hw[1], hw[2], hw[3]);
                pl[c] = as_half8(lw[0], lw[1], lw[2], lw[3]);
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const half8 vh = *reinterpret_cast<const half8*>(st.v[b][e][0][lane]);
                    const half8 vl = *reinterpret_cast<const half8*>(st.v[b][e][1][lane]);
#pragma unroll
                    for (int c = 0; c < CT; c++)
                        o[c][b][e] = mfma(vh, ph[c], mfma(vh, pl[c], mfma(vl, ph[c], o[c][b][e])));
                }
        }
        if (t + 1 < t1) store_part<HD>(t + 1, part, ld, room);
        if (wave == (t & 3)) key_factors(t + 2);
    }
    // Each lane has 8 channels of every block of its columns: 32 b + 8 g + i at o[b][i & 1][i >> 1] * 2^-kLift.
#pragma unroll
    for (int c = 0; c < CT; c++) l[c] = across_groups_sum(l[c]);
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const Place at = room.place[(wave * CT + c) * 16 + n];
        if (at.row == ~0u) continue;
        const size_t to = static_cast<size_t>(at.row) * a.n_heads + (at.head & 0x7FFFFFFFu);
        const bool bad = at.head >> 31;
        float* out = a.out + to * HD + g * 8;
        const float f = bad ? __builtin_nanf("") : l[c] == 0.0f ? 0.0f : 1.0f / (static_cast<float>(1 << kLift) * l[c]);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 8; i++) out[32 * b + i] = o[c][b][i & 1][i >> 1] * f;
        if (a.lse && g == 0) a.lse[to] = bad ? __builtin_nanf("") : (base[c] + log2f(l[c])) * kLn2;
    }
}

// Adds to each key's weight what every (query row, head of its group) gave it: exp(score - lse), the
// lse rounded to f32 between the two calls, so that a row's weights share an error of 2^-24 |lse|
// of themselves beside the scores' own.  (A sum over the keys again would cost the attention's first
// half once more.)
// Two forms: k_kv4_weigh_step for a single tile of 16 columns, whose queries are
// split once for all the keys that a wave walks, and k_kv4_weigh_prompt.

// The score of 32 keys and 16 columns as weights, added to acc.
template <int HD, bool MODS, bool MASKED, typename Scales>
__device__ __forceinline__ void add_weights(const AttnArgs& a, const half8 (&lv)[2][Shape<HD>::NB], const Scales& scales,
                                            const Column<HD>& col, float lse, const uint32_t* kpos, int key0,
                                            float (&acc)[8]) {
    float x[8];
#pragma unroll
    for (int b = 0; b < Shape<HD>::NB; b++) {
        const u32x4 kd = scales(b);  // of the lane's eight keys
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f32x4 d = mfma(lv[h][b], col.hi[b], mfma(lv[h][b], col.lo[b], f32x4{0, 0, 0, 0}));
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[4 * h + j] = b == 0 ? half_at(kd, 4 * h + j) * d[j] : fmaf(half_at(kd, 4 * h + j), d[j], x[4 * h + j]);
        }
    }
    finish_scores<HD, MODS>(a, col, kpos, key0, x);
    const float f = MODS ? 1.0f : col.factor * kLog2e;
#pragma unroll
    for (int j = 0; j < 8; j++)
        acc[j] += !MASKED || static_cast<uint32_t>(key0 + j - col.first) < static_cast<uint32_t>(col.wide)
                      ? __builtin_amdgcn_exp2f(fmaf(x[j], f, -lse)) : 0.0f;
}

// A workgroup: every fourth tile of its share of the keys to a wave, the next on its way.
// 8 x 16000 keys of 32 and 8 heads of width 128 24 us (68 with the queries split again for
// every two tiles), 64 x <= 1023 of 14 and 2 heads of width 64 6: load latency.
template <int HD, bool MODS>
__global__ void __launch_bounds__(kThreads, 2) k_kv4_weigh_step(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int split = static_cast<int>(blockIdx.x) % a.splits, id = static_cast<int>(blockIdx.x) / a.splits;
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    Column<HD> col;
    column_place<HD, MODS>(a, r, kv, n, col);
    int lo, hi, flo, fhi;
    column_range(col.on, col.first, col.wide, lo, hi, flo, fhi);
    if (lo >= hi) return;
    const int first = lo / 32, tiles = (hi + 31) / 32 - first;
    // (at most 2^20 tiles and 2^10 splits)
    const uint32_t each = static_cast<uint32_t>(tiles), of = static_cast<uint32_t>(a.splits);
    const int t1 = first + static_cast<int>(each * (split + 1) / of);
    int t = first + static_cast<int>(each * split / of) + wave;
    if (t >= t1) return;
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + static_cast<size_t>(id) * a.c.cap : nullptr;
    float* weight = a.c.weight + static_cast<size_t>(id) * a.c.cap;
    uint32_t k[2][NB];
    u32x4 kd[NB];
    load_k<HD>(p, a.c.cap, t, lane, k);
    load_kd<HD>(p, a.c.cap, t, lane, kd);
    column_query<HD>(a, lane, col);
    const float lse = col.on ? a.lse_in[static_cast<size_t>(col.row) * a.n_heads + col.head] * kLog2e : 0.0f;
    for (; t < t1; t += 4) {
        half8 lv[2][NB];
        u32x4 sc[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            lv[0][b] = k_levels(k[0][b]);
            lv[1][b] = k_levels(k[1][b]);
            sc[b] = kd[b];
        }
        const int next = min(t + 4, t1 - 1);
        load_k<HD>(p, a.c.cap, next, lane, k);
        load_kd<HD>(p, a.c.cap, next, lane, kd);
        const int key = t * 32 + 8 * g + (n & 7);  // (lanes n and n + 8 have the same; n < 8 add it)
        const bool mine = n < 8 && key >= lo && key < hi;
        const float old = mine ? weight[key] : 0.0f;
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        add_weights<HD, MODS, true>(a, lv, [&](int b) { return sc[b]; }, col, lse, kpos, t * 32 + 8 * g, acc);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = fh::group_sum<16>(acc[j]);
            sum = (n & 7) == j ? v : sum;
        }
        if (mine) weight[key] = old + sum;
    }
}

// A workgroup has 8 KT tiles of keys, KT to a wave (every eighth of them, so that a causal
// prompt's diagonal is shared out), and takes 4 or 8 tiles of 16 columns at a time of its share
// (of `splits`; their sums then go to a.part and k_kv4_add_weights adds them up in
// order): each wave splits the queries of one into LDS for all of them, while the
// next batch is on its way.  (Split by every wave for itself, 1 x 1000 rows of 32 and 8
// heads of width 128 took 54 us; they take 31, 132 TFLOP/s of products of two terms.)
// Bound by its waits (49 % of the waves' cycles; VALU 45 % busy, MFMA 17 %): a workgroup has two
// batches there, each with two barriers, and nothing of the next one's split behind the products.
constexpr int kWeighTiles = 2;  // KT

template <int HD>
struct WeighRoom {
    half8 q[8][Shape<HD>::NB][2][64];
    f32x4 unit[8][16];  // factor, slope, log-sum-exp (log2), position
    int first[8][16], wide[8][16];
    int range[4][8];  // of a tile's columns: keys that one sees, keys that all see
    u32x4 kd[8][kWeighTiles][Shape<HD>::NB][4];  // (in registers they would crowd the queries on their way out)
};

template <int HD, bool MODS>
__global__ void __launch_bounds__(512, 2) k_kv4_weigh_prompt(AttnArgs a) {
    constexpr int NB = Shape<HD>::NB, KT = kWeighTiles;
    extern __shared__ __align__(16) char smem[];
    WeighRoom<HD>& room = *reinterpret_cast<WeighRoom<HD>*>(smem);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int limit = static_cast<int>(a.max_keys), heads = a.c.seqs * a.c.n_kv;
    int id = static_cast<int>(blockIdx.x);
    const int split = id % a.splits;
    id /= a.splits;
    const int tile0 = id / heads * (8 * KT);  // (the most seen keys first)
    id %= heads;
    const int kv = id % a.c.n_kv, s = id / a.c.n_kv;
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, s);
    const Planes p = planes_of<HD>(a.c, s, kv);
    const uint32_t* kpos = MODS && a.c.pos ? a.c.pos + static_cast<size_t>(id) * a.c.cap : nullptr;
    half8 lv[KT][2][NB];
    float acc[KT][8];
#pragma unroll
    for (int i = 0; i < KT; i++) {
        const int tile = tile0 + i * 8 + wave;
        if (lane < NB * 4)
            room.kd[wave][i][lane / 4][lane % 4] = *reinterpret_cast<const u32x4*>(
                p.kd + (static_cast<uint32_t>(min(tile * 4 + lane % 4, a.c.cap / 8 - 1)) * (NB * 8) + lane / 4 * 8));
        uint32_t k[2][NB];
        load_k<HD>(p, a.c.cap, tile, lane, k);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int b = 0; b < NB; b++) lv[i][h][b] = k_levels(k[h][b]);
#pragma unroll
        for (int j = 0; j < 8; j++) acc[i][j] = 0.0f;
    }
    const uint32_t tiles = (r.count * a.group + 15) / 16;  // (below 2^31: total * n_heads is)
    const uint32_t per = static_cast<uint32_t>(a.weigh_cols), batches = (tiles + per - 1) / per;
    // (rows above the first key do not see it, unless the call says where their keys end)
    const uint64_t key0 = static_cast<uint64_t>(tile0) * 32;
    const uint32_t none = a.end || key0 <= r.at ? 0 : static_cast<uint32_t>(min(
        (key0 - r.at) * static_cast<uint32_t>(a.group) / (16 * per), static_cast<uint64_t>(batches)));
    const uint32_t some = batches - none;
    const uint32_t b0 = none + static_cast<uint32_t>(static_cast<uint64_t>(some) * split / a.splits);
    const uint32_t b1 = none + static_cast<uint32_t>(static_cast<uint64_t>(some) * (split + 1) / a.splits);
    Column<HD> col;  // of the tile that this wave splits next
    float raw[NB][8], lse = 0.0f;
    int lo = 0, hi = 0, flo = 0, fhi = 0;
    const auto load = [&](uint32_t batch) {
        hi = 0;
        if (wave >= a.weigh_cols) return;
        column_place<HD, MODS>(a, r, kv, (batch * per + wave) * 16 + n, col);
        column_range(true, col.first, col.wide, lo, hi, flo, fhi);  // (one that is not the call's sees nothing)
        if (lo < (tile0 + 8 * KT) * 32 && hi > tile0 * 32) {
            load_query<HD>(a, lane, col, raw);
            lse = col.on ? a.lse_in[static_cast<size_t>(col.row) * a.n_heads + col.head] * kLog2e : 0.0f;
        } else {
            hi = 0;
        }
    };
    if (b0 < b1) load(b0);
    for (uint32_t batch = b0; batch < b1; batch++) {
        if (hi) {
            split_query<HD>(a, raw, col);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                room.q[wave][b][0][lane] = col.hi[b];
                room.q[wave][b][1][lane] = col.lo[b];
            }
            if (g == 0) {
                room.unit[wave][n] = f32x4{col.factor, MODS ? col.slope : 0.0f, lse, MODS ? __int_as_float(col.qpos) : 0.0f};
                room.first[wave][n] = col.first;
                room.wide[wave][n] = col.wide;
            }
        }
        if (lane == 0) {
            room.range[0][wave] = lo;
            room.range[1][wave] = hi;
            room.range[2][wave] = flo;
            room.range[3][wave] = fhi;
        }
        __syncthreads();
        if (batch + 1 < b1) load(batch + 1);
        const int ranges = room.range[lane / 8 & 3][lane % 8];
        for (int c = 0; c < a.weigh_cols; c++) {
            const int from = __builtin_amdgcn_readlane(ranges, c), to = __builtin_amdgcn_readlane(ranges, 8 + c);
            const int all_from = __builtin_amdgcn_readlane(ranges, 16 + c), all_to = __builtin_amdgcn_readlane(ranges, 24 + c);
            const auto seen = [&](int i) {
                const int key = (tile0 + i * 8 + wave) * 32;
                return from < key + 32 && to > key;
            };
            bool any = false;
#pragma unroll
            for (int i = 0; i < KT; i++) any = any || seen(i);
            if (!any) continue;
            Column<HD> now;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                now.hi[b] = room.q[c][b][0][lane];
                now.lo[b] = room.q[c][b][1][lane];
            }
            const f32x4 unit = room.unit[c][n];
            now.factor = unit[0];
            now.slope = unit[1];
            now.qpos = __float_as_int(unit[3]);
            now.first = room.first[c][n];
            now.wide = room.wide[c][n];
            const auto add = [&](int i, auto masked) {
                const auto scales = [&](int b) { return room.kd[wave][i][b][g]; };
                add_weights<HD, MODS, masked.value>(a, lv[i], scales, now, unit[2], kpos, (tile0 + i * 8 + wave) * 32 + 8 * g, acc[i]);
            };
            if ((tile0 + wave) * 32 >= all_from && (tile0 + (KT - 1) * 8 + wave) * 32 + 32 <= all_to) {
                // (side by side: one's products hide behind what follows the other's)
#pragma unroll
                for (int i = 0; i < KT; i++) add(i, std::false_type{});
            } else {
#pragma unroll
                for (int i = 0; i < KT; i++)
                    if (seen(i)) add(i, std::true_type{});
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < KT; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float sum = fh::group_sum<16>(acc[i][j]);
            const int key = (tile0 + i * 8 + wave) * 32 + 8 * g + j;
            if (n != j || key >= limit || static_cast<uint64_t>(key) >= r.at + r.count) continue;
            if (a.splits > 1) a.part[(static_cast<size_t>(split) * heads + id) * limit + key] = sum;
            else a.c.weight[static_cast<size_t>(id) * a.c.cap + key] += sum;
        }
}

// (2 x 1000 weights of 55 parts, a load at a time: 15.6 us; 8 x 1000 of 16, eight at once: 4.8.)
__global__ void __launch_bounds__(kThreads) k_kv4_add_weights(AttnArgs a) {
    const uint32_t heads = static_cast<uint32_t>(a.c.seqs) * a.c.n_kv;
    const size_t i = blockIdx.x * static_cast<size_t>(kThreads) + threadIdx.x, all = static_cast<size_t>(heads) * a.max_keys;
    if (i >= all) return;
    const uint32_t id = static_cast<uint32_t>(i / a.max_keys), key = static_cast<uint32_t>(i % a.max_keys);
    const Rows r = rows_of(a.off, a.len, a.total, a.max_rows, a.c.seqs, static_cast<int>(id) / a.c.n_kv);
    if (key >= r.at + r.count) return;
    float sum = 0.0f;
    for (int s = 0; s < a.splits; s += 8) {  // (eight on their way at once)
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = a.part[min(s + j, a.splits - 1) * all + i];
#pragma unroll
        for (int j = 0; j < 8; j++) sum += s + j < a.splits ? x[j] : 0.0f;
    }
    a.c.weight[static_cast<size_t>(id) * a.c.cap + key] += sum;
}

// ---- append -------------------------------------------------------------------

struct AppendArgs {
    Cache c;
    const float* qkv;
    size_t ld;
    uint32_t total, max_rows;
    int n_heads, octets, heads;  // heads: kv heads of a workgroup, with their query heads
    const uint32_t *off, *len, *pos;
    int rope_dim, neox;
    double log2_base;
    float linear;
    const float* ff;
    float* q;
};

// The frequency of pair i and the angle at a position: apply_rope's (llm.rs:146-175, RopeScaling::angle,
// llm.rs:118-121), in 32 bits as there.
__device__ __forceinline__ float rope_frequency(int i, const AppendArgs& a) {
    return i == 0 ? 1.0f : static_cast<float>(exp2(static_cast<double>(-2 * i) / a.rope_dim * a.log2_base));
}
__device__ __forceinline__ float rope_angle(uint32_t pos, int i, float freq, const AppendArgs& a) {
#pragma clang fp contract(off)
    const float f = a.ff ? a.ff[i] : 1.0f;
    return static_cast<float>(static_cast<int>(pos)) * freq / f * (1.0f / a.linear);
}

// Four channels from ch (a multiple of 4) of a head row and those they are rotated with.
struct Quad {
    f32x4 own, other;
};
template <bool QUADS>  // 16-byte accesses
__device__ __forceinline__ Quad load_quad(const float* x, int ch, bool turned, const AppendArgs& a) {
    const int half = a.rope_dim / 2;
    Quad q;
    if constexpr (QUADS) {
        const bool apart = turned && a.neox && ch < a.rope_dim;
        q.own = *reinterpret_cast<const f32x4*>(x + ch);
        const f32x4 v = *reinterpret_cast<const f32x4*>(x + (!apart ? ch : ch >= half ? ch - half : ch + half));
        q.other = apart ? v : f32x4{v[1], v[0], v[3], v[2]};
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int c = ch + k;
            q.own[k] = x[c];
            q.other[k] = turned && c < a.rope_dim ? x[a.neox ? (c >= half ? c - half : c + half) : c ^ 1] : 0.0f;
        }
    }
    return q;
}
// Rotated where they are among the first rope_dim: angles in 32 bits as
// fh_rope_async's, sine, cosine and products in 64, since a key's channel goes on
// to the border between two levels, where its last bit decides.
template <bool QUADS>
__device__ __forceinline__ f32x4 rotate_quad(const Quad& q, int ch, const AppendArgs& a, const double2* turn) {
#pragma clang fp contract(off)
    const int half = a.rope_dim / 2;
    f32x4 y = q.own;
    if (QUADS && ch >= a.rope_dim) return y;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int c = ch + k;
        if (QUADS || c < a.rope_dim) {
            const bool hi = a.neox ? c >= half : c & 1;
            const double2 t = turn[a.neox ? (hi ? c - half : c) : c >> 1];  // (cosine, sine)
            const double u = q.own[k], v = q.other[k];
            y[k] = static_cast<float>(fma(u, t.x, v * (hi ? t.y : -t.y)));
        }
    }
    return y;
}

// Exchange within eight consecutive lanes.
__device__ __forceinline__ float max8(float v) {
    v = fmaxf(v, fh::dpp<0xB1>(v));
    v = fmaxf(v, fh::dpp<0x4E>(v));
    return fmaxf(v, fh::dpp<0x141>(v));
}
__device__ __forceinline__ int min8(int v) {
    v = min(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false));
    return min(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false));
}

// The scale (f16 bits) and levels of a block whose channels 4 l .. 4 l + 3 lane l of
// eight holds: nibbles of channels 0, 1 (bits 0 .. 7) and 2, 3 (8 .. 15) of the lane's four.
__device__ __forceinline__ void quantise4(const f32x4& x, uint16_t& scale, uint32_t& levels) {
    const int l = threadIdx.x & 7;
    float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    const bool fine = fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY && fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY;
    top = max8(fine ? top : INFINITY);
    int at = 127;  // 2 * (first channel of that magnitude) + its sign
#pragma unroll
    for (int k = 3; k >= 0; k--)
        if (fabsf(x[k]) == top) at = 2 * (4 * l + k) + (x[k] < 0.0f);
    at = min8(at);
    const float m = at & 1 ? -top : top;
    const bool odd = !(top < INFINITY);
    _Float16 dh = static_cast<_Float16>(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
    if (odd) dh = __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x7E00));
    const float d = static_cast<float>(dh), inv = __builtin_amdgcn_rcpf(d), lim = 0.5f * fabsf(d);
    const bool flat = odd || d == 0.0f;
    levels = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        // the nearest level, ties to even: from an approximate quotient, put right by the
        // remainder, which one FMA gives exactly
        float t = rintf(x[k] * inv);
        const float rest = fmaf(-t, d, x[k]), over = fabsf(rest) - lim;
        const bool odd_t = static_cast<int>(t) & 1;
        if (over > 0.0f || (over == 0.0f && odd_t)) t += (rest > 0.0f) == (d > 0.0f) ? 1.0f : -1.0f;
        const uint32_t q = flat ? 8u : static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(t, -8.0f), 7.0f)) + 8);
        levels |= q << (4 * k);
    }
    scale = __builtin_bit_cast(uint16_t, dh);
}

// The eight cache rows of one octet: rotate and store their queries, quantise
// their keys and values, eight lanes a block.  Whole octets leave as they lie in the
// planes, through LDS; four quads a thread are on their way at once (8 x <= 1000 rows of
// 32 and 8 heads of width 128: 213 us with one channel a thread and one load, 62 so, which
// is 4.4 TB/s, 94 % of a large copy's; VALU issue, the rotation in 64 bits and the
// quantiser, is as full).  A token's row is a chain of latencies, 5.5 us: loads before the
// angles spill and gain nothing.
template <int HD, bool QUADS>
__global__ void __launch_bounds__(kThreads, 4) k_kv4_append(AppendArgs a) {
    constexpr int NB = Shape<HD>::NB, VN = Shape<HD>::N, BP = Shape<HD>::BP, KW = HD / 8, VU = HD / 4;
    extern __shared__ __align__(16) char smem[];
    const int half = a.rope_dim / 2;
    double2* turn = reinterpret_cast<double2*>(smem);           // [8][half]
    uint8_t* kl = reinterpret_cast<uint8_t*>(turn + 8 * half);  // [heads][8][HD / 2]
    uint8_t* vl = kl + a.heads * 4 * HD;                        // [heads][VN][BP][8][2]
    uint16_t* kdl = reinterpret_cast<uint16_t*>(vl + a.heads * 4 * HD);  // [heads][NB][8]
    uint16_t* vdl = kdl + a.heads * NB * 8;
    float* freq = reinterpret_cast<float*>(vdl + a.heads * NB * 8);  // [half]
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
    if (half) {
        for (int i = threadIdx.x; i < half; i += kThreads) freq[i] = rope_frequency(i, a);
        __syncthreads();
        for (int i = threadIdx.x; i < (j1 - j0) * half; i += kThreads) {
            const int j = j0 + i / half;
            const uint32_t row = row0 + (j - j0);
            const uint32_t pos = a.pos ? a.pos[row] : static_cast<uint32_t>(oct * 8 + j);
            double sn, cs;
            sincos(static_cast<double>(rope_angle(pos, i % half, freq[i % half], a)), &sn, &cs);
            turn[j * half + i % half] = make_double2(cs, sn);
        }
        __syncthreads();
    }
    // Keys and values from the first wave on, queries from the wave after them on: of a
    // single token each wave has one or the other.
    const int l = threadIdx.x & 7, blocks = heads * NB;
    constexpr int R = 4;
    const int per = 2 * blocks, all = store ? (j1 - j0) * per : 0;
    const bool one = j1 - j0 == 1;
    const size_t plane = static_cast<size_t>(s) * a.c.n_kv + h0;
    for (int u0 = threadIdx.x >> 3; u0 < all; u0 += R * (kThreads / 8)) {
        Quad q[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int w = min(u0 + i * (kThreads / 8), all - 1), jj = w / per, u = w - jj * per;
            const bool v = u >= blocks;
            const int hb = v ? u - blocks : u;
            q[i] = load_quad<QUADS>(a.qkv + (row0 + jj) * a.ld + static_cast<size_t>(a.n_heads + h0 + (v ? a.c.n_kv : 0) + hb / NB) * HD,
                             hb % NB * 32 + 4 * l, !v, a);
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            // (the eight lanes of a block leave together, which is all that their exchange needs)
            const int w = u0 + i * (kThreads / 8), jj = w / per, u = w - jj * per, j = j0 + jj;
            if (w >= all) break;
            const bool v = u >= blocks;
            const int hb = v ? u - blocks : u, h = hb / NB, b = hb % NB;
            const f32x4 y = v ? q[i].own : rotate_quad<QUADS>(q[i], 32 * b + 4 * l, a, turn + j * half);
            uint16_t scale;
            uint32_t lev;
            quantise4(y, scale, lev);
            const auto lay_down = [&](uint8_t* to, uint16_t* to_d) {
                if (v) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int n = 2 * l + k;
                        to[(HD >= 64 ? (n * BP + b / 2) * 16 + b % 2 : n % VN * 16 + n / VN) + j * 2] =
                            static_cast<uint8_t>(lev >> (8 * k));
                    }
                } else {
                    *reinterpret_cast<uint16_t*>(to + j * (HD / 2) + ((l >> 1) * NB + b) * 4 + (l & 1) * 2) =
                        static_cast<uint16_t>(lev);
                }
                if (l == 0) to_d[b * 8 + j] = scale;
            };
            if (one) {
                const size_t o = (plane + h) * (a.c.cap / 8) + oct;
                lay_down((v ? a.c.v : a.c.k) + o * (4 * HD), (v ? a.c.vd : a.c.kd) + o * (NB * 8));
            } else {
                lay_down((v ? vl : kl) + h * 4 * HD, (v ? vdl : kdl) + h * NB * 8);
            }
        }
    }
    if (a.q) {
        // four quads a thread on their way at once
        constexpr int PER = HD / 4;
        const int wide = heads * group * PER, all_q = (j1 - j0) * wide, ahead = (all * 8 + 63) / 64 * 64 % kThreads;
        for (int u0 = (threadIdx.x + kThreads - ahead) % kThreads; u0 < all_q; u0 += R * kThreads) {
            Quad q[R];
            int jj[R], u[R];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int v = min(u0 + i * kThreads, all_q - 1);
                jj[i] = v / wide;
                u[i] = v - jj[i] * wide;
                q[i] = load_quad<QUADS>(a.qkv + (row0 + jj[i]) * a.ld + static_cast<size_t>(h0) * group * HD + u[i] / PER * HD,
                                 u[i] % PER * 4, true, a);
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (u0 + i * kThreads >= all_q) continue;
                const f32x4 v = rotate_quad<QUADS>(q[i], u[i] % PER * 4, a, turn + (j0 + jj[i]) * half);
                float* y = a.q + ((row0 + jj[i]) * static_cast<size_t>(a.n_heads) + static_cast<size_t>(h0) * group) * HD + u[i] * 4;
                if constexpr (QUADS) *reinterpret_cast<f32x4*>(y) = v;
                else
#pragma unroll
                    for (int k = 0; k < 4; k++) y[k] = v[k];
            }
        }
    }
    if (!store) return;
    for (int u = threadIdx.x; u < heads * 8; u += kThreads) {
        const int h = u / 8, j = u % 8;
        if (j < j0 || j >= j1) continue;
        const size_t to = (plane + h) * a.c.cap + oct * 8 + j;
        if (a.c.pos) a.c.pos[to] = a.pos ? a.pos[row0 + (j - j0)] : static_cast<uint32_t>(oct * 8 + j);
        if (a.c.weight) a.c.weight[to] = 0.0f;
    }
    if (one) return;
    __syncthreads();
    // keys: words of whole rows
    for (int u = threadIdx.x; u < heads * 8 * KW; u += kThreads) {
        const int h = u / (8 * KW), j = u / KW % 8, w = u % KW;
        if (j >= j0 && j < j1)
            reinterpret_cast<uint32_t*>(a.c.k + ((plane + h) * a.c.cap + oct * 8 + j) * (HD / 2))[w] =
                reinterpret_cast<const uint32_t*>(kl)[u];
    }
    // values and scales: 2-byte units, eight keys side by side, at once where all eight are new
    const bool whole = j0 == 0 && j1 == 8;
    const int rows8 = heads * (VU + 2 * NB);
    for (int u = threadIdx.x; u < rows8 * (whole ? 1 : 8); u += kThreads) {
        const int j = whole ? 0 : u % 8, q = whole ? u : u / 8, h = q / (VU + 2 * NB), w = q % (VU + 2 * NB);
        const size_t o = (plane + h) * (a.c.cap / 8) + oct;
        const uint16_t* from;
        uint16_t* to;
        if (w < VU) {
            from = reinterpret_cast<const uint16_t*>(vl) + (h * VU + w) * 8;
            to = reinterpret_cast<uint16_t*>(a.c.v) + (o * VU + w) * 8;
        } else if (w < VU + NB) {
            from = kdl + (h * NB + w - VU) * 8;
            to = a.c.kd + (o * NB + w - VU) * 8;
        } else {
            from = vdl + (h * NB + w - VU - NB) * 8;
            to = a.c.vd + (o * NB + w - VU - NB) * 8;
        }
        if (whole) *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
        else if (j >= j0 && j < j1) to[j] = from[j];
    }
}

// ---- read back ----------------------------------------------------------------

// Rows first[s] .. + rows - 1 of every head as f32 rows of n_kv * HD, the f32
// cache's layout.  One thread: four channels of a key and of its value, so that
// a wave's stores are whole lines, and past the caches (what is written is larger than
// they are): 8 x 8192 rows of 8 heads of width 128 130 us, 4.7 TB/s, 210 with neither.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_read(Cache c, const uint32_t* __restrict__ first, uint32_t rows,
                                                      float* __restrict__ ko, float* __restrict__ vo) {
    constexpr int NB = Shape<HD>::NB, N = Shape<HD>::N, BP = Shape<HD>::BP, VU = HD / 4, PER = HD / 4;
    const int s = static_cast<int>(blockIdx.y);
    const size_t id = blockIdx.x * static_cast<size_t>(kThreads) + threadIdx.x;
    const size_t head = id / PER;  // (row, kv head)
    if (head >= static_cast<size_t>(rows) * c.n_kv) return;
    const uint32_t t = static_cast<uint32_t>(head / c.n_kv);
    const int h = static_cast<int>(head - static_cast<size_t>(t) * c.n_kv), ch = static_cast<int>(id % PER) * 4;
    const uint64_t key = static_cast<uint64_t>(first ? first[s] : 0) + t;
    const bool ok = key < static_cast<uint64_t>(c.cap);
    const size_t at = (static_cast<size_t>(s) * c.n_kv + h) * c.cap + (ok ? key : 0), oct = at / 8, j = at % 8;
    const int b = ch / 32, g = ch % 32 / 8, n = ch % 32 / 2;
    const uint32_t kw = *reinterpret_cast<const uint16_t*>(c.k + at * (HD / 2) + (g * NB + b) * 4 + ch % 8 / 2);
    const uint8_t* v = c.v + oct * (VU * 16) + j * 2;
    const uint32_t v0 = v[HD >= 64 ? (n * BP + b / 2) * 16 + b % 2 : n % N * 16 + n / N];
    const uint32_t v1 = v[HD >= 64 ? ((n + 1) * BP + b / 2) * 16 + b % 2 : (n + 1) % N * 16 + (n + 1) / N];
    const float kd = ok ? fh_h2f(c.kd[(oct * NB + b) * 8 + j]) : __builtin_nanf("");
    const float vd = ok ? fh_h2f(c.vd[(oct * NB + b) * 8 + j]) : __builtin_nanf("");
    const uint32_t vw = v0 | v1 << 8;
    const size_t to = (static_cast<size_t>(s) * rows * c.n_kv + head) * HD + ch;
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    f32x4u x, y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] = static_cast<float>(static_cast<int>(kw >> (4 * i) & 15) - 8) * kd;
        y[i] = static_cast<float>(static_cast<int>(vw >> (4 * i) & 15) - 8) * vd;
    }
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4u*>(ko + to));
    __builtin_nontemporal_store(y, reinterpret_cast<f32x4u*>(vo + to));
}

// ---- eviction -----------------------------------------------------------------

// A weight as an unsigned number of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t b = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

}  // namespace

namespace fh {
// The sum over a wave's lanes up to each.
__device__ __forceinline__ uint32_t wave_upto(uint32_t u) {
    uint32_t v = u;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t x = __shfl_up(v, m, 64);
        if (static_cast<int>(threadIdx.x & 63) >= m) v += x;
    }
    return v;
}
}  // namespace fh

namespace {

constexpr int kSelect = 1024, kHeld = 16;  // threads, and weights that each keeps in registers

// Which rows of a (sequence, kv head) stay: the last `recent` and the heaviest
// of the others up to `keep`, in order; idx gets their cache rows, *count how
// many.  The lightest weight that stays is found by a radix select of 8-bit digits,
// until what is left of a digit all stays, from registers up to 16384 rows (a bit at a
// time by counting, without atomics, the 32 rounds of barriers cost more: 19 us, and 30
// at 16384 rows).  Row k * 1024 + t is thread t's k-th, so places follow from counts per
// (k, wave).
__global__ void __launch_bounds__(kSelect) k_kv4_select(Cache c, const uint32_t* __restrict__ len, uint32_t max_len,
                                                       uint32_t keep, uint32_t recent, uint32_t* __restrict__ idx,
                                                       uint32_t* __restrict__ counts) {
    constexpr int W = kSelect / 64;
    __shared__ uint32_t hist[256], pick[3], slot[kHeld * W], base;
    const int s = static_cast<int>(blockIdx.x) / c.n_kv;
    const uint32_t n = min(min(len[s], max_len), static_cast<uint32_t>(c.cap));
    uint32_t* to = idx + static_cast<size_t>(blockIdx.x) * keep;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (tid == 0) counts[blockIdx.x] = min(n, keep);
    if (n <= keep) {
        for (uint32_t i = tid; i < n; i += kSelect) to[i] = i;
        return;
    }
    const uint32_t free = n - recent, want = keep - recent;  // `want` of the free rows stay
    for (uint32_t i = tid; i < recent; i += kSelect) to[want + i] = free + i;
    if (want == 0) return;
    const float* w = c.weight + static_cast<size_t>(blockIdx.x) * c.cap;
    uint32_t held[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
        const uint32_t i = k * kSelect + tid;
        held[k] = i < free ? ordered(w[i]) : 0;  // (0 is below every weight's number: -NaN has none of its own)
    }
    // the largest `cut` that at least `want` rows reach, 8 bits at a time
    uint32_t cut = 0, mask = 0, left = want;  // `left` of the rows that agree with `cut` so far
    bool whole = false;                       // all of them: then every row from `cut` up stays
    for (int shift = 24; shift >= 0 && !whole; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kHeld; k++) {
            if (static_cast<uint32_t>(k * kSelect) >= free) continue;
            if (static_cast<uint32_t>(k * kSelect + tid) < free && (held[k] & mask) == cut)
                atomicAdd(&hist[held[k] >> shift & 255], 1u);
        }
        for (uint32_t i = kHeld * kSelect + tid; i < free; i += kSelect) {
            const uint32_t o = ordered(w[i]);
            if ((o & mask) == cut) atomicAdd(&hist[o >> shift & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // from the heaviest digit down: the one at which the count reaches `left`
            uint32_t h[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) sum += h[i] = hist[255 - (lane * 4 + i)];
            uint32_t before = fh::wave_upto(sum) - sum;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (before < left && before + h[i] >= left) {
                    pick[0] = 255 - (lane * 4 + i);
                    pick[1] = left - before;
                    pick[2] = before + h[i] == left;
                }
                before += h[i];
            }
        }
        __syncthreads();
        cut |= pick[0] << shift;
        left = pick[1];
        whole = pick[2] != 0;
        mask |= 255u << shift;
    }
    // rows above `cut` all stay, and the first `left` of those at it
    const uint64_t below = (uint64_t(1) << lane) - 1;
    uint32_t equal = 0, kept = 0;  // before the chunk at hand
    for (uint32_t c0 = 0; c0 < free; c0 += kHeld * kSelect) {
        if (c0) {
#pragma unroll
            for (int k = 0; k < kHeld; k++) {
                const uint32_t i = c0 + k * kSelect + tid;
                held[k] = i < free ? ordered(w[i]) : 0;
            }
        }
        // twice: places among the equals (if some go), then among the rows that stay
        uint32_t stay = 0;
#pragma unroll
        for (int pass = 0; pass < 2; pass++) {
            if (pass == 0 && whole) {
#pragma unroll
                for (int k = 0; k < kHeld; k++)
                    if (c0 + k * kSelect + tid < free && held[k] >= cut) stay |= 1u << k;
                continue;
            }
            uint64_t votes[kHeld];
#pragma unroll
            for (int k = 0; k < kHeld; k++) {
                votes[k] = 0;
                if (c0 + k * kSelect >= free) continue;
                const bool in = c0 + k * kSelect + tid < free;
                votes[k] = __ballot(pass == 0 ? in && held[k] == cut : (stay >> k & 1) != 0);
                if (lane == 0) slot[k * W + wave] = __popcll(votes[k]);
            }
            __syncthreads();
            if (wave == 0) {  // exclusive sums over the 256 counts, four a lane
                uint32_t v[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[i] = sum;
                    sum += c0 + (lane / 4) * kSelect < free ? slot[lane * 4 + i] : 0;  // (k = lane / 4)
                }
                const uint32_t upto = fh::wave_upto(sum);
#pragma unroll
                for (int i = 0; i < 4; i++) slot[lane * 4 + i] = v[i] + upto - sum;
                if (lane == 63) base = upto;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kHeld; k++) {
                if (c0 + k * kSelect >= free) continue;
                const uint32_t place = slot[k * W + wave] + __popcll(votes[k] & below), i = c0 + k * kSelect + tid;
                if (pass == 0) {
                    const bool in = i < free;
                    if (in && (held[k] > cut || (held[k] == cut && equal + place < left))) stay |= 1u << k;
                } else if (stay >> k & 1) {
                    to[kept + place] = i;
                }
            }
            if (pass == 0) equal += base;
            else kept += base;
            __syncthreads();
        }
    }
}

// Moves the rows that stay.  A workgroup: 64 rows of one (sequence, kv head),
// keys in 16-byte pieces of a row, values and scales eight rows' units at once (2-byte
// reads, 16-byte writes): 64 x 8192 rows of width 128 34 us, 4.4 TB/s.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_move(Cache c, Cache d, uint32_t keep, int chunks,
                                                      const uint32_t* __restrict__ idx,
                                                      const uint32_t* __restrict__ counts,
                                                      uint32_t* __restrict__ new_len) {
    constexpr int NB = Shape<HD>::NB, VU = HD / 4, KP = HD / 32;  // KP: 16-byte pieces of a key row
    const int sh = static_cast<int>(blockIdx.x) / chunks, ck = static_cast<int>(blockIdx.x) % chunks;
    const uint32_t n = counts[sh], r0 = static_cast<uint32_t>(ck) * 64;
    if (ck == 0 && threadIdx.x == 0 && sh % c.n_kv == 0) new_len[sh / c.n_kv] = n;
    if (r0 >= n) return;
    __shared__ uint32_t src[64];
    const int rows = static_cast<int>(min(n - r0, 64u));
    if (threadIdx.x < 64) src[threadIdx.x] = idx[static_cast<size_t>(sh) * keep + r0 + min(static_cast<int>(threadIdx.x), rows - 1)];
    __syncthreads();
    const size_t from = static_cast<size_t>(sh) * c.cap, to = static_cast<size_t>(sh) * d.cap;
    for (int u = threadIdx.x; u < rows * KP; u += kThreads)
        reinterpret_cast<u32x4*>(d.k)[(to + r0 + u / KP) * KP + u % KP] =
            reinterpret_cast<const u32x4*>(c.k)[(from + src[u / KP]) * KP + u % KP];
    for (int u = threadIdx.x; u < (VU + 2 * NB) * 8; u += kThreads) {
        const int w = u % (VU + 2 * NB), o = u / (VU + 2 * NB);
        if (o * 8 >= rows) break;
        const uint16_t* sp;
        uint16_t* tp;
        int wide;  // units of an octet
        if (w < VU) {
            sp = reinterpret_cast<const uint16_t*>(c.v) + w * 8;
            tp = reinterpret_cast<uint16_t*>(d.v) + w * 8;
            wide = VU;
        } else {
            const bool k = w < VU + NB;
            const int x = (k ? w - VU : w - VU - NB) * 8;
            sp = (k ? c.kd : c.vd) + x;
            tp = (k ? d.kd : d.vd) + x;
            wide = NB;
        }
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t r = src[o * 8 + j];  // (rows past the end repeat the last)
            v[j] = sp[(from / 8 + r / 8) * (wide * 8) + r % 8];
        }
        tp += (to / 8 + r0 / 8 + o) * (wide * 8);
        if (o * 8 + 8 <= rows) {
            *reinterpret_cast<u32x4*>(tp) = u32x4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (o * 8 + j < rows) tp[j] = static_cast<uint16_t>(v[j]);
        }
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
constexpr size_t kUnits = 1024;
constexpr size_t kPartBytes = kUnits * 16 * (128 + 2) * sizeof(float);

// Over how many workgroups the keys of a unit (16 columns, or eight) are dealt: that power
// of two of which least time is expected.  A wave's tile, or pair of them, takes `step` us
// alone on its SIMD and `crowd` of it with each further wave there, a workgroup two
// steps' time besides, and joining the splits 2.8 us and 2 for every pass of the last
// workgroup but the first.  us measured, by splits of 1 / 2 / 4 / 8 / 16 / 32 (the one
// taken in brackets):
//   14 and 2 heads of width 64, 1 x 511      (6.2)  7.4  7.8  7.5  7.6  8.8
//   14 and 2 heads of width 64, 1 x 4000     19.2  14.2  10.6  8.8  (7.7)  9.0
//   14 and 2 heads of width 64, 64 x <= 1023 (8.1)  9.2  10.2  18.1
//   14 and 2 heads of width 64, 64 x <= 4000 20.0  15.8  (14.4)  21.3
//   12 and 12 heads of width 64, 16 x <= 2999 (16.4)  16.5  19.4
//   32 and 8 heads of width 128, 8 x <= 2000 20.8  16.0  (12.9)  15.0
//   32 and 8 heads of width 128, 8 x <= 32767 269  139  74  (59)  62
// and of single units, by splits of 16 / 32 / 64 / 128 / 256:
//   1 head of width 128, 1 x 32760            23.7  16.1  12.9  (12.4)  15.9
//   5 and 1 heads of width 128, 1 x 32760     24.0  18.4  (18.0)  23.5  37.5
//   8 and 1 heads of width 32, 1 x 262144     47.5  28.0  (19.3)  17.3  21.2
//   16 and 1 heads of width 64, 1 x 65536     27.3  (19.2)  17.8  22.5
size_t attention_splits(size_t units, size_t tiles, size_t cols, size_t width, bool pairs, size_t cus) {
    const double step = pairs ? (width == 32 ? 0.63 : 0.95) : width == 32 ? 0.48 : width == 64 ? 0.66 : 1.03;
    const double crowd = pairs ? 0.75 : 0.85;
    const size_t pass = 8 * (cols > 8 ? 1 : cols > 4 ? 2 : cols > 2 ? 4 : 16 / cols);  // splits that are joined at once
    const size_t round = pairs ? 8 : 4;                                               // tiles that four waves take at once
    size_t best = 1;
    double least = 0;
    for (size_t n = 1; n == 1 || (n <= tiles && n * units <= kUnits); n *= 2) {
        const double there = static_cast<double>((units * n + cus - 1) / cus);
        const double walk = static_cast<double>((tiles + round * n - 1) / (round * n));
        const double t = step * (walk + 2) * std::max(1.0, crowd * there) +
                         (n > 1 ? 2.8 + 2.0 * static_cast<double>((n - 1) / pass) : 0.0);
        if (n == 1 || t < least) {
            best = n;
            least = t;
        }
    }
    return best;
}

template <int HD, bool MODS>
void launch_attention(fh_ctx* ctx, const AttnArgs& a, bool prompt, bool pairs, size_t grid) {
    const dim3 g(static_cast<unsigned>(grid));
    if (prompt) {
        if constexpr (HD >= 64)
            hipLaunchKernelGGL((k_kv4_prompt<HD, MODS>), g, dim3(kThreads), sizeof(Room<HD>), ctx->stream, a);
    } else {
        if constexpr (HD <= 64)
            if (pairs) {
                hipLaunchKernelGGL((k_kv4_attention<HD, MODS, 2>), g, dim3(kThreads), 0, ctx->stream, a);
                return;
            }
        hipLaunchKernelGGL((k_kv4_attention<HD, MODS, 1>), g, dim3(kThreads), 0, ctx->stream, a);
    }
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
    a.octets = static_cast<int>((max_rows + 14) / 8);  // a block of rows touches that many at most
    a.off = off;
    a.len = len;
    a.pos = pos;
    a.rope_dim = static_cast<int>(rope_dim);
    a.neox = rope_type == FH_ROPE_NEOX;
    a.log2_base = std::log2(static_cast<double>(base));
    a.linear = linear;
    a.ff = ff;
    a.q = q;
    // Two kv heads a workgroup (8 x 1000 rows of 32 and 8 heads of width 128: 63 us, by ones 80, by
    // eights 78), single tokens one (64 of 14 and 2 heads of width 64: 5.8 us, by twos 7.0).
    a.heads = static_cast<int>(std::min<size_t>(c.n_kv, max_rows == 1 ? 1 : 2));
    // 16-byte accesses: every four channels from a multiple of 4 are aligned, and so are their partners
    const bool quads = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q)) % 16 == 0 &&
              (rope_type != FH_ROPE_NEOX || rope_dim % 8 == 0) && rope_dim % 4 == 0;
    const size_t lds = 8 * (rope_dim / 2) * sizeof(double2) + rope_dim / 2 * sizeof(float) +
                       a.heads * (8 * c.head_dim + c.head_dim / 32 * 8 * 2 * 2);
    const dim3 grid(static_cast<unsigned>(c.seqs * a.octets), static_cast<unsigned>((c.n_kv + a.heads - 1) / a.heads));
    const auto go = [&](auto width) {
        constexpr int HD = decltype(width)::value;
        if (quads) hipLaunchKernelGGL((k_kv4_append<HD, true>), grid, dim3(kThreads), lds, ctx->stream, a);
        else hipLaunchKernelGGL((k_kv4_append<HD, false>), grid, dim3(kThreads), lds, ctx->stream, a);
    };
    switch (c.head_dim) {
        case 32: go(std::integral_constant<int, 32>{}); break;
        case 64: go(std::integral_constant<int, 64>{}); break;
        default: go(std::integral_constant<int, 128>{}); break;
    }
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
    // Many columns share each key's expansion (128 to a workgroup) where that still fills the
    // GPU twice over, so that one workgroup's barriers hide behind another's work.  us, and by 16
    // columns: 8 x 500 rows of 32 and 8 heads of width 128 (1024 such workgroups) 75, 122; 3 x
    // 1000 (768) 87, 119; 2 x 1000 (512) 80, 81; 1 x 1000 (256) 73, 43; 8 x 1001 rows of 14 and 2
    // heads of width 64 (880) 73, 83; 4 x 1000 (440) 58, 40.  (Width 32 has one form only: a tile of
    // it is half a workgroup's parts.  8 x 500 rows of 32 and 8 heads of it take 45, of width 64 60
    // by 16 columns and 51 shared.)
    const size_t shared = c.seqs * c.n_kv * ((tiles16 + 4 * kPromptTiles - 1) / (4 * kPromptTiles));
    // (and only with three quarters of those columns in use: its cost is a workgroup's.  us, and by
    // 16 columns, 32 sequences of 32 and 8 heads of width 128 behind 1000 keys: 36 rows, 56 % in use,
    // 100, 82; 40, 62 %, 103, 92; 44, 69 %, 104, 99; 48, 75 %, 104, 109; 56, 88 %, 107, 124.  The
    // fewer the keys, the sooner it wins: 40 rows behind none 17, 25.)
    const bool prompt = c.head_dim >= 64 && shared >= 2 * static_cast<size_t>(ctx->num_cus) &&
                        4 * tiles16 * c.seqs * c.n_kv >= 3 * 4 * kPromptTiles * shared;
    // At most eight columns take the keys two tiles at a time.  us, 64 x <= 8000 keys of 12 heads of
    // width 64: 81, and 97 by single tiles; 64 x <= 1023 of 14 and 2 heads 8.1 and 9.4.  At width 128
    // a pair's registers would be spilled: 8 x <= 32767 of 32 and 8 heads 125 and 60.
    const bool pairs = cols <= 8 && c.head_dim <= 64;
    size_t grid = shared;
    if (prompt) {
        a.col_tiles = static_cast<int>((tiles16 + 4 * kPromptTiles - 1) / (4 * kPromptTiles));
        a.splits = 1;
    } else {
        a.col_tiles = static_cast<int>(tiles16);
        const size_t units = c.seqs * c.n_kv * tiles16;
        const size_t splits = attention_splits(units, key_tiles, std::min<size_t>(cols, 16), c.head_dim, pairs,
                                               static_cast<size_t>(ctx->num_cus));
        a.splits = static_cast<int>(splits);
        grid = units * splits;
        if (splits > 1) {
            void* area = nullptr;
            const int rc = fh_kv4_area(ctx, kUnits * sizeof(unsigned) + kPartBytes, &area);
            if (rc) return rc;
            a.counters = static_cast<unsigned*>(area);
            a.part = reinterpret_cast<float*>(a.counters + kUnits);
        }
    }
    if (grid > 0x7FFFFFFF) return fh_fail(ctx, FH_ERR_LIMIT, "fh_kv4_attention: more than 2^31 - 1 workgroups");
    const bool mods = a.softcap > 0.0f || a.slopes;
    switch (c.head_dim) {
        case 32: mods ? launch_attention<32, true>(ctx, a, prompt, pairs, grid) : launch_attention<32, false>(ctx, a, prompt, pairs, grid); break;
        case 64: mods ? launch_attention<64, true>(ctx, a, prompt, pairs, grid) : launch_attention<64, false>(ctx, a, prompt, pairs, grid); break;
        default: mods ? launch_attention<128, true>(ctx, a, prompt, pairs, grid) : launch_attention<128, false>(ctx, a, prompt, pairs, grid); break;
    }
    FH_HIP(ctx, hipGetLastError());
    return FH_OK;
}

template <int HD, bool MODS>
static int launch_weigh(fh_ctx* ctx, AttnArgs& a, size_t tiles16) {
    const size_t heads = static_cast<size_t>(a.c.seqs) * a.c.n_kv, tiles = (a.max_keys + 31) / 32;
    if (tiles16 == 1) {
        // One workgroup for each CU, of four tiles of keys at least, or four, of eight.  us, by this
        // rule and by four of four: 64 x <= 1023 keys of 14 and 2 heads of width 64 5.7, 6.3; 8 x <=
        // 2000 of 32 and 8 heads of width 128 7.3, 8.6; by it and by four of eight: 1 x 8000 4.7,
        // 5.2; 4 x <= 700 of 12 heads of width 64 5.1, 5.5; and by one only: 8 x 16000 23.6, 31.1.
        const size_t cus = static_cast<size_t>(ctx->num_cus);
        const size_t splits = std::max<size_t>(1, std::max(std::min(cus / heads, tiles / 4), std::min(4 * cus / heads, tiles / 8)));
        a.splits = static_cast<int>(splits);
        hipLaunchKernelGGL((k_kv4_weigh_step<HD, MODS>), dim3(static_cast<unsigned>(heads * splits)), dim3(kThreads), 0,
                           ctx->stream, a);
        FH_HIP(ctx, hipGetLastError());
        return FH_OK;
    }
    // The columns are shared out too, over as many workgroups as the GPU holds at once, or, where
    // that is not four times as many, over four times that (us, 1 x 1000 rows of 32 and 8 heads of
    // width 128: 16 parts 34, 31 38; 4 x 2000: two parts 360, eight 345).  Eight tiles of
    // columns a batch, four where that leaves the GPU half empty (8 x 16 rows behind 2000 of
    // 14 and 2 heads of width 64: 14.0 and 12.1; 16 x 100, 192 workgroups by eights: 12.7 and 16.5).
    const size_t cus = static_cast<size_t>(ctx->num_cus), groups = (tiles + 8 * kWeighTiles - 1) / (8 * kWeighTiles);
    const size_t batch = heads * groups * ((tiles16 + 7) / 8) < cus / 2 ? 4 : 8, batches = (tiles16 + batch - 1) / batch;
    const size_t room = cus / (heads * groups);
    const size_t splits = std::max<size_t>(1, std::min(room >= 4 ? room : 4 * cus / (heads * groups), batches));
    a.weigh_cols = static_cast<int>(batch);
    const size_t grid = heads * groups * splits;
    if (grid > 0x7FFFFFFF) return fh_fail(ctx, FH_ERR_LIMIT, "fh_kv4_weigh: more than 2^31 - 1 workgroups");
    a.splits = static_cast<int>(splits);
    if (splits > 1) {
        void* ws = nullptr;
        const int rc = fh_kv4_room(ctx, splits * heads * a.max_keys * sizeof(float), &ws);
        if (rc) return rc;
        a.part = static_cast<float*>(ws);
    }
    hipLaunchKernelGGL((k_kv4_weigh_prompt<HD, MODS>), dim3(static_cast<unsigned>(grid)), dim3(512),
                       sizeof(WeighRoom<HD>), ctx->stream, a);
    FH_HIP(ctx, hipGetLastError());
    if (splits > 1) {
        const size_t n = heads * a.max_keys;
        hipLaunchKernelGGL(k_kv4_add_weights, dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           ctx->stream, a);
        FH_HIP(ctx, hipGetLastError());
    }
    return FH_OK;
}

int fh_launch_kv4_weigh(fh_ctx* ctx, const fh_kv4_cache& c, const float* q, size_t ld, size_t total, size_t n_heads,
                        const uint32_t* off, size_t max_rows, const uint32_t* len, size_t max_keys,
                        const fh_attn_score* sc, const float* lse) {
    AttnArgs a = attn_args(c, q, ld, total, n_heads, off, max_rows, len, max_keys, sc);
    a.lse_in = lse;
    const size_t tiles16 = (max_rows * a.group + 15) / 16;
    const bool mods = a.softcap > 0.0f || a.slopes;
    switch (c.head_dim) {
        case 32: return mods ? launch_weigh<32, true>(ctx, a, tiles16) : launch_weigh<32, false>(ctx, a, tiles16);
        case 64: return mods ? launch_weigh<64, true>(ctx, a, tiles16) : launch_weigh<64, false>(ctx, a, tiles16);
        default: return mods ? launch_weigh<128, true>(ctx, a, tiles16) : launch_weigh<128, false>(ctx, a, tiles16);
    }
}

int fh_launch_kv4_read(fh_ctx* ctx, const fh_kv4_cache& c, const uint32_t* first, size_t rows, float* k, float* v) {
    const Cache d = device_cache(c);
    const size_t n = rows * c.n_kv * (c.head_dim / 4);
    const dim3 grid(static_cast<unsigned>((n + kThreads - 1) / kThreads), static_cast<unsigned>(c.seqs));
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
    const int rc = fh_kv4_room(ctx, idx_bytes + heads * sizeof(uint32_t), &ws);
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
