// What the attention kernels over K / V pages of 16-bit numbers share: which keys a
// query sees, and the scores' functions.
#pragma once
#include "paged.h"

namespace v1 {
namespace paged {

// The subtracted maximum, and how far above it a score may lie (base 2): bf16 holds
// every probability up to 2^kLag.  fp16 holds numbers from 2^-24 to 65504, so its
// probabilities are made 2^7 larger than the maximum's 1 and may grow to 2^15: a key
// 2^-31 of the largest still counts (2^-24 would lose a million keys of 2^-25 each).
template <class T>
struct Range;
template <>
struct Range<__bf16> {
    static constexpr float head = 0.f, most = kLag;
};
template <>
struct Range<_Float16> {
    static constexpr float head = 7.f, most = 15.f;
};

template <class T>
__device__ __forceinline__ f32x4 mfma16(const Frag& a, const Frag& b, f32x4 c) {
    if constexpr (__is_same(T, __bf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
    } else {
        using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
    }
}

// tanh(t) / t in t^2 for |t| up to 0.16, 0.33 and 0.75, and the same polynomials of
// cap log2(e) tanh(d scale / cap) / d in d^2 for |d| up to so much.  The fits are off by 3e-8
// of the value at most; they are held in 64 bits, so that a coefficient is rounded once,
// with the scale and the cap in it (by 1e-7 of the value then).
constexpr double kCapLeast[3] = {0.9999999721658054, -0.3333137411469761, 0.1312851958668552};
constexpr double kCapNear[4] = {0.9999999780542091, -0.3333268647142513, 0.1330338186573907, -0.04948183016008989};
constexpr double kCapFar[6] = {0.9999999710131235, -0.33332958872695295, 0.13325405922016131, -0.053344425407917576,
                               0.019582898606222813, -0.0047162504597644895};
constexpr float kCapLeastMost = 0.16f, kCapNearMost = 0.33f, kCapFarMost = 0.75f;
struct Cap {
    float least[3], near[4], far[6];
    float least_most, near_most, far_most;
};

inline Cap cap_of(float scale, float softcap) {
    Cap c{};
    if (softcap <= 0.f) return c;
    const double in = (double)scale / softcap;
    double by = scale * 1.4426950408889634;  // (log2(e))
    for (int i = 0; i < 6; ++i, by *= in * in) {
        if (i < 3) c.least[i] = (float)(kCapLeast[i] * by);
        if (i < 4) c.near[i] = (float)(kCapNear[i] * by);
        c.far[i] = (float)(kCapFar[i] * by);
    }
    // (a cap so far from the scale that the coefficients would not be normal numbers: no polynomial)
    const bool normal = in >= 0x1p-12 && in <= 0x1p12;
    c.least_most = normal ? (float)(kCapLeastMost / in) : -1.f;
    c.near_most = normal ? (float)(kCapNearMost / in) : -1.f, c.far_most = normal ? (float)(kCapFarMost / in) : -1.f;
    return c;
}

// What a score takes: nothing, a cap, a distance, or both.
constexpr int kPlain = 0, kCapped = 1, kBiased = 2, kBoth = 3;

struct AttendParams {
    const uint16_t* q;
    int64_t q_token, q_head;
    const uint16_t* pool[2];
    int64_t page[2], token[2], head[2];  // strides, numbers
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    const int32_t* cu;        // NULL: one query for each request
    const int32_t* prefix;    // of a request; NULL: 0
    const int32_t* document;  // of a token; NULL: 0
    const int32_t* parents;   // of a token, in its request: a tree; NULL: a sequence
    const float* slopes;      // of a query head; NULL: 0
    int32_t table_len, tokens, requests, max_q, kv_heads, group;
    uint32_t group_magic;
    int32_t window;           // 0: none
    float scale2;             // scores times log2(e)
    float cap_in, cap2;       // scale / cap, cap log2(e); 0: no cap
    Cap cap;
    uint16_t* out;
    int64_t o_token, o_head;
    float* lse;
    Plan plan;                // of the requests, by their keys or those that a window leaves (a prefix is not counted)
    int32_t blocks;           // of a request's columns
    // few queries: together: KV heads of a work-group, spread: work-groups of an XCD;
    // blocks: units (items or slots, times KV heads) and those that an XCD takes together
    int32_t spread, together, units, xcds;
    int32_t slots;            // of columns' blocks of all requests; 0: `blocks` of every request
    Parts parts;
};

// ------------------------------------------------------------ what a query sees
// Queries of a request and the heads of one KV head make its columns: column m is
// query m / group, head m % group.
struct Request {
    int32_t q_lo, nq;     // its first query, and how many there are (max_q at most)
    int32_t len, before;  // its keys, and those before its first query
    int32_t pre;          // keys that every query sees
};

__device__ __forceinline__ Request request_at(const AttendParams& p, int32_t r) {
    Request w;
    int32_t n = 1;
    w.q_lo = r;
    if (p.cu) {
        w.q_lo = min(max(p.cu[r], 0), p.tokens);
        n = min(max(p.cu[r + 1], w.q_lo), p.tokens) - w.q_lo;
    }
    w.len = min(max(p.lens[r], 0), p.table_len * kTileKeys);
    w.before = w.len - n;
    w.nq = min(n, p.max_q);
    w.pre = p.prefix ? min(max(p.prefix[r], 0), w.len) : 0;
    w.q_lo = __builtin_amdgcn_readfirstlane(w.q_lo), w.nq = __builtin_amdgcn_readfirstlane(w.nq);
    w.len = __builtin_amdgcn_readfirstlane(w.len), w.before = __builtin_amdgcn_readfirstlane(w.before);
    w.pre = __builtin_amdgcn_readfirstlane(w.pre);
    return w;
}

// Drafted tokens of a request: which of them each one sees, itself and its ancestors
// (bit j of 256), and its depth.  A parent lies before its child; other numbers are no
// parent, so every path ends.
constexpr int kMostDrafts = 256;
struct Tree {
    uint64_t sees[kMostDrafts][kMostDrafts / 64];
    int32_t depth[kMostDrafts];
    int32_t parent[kMostDrafts];
};

// (All of the work-group's threads; ends behind a barrier.)
__device__ __forceinline__ void find_tree(const AttendParams& p, const Request& w, Tree& tree) {
    for (int32_t i = (int32_t)threadIdx.x; i < w.nq; i += (int32_t)blockDim.x) tree.parent[i] = p.parents[w.q_lo + i];
    __syncthreads();
    for (int32_t i = (int32_t)threadIdx.x; i < w.nq; i += (int32_t)blockDim.x) {
        uint64_t sees[kMostDrafts / 64];
#pragma unroll
        for (int k = 0; k < kMostDrafts / 64; ++k) sees[k] = i / 64 == k ? 1ull << (i % 64) : 0;
        int32_t depth = 0;
        for (int32_t at = i;;) {
            const int32_t up = tree.parent[at];
            if (up < 0 || up >= at) break;
            at = up;
            ++depth;
#pragma unroll
            for (int k = 0; k < kMostDrafts / 64; ++k) sees[k] |= at / 64 == k ? 1ull << (at % 64) : 0;
        }
#pragma unroll
        for (int k = 0; k < kMostDrafts / 64; ++k) tree.sees[i][k] = sees[k];
        tree.depth[i] = depth;
    }
    __syncthreads();
}

// Bits of 256 from number `from` on.
__device__ __forceinline__ uint64_t bits_from(const uint64_t* words, int32_t from) {
    if (from <= -64 || from >= kMostDrafts) return 0;
    if (from < 0) return words[0] << -from;
    const int32_t at = from / 64, by = from % 64;
    const uint64_t lo = words[at] >> by, hi = by && at + 1 < kMostDrafts / 64 ? words[at + 1] << (64 - by) : 0;
    return lo | hi;
}

// Bits a - k0 .. b - k0 - 1 of 64.
__device__ __forceinline__ uint64_t bits_between(int32_t a, int32_t b, int32_t k0) {
    auto below = [&](int32_t x) __attribute__((always_inline)) -> uint64_t {
        const int32_t n = min(max(x - k0, 0), 64);
        return n == 64 ? ~0ull : (1ull << n) - 1;
    };
    return below(b) & ~below(a);
}

// What a column sees: the prefix, keys lo .. hi - 1, and of a tree its own drafts.
struct Column {
    int32_t query, head;  // within the request, within the KV head
    int32_t position;     // of the query
    int32_t lo, hi;
};

// Column x of the block whose first column is m0.  Columns past the last see nothing
// and are query 0 (whose numbers may be read).
__device__ __forceinline__ Column column_at(const AttendParams& p, const Request& w, const Tree& tree, int32_t m0, int32_t x) {
    Column c;
    const int32_t i0 = m0 / p.group, y = m0 - i0 * p.group + x;
    const int32_t d = p.group == 1 ? y : (int32_t)small_div((uint32_t)y, p.group_magic);
    c.query = i0 + d, c.head = y - d * p.group;
    const bool there = c.query < w.nq;
    if (!there) c.query = c.head = 0;
    c.position = w.before + (p.parents ? tree.depth[c.query] : c.query);
    c.hi = there ? min(max(p.parents ? w.before : c.position + 1, 0), w.len) : 0;
    c.lo = p.window > 0 ? max(c.position - p.window + 1, 0) : 0;
    if (p.document && there) c.lo = max(c.lo, p.document[w.q_lo + c.query]);
    c.lo = min(c.lo, c.hi);
    return c;
}

__device__ __forceinline__ uint64_t column_sees(const AttendParams& p, const Request& w, const Tree& tree, const Column& c, int32_t k0) {
    uint64_t bits = bits_between(c.lo, c.hi, k0) | bits_between(0, w.pre, k0);
    if (p.parents && k0 + kTileKeys > w.before) bits |= bits_from(tree.sees[c.query], k0 - w.before);
    return bits;
}

// The tiles that some column of a block sees: those of the prefix, then from the
// first key on.  least_lo .. most_hi: over the block's columns.
struct Tiles {
    int32_t pre, shift, count;
    __device__ __forceinline__ int32_t at(int32_t t) const { return t < pre ? t : t + shift; }
};

__device__ __forceinline__ Tiles tiles_seen(const AttendParams& p, const Request& w, int32_t least_lo, int32_t most_hi) {
    Tiles t;
    const int32_t end = tiles_of(p.parents ? w.len : most_hi);
    t.pre = tiles_of(w.pre);
    const int32_t begin = max(t.pre, least_lo / kTileKeys);
    t.shift = begin - t.pre;
    t.count = t.pre + max(0, end - begin);
    return t;
}

__device__ __forceinline__ int32_t wave_min(int32_t x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
    return __builtin_amdgcn_readfirstlane(x);
}

// Bounds of what the columns of lanes 0 .. n - 1 see.  They ascend with the columns,
// unless documents or depths decide.
struct Bounds {
    int32_t least_lo, most_lo, least_hi, most_hi;
};

__device__ __forceinline__ Bounds bounds_of(const AttendParams& p, const Column& c, int32_t lane, int32_t n) {
    if (n <= 0) return {INT32_MAX, 0, INT32_MAX, 0};
    const int32_t last = min(n, kWave) - 1;
    Bounds b;
    b.least_hi = __builtin_amdgcn_readlane(c.hi, 0), b.most_hi = __builtin_amdgcn_readlane(c.hi, last);
    if (p.document || (p.parents && p.window > 0)) {
        b.least_lo = wave_min(lane <= last ? c.lo : INT32_MAX);
        b.most_lo = -wave_min(lane <= last ? -c.lo : 0);
    } else {
        b.least_lo = __builtin_amdgcn_readlane(c.lo, 0), b.most_lo = __builtin_amdgcn_readlane(c.lo, last);
    }
    return b;
}

// All bits of a register where the bit of a key among 64 is set.
__device__ __forceinline__ uint32_t mask_of(uint64_t seen, int key) {
    return (uint32_t)__builtin_amdgcn_sbfe((int)(uint32_t)(key < 32 ? seen : seen >> 32), key & 31, 1);
}
__device__ __forceinline__ float if_seen(uint32_t mask, float x) { return __uint_as_float(mask & __float_as_uint(x)); }
__device__ __forceinline__ float if_seen_or_least(uint32_t mask, float x) {
    return __uint_as_float((mask & __float_as_uint(x)) | (~mask & 0xff800000u));
}

// ------------------------------------------------------------------ capped scores
// cap tanh(x / cap), base 2, of a product d = q . k, t = d scale / cap: past |t| = 0.75
// cap (1 - 2 / (e^2t + 1)), below it t G(t^2) with a polynomial G fitted to tanh(t) / t, its
// coefficients in fp32 (off by 7e-8 of the value, a step of fp32, beside the roundings of its
// evaluation; the other form there is off by as much of the cap, many times a small value).
__device__ __forceinline__ float capped(float t, float cap2) {
    const float z = t * t;
    float g = (float)kCapFar[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) g = fmaf(g, z, (float)kCapFar[i]);
    const float e = __builtin_amdgcn_exp2f(2.f * kLog2e * t);
    const float past = fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(e + 1.f), cap2);
    return fabsf(t) <= kCapFarMost ? t * cap2 * g : past;
}

// capped(d scale / cap) - sub of a tile's scores: where all of them are small, as those of
// a model trained with a cap far above them are, by the shortest of three polynomials in
// d^2, whose coefficients have the scale and the cap in them: four operations a score
// where `capped` takes fifteen and two of the quarter-rate ones.
// `far`: the largest |d| of the lane's; each(f): d := f(d) for all of them.
template <class Each>
__device__ __forceinline__ void cap_scores(const Cap& cap, float cap_in, float cap2, float far, Each each) {
    if (__ballot(far > cap.least_most) == 0) {
        each([&](float d, float sub) __attribute__((always_inline)) {
            const float z = d * d;
            return fmaf(d, fmaf(fmaf(cap.least[2], z, cap.least[1]), z, cap.least[0]), -sub);
        });
    } else if (__ballot(far > cap.near_most) == 0) {
        each([&](float d, float sub) __attribute__((always_inline)) {
            const float z = d * d;
            return fmaf(d, fmaf(fmaf(fmaf(cap.near[3], z, cap.near[2]), z, cap.near[1]), z, cap.near[0]), -sub);
        });
    } else if (__ballot(far > cap.far_most) == 0) {
        each([&](float d, float sub) __attribute__((always_inline)) {
            const float z = d * d;
            float g = fmaf(cap.far[5], z, cap.far[4]);
#pragma unroll
            for (int i = 3; i >= 0; --i) g = fmaf(g, z, cap.far[i]);
            return fmaf(d, g, -sub);
        });
    } else {
        each([&](float d, float sub) __attribute__((always_inline)) { return capped(d * cap_in, cap2) - sub; });
    }
}

// ----------------------------------------------- infinite and NaN values that are masked
// Pairs of numbers of T without their infinities and NaN (zeros there), and with 1.0
// where the number is +inf or NaN, or -inf or NaN.
template <class T>
__device__ __forceinline__ void split_odd(uint32_t w, uint32_t& plain, uint32_t& pos, uint32_t& neg) {
    constexpr uint32_t inf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u, one = __is_same(T, __bf16) ? 0x3f80u : 0x3c00u;
    plain = pos = neg = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t x = (w >> (16 * half)) & 0xffffu;
        const bool odd = (x & inf) == inf, nan = odd && (x & 0x7fffu) != inf;
        plain |= (odd ? 0u : x) << (16 * half);
        pos |= (odd && (nan || x == inf) ? one : 0u) << (16 * half);
        neg |= (odd && (nan || x == (inf | 0x8000u)) ? one : 0u) << (16 * half);
    }
}

template <class T>
constexpr uint32_t kOne = __is_same(T, __bf16) ? 0x3f80u : 0x3c00u;

// Columns of a work-group for many queries: 256, or 128 for work that leaves CUs idle.
constexpr int kBlockColumns = 256, kSmallBlockColumns = 128;

// The launch of paged_blocks.hip.
int launch_blocks(bool fp16, int columns, int mode, const AttendParams& p, int64_t groups, hipStream_t st);

}  // namespace paged
}  // namespace v1
