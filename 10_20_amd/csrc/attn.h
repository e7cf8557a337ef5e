// What the attention kernels over 8-bit and latent caches share: fragments of
// v_mfma_f32_16x16x32_bf16, copies from memory to LDS, and the join of the
// parts that a row's keys were split into.
#pragma once
#include "common.h"

namespace v1 {
namespace attn {

using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x2 = __attribute__((ext_vector_type(2))) int;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// The maximum that is subtracted may lag the true one by 2^kLag: sums are
// rescaled only past that (probabilities keep their relative precision; at 2^6
// every third tile of 64 heads had a head to rescale, 4% of the time).  So sums
// hold up to 2^16 times the number of keys times a value before they are divided
// by their total: values past some 2^100 may overflow where their mean does not.
constexpr float kLag = 16.f;
// The maximum of keys whose scores are all -inf, which give 0 / 0 as the formula
// does, told from that of no keys, -inf, which give zeros.
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

union Frag {
    u32x4 u;
    uint32_t w[4];
    bf16x8 v;
};

__device__ __forceinline__ f32x4 mfma16(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}

// Two fp32 -> two bf16, round to nearest even.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// Two e4m3 codes (the low or the high pair of four) -> two bf16, exact: 4
// significant bits, exponents -9 .. 8.
template <int HIGH>
__device__ __forceinline__ uint32_t codes_pair(uint32_t four) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, HIGH != 0));
}

__device__ __forceinline__ Frag bf16_of_codes(uint32_t lo, uint32_t hi) {
    Frag f;
    f.w[0] = codes_pair<0>(lo);
    f.w[1] = codes_pair<1>(lo);
    f.w[2] = codes_pair<0>(hi);
    f.w[3] = codes_pair<1>(hi);
    return f;
}

// Exponent e of the scale 2^e of codes whose largest magnitude is `amax`
// (finite): the smallest with amax <= 448 * 2^e, at least -126.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four values, scaled, -> e4m3 codes: round to nearest even, past +-448 and
// infinities to +-448, NaN stays NaN.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    auto clip = [](float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(clip(a), clip(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clip(c), clip(d), r, true);
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.f;  // (NaN compares false)
}

// f(Number<0>{}), .., f(Number<N - 1>{})
template <int I>
struct Number {
    static constexpr int value = I;
};

template <int N, int I = 0, class F>
__device__ __forceinline__ void each_of(F&& f) {
    if constexpr (I < N) {
        f(Number<I>{});
        each_of<N, I + 1>(f);
    }
}

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return (uint32_t)reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p);
}

// 16 bytes per lane, memory -> LDS at `lds` + 16 * lane (`lds` the same for the
// wave).  Written as asm so that the compiler puts no waits of its own before
// LDS reads; the caller waits for them (wait_copies, wait_barrier).  There is no output
// register that could be reused while the copy is in flight.
__device__ __forceinline__ void copy_to_lds(const void* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :: "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}

// 4 bytes per lane.
__device__ __forceinline__ void copy4_to_lds(const void* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 :: "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}

// Waits until at most N vector memory operations of this wave are in flight and
// its LDS operations are done.
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Waits until at most N vector memory operations of this wave are in flight
// and its LDS operations are done, then joins the work-group's barrier.
template <int N>
__device__ __forceinline__ void wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The work-group's barrier for LDS data alone: copies stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Whether one launch holds so many work-groups (fewer than 2^32 work-items a dimension).
inline bool launchable(int64_t groups, int threads) { return groups < (1ll << 32) / threads; }

// ------------------------------------------------ parts of a row's keys
// A row's keys, in tiles of 64, are split over several work-groups where the
// rows alone would not fill the GPU.  Each part leaves its unnormalised sums
// with their maximum (base 2) and total in a workspace, and join_kernel adds
// them.  Two rules, both functions of the call's shapes and lengths alone:
//   chunk > 0  every row in the same number of parts (rows of one capacity);
//   chunk == 0 rows of different lengths (`lens` on the device, at most
//              kPlanRows of them): the smallest of nine sizes of a part, from
//              sum(tiles) / slots to sum(tiles) / target, with no more than
//              `slots` parts, else the last (at most target + rows parts), found
//              by every work-group from the lengths.  Where the rows alone are
//              `slots` or more, or past kPlanRows, the first rule holds, one part a
//              row, and the longest row is a work-group's: contexts of 4096 to
//              131072, us on both sides of that: 127 and 128 rows of 128 heads 2330,
//              4240; 255 and 256 of 16 1600, 2760; 8-bit, 255 and 256 of 8 KV heads
//              4090, 6130, 256 and 257 of 4 1540, 4400.  By the capacity instead below it, 7 rows
//              of 64 heads and up to 60000 latent rows take 69 us (58 so), 40 rows of
//              up to 30000 171 (89), 48 contexts of 4 KV heads in 8 bits 337 (202).
//              Parts go to the XCDs in turn, since their number is known there alone:
//              a range of the most there could be for each XCD left the last ones
//              without work (200 rows of 16 heads, up to 8000 latent rows: 157 us, 102
//              so, and 98 with as many parts as run at once).
constexpr int kTileKeys = 64;
constexpr int kPlanRows = 256;
constexpr int32_t kMostKeys = INT32_MAX - 32 * kTileKeys;  // (positions of the tiles asked for ahead stay below 2^31)

struct Plan {
    const int32_t* lens;  // NULL: `keys` keys in every row
    int32_t rows, keys, chunk, target, slots;
};

struct Item {
    int32_t row, keys;           // keys: of the row
    int32_t first, tiles, parts; // tiles [first, first + tiles) of the row; parts of the row
    int32_t part;
};

__device__ __forceinline__ int32_t tiles_of(int32_t keys) { return (keys + kTileKeys - 1) / kTileKeys; }
__device__ __forceinline__ int32_t keys_of(const Plan& p, int32_t row) {
    return p.lens ? min(max(p.lens[row], 0), p.keys) : p.keys;
}

__device__ __forceinline__ void cut(Item& it) {
    const int32_t tiles = tiles_of(it.keys), each = (tiles + it.parts - 1) / it.parts;
    it.first = min(it.part * each, tiles);
    it.tiles = min(each, tiles - it.first);
}

// The planned parts of up to kPlanRows rows, four rows a lane (row 4 lane + i);
// returns the number of parts before the lane's first row.
__device__ __forceinline__ int32_t plan_parts(const Plan& p, int32_t (&keys)[4], int32_t (&parts)[4]) {
    const int32_t lane = (int32_t)threadIdx.x % kWave;
    int32_t tiles = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t r = 4 * lane + i;
        keys[i] = min(max(p.lens[min(r, p.rows - 1)], 0), p.keys);
        if (r >= p.rows) keys[i] = 0;
        tiles += tiles_of(keys[i]);
    }
    const int32_t all = __shfl((int32_t)wave_inclusive_sum((uint32_t)tiles), kWave - 1, kWave);
    const int32_t most = max(1, (all + p.target - 1) / p.target), least = max(1, (all + p.slots - 1) / p.slots);
    const int32_t step = max(1, (most - least + 7) / 8);
    int32_t mine, upto, lo = 0, hi = 8;
    for (;;) {
        const int32_t at = (lo + hi) / 2, chunk = at == 8 ? most : min(least + at * step, most);
        const float inv = 1.0f / (float)chunk;
        mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // ceil(tiles / chunk): the product is off by less than one (tiles stay below 2^26, parts below 2^22)
            const int32_t n = tiles_of(keys[i]);
            int32_t q = (int32_t)((float)n * inv);
            q -= q * chunk > n;
            q += q * chunk < n;
            q += q * chunk < n;
            parts[i] = 4 * lane + i < p.rows ? max(1, q) : 0;
            mine += parts[i];
        }
        upto = (int32_t)wave_inclusive_sum((uint32_t)mine);
        if (lo == hi) break;
        if (__shfl(upto, kWave - 1, kWave) <= p.slots) hi = at;
        else lo = at + 1;
    }
    return upto - mine;
}

// Work item `index`; false: there is none.  (Every wave finds it by itself.)
__device__ __forceinline__ bool find_item(const Plan& p, int32_t index, Item& it) {
    if (p.chunk > 0) {
        it.parts = max(1, (tiles_of(p.keys) + p.chunk - 1) / p.chunk);
        it.row = index / it.parts;
        it.part = index - it.row * it.parts;
        if (it.row >= p.rows) return false;
        it.keys = keys_of(p, it.row);
    } else {
        int32_t keys[4], parts[4];
        const int32_t lane = (int32_t)threadIdx.x % kWave;
        int32_t at = plan_parts(p, keys, parts);
        int32_t row = -1, part = 0, n = 0, of = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (index >= at && index < at + parts[i]) {
                row = 4 * lane + i;
                part = index - at;
                n = keys[i];
                of = parts[i];
            }
            at += parts[i];
        }
        const uint64_t who = __ballot(row >= 0);
        if (who == 0) return false;
        const int src = __ffsll((unsigned long long)who) - 1;
        it.row = __shfl(row, src, kWave);
        it.part = __shfl(part, src, kWave);
        it.keys = __shfl(n, src, kWave);
        it.parts = __shfl(of, src, kWave);
    }
    it.row = __builtin_amdgcn_readfirstlane(it.row);
    it.part = __builtin_amdgcn_readfirstlane(it.part);
    it.keys = __builtin_amdgcn_readfirstlane(it.keys);
    it.parts = __builtin_amdgcn_readfirstlane(it.parts);
    cut(it);
    return true;
}

// Whether the device's lengths may decide: few rows, and their tiles can be added in 32 bits.
inline bool planned(int64_t rows, int64_t tiles) { return rows <= kPlanRows && rows * tiles < 1ll << 30; }

// Most work items that a call can have.
inline int64_t items_at_most(const Plan& p) {
    if (p.chunk > 0) return (int64_t)p.rows * std::max<int64_t>(1, cdiv(cdiv(p.keys, kTileKeys), p.chunk));
    return std::max<int64_t>(p.slots, (int64_t)p.rows + p.target);
}

// Tiles of a part of rows of `tiles` tiles: the number of parts whose work-groups
// end first, `slots` of them running at a time, where a part costs `start` tiles'
// time beside its own and each part of several another `leave` (its sums, written
// and joined).  128 rows of 16 heads over 2048 of two million latent rows take 43 us in
// the two parts a row that this finds, 51 in one, 52 in four, 69 in eight.
inline int32_t chunk_for(int64_t rows, int64_t tiles, int64_t slots, int64_t start, int64_t leave) {
    int64_t best = tiles, least = cdiv(rows, slots) * (tiles + start);
    for (int64_t parts = 2; parts <= tiles && rows * (parts - 1) < slots; ++parts) {
        const int64_t chunk = cdiv(tiles, parts), cost = cdiv(rows * cdiv(tiles, chunk), slots) * (chunk + start + leave);
        if (cost < least) least = cost, best = chunk;
    }
    return (int32_t)std::max<int64_t>(1, best);
}

// Workspace: sums [items][heads][dims], maxima and totals [items][heads], and of a
// planned call each row's first item and number of parts, written with its first part.
struct Parts {
    float* sums;
    f32x2* stats;
    i32x2* of_row;
};

inline int64_t parts_bytes(const Plan& plan, int32_t heads, int32_t dims) {
    return items_at_most(plan) * heads * (dims + 2) * (int64_t)sizeof(float) + (plan.chunk > 0 ? 0 : plan.rows * (int64_t)sizeof(i32x2));
}

inline Parts parts_at(void* ws, const Plan& plan, int32_t heads, int32_t dims) {
    const int64_t items = items_at_most(plan);
    float* sums = static_cast<float*>(ws);
    f32x2* stats = reinterpret_cast<f32x2*>(sums + items * heads * dims);
    return {sums, stats, reinterpret_cast<i32x2*>(stats + items * heads)};
}

struct JoinParams {
    Plan plan;
    Parts parts;
    uint16_t* out;
    int64_t o_row, o_head;
    float* lse;
    int32_t heads;
    // not NULL: only rows cu[b] .. min(cu[b + 1], cu[b] + most) - 1 of the output have parts (the
    // ends taken within [0, tokens]), the others are left as they are.  The plan's rows are those
    // of the output, or (by_sequence) `most` for each of the sequences.
    const int32_t* cu;
    int32_t tokens, batch, most;
    bool by_sequence;
};

// The output's row of a row of the plan; -1: it has no parts (asked by a whole work-group).
__device__ __forceinline__ int32_t joined_row(const JoinParams& p, int32_t row) {
    if (!p.cu) return row;
    auto begin = [&](int32_t b) __attribute__((always_inline)) { return min(max(p.cu[b], 0), p.tokens); };
    if (p.by_sequence) {
        const int32_t b = row / p.most, i = row - b * p.most, lo = begin(b);
        return i < begin(b + 1) - lo ? lo + i : -1;
    }
    int mine = 0;
    for (int32_t b = (int32_t)threadIdx.x; b < p.batch; b += 256) {
        const int32_t lo = begin(b), hi = begin(b + 1);
        mine |= row >= lo && row < hi && row - lo < p.most;
    }
    return __syncthreads_or(mine) ? row : -1;
}

__device__ __forceinline__ void write_joined(const JoinParams& p, int32_t row, int32_t h, int32_t at4, f32x4 o, float top, float total) {
    const bool none = top == -__builtin_inff() && total == 0.f;  // no key attended
    const float inv = none ? 0.f : 1.0f / total;
    *reinterpret_cast<u32x2*>(p.out + row * p.o_row + h * p.o_head + 4 * at4) =
        none ? u32x2{0, 0} : u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    if (p.lse && at4 == 0)
        p.lse[(int64_t)row * p.heads + h] = none ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

constexpr int kFewParts = 8;

// One work-group per (row, head): D / 4 threads add four dims of every (1024 / D)-th
// part, scaled to the largest of the parts' maxima, and the groups meet in LDS (one
// thread per two dims over all parts took 30 us for 37 parts of 7 rows x 64 heads x
// 512: a chain of memory latencies; this takes 9, 34 MB at 3.7 TB/s).  Rows of one
// part have been written.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(JoinParams p) {
    constexpr int T = D / 4, G = 256 / T;
    __shared__ f32x4 sums[G][T];
    __shared__ float totals[G];
    const int32_t row = (int32_t)blockIdx.x, h = (int32_t)blockIdx.y, lane = (int32_t)threadIdx.x % kWave;
    const int32_t group = (int32_t)threadIdx.x / T, at4 = (int32_t)threadIdx.x % T;
    const int32_t to = joined_row(p, row);
    if (to < 0) return;
    int32_t parts, first;
    if (p.plan.chunk > 0) {
        parts = (tiles_of(p.plan.keys) + p.plan.chunk - 1) / p.plan.chunk;
        first = row * parts;
    } else {
        const i32x2 of = p.parts.of_row[row];
        first = of[0], parts = of[1];
    }
    if (parts <= 1) return;
    float top = -__builtin_inff(), total = 0.f;
    for (int32_t i = lane; i < parts; i += kWave) top = fmaxf(top, p.parts.stats[(int64_t)(first + i) * p.heads + h][0]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    const float sub = top == -__builtin_inff() ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int32_t i = group; i < parts; i += G) {
        const int64_t at = (int64_t)(first + i) * p.heads + h;
        const f32x2 st = p.parts.stats[at];
        const f32x4 x = *reinterpret_cast<const f32x4*>(p.parts.sums + at * D + 4 * at4);
        const float f = __builtin_amdgcn_exp2f(st[0] - sub);
        total = fmaf(f, st[1], total);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(f, x[k], o[k]);
    }
    sums[group][at4] = o;
    if (at4 == 0) totals[group] = total;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
        o += sums[k][at4];
        total += totals[k];
    }
    write_joined(p, to, h, at4, o, top, total);
}

// The same for rows of a few parts, known on the host: D / 4 threads for each (row,
// head), several of them a work-group.  (1024 rows of 16 heads x 128, four parts: 22 us
// a work-group each, 8 so.)
template <int D>
__global__ __launch_bounds__(256) void join_few_kernel(JoinParams p) {
    constexpr int T = D / 4, G = 256 / T;
    const int32_t row = (int32_t)blockIdx.x, h = (int32_t)blockIdx.y * G + (int32_t)threadIdx.x / T, at4 = (int32_t)threadIdx.x % T;
    const int32_t to = joined_row(p, row);
    if (to < 0 || h >= p.heads) return;
    const int32_t parts = (tiles_of(p.plan.keys) + p.plan.chunk - 1) / p.plan.chunk;
    const int64_t first = (int64_t)row * parts * p.heads + h;
    f32x2 st[kFewParts];
    f32x4 x[kFewParts];
    float top = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int i = 0; i < kFewParts; ++i) {
        const int64_t at = first + (int64_t)min(i, parts - 1) * p.heads;
        st[i] = p.parts.stats[at];
        x[i] = *reinterpret_cast<const f32x4*>(p.parts.sums + at * D + 4 * at4);
        top = fmaxf(top, st[i][0]);
    }
    const float sub = top == -__builtin_inff() ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kFewParts; ++i) {
        if (i >= parts) break;
        const float f = __builtin_amdgcn_exp2f(st[i][0] - sub);
        total = fmaf(f, st[i][1], total);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(f, x[i][k], o[k]);
    }
    write_joined(p, to, h, at4, o, top, total);
}

template <int D>
int launch_join(const JoinParams& p, hipStream_t st, const char* what) {
    const int64_t parts = p.plan.chunk > 0 ? cdiv(cdiv(p.plan.keys, kTileKeys), p.plan.chunk) : kPlanRows;
    constexpr int G = 256 / (D / 4);
    if (parts <= kFewParts)
        hipLaunchKernelGGL(join_few_kernel<D>, dim3((uint32_t)p.plan.rows, (uint32_t)cdiv(p.heads, G)), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL(join_kernel<D>, dim3((uint32_t)p.plan.rows, (uint32_t)p.heads), dim3(256), 0, st, p);
    return V1_LAUNCHED(what);
}

}  // namespace attn
}  // namespace v1
