// Attention of many queries of each request over K / V pages of 16-bit numbers: the
// sums of paged_rows.hip, with the tiles of keys shared by the waves of a work-group.
//
// A work-group takes 256 columns (queries times the heads of a KV head, so that heads
// that share keys share their tiles too) or 128, a wave 32 of them, as columns of
// v_mfma_f32_32x32x16:
//   scores  S^T = K Q^T, a page of 64 keys at a time from LDS;
//   output  O^T = V^T P^T: a lane's scores are already the probabilities of its B
//           fragment (the key order inside 16 keys is chosen so), rounded to the pages'
//           type once, half a step of each, as the output is (1.3-1.4 times the error of a
//           rounded exact result; a second number for the rest would be 16 products
//           more beside a tile's 32); values come transposed from LDS.
// Scores, maxima and sums are fp32, exponentials base 2.  Rows are laid with their
// 16-byte chunks XORed by the row so that the fragments' reads meet different banks.
// Tiles are those that some column of the block sees: the prefix's pages, then from the
// first key of the window or document on.
//
// Bound by vector issue where scores are capped, by products and their fragments else:
// 4096 queries of 32 heads, 8 KV heads, over 32768 keys, us (TFLOP/s):
//   plain 1813-1900 (1137-1085; an 8192^3 library product 1404 on such a card), a cap of 50
//   2148-2230, distances 1887-2050, both 2470-2570, a cap of 2 (scores past it) 3590.
//   Matrix units are busy 40% of the time and vector units 58% when capped; without
//   probabilities a copy takes 1614, without products 1251 plain and 1761 capped (with the polynomial of three steps).
// On the way there (capped): fragments' reads left to the compiler, which waits for each
// one, 2657; copies whose addresses are made between the products 2700; capped scores by
// one polynomial of degree 5 2690, by the shorter where they are small 2394, and maxima
// looked for only where the largest magnitude may pass the subtracted one 2205; by a
// still shorter one below 0.16 of the cap 2148.  Keys from the last one back where
// distances count, so that the first maximum stays: 2350 -> 2050.
#include "paged_attend.h"

namespace v1 {
namespace {

using namespace paged;

constexpr int kRows = 32;  // columns of a wave

using f32x16 = __attribute__((ext_vector_type(16))) float;
using i16x4 = __attribute__((ext_vector_type(4))) short;

struct PageTile {
    uint8_t key[kTileKeys][2 * kDim];
    uint8_t value[kTileKeys][2 * kDim];
};

// Work-groups of WAVES waves: eight, which take all of a CU's LDS for four tiles, or
// four, two work-groups a CU with two tiles each.
template <int WAVES>
struct BlocksLds {
    PageTile tile[WAVES / 2];
    Tree tree;
    int32_t lo[WAVES], hi[WAVES];
};

template <class T>
__device__ __forceinline__ f32x16 mfma32(const Frag& a, const Frag& b, f32x16 c) {
    if constexpr (__is_same(T, __bf16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
    } else {
        using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
    }
}

// A fragment of V^T, rows 32 d .., of 16 keys 16 kk ..: lanes 4r .. 4r + 3 of a
// group of 16 hand in 16 columns of a key, lane n gets column n of four keys.
__device__ __forceinline__ Frag values(const PageTile& tile, int kk, int d) {
    const int32_t lane = (int32_t)threadIdx.x % kWave;
    const int32_t r = 16 * kk + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int32_t chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    Frag v;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint8_t* at = &tile.value[r + 8 * e][16 * (chunk ^ (4 * (r & 3))) + 8 * (lane & 1)];
        const u32x2 w = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at));
        v.w[2 * e] = w[0];
        v.w[2 * e + 1] = w[1];
    }
    return v;
}

// 16 bytes per lane, memory -> LDS as copy_to_lds does, from a base of the whole wave's.
__device__ __forceinline__ void copy_from(const void* base, uint32_t offset, uint32_t lds) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const uint64_t same = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(offset), "s"(same), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}

// Products between the read of a fragment from LDS and its own.
constexpr int kAhead = 5;

struct BlocksWork {
    Request w;
    int32_t request, kv, block;  // block: of columns
    int32_t part, parts;
    int64_t unit;  // its sums' place in the workspace
};

// The work-group's part of the attention; false: there is none.
template <int WAVES>
__device__ __forceinline__ bool find_work(const AttendParams& p, BlocksWork& work) {
    // Work-groups reach the XCDs in turn.  An XCD takes whole units, a KV head of an item
    // (a request, or a part of its keys), `together` of them at a time, the longest
    // blocks of all of them first: blocks of the same keys meet in one L2, and the last
    // ones to end are short.
    constexpr int kBlock = WAVES * kRows;
    const int32_t units = (p.units + p.xcds - 1) / p.xcds, turn = (int32_t)blockIdx.x / p.xcds;
    const int32_t before = turn / (p.together * p.blocks) * p.together, size = min(p.together, units - before);
    const int32_t within = turn - before * p.blocks, rank = within / size;
    const int32_t unit = (before + within % size) * p.xcds + (int32_t)blockIdx.x % p.xcds;
    if (unit >= p.units) return false;
    work.kv = unit % p.kv_heads;
    if (p.slots > 0) {
        // slots: request r's blocks lie in slots cu[r] group / 256 + r and on, as many as it can need wherever it begins
        const int32_t slot = p.slots - 1 - unit / p.kv_heads;
        auto start = [&](int32_t r) __attribute__((always_inline)) {
            return (int32_t)((int64_t)min(max(p.cu[r], 0), p.tokens) * p.group / kBlock) + r;
        };
        const int32_t r = last_at_most(p.requests, slot, start);
        work.request = r;
        work.block = slot - __builtin_amdgcn_readfirstlane(start(r));
        work.part = 0, work.parts = 1, work.unit = 0;
        if (work.block < 0) return false;
    } else {
        Item it;
        const int32_t index = unit / p.kv_heads;
        if (!find_item(p.plan, index, it)) return false;
        work.block = p.blocks - 1 - rank;
        work.request = it.row, work.part = it.part, work.parts = it.parts;
        work.unit = ((int64_t)index * p.kv_heads + work.kv) * p.blocks + work.block;
        if (p.plan.chunk == 0 && it.part == 0 && work.kv == 0 && rank == 0 && threadIdx.x == 0)
            p.parts.of_row[it.row] = i32x2{index, it.parts};
    }
    work.w = request_at(p, work.request);
    return (int64_t)work.block * kBlock < (int64_t)work.w.nq * p.group;
}

// Masked keys of infinite or NaN values: sums that end up not finite (true is returned,
// nothing written) are found again by the CAREFUL form.
template <class T, int MODE, int WAVES, bool CAREFUL>
__device__ __forceinline__ bool blocks_part(const AttendParams& p, const BlocksWork& work, BlocksLds<WAVES>& lds) {
    constexpr int kWaves = WAVES, kBlock = WAVES * kRows, kBuffers = WAVES / 2;
    constexpr int COPIES = (int)(sizeof(PageTile) / 1024) / kWaves;
    static_assert(COPIES * kWaves == 32, "copies of a tile");
    const Request& w = work.w;
    const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave);
    const int32_t lane = (int32_t)threadIdx.x % kWave, c = lane & 31, h = lane >> 5;
    const int32_t m0 = work.block * kBlock, columns = min(w.nq * p.group - m0, kBlock) - wave * kRows;  // (of this wave, or less)
    const int32_t* table = p.table + work.request * p.table_stride;

    const Column col = column_at(p, w, lds.tree, m0, wave * kRows + c);
    const Bounds mine = bounds_of(p, col, c, min(columns, kRows));
    const int32_t least_lo = mine.least_lo, most_lo = mine.most_lo, least_hi = mine.least_hi, most_hi = mine.most_hi;
    float slope = 0.f;
    if ((MODE == kBiased || MODE == kBoth) && p.slopes) slope = p.slopes[work.kv * p.group + col.head] * kLog2e;
    if (lane == 0) lds.lo[wave] = least_lo, lds.hi[wave] = most_hi;
    lds_barrier();
    int32_t all_lo = INT32_MAX, all_hi = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all_lo = min(all_lo, lds.lo[i]), all_hi = max(all_hi, lds.hi[i]);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    const Tiles list = tiles_seen(p, w, all_lo, all_hi);
    const int32_t each = (list.count + work.parts - 1) / work.parts;
    const int32_t first = min(work.part * each, list.count), tiles = min(each, list.count - first);
    const int32_t end = p.parents ? w.len : max(all_hi, w.pre);  // no column sees a key from here on

    // pages of the next 64 tiles, one a lane; -1: no page
    int32_t page_of = -1;
    constexpr bool BACK = MODE == kBiased || MODE == kBoth;
    auto tile_at = [&](int32_t t) __attribute__((always_inline)) { return list.at(first + (BACK ? tiles - 1 - t : t)); };
    auto fetch_pages = [&](int32_t t) __attribute__((always_inline)) {
        page_of = table[tile_at(min(t + lane, tiles - 1))];
        if (page_of >= p.pages) page_of = -1;
    };
    auto page_at = [&](int32_t t) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(page_of, t & 63); };
    auto first_key = [&](int32_t t) __attribute__((always_inline)) { return tile_at(t) * kTileKeys; };

    // Copy j of the wave's of a tile: four keys each in the first half, four values in the second.  (Rows that no column
    // sees are copies of the last that one may; tiles without a page, which nobody reads, are page 0's.)
    struct From {
        const uint16_t* page[2];  // of keys, of values
        int32_t rows;             // of it that may be seen
    };
    auto from_page = [&](int32_t k0, int32_t page) __attribute__((always_inline)) {
        From f;
#pragma unroll
        for (int v = 0; v < 2; ++v) f.page[v] = p.pool[v] + work.kv * p.head[v] + max(page, 0) * p.page[v];
        f.rows = end - k0;
        return f;
    };
    const int32_t row0 = 4 * wave + (lane >> 4);
    const uint32_t stride[2] = {(uint32_t)p.token[0] * 2, (uint32_t)p.token[1] * 2};  // (below 2^26: a page's rows lie within 2^32 bytes)
    // (rows 16 and 32 apart have the same chunks)
    const uint32_t chunk[2] = {16u * ((lane & 15) ^ (row0 & 15)), 16u * ((lane & 15) ^ (4 * (row0 & 3)))};
    auto copy = [&](int32_t t, const From& f, auto which) __attribute__((always_inline)) {
        constexpr int HALF = COPIES / 2, j = which.value % HALF, v = which.value / HALF;
        PageTile& to = lds.tile[t % kBuffers];
        const int32_t i = j * kWaves + wave;
        copy_from(f.page[v], (uint32_t)min(row0 + 4 * kWaves * j, f.rows - 1) * stride[v] + chunk[v],
                  lds_offset(v == 0 ? &to.key[4 * i][0] : &to.value[4 * i][0]));
    };
    auto copy_tile = [&](int32_t t, const From& f) __attribute__((always_inline)) {
        each_of<COPIES>([&](auto j) __attribute__((always_inline)) { copy(t, f, j); });
    };

    // B fragments of Q^T: column c.  The rows come through LDS (rows of 16 chunks of 16
    // bytes end to end, XORed by the row, in the later buffers): fragments read from
    // memory are 32 rows' lines for every one.
    Frag q[8];
    int32_t page0 = -1, page1 = -1, key0 = 0, key1 = 0;  // of this tile and the next
    {
        uint8_t* const rows = &lds.tile[kBuffers / 2].key[0][0] + wave * (kRows * 2 * kDim);
        static_assert(kWaves * kRows * 2 * kDim == kBuffers / 2 * sizeof(PageTile), "queries in the later half of the buffers");
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int32_t r = 4 * j + (lane >> 4), chunk = (lane & 15) ^ (r & 15);
            const int32_t query = __shfl(col.query, r, kWave), head = __shfl(col.head, r, kWave);
            copy_to_lds(p.q + (w.q_lo + (int64_t)query) * p.q_token + (int64_t)(work.kv * p.group + head) * p.q_head + 8 * chunk,
                        lds_offset(rows + 1024 * j));
        }
        if (tiles > 0) {
            fetch_pages(0);
            page0 = page_at(0), key0 = first_key(0);
            page1 = page_at(min(1, tiles - 1)), key1 = first_key(min(1, tiles - 1));
            copy_tile(0, from_page(key0, page0));
            wait_copies<COPIES>();
        } else {
            wait_copies<0>();
        }
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s].u = *reinterpret_cast<const u32x4*>(rows + 256 * c + 16 * ((2 * s + h) ^ (c & 15)));
        lds_barrier();
        if (WAVES == 8 && tiles > 0) copy_tile(1, from_page(key1, page1));
    }
    f32x16 acc[4], s[2];
    Frag pf[4];
    float mx = -__builtin_inff(), total = 0.f;
    bool some = false;  // a key of the column is attended
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    // whether the wave sees a key of a tile, and whether all of its columns see all of them
    auto sees = [&](int32_t k0, int32_t page) __attribute__((always_inline)) {
        return page >= 0 && columns > 0 &&
               ((k0 + kTileKeys > least_lo && k0 < most_hi) || k0 < w.pre || (p.parents && k0 + kTileKeys > w.before));
    };
    auto sees_all = [&](int32_t k0) __attribute__((always_inline)) {
        return (k0 >= most_lo && k0 + kTileKeys <= least_hi) || k0 + kTileKeys <= w.pre;
    };
    // Sixteen products, of tile t's values (which 0) or keys (1), each fragment read kAhead
    // products before its own; beside those of the keys the copies of tile `next`.  Scores:
    // register i of half u is key 32u + 8 (i / 4) + 4h + i % 4.
    auto multiply = [&](int32_t t, int32_t next, const From& f, auto which) __attribute__((always_inline)) {
        constexpr bool SCORES = which.value != 0;
        const PageTile& tile = lds.tile[t % kBuffers];
        Frag x[kAhead];
        auto fetch = [&](auto number) __attribute__((always_inline)) {
            constexpr int n = number.value;
            if constexpr (!SCORES) {
                x[n % kAhead] = values(tile, n / 4, n % 4);
            } else {  // key rows 32 (n & 1) .., numbers 16 (n / 2) ..
                const int32_t r = 32 * (n & 1) + c;
                x[n % kAhead].u = *reinterpret_cast<const u32x4*>(&tile.key[r][16 * ((n - (n & 1) + h) ^ (r & 15))]);
            }
        };
        if constexpr (SCORES) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
        }
        each_of<kAhead>(fetch);
        __builtin_amdgcn_sched_barrier(0);
        each_of<16>([&](auto number) __attribute__((always_inline)) {
            constexpr int n = number.value;
            if constexpr (!SCORES) acc[n % 4] = mfma32<T>(x[n % kAhead], pf[n / 4], acc[n % 4]);
            else s[n & 1] = mfma32<T>(x[n % kAhead], q[n / 2], s[n & 1]);
            if constexpr (n + kAhead < 16) fetch(Number<n + kAhead>{});
            if constexpr (SCORES && n % (16 / COPIES) == 1) copy(next, f, Number<n / (16 / COPIES)>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto each_score = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = f(s[u][i], 32 * u + 8 * (i / 4) + i % 4);  // (the key, but for 4h)
    };
    Cap cap = p.cap;
    if constexpr (MODE == kCapped) {  // (in registers of the loop's own: there are too few scalar ones)
#pragma unroll
        for (int i = 0; i < 3; ++i) asm volatile("" : "+v"(cap.least[i]));
    }
    uint64_t seen = ~0ull;  // bit 32u + 8 a + i: key 32u + 8a + 4h + i of the tile in `pf`
    auto softmax = [&](int32_t k0) __attribute__((always_inline)) {
        if constexpr (MODE == kBoth) {
            float far = 0.f;
            each_score([&](float x, int) { far = fmaxf(far, fabsf(x)); return x; });
            cap_scores(p.cap, p.cap_in, p.cap2, far, [&](auto f) __attribute__((always_inline)) { each_score([&](float x, int) { return f(x, 0.f); }); });
        }
        if constexpr (MODE == kBiased || MODE == kBoth) {
            const float factor = MODE == kBoth ? 1.f : p.scale2;
            if (k0 + kTileKeys <= least_hi) {  // (no key behind a query: the distances fall by one a key)
                const float base = -slope * (float)(col.position - k0 - 4 * h);
                each_score([&](float x, int key) { return fmaf(x, factor, fmaf(slope, (float)key, base)); });
            } else {
                // (a draft's depth in place of its number; read for every key, without branches)
                const int32_t draft0 = k0 + 4 * h - w.before, from = p.parents ? 0 : INT32_MAX;
                each_score([&](float x, int key) {
                    const int32_t draft = draft0 + key, depth = lds.tree.depth[min(max(draft, 0), kMostDrafts - 1)];
                    return fmaf(-slope, fabsf((float)(col.position - w.before - (draft >= from ? depth : draft))), x * factor);
                });
            }
        }
        const bool whole = sees_all(k0);
        bool sees_some = true;
        seen = ~0ull;
        if (!whole) {
            seen = column_sees(p, w, lds.tree, col, k0);
            sees_some = seen != 0;
            seen >>= 4 * h;
        }
        some |= sees_some;
        // The largest magnitude bounds the scores; their maximum is looked for where the bound may pass the subtracted one.
        float far = BACK ? -__builtin_inff() : 0.f;
        each_score([&](float x, int) { far = fmaxf(far, BACK ? x : fabsf(x)); return x; });
        const float bound = MODE == kPlain ? far * p.scale2 : MODE == kCapped ? far * p.cap.far[0] : far;
        if (__ballot(bound > mx + Range<T>::most || mx == -__builtin_inff())) {
            float top = -__builtin_inff();
            if (whole) each_score([&](float x, int) { top = fmaxf(top, x); return x; });
            else each_score([&](float x, int key) { top = fmaxf(top, if_seen_or_least(mask_of(seen, key), x)); return x; });
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            if (MODE == kPlain) top *= p.scale2;
            if (MODE == kCapped) top = sees_some ? capped(top * p.cap_in, p.cap2) : -__builtin_inff();
            if (__ballot(top > mx + Range<T>::most)) {
                const float next = top > mx + Range<T>::most ? top - Range<T>::head : mx;
                const float keep = mx == -__builtin_inff() ? (next == mx ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mx - next);
                mx = next;
                total *= keep;
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[d] *= keep;
            }
        }
        const float sub = mx == -__builtin_inff() ? 0.f : mx;
        if constexpr (MODE == kCapped) {
            cap_scores(cap, p.cap_in, p.cap2, far, [&](auto f) __attribute__((always_inline)) { each_score([&](float x, int) { return f(x, sub); }); });
        }
        each_score([&](float x, int) {
            return __builtin_amdgcn_exp2f(MODE == kPlain ? fmaf(x, p.scale2, -sub) : MODE == kCapped ? x : x - sub);
        });
        if (!whole) each_score([&](float x, int key) { return if_seen(mask_of(seen, key), x); });
        each_score([&](float x, int) { total += x; return x; });
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pf[kk].w[i] = pack<T>(s[kk / 2][8 * (kk & 1) + 2 * i], s[kk / 2][8 * (kk & 1) + 2 * i + 1]);
    };
    auto careful_products = [&](int32_t t) __attribute__((always_inline)) {
        const PageTile& tile = lds.tile[t % kBuffers];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            f32x16 up, down;
#pragma unroll
            for (int i = 0; i < 16; ++i) up[i] = down[i] = 0.f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                const Frag v = values(tile, kk, d);
                Frag plain, pos, neg, see;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    split_odd<T>(v.w[i], plain.w[i], pos.w[i], neg.w[i]);
                    const int32_t bit = 16 * kk + 8 * (i / 2) + 2 * (i & 1);  // (of the lane's numbers 2i, 2i + 1)
                    see.w[i] = ((seen >> bit) & 1 ? kOne<T> : 0u) | ((seen >> (bit + 1)) & 1 ? kOne<T> << 16 : 0u);
                }
                acc[d] = mfma32<T>(plain, pf[kk], acc[d]);
                up = mfma32<T>(pos, see, up);
                down = mfma32<T>(neg, see, down);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[d][i] += (up[i] > 0.f ? __builtin_inff() : 0.f) - (down[i] > 0.f ? __builtin_inff() : 0.f);
        }
    };
    constexpr Number<0> of_values;
    constexpr Number<1> of_keys;
    auto values_of = [&](int32_t t, const From& f) __attribute__((always_inline)) {
        if constexpr (CAREFUL) careful_products(t);
        else multiply(t, 0, f, of_values);
    };
    if constexpr (WAVES == 8) {
        // The two waves of a SIMD half a tile apart: one multiplies (the last tile's
        // values, this one's keys) and asks for its copies of the tile after the next,
        // whose buffer was read until two steps ago, while the other makes
        // probabilities.  Steps are divided by barriers, every other one of them behind a
        // wait for the copies of the tile whose keys come next.
        const bool second = wave >= kWaves / 2;
        auto sync = [&](bool landed) __attribute__((always_inline)) {
            if (landed) wait_barrier<COPIES>();
            else lds_barrier();
        };
        if (second) sync(true);
        bool saw = false;
#pragma unroll 1
        for (int32_t t = 0; t <= tiles; ++t) {
            const bool now = t < tiles && sees(key0, page0);
            const int32_t later = min(t + 2, tiles - 1);
            if (((t + 2) & 63) == 0 && t + 2 < tiles) fetch_pages(t + 2);
            const int32_t page2 = page_at(later), key2 = first_key(later);
            const From f = from_page(key2, page2);
            sync(!second);
            // (one place for each: variants of both together cost copies of the sums between them)
            if (saw) values_of(t - 1, f);
            if (now) multiply(t, t + 2, f, of_keys);
            else if (t < tiles) copy_tile(t + 2, f);
            sync(second);
            if (now) softmax(key0);
            saw = now;
            key0 = key1, page0 = page1, key1 = key2, page1 = page2;
        }
        if (!second) lds_barrier();
    } else {
        // A tile after the other; the CU's other work-group multiplies meanwhile.
#pragma unroll 1
        for (int32_t t = 0; t < tiles; ++t) {
            const bool now = sees(key0, page0);
            if (((t + 1) & 63) == 0 && t + 1 < tiles) fetch_pages(t + 1);
            const int32_t later = min(t + 1, tiles - 1), page = page_at(later), key = first_key(later);
            const From f = from_page(key, page);
            wait_barrier<0>();  // (this tile is there, and nobody reads the last one)
            if (now) {
                multiply(t, t + 1, f, of_keys);
                softmax(key0);
                values_of(t, f);
            } else {
                copy_tile(t + 1, f);
            }
            key0 = key, page0 = page;
        }
    }
    wait_copies<0>();
    __syncthreads();  // the tiles' memory is free
    if constexpr (!CAREFUL) {
        float odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d) odd[d] = fmaf(acc[d][i], 0.f, odd[d]);
        const float sum = (odd[0] + odd[1]) + (odd[2] + odd[3]);
        if (__syncthreads_or(sum != sum)) return true;
    }
    total += __shfl_xor(total, 32, kWave);
    const bool none = !some;  // no key seen
    // Rows leave through LDS as well, whole ones at a time: row c's numbers 32 d + 8 a
    // + 4 h .. are its piece 8 d + 2 a + h of four, pieces XORed by the row.
    static_assert(sizeof(PageTile) * kBuffers >= kWaves * kRows * 4 * kDim, "rows");
    uint8_t* const rows = &lds.tile[0].key[0][0] + wave * (kRows * 4 * kDim);
    if (work.parts == 1) {
        const float inv = none ? 0.f : 1.0f / total;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                *reinterpret_cast<u32x2*>(rows + 256 * c + 8 * ((8 * d + 2 * a + h) ^ c)) =
                    none ? u32x2{0, 0} : u32x2{pack<T>(acc[d][4 * a] * inv, acc[d][4 * a + 1] * inv),
                                               pack<T>(acc[d][4 * a + 2] * inv, acc[d][4 * a + 3] * inv)};
        wait_lds();
#pragma unroll
        for (int j = 0; j < kRows / 2; ++j) {
            const int32_t r = 2 * j + h;
            const u32x2 x = *reinterpret_cast<const u32x2*>(rows + 256 * r + 8 * (c ^ r));
            const int32_t query = __shfl(col.query, r, kWave), head = work.kv * p.group + __shfl(col.head, r, kWave);
            if (r < columns) *reinterpret_cast<u32x2*>(p.out + (w.q_lo + (int64_t)query) * p.o_token + head * p.o_head + 4 * c) = x;
        }
        if (p.lse && h == 0 && c < columns)
            p.lse[(w.q_lo + (int64_t)col.query) * p.kv_heads * p.group + work.kv * p.group + col.head] =
                none ? -__builtin_inff() : (mx + __builtin_amdgcn_logf(total)) * kLn2;
    } else {
        const int64_t at = work.unit * kBlock + wave * kRows;
        if (tiles > 0) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<f32x4*>(rows + 512 * c + 16 * ((8 * d + 2 * a + h) ^ c)) =
                        f32x4{acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]};
            wait_lds();
#pragma unroll
            for (int j = 0; j < kRows / 2; ++j) {
                const int32_t r = 2 * j + h;
                const f32x4 x = *reinterpret_cast<const f32x4*>(rows + 512 * r + 16 * (c ^ r));
                if (r < columns) *reinterpret_cast<f32x4*>(p.parts.sums + (at + r) * kDim + 4 * c) = x;
            }
        }
        if (h == 0 && c < columns) p.parts.stats[at + c] = f32x2{none ? -__builtin_inff() : fmaxf(mx, kLowest), none ? 0.f : total};
    }
    return false;
}

// (A call, so that its registers are not the common form's.)
template <class T, int MODE, int WAVES>
__device__ __attribute__((noinline)) void careful_block(AttendParams p, BlocksLds<WAVES>* lds) {
    BlocksWork work;
    if (find_work<WAVES>(p, work)) blocks_part<T, MODE, WAVES, true>(p, work, *lds);
}

template <class T, int MODE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void blocks_kernel(AttendParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto& lds = *reinterpret_cast<BlocksLds<WAVES>*>(lds_raw);
    BlocksWork work;
    if (!find_work<WAVES>(p, work)) return;
    // (the same for the work-group, and in scalar registers from here on)
    for (int32_t* x : {&work.request, &work.kv, &work.block, &work.part, &work.parts}) *x = __builtin_amdgcn_readfirstlane(*x);
    if (p.parents) find_tree(p, work.w, lds.tree);
    if (__builtin_expect(blocks_part<T, MODE, WAVES, false>(p, work, lds), 0)) careful_block<T, MODE, WAVES>(p, &lds);
}

template <class T, int MODE, int WAVES>
int launch(const AttendParams& p, int64_t groups, hipStream_t st) {
    static OncePerDevice once;
    const auto kernel = blocks_kernel<T, MODE, WAVES>;
    const int rc = allow_lds(once, reinterpret_cast<const void*>(kernel), sizeof(BlocksLds<WAVES>), "paged_attend: LDS");
    if (rc != V1_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)groups), dim3(64 * WAVES), sizeof(BlocksLds<WAVES>), st, p);
    return V1_LAUNCHED("paged_attend: blocks");
}

template <class T, int WAVES>
int launch(int mode, const AttendParams& p, int64_t groups, hipStream_t st) {
    return mode == kPlain ? launch<T, kPlain, WAVES>(p, groups, st) : mode == kCapped ? launch<T, kCapped, WAVES>(p, groups, st)
         : mode == kBiased ? launch<T, kBiased, WAVES>(p, groups, st) : launch<T, kBoth, WAVES>(p, groups, st);
}

template <class T>
int launch(int columns, int mode, const AttendParams& p, int64_t groups, hipStream_t st) {
    return columns == 4 * kRows ? launch<T, 4>(mode, p, groups, st) : launch<T, 8>(mode, p, groups, st);
}

}  // namespace

int paged::launch_blocks(bool fp16, int columns, int mode, const AttendParams& p, int64_t groups, hipStream_t st) {
    return fp16 ? launch<_Float16>(columns, mode, p, groups, st) : launch<__bf16>(columns, mode, p, groups, st);
}

}  // namespace v1
