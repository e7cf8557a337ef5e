// Attention of a few queries of each request over K / V pages of 16-bit numbers:
//   S[m, j] = scale q_m . k_j, capped and biased, O[m] = sum_j softmax_j(S[m, :]) v_j
// for the columns m of a request (its queries times the heads of a KV head), at most 32
// of them, and the keys j that column m sees; and the host's side of both kernels.
//
// A work-group attends one, two or four KV heads of a request over one part of its
// pages, a wave each; waves of one head take the part's pages in turn, each with its own
// running maximum, and join through LDS.  A page is a tile of 64 keys.
//   scores  S^T = K Q^T (v_mfma_f32_16x16x32): keys come straight into registers, 64
//           bytes of 16 rows an instruction; column c of a fragment is column c of 16.
//   output  O^T = V^T P^T: values go memory -> LDS and come back transposed
//           (ds_read_b64_tr_b16); the lane's own scores are its B fragment's
//           probabilities, each in two numbers of the pages' type, so that the output's
//           rounding is all that is left (error against 64 bits 1.0 times a rounded exact
//           result's).
// Whether a tile is seen whole is known for the wave; else each column's 64 bits of it
// are made once.  A masked key's probability is zero, which an infinite or NaN value
// would turn into NaN: sums that end up not finite are found again by a careful form
// (CAREFUL), which counts the infinities that each column sees.
//
// Bound by memory: 48 contexts of 4096 to 65536 tokens, 4 KV heads of 8 query heads,
// 383 us for 2.18 GB, 5.7 TB/s (a copy of 512 MiB moves 5.3); 128 requests of which a
// window leaves 4096 tokens, 8 KV heads, 316 us for 1.8 GB.  Few keys are bound by latency: 8
// requests of 1500 to 16384 tokens, one KV head, 10.5 us and 4.5 for the join, of which a
// work-group's own chain is lengths and plan 1.6, table and keys 2.7, a tile 1.5, the
// join of its waves 1.8.
// Loads of keys that pass the caches gain 5% at 2 GB (363 us) and lose 5-13% where the
// keys fit the last cache (128 contexts of 45 to 500 tokens, 8 KV heads, 32 and 37 us).
#include "paged_attend.h"

namespace v1 {
namespace {

using namespace paged;

constexpr int kWaves = 4;

template <int NC>
struct RowsLds {
    union {
        uint8_t value[2][kTileKeys][2 * kDim];
        float out[16 * NC][kDim + 4];
    } u[kWaves];
    float top[kWaves][16 * NC], total[kWaves][16 * NC];
    Tree tree;
};

// What the kernel has found of its work.
struct RowsWork {
    Item item;
    Request w;
    int32_t index, set, block;  // work item, KV heads, block of columns
};

template <class T, int NC, int MODE, bool CAREFUL>
__device__ __forceinline__ bool rows_part(const AttendParams& p, const RowsWork& work, RowsLds<NC>& lds) {
    constexpr int COLS = 16 * NC;
    const Item& it = work.item;
    const Request& w = work.w;
    const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave);
    const int32_t lane = (int32_t)threadIdx.x % kWave, g = lane >> 4, c = lane & 15;
    const int32_t streams = kWaves / p.together, stream = wave / p.together, kvh = work.set * p.together + wave % p.together;
    const int32_t m0 = work.block * COLS, columns = min(w.nq * p.group - m0, COLS);
    const int32_t* table = p.table + it.row * p.table_stride;
    const uint16_t* kb = p.pool[0] + kvh * p.head[0];
    const uint16_t* vb = p.pool[1] + kvh * p.head[1];

    Column col[NC];
    int32_t least_lo = INT32_MAX, most_lo = 0, least_hi = INT32_MAX, most_hi = 0;
    float slope[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        col[n] = column_at(p, w, lds.tree, m0, 16 * n + c);
        const Bounds b = bounds_of(p, col[n], c, min(columns - 16 * n, 16));
        least_lo = min(least_lo, b.least_lo), most_lo = max(most_lo, b.most_lo);
        least_hi = min(least_hi, b.least_hi), most_hi = max(most_hi, b.most_hi);
        slope[n] = 0.f;
        if ((MODE == kBiased || MODE == kBoth) && p.slopes) slope[n] = p.slopes[kvh * p.group + col[n].head] * kLog2e;
    }
    const Tiles tiles = tiles_seen(p, w, least_lo, most_hi);
    const int32_t each = (tiles.count + it.parts - 1) / it.parts;
    const int32_t first = min(it.part * each, tiles.count), count = min(each, tiles.count - first);
    const int32_t mine = (count - stream + streams - 1) / streams;  // this wave's tiles: stream, stream + streams, ...
    const int32_t end = p.parents ? w.len : max(most_hi, w.pre);    // no column sees a key from here on

    // pages of the wave's next 64 tiles, one a lane; -1: no page
    int32_t page_of = -1;
    auto fetch_pages = [&](int32_t t) __attribute__((always_inline)) {
        page_of = -1;
        if (t + lane < mine) page_of = table[tiles.at(first + stream + streams * (t + lane))];
        if (page_of >= p.pages) page_of = -1;
    };
    auto page_at = [&](int32_t t) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(page_of, t & 63); };
    auto first_key = [&](int32_t t) __attribute__((always_inline)) { return tiles.at(first + stream + streams * t) * kTileKeys; };
    // A fragments of K: key 16u + c, numbers 32 s + 8 g ..  (Rows that no column sees are copies of the last that one may.)
    auto load_keys = [&](u32x4 (&k)[4][4], int32_t k0, int32_t page) __attribute__((always_inline)) {
        const uint16_t* at = kb + max(page, 0) * p.page[0] + 8 * g;
        const int32_t last = min(end - k0, kTileKeys) - 1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint16_t* row = at + min(16 * u + c, last) * p.token[0];
#pragma unroll
            for (int s = 0; s < 4; ++s) k[u][s] = *reinterpret_cast<const u32x4*>(row + 32 * s);
        }
    };
    // V rows, memory -> LDS, chunk n of row r at n ^ 2 (r % 8)
    auto copy_values = [&](int32_t t, int32_t k0, int32_t page) __attribute__((always_inline)) {
        const uint16_t* at = vb + max(page, 0) * p.page[1];
        const int32_t last = min(end - k0, kTileKeys) - 1;
        const uint32_t to = lds_offset(&lds.u[wave].value[t & 1][0][0]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int32_t r = 4 * j + g;
            copy_to_lds(at + min(r, last) * p.token[1] + 8 * (c ^ (2 * (r & 7))), to + 1024 * j);
        }
    };

    // B fragments of Q^T: column 16 n + c, numbers 32 s + 8 g ..
    Frag q[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const uint16_t* src = p.q + (w.q_lo + (int64_t)col[n].query) * p.q_token + (int64_t)(kvh * p.group + col[n].head) * p.q_head + 8 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) q[n][s].u = *reinterpret_cast<const u32x4*>(src + 32 * s);
    }
    f32x4 acc[NC][8];
    float mx[NC], total[NC];
    int32_t some = 0;  // bit n: a key of column n is attended
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        mx[n] = -__builtin_inff(), total[n] = 0.f;
    }
    u32x4 k[4][4];
    int32_t page = -1;
    if (mine > 0) {
        fetch_pages(0);
        page = page_at(0);
        load_keys(k, first_key(0), page);
        copy_values(0, first_key(0), page);
    }
#pragma unroll 1
    for (int32_t t = 0; t < mine; ++t) {
        const int32_t k0 = first_key(t);
        const bool there = page >= 0;
        const bool whole = there && ((k0 >= most_lo && k0 + kTileKeys <= least_hi) || k0 + kTileKeys <= w.pre);
        float s[NC][4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    Frag a;
                    a.u = k[u][st];
                    d = mfma16<T>(a, q[n][st], d);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][u][i] = d[i];
            }
        // the next tile's keys, then its values
        int32_t next_page = -1;
        if (t + 1 < mine) {
            if (((t + 1) & 63) == 0) fetch_pages(t + 1);
            next_page = page_at(t + 1);
            load_keys(k, first_key(t + 1), next_page);
        }
        if constexpr (MODE == kPlain) {
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][u][i] *= p.scale2;
        } else {
            if constexpr (MODE == kCapped || MODE == kBoth) {
                float far = 0.f;
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) far = fmaxf(far, fabsf(s[n][u][i]));
                cap_scores(p.cap, p.cap_in, p.cap2, far, [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                    for (int n = 0; n < NC; ++n)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[n][u][i] = f(s[n][u][i], 0.f);
                });
            } else {
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[n][u][i] *= p.scale2;
            }
            if constexpr (MODE == kBiased || MODE == kBoth) {
                // (a draft's depth in place of its number; read for every key, without branches)
                const int32_t draft0 = k0 + 4 * g - w.before, from = p.parents ? 0 : INT32_MAX;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int32_t draft = draft0 + 16 * u + i, depth = lds.tree.depth[min(max(draft, 0), kMostDrafts - 1)];
                        const int32_t at = w.before + (draft >= from ? depth : draft);
#pragma unroll
                        for (int n = 0; n < NC; ++n)
                            s[n][u][i] = fmaf(-slope[n], fabsf((float)(col[n].position - at)), s[n][u][i]);
                    }
            }
        }
        uint64_t seen[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) seen[n] = ~0ull;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const uint64_t bits = there ? column_sees(p, w, lds.tree, col[n], k0) : 0;
                some |= (bits != 0) << n;
                seen[n] = bits >> (4 * g);  // bit 16u + i: key 16u + 4g + i
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][u][i] = if_seen_or_least(mask_of(seen[n], 16 * u + i), s[n][u][i]);
            }
        } else {
            some = -1;
        }
        Frag pf[NC][2], rest[NC][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float top = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][u][i]);
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            if (__ballot(top > mx[n] + Range<T>::most)) {
                const float next = top > mx[n] + Range<T>::most ? top - Range<T>::head : mx[n];
                const float keep = mx[n] == -__builtin_inff() ? (next == mx[n] ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mx[n] - next);
                mx[n] = next;
                total[n] *= keep;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[n][i] *= keep;
            }
            const float sub = mx[n] == -__builtin_inff() ? 0.f : mx[n];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = __builtin_amdgcn_exp2f(s[n][u][i] - sub);
                    total[n] += x[i];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t b = pack<T>(x[2 * i], x[2 * i + 1]);
                    const f32x2 back = unpack<T>(b);
                    pf[n][u / 2].w[2 * (u & 1) + i] = b;
                    rest[n][u / 2].w[2 * (u & 1) + i] = pack<T>(x[2 * i] - back[0], x[2 * i + 1] - back[1]);
                }
            }
        }
        // this tile's values have landed: behind them at least the next tile's 16 loads of keys were issued, if there is one
        if (t + 1 < mine) {
            asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
            copy_values(t + 1, first_key(t + 1), next_page);
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        page = next_page;
        // number j of a lane's eight keys is 32 step + 16 (j / 4) + 4g + j % 4: of the four keys 4g .. a
        // group of 16 lanes hands in 16 columns each (lane n: key n / 4, columns 4 (n % 4) ..) and gets column n of all
#pragma unroll
        for (int step = 0; step < 2; ++step) {
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                Frag v;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int32_t r = 32 * step + 16 * e + 4 * g + (c >> 2), chunk = 2 * d + ((c & 3) >> 1);
                    const uint8_t* at = &lds.u[wave].value[t & 1][r][16 * (chunk ^ (2 * (r & 7))) + 8 * (c & 1)];
                    using i16x4 = __attribute__((ext_vector_type(4))) short;
                    const u32x2 x = __builtin_bit_cast(
                        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at));
                    v.w[2 * e] = x[0], v.w[2 * e + 1] = x[1];
                }
                if constexpr (CAREFUL) {
                    Frag plain, pos, neg;
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_odd<T>(v.w[i], plain.w[i], pos.w[i], neg.w[i]);
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        Frag see;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int32_t bit = 32 * step + 16 * (i / 2) + 2 * (i & 1);  // (of the lane's numbers 2i, 2i + 1)
                            see.w[i] = ((seen[n] >> bit) & 1 ? kOne<T> : 0u) | ((seen[n] >> (bit + 1)) & 1 ? kOne<T> << 16 : 0u);
                        }
                        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                        const f32x4 up = mfma16<T>(pos, see, zero), down = mfma16<T>(neg, see, zero);
                        acc[n][d] = mfma16<T>(plain, pf[n][step], acc[n][d]);
                        acc[n][d] = mfma16<T>(plain, rest[n][step], acc[n][d]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[n][d][i] += (up[i] > 0.f ? __builtin_inff() : 0.f) - (down[i] > 0.f ? __builtin_inff() : 0.f);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        acc[n][d] = mfma16<T>(v, pf[n][step], acc[n][d]);
                        acc[n][d] = mfma16<T>(v, rest[n][step], acc[n][d]);
                    }
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the values' buffers become the sums'
    if constexpr (!CAREFUL) {
        float odd = 0.f;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) odd = fmaf(acc[n][d][i], 0.f, odd);
        if (__syncthreads_or(odd != odd)) return true;
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        total[n] += __shfl_xor(total[n], 16, kWave);
        total[n] += __shfl_xor(total[n], 32, kWave);
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&lds.u[wave].out[16 * n + c][16 * d + 4 * g]) = acc[n][d];
        if (g == 0) {
            lds.top[wave][16 * n + c] = (some >> n) & 1 ? fmaxf(mx[n], kLowest) : mx[n];
            lds.total[wave][16 * n + c] = total[n];
        }
    }
    __syncthreads();
    for (int32_t i = (int32_t)threadIdx.x; i < p.together * COLS * (kDim / 2); i += 64 * kWaves) {
        const int32_t row = i / (kDim / 2), dim = 2 * (i % (kDim / 2)), sub_head = row / COLS, x = row % COLS;
        if (x >= columns) continue;
        const int32_t kv = work.set * p.together + sub_head;
        float top = -__builtin_inff();
        for (int32_t v = sub_head; v < kWaves; v += p.together) top = fmaxf(top, lds.top[v][x]);
        const float sub = top == -__builtin_inff() ? 0.f : top;
        float sum = 0.f, o0 = 0.f, o1 = 0.f;
        for (int32_t v = sub_head; v < kWaves; v += p.together) {
            const float f = __builtin_amdgcn_exp2f(lds.top[v][x] - sub);
            sum = fmaf(f, lds.total[v][x], sum);
            o0 = fmaf(f, lds.u[v].out[x][dim], o0);
            o1 = fmaf(f, lds.u[v].out[x][dim + 1], o1);
        }
        if (it.parts == 1) {
            const int32_t i0 = m0 / p.group, y = m0 - i0 * p.group + x;
            const int32_t by = p.group == 1 ? y : (int32_t)small_div((uint32_t)y, p.group_magic);
            const int64_t token = w.q_lo + i0 + by;
            const int32_t head = kv * p.group + y - by * p.group;
            const bool none = top == -__builtin_inff() && sum == 0.f;  // no key attended
            const float inv = none ? 0.f : 1.0f / sum;
            *reinterpret_cast<uint32_t*>(p.out + token * p.o_token + head * p.o_head + dim) = none ? 0u : pack<T>(o0 * inv, o1 * inv);
            if (p.lse && dim == 0)
                p.lse[token * p.kv_heads * p.group + head] = none ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        } else {
            const int64_t at = (((int64_t)work.index * p.kv_heads + kv) * p.blocks + work.block) * COLS + x;
            *reinterpret_cast<f32x2*>(p.parts.sums + at * kDim + dim) = f32x2{o0, o1};
            if (dim == 0) p.parts.stats[at] = f32x2{top, sum};
        }
    }
    return false;
}

// (A call, so that its registers are not the common form's.)
template <class T, int NC, int MODE>
__device__ __attribute__((noinline)) void careful_rows(AttendParams p, RowsWork work, RowsLds<NC>* lds) {
    rows_part<T, NC, MODE, true>(p, work, *lds);
}

template <class T, int NC, int MODE>
__global__ __launch_bounds__(64 * kWaves, 1) void rows_kernel(AttendParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto& lds = *reinterpret_cast<RowsLds<NC>*>(lds_raw);
    const int32_t xcd = (int32_t)blockIdx.x % 8, turn = (int32_t)blockIdx.x / 8, sets = p.kv_heads / p.together * p.blocks;
    RowsWork work;
    const int32_t which = p.plan.chunk > 0 ? (xcd * p.spread + turn) % sets : turn % sets;
    work.index = p.plan.chunk > 0 ? (xcd * p.spread + turn) / sets : turn / sets * 8 + xcd;
    work.block = which % p.blocks, work.set = which / p.blocks;
    if (!find_item(p.plan, work.index, work.item)) return;
    if (p.plan.chunk == 0 && work.item.part == 0 && which == 0 && threadIdx.x == 0)
        p.parts.of_row[work.item.row] = i32x2{work.index, work.item.parts};
    work.w = request_at(p, work.item.row);
    if (work.block * 16 * NC >= work.w.nq * p.group) return;
    if (p.parents) find_tree(p, work.w, lds.tree);
    if (__builtin_expect(rows_part<T, NC, MODE, false>(p, work, lds), 0)) careful_rows<T, NC, MODE>(p, work, &lds);
}

// A work-group of the join: 8 / G columns of a request and KV head, G groups of 32
// threads for each, every group every G-th part.
struct RowsJoin {
    AttendParams a;
    int32_t cols;  // of a block
};

template <class T, int G>
__global__ __launch_bounds__(256) void rows_join(RowsJoin j) {
    __shared__ f32x4 sums[8][32];
    __shared__ float totals[8];
    const AttendParams& p = j.a;
    constexpr int C = 8 / G;
    const int32_t r = (int32_t)blockIdx.y, each = p.blocks * j.cols / C, kv = (int32_t)blockIdx.x / each;
    const int32_t who = (int32_t)threadIdx.x / 32, at4 = (int32_t)threadIdx.x % 32, group = who % G;
    const int32_t m = (int32_t)blockIdx.x % each * C + who / G;
    int32_t parts, first;
    if (p.plan.chunk > 0) {
        parts = (tiles_of(p.plan.keys) + p.plan.chunk - 1) / p.plan.chunk;
        first = r * parts;
    } else {
        const i32x2 of = p.parts.of_row[r];
        first = of[0], parts = of[1];
    }
    const Request w = request_at(p, r);
    if (parts <= 1 || (m - who / G) >= w.nq * p.group) return;
    const int64_t step = (int64_t)p.kv_heads * p.blocks * j.cols, base = first * step + (int64_t)kv * p.blocks * j.cols + m;
    float top = -__builtin_inff(), total = 0.f;
    const bool there = m < w.nq * p.group;
    if (!there) parts = 0;
    for (int32_t i = at4; i < parts; i += 32) top = fmaxf(top, p.parts.stats[base + i * step][0]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    const float sub = top == -__builtin_inff() ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int32_t i = group; i < parts; i += G) {
        const int64_t at = base + i * step;
        const f32x2 st = p.parts.stats[at];
        f32x4 x = *reinterpret_cast<const f32x4*>(p.parts.sums + at * kDim + 4 * at4);
        const bool none = st[0] == -__builtin_inff() && st[1] == 0.f;  // (no key of it is seen: its sums may not be written)
        const float f = __builtin_amdgcn_exp2f(st[0] - sub);
        total = fmaf(f, st[1], total);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(f, none ? 0.f : x[k], o[k]);
    }
    if constexpr (G > 1) {
        sums[who][at4] = o;
        if (at4 == 0) totals[who] = total;
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int k = 1; k < G; ++k) {
            o += sums[who + k][at4];
            total += totals[who + k];
        }
    }
    if (!there) return;
    const int32_t i = m / p.group, head = kv * p.group + m % p.group;
    const int64_t token = w.q_lo + i;
    const bool none = top == -__builtin_inff() && total == 0.f;  // no key attended
    const float inv = none ? 0.f : 1.0f / total;
    *reinterpret_cast<u32x2*>(p.out + token * p.o_token + head * p.o_head + 4 * at4) =
        none ? u32x2{0, 0} : u32x2{pack<T>(o[0] * inv, o[1] * inv), pack<T>(o[2] * inv, o[3] * inv)};
    if (p.lse && at4 == 0)
        p.lse[token * p.kv_heads * p.group + head] = none ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

template <class T, int G>
int launch_join(const AttendParams& p, int32_t cols, hipStream_t st) {
    const int64_t groups = (int64_t)p.kv_heads * p.blocks * cols / (8 / G);
    hipLaunchKernelGGL((rows_join<T, G>), dim3((uint32_t)groups, (uint32_t)p.requests), dim3(256), 0, st, RowsJoin{p, cols});
    return V1_LAUNCHED("paged_attend: join");
}

// -------------------------------------------------------------- the host's side
// Keys at the end of a request that a window leaves, with the rest of their first tile.  The parts are planned for
// these alone: a prefix beside a window, usually a few positions, is read by as few work-groups, however long it is
// (8 single tokens, one KV head, a window of 64: 15 us with a prefix of 4, 50 of 4096, 646 of 60000).
inline int32_t reach_of(int32_t window, int32_t max_q) {
    return window > 0 ? (int32_t)std::min<int64_t>((int64_t)window + max_q + kTileKeys, INT32_MAX) : 0;
}

// Whether work-groups of 128 columns are better than ones of 256, of which there would
// be `groups` without parts, over at most `tiles` tiles of keys (those of the table's width
// or of a window: the lengths are on the device).  Two of 128 share a CU, so that one's
// first and last steps (12 us of a work-group) pass beside the other's products; those of
// 256 read the keys half as often and overlap products and exponentials by their turns.
// 256 and 128 columns, us, 32 heads of 8 KV heads unless said:
//   fewer than half of the CUs
//     8 trees of 16 drafts, 4 heads         29, 24
//   up to four a CU, up to 128 tiles
//     nine prompts of 1-1500, 16 heads      27, 22     one of 2000                       78, 60
//     four of 1193-3434, 16, distances     200, 166    16 of 300                         64, 47
//     8 chunks of 500 behind 4000          336, 289    32 chunks of 100 behind 4000     335, 290
//   where that is the slower side
//     one prompt of 4096                   148, 161    two of 4096                      287, 291
//     32 chunks of 64 behind 4000          175, 198    behind 8000                      340, 403
//     32 chunks of 40 behind 4000          160, 190    64 of 64 behind 4000             388, 400
//   past both
//     four prompts of 4096                 572, 573    32 trees of 64, 4 KV heads      1081, 1163
//   the second list in tables for 128K positions, which take 256 columns for it: 16
//   prompts of 300 67 us (48 in tables of their own width), 8 chunks of 500 341 (295)
inline bool small_blocks(double groups, int64_t tiles) { return groups < device_cus() / 2 || (tiles <= 128 && groups <= 4 * device_cus()); }

struct Shape {
    int32_t cols, blocks, together, reach;  // cols: of a block; 256: the kernel of many queries
    int32_t slots, units, xcds;
    int64_t items;
    Plan plan;
};

// The most columns that the kernel of few queries takes.  64 of them in two blocks of 32 (in one block of 64 a wave's
// registers spill: 8 trees of 16 drafts, 4 heads, 33 us in place of 24) and by the kernel of many queries: 32 trees of 8 drafts, 8 heads a
// KV head, 379 and 354 us; 128 trees of 16 drafts, 4 heads a KV head, 412 and 303; 8 trees of 16, 26.6 and 24.
constexpr int kFewColumns = 32;
constexpr int32_t kMostRequests = 1 << 24;  // (so many and one head are past the grid of either kernel)

inline Shape shape_of(const int32_t* lens, int32_t tokens, int32_t requests, int32_t kv_heads, int32_t group, int32_t max_q, int32_t keys,
                      int32_t window) {
    Shape s;
    s.reach = reach_of(window, max_q);
    const int64_t columns = (int64_t)max_q * group;
    const bool few = columns <= kFewColumns;
    const double groups = (double)requests * cdiv(columns, kBlockColumns) * kv_heads;  // (the largest sizes: past 64 bits)
    const bool small = !few && small_blocks(groups, cdiv(s.reach > 0 ? std::min(keys, s.reach) : keys, kTileKeys));
    s.cols = !few ? (small ? kSmallBlockColumns : kBlockColumns) : columns <= 16 ? 16 : 32;
    s.blocks = (int32_t)cdiv(columns, s.cols);
    s.together = !few ? 1 : kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
    s.slots = s.units = 0, s.xcds = 1;
    if (s.reach > 0) keys = std::min(keys, s.reach);
    const int64_t sets = (int64_t)kv_heads / s.together * s.blocks, streams = few ? kWaves / s.together : 1;
    const int64_t running = std::max<int64_t>(1, device_cus() / sets), tiles = cdiv(keys, kTileKeys);
    // Parts at most, and tiles of a part at least.  Few queries: as many as run at once; where the requests alone are half that
    // many, two for each of the longer ones, unless a window makes them alike: 130 requests of 1000 to 20000 tokens, 32 heads
    // of 8 KV heads, 1013 us in one part each and 625 so; 250 of 8000, 4 KV heads, 685 and 694; 128 of 500, which parts of
    // less than 32 tiles would cut, 46 and 59.  Many queries: enough for two work-groups of 256 columns a CU (32 trees of 64 drafts over
    // 4K-64K tokens 1110 us, three a CU 1056, four 1085; 8 such trees 282, 303, 313), or for twice several requests where that is
    // four a CU or less (8 chunks of 512 behind 1000 to 32000 tokens, 32 heads: 1250 us in one part each, 706 so).
    const bool crowded = few && 2ll * requests > running;
    const int64_t most = !few ? std::max<int64_t>({1, 2 * device_cus() / sets, requests > 1 ? std::min<int64_t>(4 * device_cus() / sets, 2ll * requests) : 0})
                       : crowded && s.reach == 0 ? std::max<int64_t>(running, std::min<int64_t>(4 * running, 2ll * requests)) : running;
    s.plan = Plan{lens, requests, keys, 0, 0, (int32_t)most, !few ? 4 : crowded ? (int32_t)(32 * streams) : 1};
    // (a request of few tiles is one work-group's: the join would take longer than its tiles)
    if (few && tiles <= std::max<int64_t>(4 * streams, s.plan.least)) s.plan.chunk = (int32_t)std::max<int64_t>(1, tiles);
    else if (keys > 0 && planned(requests, tiles) && requests < most)
        s.plan.target = (int32_t)std::max(most - requests, (most + 1) / 2);
    else s.plan.chunk = (int32_t)streams * chunk_for(requests, cdiv(tiles, streams), running, few ? 2 : 6, few ? 1 : 2);
    s.items = items_at_most(s.plan);
    if (!few) {
        // Every request gets as many blocks as the longest can have, unless the blocks that the queries can need are
        // less than a third of those.  Contexts are not cut then: a chunk of 512 tokens and 16 single ones, 32 heads of 8
        // KV heads over 64K each, 1590 us, as two calls 590 and 715.
        const int64_t slots = (int64_t)tokens * group / s.cols + requests;
        if (max_q > 1 && ((int64_t)requests * s.blocks > 3 * slots || (double)(s.items * kv_heads + 7) * s.blocks >= 0x1p32 / 512)) {
            s.slots = (int32_t)slots, s.blocks = 1, s.items = slots;
            s.plan.chunk = (int32_t)std::max<int64_t>(1, tiles);
        }
        const int64_t units = s.items * kv_heads;
        s.xcds = units % 8 == 0 || units >= 64 ? 8 : 1;
        s.units = (int32_t)std::min<int64_t>(units, INT32_MAX);
        s.together = (int32_t)std::max<int64_t>(1, std::min(cdiv(units, s.xcds), cdiv(2 * device_cus() / s.xcds, s.blocks)));
    }
    return s;
}

inline int64_t workspace_of(const Shape& s, int32_t kv_heads) {
    if (s.slots > 0 || (s.plan.chunk > 0 && s.items == s.plan.rows)) return 0;
    return s.items * kv_heads * s.blocks * s.cols * (kDim + 2) * (int64_t)sizeof(float) + (s.plan.chunk > 0 ? 0 : s.plan.rows * (int64_t)sizeof(i32x2));
}

inline Parts parts_of(void* ws, const Shape& s, int32_t kv_heads) {
    const int64_t columns = s.items * kv_heads * s.blocks * s.cols;
    float* sums = static_cast<float*>(ws);
    f32x2* stats = reinterpret_cast<f32x2*>(sums + columns * kDim);
    return {sums, stats, reinterpret_cast<i32x2*>(stats + columns)};
}

template <class T, int NC, int MODE>
int launch_rows(const AttendParams& p, int64_t groups, hipStream_t st) {
    static OncePerDevice once;
    const auto kernel = rows_kernel<T, NC, MODE>;
    const int rc = allow_lds(once, reinterpret_cast<const void*>(kernel), sizeof(RowsLds<NC>), "paged_attend: LDS");
    if (rc != V1_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)groups), dim3(64 * kWaves), sizeof(RowsLds<NC>), st, p);
    return V1_LAUNCHED("paged_attend");
}

template <class T, int NC>
int launch_rows(int mode, const AttendParams& p, int64_t groups, hipStream_t st) {
    return mode == kPlain ? launch_rows<T, NC, kPlain>(p, groups, st) : mode == kCapped ? launch_rows<T, NC, kCapped>(p, groups, st)
         : mode == kBiased ? launch_rows<T, NC, kBiased>(p, groups, st) : launch_rows<T, NC, kBoth>(p, groups, st);
}

template <class T>
int attend(AttendParams& p, const Shape& s, int mode, hipStream_t st) {
    int rc;
    if (s.cols >= kSmallBlockColumns) {
        const int64_t groups = cdiv(s.items * p.kv_heads, s.xcds) * s.xcds * s.blocks;
        V1_REQUIRE(launchable(groups, 512) && s.items * p.kv_heads <= INT32_MAX, "paged_attend: too many requests, queries and heads for a launch");
        rc = launch_blocks(__is_same(T, _Float16), s.cols, mode, p, groups, st);
    } else {
        const int64_t sets = (int64_t)p.kv_heads / s.together * s.blocks;
        const int64_t spread = s.plan.chunk > 0 ? cdiv(s.items * sets, 8) : cdiv(s.items, 8) * sets;
        V1_REQUIRE(launchable(8 * spread, 64 * kWaves), "paged_attend: too many requests and heads for a launch");
        p.spread = (int32_t)spread;
        rc = s.cols == 16 ? launch_rows<T, 1>(mode, p, 8 * spread, st) : launch_rows<T, 2>(mode, p, 8 * spread, st);
    }
    if (rc != V1_OK || workspace_of(s, p.kv_heads) == 0) return rc;
    // (about as many groups as a request has parts)
    const int64_t parts = cdiv(s.items, p.requests);
    return parts > 8 ? launch_join<T, 8>(p, s.cols, st) : parts > 2 ? launch_join<T, 2>(p, s.cols, st) : launch_join<T, 1>(p, s.cols, st);
}

}  // namespace
}  // namespace v1

using namespace v1;

extern "C" int64_t v1_paged_attend_workspace(int32_t tokens, int32_t requests, int32_t kv_heads, int32_t group, int32_t max_q,
                                             int32_t keys, int32_t window) {
    if (tokens <= 0 || requests <= 0 || kv_heads <= 0 || group <= 0 || max_q <= 0 || keys <= 0) return 0;
    if ((int64_t)kv_heads * group >= 1 << 15 || (int64_t)tokens * group > kMostKeys || keys > kMostKeys || requests >= kMostRequests)
        return 0;  // (refused by the entry)
    max_q = std::min(max_q, tokens);
    return workspace_of(shape_of(nullptr, tokens, requests, kv_heads, group, max_q, keys, window), kv_heads);
}

extern "C" int v1_paged_attend(const v1_paged_attend_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "paged_attend: null arguments");
    auto [q, q_token, q_head, k_pool, kp_page, kp_token, kp_head, v_pool, vp_page, vp_token, vp_head, pages, table,
          table_stride, lens, cu_q, prefix, document, parents, slopes, out, o_token, o_head, lse, workspace,
          workspace_bytes, table_len, tokens, requests, max_q, kv_heads, group, window, fp16, scale, softcap] = *a;
    max_q = cu_q ? std::min(max_q, tokens) : 1;
    V1_REQUIRE(tokens >= 0 && requests >= 0 && max_q >= 0 && kv_heads > 0 && group > 0 && pages >= 0 && table_len >= 0 &&
                   window >= 0 && (int64_t)kv_heads * group < 1 << 15,
               "paged_attend: bad shape");
    V1_REQUIRE((int64_t)table_len * kTileKeys <= kMostKeys && (int64_t)tokens * group <= kMostKeys, "paged_attend: too many keys or queries");
    V1_REQUIRE(requests < kMostRequests, "paged_attend: too many requests for a launch");
    V1_REQUIRE(cu_q != nullptr || tokens == requests, "paged_attend: one query for each request");
    V1_REQUIRE(parents == nullptr || (max_q <= kMostDrafts && document == nullptr && prefix == nullptr),
               "paged_attend: at most %d drafted tokens of a request", kMostDrafts);
    V1_REQUIRE(scale > 0.f && scale * kLog2e < __builtin_inff(), "paged_attend: scale must be positive and finite");
    V1_REQUIRE(softcap >= 0.f && (softcap == 0.f || (softcap >= 0x1p-126f && softcap * 4.f < __builtin_inff() && scale / softcap >= 0x1p-126f &&
                                                      scale / softcap < __builtin_inff())),
               "paged_attend: softcap must be zero or positive, and softcap and scale / softcap normal numbers");
    V1_REQUIRE(paged::aligned16(q) && (q_token | q_head) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0 && (o_token | o_head) % 4 == 0,
               "paged_attend: q must be 16-byte aligned with strides in multiples of 8, out 8-byte and 4");
    V1_REQUIRE(paged::aligned16(k_pool) && paged::aligned16(v_pool) &&
                   (kp_page | kp_token | kp_head | vp_page | vp_token | vp_head) % 8 == 0,
               "paged_attend: pools must be 16-byte aligned with strides in multiples of 8");
    V1_REQUIRE(kp_token >= 0 && kp_token < 1 << 25 && vp_token >= 0 && vp_token < 1 << 25,
               "paged_attend: a page's tokens must lie less than 2^25 numbers apart");
    if (tokens == 0 || requests == 0 || max_q == 0) return V1_OK;
    if (pages == 0) table_len = 0;
    const int32_t keys = table_len * kTileKeys;
    const Shape s = shape_of(lens, tokens, requests, kv_heads, group, max_q, keys, window);
    const int64_t need = workspace_of(s, kv_heads);
    V1_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr), "paged_attend: workspace of %lld bytes needed", (long long)need);
    const float in = softcap > 0.f ? scale / softcap : 0.f;
    const int mode = softcap == 0.f ? (slopes ? kBiased : kPlain) : slopes ? kBoth : kCapped;
    AttendParams p{static_cast<const uint16_t*>(q), q_token, q_head,
                   {static_cast<const uint16_t*>(k_pool), static_cast<const uint16_t*>(v_pool)}, {kp_page, vp_page},
                   {kp_token, vp_token}, {kp_head, vp_head}, pages, table, table_stride, lens, cu_q, prefix, document,
                   parents, slopes, table_len, tokens, requests, max_q, kv_heads, group, small_div_magic((uint32_t)group),
                   window, scale * kLog2e, in, softcap * kLog2e, cap_of(scale, softcap),
                   static_cast<uint16_t*>(out), o_token, o_head, lse, s.plan, s.blocks, 0, s.together,
                   s.units, s.xcds, s.slots, parts_of(workspace, s, kv_heads)};
    return fp16 ? attend<_Float16>(p, s, mode, as_stream(stream)) : attend<__bf16>(p, s, mode, as_stream(stream));
}
