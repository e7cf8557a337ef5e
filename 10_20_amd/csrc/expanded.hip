// Attention of ragged sequences over keys and values expanded per head from the
// latent: q [tokens, heads, 128 + 64], kv [keys, heads, 128 key | 128 value]
// numbers, one rope key [keys, 64] for all heads, bf16:
//   S[i, j] = scale * (q[i, 0:128] . k_j + q[i, 128:192] . rope_j),  O[i] = sum_j softmax_j(S[i, :]) v_j,
// query i of a sequence of nq queries and nk keys sees keys j <= nk - nq + i
// (causal) or all.
//
// A work-group of 8 waves takes 256 queries of one head; each wave its own 32, as
// columns of v_mfma_f32_32x32x16_bf16:
//   scores  S^T = K Q^T, a tile of 64 keys at a time from LDS;
//   output  O^T = V^T P^T: a lane's scores are already the probabilities of its
//           B fragment (the key order inside 16 keys is chosen so), rounded to
//           bf16 once, 2^-8 of each at most, as the output is (1.38 times the error of
//           a rounded exact result; a second number for the rest would be 16 products
//           more beside a tile's 40, of the units that bound the kernel); V comes
//           transposed from LDS (ds_read_b64_tr_b16).
// Scores, maxima and sums stay fp32, exponentials are base 2.  Tiles come memory
// -> LDS two ahead; rows are laid with their 16-byte chunks XORed by the row so
// that the fragments' reads meet different banks.
//
// Bound by the matrix units at the clock under load: 16 heads of 4096 queries over
// 32768 keys take 1136-1185 us by card, 1090-1134 TFLOP/s (an 8192^3 library product:
// 1210).  On the way there: both waves of a SIMD in the same step, products and
// exponentials by turns, 1336; fragments' reads where the compiler puts them 1233;
// copies in one piece behind the barrier 1187.  Short sequences are bound by their
// longest block, 8 us and 1.7 for each tile of its keys: 16 heads of 256 queries and
// keys 15.6 us (18.7 with queries and outputs straight from and to the fragments, 32
// rows' lines an instruction).
// Work-groups of 128 queries, two to a CU, took 1800 us where this form took 1233, 326
// against 312 for 32 sequences of 100 queries and 4096 keys, and were ahead only below
// some 300 keys a sequence (64 sequences of 300, 8 heads: 70 against 78 us).  Parts by a
// plan from the lengths, so that the longest blocks alone are cut, took 36 us for
// nine prompts of 1 to 1000 tokens (39 without parts), but 95 for nine of 1500 (54).
#include "attn.h"

namespace v1 {
namespace {

using namespace attn;

constexpr int kKey = 128, kValue = 128, kRopeDims = 64;
constexpr int kRows = 32;  // queries of a wave
constexpr int kWaves = 8, kBlock = kWaves * kRows;  // of a work-group
constexpr int kBuffers = 4;  // tiles in LDS: all of its 160 KB

using f32x16 = __attribute__((ext_vector_type(16))) float;
using i16x4 = __attribute__((ext_vector_type(4))) short;

struct ExpandedParams {
    const uint16_t* q;
    int64_t q_row, q_head;
    const uint16_t* kv;
    int64_t kv_row, kv_head;
    const uint16_t* rope;
    int64_t rope_row;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int32_t tokens, keys, batch, heads, max_q;
    int32_t blocks;           // of every sequence; 0: windows of slots
    int32_t window, windows;  // blocks or slots of one, and their number
    int32_t causal, parts, xcds, group;
    float scale2;
    uint16_t* out;
    int64_t o_row, o_head;
    float* lse;
    bool by_sequence;  // workspace rows: max_q for each sequence, else one for each token
    Parts partial;
};

struct ExpandedTile {
    uint8_t key[kTileKeys][2 * kKey];
    uint8_t value[kTileKeys][2 * kValue];
    uint8_t rope[kTileKeys][2 * kRopeDims];
};

__device__ __forceinline__ f32x16 mfma32(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}

// Keys that query i of a sequence sees: the first of them.
__device__ __forceinline__ int32_t keys_seen(const ExpandedParams& p, int32_t before, int32_t nk, int32_t i) {
    return p.causal ? min(max(before + i + 1, 0), nk) : nk;
}

struct Work {
    // the sequence of its block: where its queries begin, how many there are (max_q at
    // most), its keys, and those before its first query (nk less all of its queries)
    int32_t q_lo, nq, k_lo, nk, before;
    int32_t q0;   // the block's first query there
    int32_t row;  // its row in the workspace
    int32_t head, part;
};

// Slots: sequence b's blocks of queries lie in slots cu_q[b] / kBlock + b and on, as many as
// its queries can need wherever they begin; tokens / kBlock + batch in all, taken in
// windows of a wave's lanes.
constexpr int kWindow = kWave;

// The block of the window with the rank-th most tiles of keys (equal ones in the
// slots' order); false: there are no more.  Every wave finds it by itself, in two
// rounds of loads for up to 64 sequences and one more for every factor of 64.
__device__ __forceinline__ bool find_block(const ExpandedParams& p, int32_t window, int32_t rank, Work& w) {
    const int32_t lane = (int32_t)threadIdx.x % kWave, first = window * kWindow, slot = first + lane;
    int32_t from = 0;  // a sequence whose slots begin at the first one or before: the lanes take 64 from there on
    if (p.batch > kWave) {
        auto start = [&](int32_t b) __attribute__((always_inline)) { return min(max(p.cu_q[b], 0), p.tokens) / kBlock + b; };
        for (int32_t n = p.batch; n > 1;) {
            const int32_t step = (n + kWave - 1) / kWave;
            const bool past = lane * step >= n || start(from + min(lane * step, n - 1)) > first;
            const int32_t skip = (max(__popcll(__ballot(!past)), 1) - 1) * step;
            from += skip;
            n = min(step, n - skip);
        }
        from = __builtin_amdgcn_readfirstlane(from);
    }
    const int32_t b = from + lane, at = min(b, p.batch - 1);
    int32_t ends[4] = {p.cu_q[at], p.cu_q[at + 1], p.cu_k[at], p.cu_k[at + 1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(ends[i]));  // (one wait for the four)
    int32_t q_lo = min(max(ends[0], 0), p.tokens), nq = min(max(ends[1], q_lo), p.tokens) - q_lo;
    int32_t k_lo = min(max(ends[2], 0), p.keys), nk = min(max(ends[3], k_lo), p.keys) - k_lo, before = nk - nq;
    nq = min(nq, p.max_q);
    int32_t begin = b >= p.batch ? INT32_MAX : q_lo / kBlock + b;
    int32_t j = 0;  // from the sequences' lanes to the slots'
#pragma unroll
    for (int step = kWave / 2; step > 0; step /= 2)
        if (__shfl(begin, j + step, kWave) <= slot) j += step;
    q_lo = __shfl(q_lo, j, kWave), nq = __shfl(nq, j, kWave);
    k_lo = __shfl(k_lo, j, kWave), nk = __shfl(nk, j, kWave);
    begin = __shfl(begin, j, kWave), before = __shfl(before, j, kWave);
    const int32_t q0 = slot < begin ? nq : (slot - begin) * kBlock;
    // bit by bit of the number of tiles, from the largest: those with the bit come first
    const int32_t tiles = tiles_of(keys_seen(p, before, nk, min(q0 + kBlock, nq) - 1));
    uint64_t left = __ballot(lane < p.window && q0 < nq);
    if (rank >= __popcll(left)) return false;
    for (int32_t bit = 31 - __clz(tiles_of(p.keys) | 1); bit >= 0; --bit) {
        const uint64_t more = __ballot((tiles >> bit) & 1) & left;
        const int32_t n = __popcll(more);
        left = rank < n ? more : left & ~more;
        rank -= rank < n ? 0 : n;
    }
    const uint64_t who = __ballot(((left >> lane) & 1) && (int32_t)lanes_below(left) == rank);
    const int32_t src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
    w.q_lo = __builtin_amdgcn_readlane(q_lo, src), w.nq = __builtin_amdgcn_readlane(nq, src);
    w.k_lo = __builtin_amdgcn_readlane(k_lo, src), w.nk = __builtin_amdgcn_readlane(nk, src);
    w.before = __builtin_amdgcn_readlane(before, src), w.q0 = __builtin_amdgcn_readlane(q0, src);
    w.row = w.q_lo + w.q0;  // (by_sequence has fewer rows than tokens, batch x max_q, and then blocks are fewer than slots)
    return true;
}

// The work-group's part of the attention; false: there is none.  (Found by the
// kernel before the rest: inside expanded_part its loops cost the tiles' loop its registers.)
__device__ __forceinline__ bool find_work(const ExpandedParams& p, Work& w) {
    // Work-groups reach the XCDs in turn.  An XCD takes whole units, a head of a sequence
    // or of a window, `group` of them at a time: the group's blocks longest first, so that
    // the last ones to end are short and blocks of the same keys meet in one L2.
    // Of 4 sequences of 4096, 32 heads: a pair at a time 803 us, so 740; of 2 times
    // 4096 queries, 16384 keys, 128 heads: all pairs at a time 10290 us, so 9200.
    const int32_t per = p.window * p.parts, units = (p.windows * p.heads + p.xcds - 1) / p.xcds;
    const int32_t turn = (int32_t)blockIdx.x / p.xcds, before = turn / (p.group * per) * p.group;
    const int32_t size = min(p.group, units - before), within = turn - before * per, at = within / size;
    const int32_t index = (before + within % size) * p.xcds + (int32_t)blockIdx.x % p.xcds;
    const int32_t rank = at / p.parts, b = index / p.heads;
    w.part = at % p.parts, w.head = index % p.heads;
    if (b >= p.windows) return false;
    if (p.blocks == 0) return find_block(p, p.windows - 1 - b, rank, w);
    int32_t ends[4] = {p.cu_q[b], p.cu_q[b + 1], p.cu_k[b], p.cu_k[b + 1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(ends[i]));  // (one wait for the four)
#pragma unroll
    for (int i = 0; i < 4; ++i) ends[i] = __builtin_amdgcn_readfirstlane(ends[i]);
    w.q_lo = min(max(ends[0], 0), p.tokens), w.nq = min(max(ends[1], w.q_lo), p.tokens) - w.q_lo;
    w.k_lo = min(max(ends[2], 0), p.keys), w.nk = min(max(ends[3], w.k_lo), p.keys) - w.k_lo;
    w.before = w.nk - w.nq, w.nq = min(w.nq, p.max_q);
    w.q0 = (p.blocks - 1 - rank) * kBlock;
    w.row = (p.by_sequence ? b * p.max_q : w.q_lo) + w.q0;
    return w.q0 < w.nq;
}

// Reads of LDS, EACH for one matrix product, kAhead products before it.
constexpr int kAhead = 4;
template <int N, int EACH>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, EACH * kAhead, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + kAhead < N) __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
}

// A fragment of V^T, rows 32 d .., of 16 keys 16 kk ..: lanes 4r .. 4r + 3 of a
// group of 16 hand in 16 columns of a key, lane n gets column n of four keys.
__device__ __forceinline__ Frag values(const ExpandedTile& tile, int kk, int d) {
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

// bf16 pairs without their infinities and NaN (zeros there), and with 1.0 where
// the number is +inf or NaN, or -inf or NaN.
__device__ __forceinline__ void split_odd(uint32_t w, uint32_t& plain, uint32_t& pos, uint32_t& neg) {
    plain = pos = neg = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t x = (w >> (16 * half)) & 0xffffu;
        const bool odd = (x & 0x7f80u) == 0x7f80u, nan = odd && (x & 0x7fu) != 0;
        plain |= (odd ? 0u : x) << (16 * half);
        pos |= (odd && (nan || x == 0x7f80u) ? 0x3f80u : 0u) << (16 * half);
        neg |= (odd && (nan || x == 0xff80u) ? 0x3f80u : 0u) << (16 * half);
    }
}

// The product of a tile with masked keys where a value may be infinite or NaN:
// the finite values as they are, and counts of the +inf and -inf (NaN: both)
// that each query sees.
__device__ __forceinline__ void careful_product(f32x16 (&sums)[4], const Frag (&p)[4], const ExpandedTile& tile,
                                                int32_t left) {
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
                split_odd(v.w[i], plain.w[i], pos.w[i], neg.w[i]);
                const int32_t key = 16 * kk + 8 * (i / 2) + 2 * (i & 1);  // (of the lane's numbers 2i, 2i + 1)
                see.w[i] = (key < left ? 0x3f80u : 0u) | (key + 1 < left ? 0x3f800000u : 0u);
            }
            sums[d] = mfma32(plain, p[kk], sums[d]);
            up = mfma32(pos, see, up);
            down = mfma32(neg, see, down);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sums[d][i] += (up[i] > 0.f ? __builtin_inff() : 0.f) - (down[i] > 0.f ? __builtin_inff() : 0.f);
    }
}

// The work-group's part of the attention.  A masked key's probability is zero,
// which an infinite or NaN value would turn into NaN in the product: sums that
// end up not finite (true is returned, nothing written) are found again by the
// CAREFUL form.
template <bool CAREFUL>
__device__ __forceinline__ bool expanded_part(const ExpandedParams& p, const Work& w, ExpandedTile* lds) {
    constexpr int COPIES = (int)(sizeof(ExpandedTile) / 1024) / kWaves;
    static_assert(COPIES == 5 && kWaves * 4 * 2 == kTileKeys, "copies of a tile");
    const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave);
    const int32_t lane = (int32_t)threadIdx.x % kWave, c = lane & 31, h = lane >> 5;

    const int32_t q_lo = w.q_lo, nq = w.nq, k_lo = w.k_lo, nk = w.nk, before = w.before, q0 = w.q0, head = w.head, part = w.part;
    auto seen = [&](int32_t i) __attribute__((always_inline)) { return keys_seen(p, before, nk, i); };
    const int32_t i0 = q0 + wave * kRows;                                // this wave's first query
    const int32_t my_seen = seen(min(i0 + c, nq - 1));
    const int32_t wave_least = i0 < nq ? seen(i0) : 0, wave_most = i0 < nq ? seen(min(i0 + kRows, nq) - 1) : 0;
    const int32_t all_tiles = tiles_of(seen(min(q0 + kBlock, nq) - 1));
    const int32_t each = (all_tiles + p.parts - 1) / p.parts;
    const int32_t first = min(part * each, all_tiles), tiles = min(each, all_tiles - first);

    // Copy j of the wave's five of a tile: four keys twice, four values twice, eight
    // rows of rope numbers.  (Rows and tiles past the last are copies of the last key.)
    auto copy = [&](int32_t t, auto which) __attribute__((always_inline)) {
        constexpr int j = which.value;
        ExpandedTile& to = lds[t % kBuffers];
        const int32_t k0 = (first + t) * kTileKeys;
        if constexpr (j < 4) {
            const int32_t i = (j & 1) * kWaves + wave, r = 4 * i + (lane >> 4), at = lane & 15;
            const int32_t chunk = j < 2 ? at ^ (r & 15) : 16 + (at ^ (4 * (r & 3)));
            const int64_t key = k_lo + min(k0 + r, nk - 1);
            copy_to_lds(p.kv + key * p.kv_row + head * p.kv_head + 8 * chunk,
                        lds_offset(j < 2 ? &to.key[4 * i][0] : &to.value[4 * i][0]));
        } else {
            const int32_t r = 8 * wave + (lane >> 3);
            const int64_t key = k_lo + min(k0 + r, nk - 1);
            copy_to_lds(p.rope + key * p.rope_row + 8 * ((lane & 7) ^ (r & 7)), lds_offset(&to.rope[8 * wave][0]));
        }
    };
    auto copy_tile = [&](int32_t t) __attribute__((always_inline)) {
        each_of<COPIES>([&](auto j) __attribute__((always_inline)) { copy(t, j); });
    };

    // B fragments of Q^T: column c = query i0 + c.  The rows come through LDS (rows of
    // 24 chunks of 16 bytes end to end, eight of them XORed by the row, in the last
    // three buffers): fragments read from memory are 32 rows' lines for every one.
    Frag q[12];
    {
        uint8_t* const rows = reinterpret_cast<uint8_t*>(lds + kBuffers) - (kWaves - wave) * (kRows * 2 * (kKey + kRopeDims));
#pragma unroll
        for (int j = 0; j < 12; ++j) {
            const int32_t r = (kWave * j + lane) / 24, chunk = (kWave * j + lane) % 24;
            copy_to_lds(p.q + (q_lo + (int64_t)min(i0 + r, nq - 1)) * p.q_row + head * p.q_head + 8 * (chunk ^ (r & 7)),
                        lds_offset(rows + 1024 * j));
        }
        if (tiles > 0) {
            copy_tile(0);
            wait_copies<COPIES>();
        } else {
            wait_copies<0>();
        }
#pragma unroll
        for (int s = 0; s < 12; ++s)
            q[s].u = *reinterpret_cast<const u32x4*>(rows + 384 * c + 16 * ((2 * s + h) ^ (c & 7)));
        lds_barrier();
        if (tiles > 0) copy_tile(1);
    }
    f32x16 acc[4], s[2];
    Frag pf[4];
    float mx = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    auto first_key = [&](int32_t t) __attribute__((always_inline)) { return (first + t) * kTileKeys; };
    // a key of the tile that a query of the wave does not see
    auto is_masked = [&](int32_t t) __attribute__((always_inline)) { return first_key(t) + kTileKeys > wave_least; };
    // scores: register i of half u is key 32u + 8 (i / 4) + 4h + i % 4
    auto scores = [&](int32_t t) __attribute__((always_inline)) {
        const ExpandedTile& tile = lds[t % kBuffers];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
        // key rows 32u .., numbers 16 (n / 2) ..
        Frag k[kAhead];
        auto fetch = [&](int n) __attribute__((always_inline)) {
            const int32_t st = n / 2, r = 32 * (n & 1) + c;
            k[n % kAhead].u = *reinterpret_cast<const u32x4*>(st < 8 ? &tile.key[r][16 * ((2 * st + h) ^ (r & 15))]
                                                                     : &tile.rope[r][16 * ((2 * st - 16 + h) ^ (r & 7))]);
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) fetch(n);
        each_of<24>([&](auto number) __attribute__((always_inline)) {
            constexpr int n = number.value;
            s[n & 1] = mfma32(k[n % kAhead], q[n / 2], s[n & 1]);
            if constexpr (n + kAhead < 24) fetch(n + kAhead);
            if constexpr (n % 4 == 1 && n / 4 < COPIES) copy(t + 2, Number<n / 4>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto softmax = [&](int32_t t) __attribute__((always_inline)) {
        if (is_masked(t)) {
            const int32_t left = my_seen - first_key(t) - 4 * h;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * u + 8 * (i / 4) + i % 4 >= left) s[u][i] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        top = fmaxf(top, __shfl_xor(top, 32, kWave)) * p.scale2;
        if (__ballot(top > mx + kLag)) {
            const float next = top > mx + kLag ? top : mx;
            const float keep = mx == -__builtin_inff() ? (next == mx ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mx - next);
            mx = next;
            total *= keep;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= keep;
        }
        const float sub = mx == -__builtin_inff() ? 0.f : mx;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], p.scale2, -sub));
                total += s[u][i];
            }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pf[kk].w[i] = pack_bf16(s[kk / 2][8 * (kk & 1) + 2 * i], s[kk / 2][8 * (kk & 1) + 2 * i + 1]);
    };
    auto products = [&](int32_t t) __attribute__((always_inline)) {
        const ExpandedTile& tile = lds[t % kBuffers];
        if (CAREFUL && is_masked(t)) {
            careful_product(acc, pf, tile, my_seen - first_key(t) - 4 * h);
        } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[d] = mfma32(values(tile, kk, d), pf[kk], acc[d]);
            reads_ahead<16, 2>();
        }
    };
    const int32_t mine = min(tiles, max(tiles_of(wave_most) - first, 0));  // tiles that the wave sees something of
    // The two waves of a SIMD half a tile apart: one multiplies (the last tile's
    // values, this one's keys) and asks for its copies of the tile after the next,
    // whose buffer was read until two steps ago, while the other makes
    // probabilities.  Steps are divided by barriers, every other one of them behind a
    // wait for the copies of the tile whose keys come next.  (The copies in one piece
    // behind the barrier hold both waves up: 800 of a tile's 6300 cycles.)
    const bool second = wave >= kWaves / 2;
    auto sync = [&](bool landed) __attribute__((always_inline)) {
        if (landed) wait_barrier<COPIES>();
        else lds_barrier();
    };
    if (second) sync(true);
#pragma unroll 1
    for (int32_t t = 0; t <= tiles; ++t) {
        sync(!second);
        if (t > 0 && t <= mine) products(t - 1);
        if (t < mine) scores(t);
        else if (t < tiles) copy_tile(t + 2);
        sync(second);
        if (t < mine) softmax(t);
    }
    if (!second) lds_barrier();
    wait_copies<0>();
    __syncthreads();  // the tiles' memory is free
    if constexpr (!CAREFUL) {
        float odd = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) odd = fmaf(acc[d][i], 0.f, odd);
        int32_t* const flags = reinterpret_cast<int32_t*>(lds);
        const bool mine_odd = __ballot(odd != odd) != 0;
        if (lane == 0) flags[wave] = mine_odd;
        __syncthreads();
        int32_t any = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) any |= flags[w];
        if (__builtin_amdgcn_readfirstlane(any)) {
            __syncthreads();
            return true;
        }
    }
    total += __shfl_xor(total, 32, kWave);
    const bool none = my_seen <= first * kTileKeys;  // no key seen
    // Rows leave through LDS as well, whole ones at a time: row c's numbers 32 d + 8 a
    // + 4 h .. are its piece 8 d + 2 a + h of four, pieces XORed by the row.
    static_assert(kBuffers * sizeof(ExpandedTile) >= kWaves * (kRows * 4 * kValue + 4), "rows and the flags before them");
    uint8_t* const rows = reinterpret_cast<uint8_t*>(lds + kBuffers) - (kWaves - wave) * (kRows * 4 * kValue);
    const int32_t left = nq - i0;
    if (p.parts == 1) {
        const float inv = none ? 0.f : 1.0f / total;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                *reinterpret_cast<u32x2*>(rows + 256 * c + 8 * ((8 * d + 2 * a + h) ^ c)) =
                    none ? u32x2{0, 0} : u32x2{pack_bf16(acc[d][4 * a] * inv, acc[d][4 * a + 1] * inv),
                                               pack_bf16(acc[d][4 * a + 2] * inv, acc[d][4 * a + 3] * inv)};
        wait_lds();
#pragma unroll
        for (int j = 0; j < kRows / 2; ++j) {
            const int32_t r = 2 * j + h;
            const u32x2 x = *reinterpret_cast<const u32x2*>(rows + 256 * r + 8 * (c ^ r));
            if (r < left) *reinterpret_cast<u32x2*>(p.out + (q_lo + i0 + r) * p.o_row + head * p.o_head + 4 * c) = x;
        }
        if (p.lse && h == 0 && c < left)
            p.lse[(int64_t)(q_lo + i0 + c) * p.heads + head] = none ? -__builtin_inff() : (mx + __builtin_amdgcn_logf(total)) * kLn2;
    } else {
        const int64_t at = ((int64_t)(w.row + wave * kRows) * p.parts + part) * p.heads + head, step = (int64_t)p.parts * p.heads;
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
            if (r < left) *reinterpret_cast<f32x4*>(p.partial.sums + (at + r * step) * kValue + 4 * c) = x;
        }
        if (h == 0 && c < left) p.partial.stats[at + c * step] = f32x2{none ? mx : fmaxf(mx, kLowest), total};
    }
    return false;
}

// (A call, so that its registers are not the common form's.)
__device__ __attribute__((noinline)) void careful_part(ExpandedParams p, ExpandedTile* lds) {
    Work w;
    if (find_work(p, w)) expanded_part<true>(p, w, lds);
}

__global__ __launch_bounds__(64 * kWaves, 2) void expanded_kernel(ExpandedParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    ExpandedTile* const lds = reinterpret_cast<ExpandedTile*>(lds_raw);
    Work w;
    if (!find_work(p, w)) return;
    // (as they are from here on: without this line 27 more scalar registers spill, 0.7 us of a work-group)
    asm volatile("" : "+s"(w.q_lo), "+s"(w.nq), "+s"(w.k_lo), "+s"(w.nk), "+s"(w.before), "+s"(w.q0), "+s"(w.row), "+s"(w.head), "+s"(w.part));
    if (__builtin_expect(expanded_part<false>(p, w, lds), 0)) careful_part(p, lds);
}

// Blocks of queries, and the parts that the keys are cut into where the blocks
// leave CUs without one (of four tiles or more each): 512 queries of 16 heads over
// 32768 keys 187 us in eight parts, one for each CU; in sixteen 202.
//
// Every sequence gets as many blocks as the longest can have, unless the slots are less
// than a third of those: an empty work-group takes all of a CU's LDS for the time of its
// loads, finding a slot's block takes 2-3 us of a work-group.  Blocks and slots, us:
//   9 prompts of 1 to 1000 tokens, 16 heads      36, 16          35.7, 36.7
//   200 of 10 to 3000, 8 heads                   2400, 609        610, 592
//   64 of 512, 16 heads, max_q not given         8192, 192        737, 221
//   1000 of 100, 16 heads, max_q not given       391000, 1390   21100, 774
//   63 of 100 and one of 16000, 16 heads         4032, 150       1426, 1301
struct ExpandedShape {
    int32_t blocks, window, windows, parts;
};

inline ExpandedShape expanded_shape(int32_t tokens, int32_t keys, int32_t batch, int32_t heads, int32_t max_q) {
    const int64_t blocks = cdiv(max_q, kBlock), slots = (int64_t)tokens / kBlock + batch, tiles = cdiv(keys, kTileKeys);
    const int64_t groups = std::min(batch * blocks, slots) * heads;
    ExpandedShape s;
    s.parts = (int32_t)std::max<int64_t>(1, std::min(device_cus() / std::max<int64_t>(1, groups), tiles / (4 * (int64_t)batch)));
    if (batch * blocks <= 3 * slots && launchable(((int64_t)batch * heads + 7) * blocks * s.parts, 64 * kWaves)) {
        s.blocks = s.window = (int32_t)blocks;
        s.windows = batch;
    } else {
        s.blocks = 0;
        s.window = (int32_t)std::min<int64_t>(slots, kWindow);
        s.windows = (int32_t)cdiv(slots, s.window);
    }
    return s;
}

// For the join: as many rows of s.parts parts of a tile each as there are tokens, or, if that is less
// (a padded buffer), max_q for each sequence: 256 rows for every work-group at most, 34 MB.
inline Plan rows_of_parts(int32_t tokens, int32_t batch, int32_t max_q, const ExpandedShape& s) {
    return Plan{nullptr, (int32_t)std::min<int64_t>(tokens, (int64_t)batch * max_q), s.parts * kTileKeys, 1, 0, 0};
}

}  // namespace
}  // namespace v1

using namespace v1;

extern "C" int64_t v1_latent_expanded_workspace(int32_t tokens, int32_t keys, int32_t batch, int32_t heads,
                                                int32_t max_q) {
    if (tokens <= 0 || keys <= 0 || batch <= 0 || heads <= 0 || max_q <= 0) return 0;
    const ExpandedShape s = expanded_shape(tokens, keys, batch, heads, max_q);
    return s.parts == 1 ? 0 : attn::parts_bytes(rows_of_parts(tokens, batch, max_q, s), heads, kValue);
}

extern "C" int v1_latent_expanded(const v1_latent_expanded_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "latent_expanded: null arguments");
    auto [q, q_row, q_head, kv, kv_row, kv_head, rope, rope_row, cu_q, cu_k, out, o_row, o_head, lse, workspace,
          workspace_bytes, tokens, keys, batch, heads, max_q, causal, scale] = *a;
    V1_REQUIRE(tokens >= 0 && keys >= 0 && batch >= 0 && heads > 0 && max_q >= 0, "latent_expanded: bad shape");
    V1_REQUIRE(heads < 1 << 16, "latent_expanded: too many heads");
    V1_REQUIRE(keys <= kMostKeys && tokens <= kMostKeys, "latent_expanded: too many tokens or keys");
    V1_REQUIRE(scale > 0.f && scale * kLog2e < __builtin_inff(), "latent_expanded: scale must be positive and finite");
    const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv) | reinterpret_cast<uintptr_t>(rope);
    V1_REQUIRE(all % 16 == 0 && (q_row | q_head | kv_row | kv_head | rope_row) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 8 == 0 && (o_row | o_head) % 4 == 0,
               "latent_expanded: q, kv and rope must be 16-byte aligned with strides in multiples of 8, out 8-byte and 4");
    if (tokens == 0 || batch == 0 || max_q == 0) return V1_OK;
    const ExpandedShape s = expanded_shape(tokens, std::max(keys, 1), batch, heads, max_q);
    const int64_t need = v1_latent_expanded_workspace(tokens, keys, batch, heads, max_q);
    V1_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr),
               "latent_expanded: workspace of %lld bytes needed", (long long)need);
    // XCD by XCD where that leaves few of them short of work (12 heads of 8192 queries
    // 338 us so, 295 in turn; 9 sequences of 1500, 4 heads, 59 either way); groups of
    // two work-groups for each of an XCD's CUs
    const int64_t units = (int64_t)s.windows * heads;
    const int32_t xcds = units % 8 == 0 || units >= 64 ? 8 : 1;
    const int64_t items = cdiv(units, xcds) * xcds * s.window * s.parts;
    V1_REQUIRE(launchable(items, 64 * kWaves), "latent_expanded: too many sequences, queries and heads for a launch");
    const int64_t group = std::min(cdiv(units, xcds), cdiv(2 * device_cus() / xcds, (int64_t)s.window * s.parts));
    const Plan plan = rows_of_parts(tokens, batch, max_q, s);
    const bool by_sequence = plan.rows < tokens;
    ExpandedParams p{static_cast<const uint16_t*>(q), q_row, q_head, static_cast<const uint16_t*>(kv), kv_row, kv_head,
                     static_cast<const uint16_t*>(rope), rope_row, cu_q, cu_k, tokens, keys, batch, heads, max_q, s.blocks, s.window,
                     s.windows, causal, s.parts, xcds, (int32_t)group, scale * kLog2e, static_cast<uint16_t*>(out), o_row, o_head, lse,
                     by_sequence, parts_at(workspace, plan, heads, kValue)};
    const hipStream_t st = as_stream(stream);
    static OncePerDevice once;
    constexpr size_t bytes = kBuffers * sizeof(ExpandedTile);
    int rc = allow_lds(once, reinterpret_cast<const void*>(expanded_kernel), bytes, "latent_expanded: LDS");
    if (rc != V1_OK) return rc;
    hipLaunchKernelGGL(expanded_kernel, dim3((uint32_t)items), dim3(64 * kWaves), bytes, st, p);
    rc = V1_LAUNCHED("latent_expanded");
    if (rc != V1_OK || s.parts == 1) return rc;
    JoinParams j{plan, p.partial, p.out, o_row, o_head, lse, heads, cu_q, tokens, batch, max_q, by_sequence};
    return launch_join<kValue>(j, st, "latent_expanded: join");
}
