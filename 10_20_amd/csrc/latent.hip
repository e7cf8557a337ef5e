// Latent K/V cache rows of 656 bytes (512 e4m3 codes, 64 bf16 rope numbers, 4
// fp32 scales, one for 128 codes) and attention over them with queries that
// already carry the key projection ("absorbed" form): one shared row of 512 + 64
// numbers is every head's key, its first 512 every head's value,
//   S[h, j] = scale * (q[h, 0:512] . c_j + q[h, 512:576] . r_j),
//   O[h] = sum_j softmax_j(S[h, :]) c_j,  c_j[d] = code_j[d] * s_j[d / 128].
#include "attn.h"

namespace v1 {
namespace {

using namespace attn;

constexpr int kLatent = 512, kRope = 64, kRowBytes = 656, kScaleBlocks = 4;
constexpr int kRopeAt = kLatent, kScaleAt = kLatent + 2 * kRope;
constexpr int kChunks = kRowBytes / 16;
constexpr int kTileBytes = kTileKeys * kRowBytes;

// ------------------------------------------------------------------ store
// One wave per token: lane l holds numbers 8l .. 8l + 7; the 16 lanes of a
// block of 128 find its largest magnitude (four lanes' worth of shuffles; a token
// per work-group would leave the loads of one wave to wait for).  Codes are rounded
// once, to nearest even, at a power of two: x / s is exact.  Bound by memory, 1152
// bytes read and 656 written a token: 16384 tokens to random rows 8.5 us, 3.5 TB/s;
// 128 tokens 2.9 us, a launch and two dependent loads.
struct StoreParams {
    const uint16_t* latent;
    int64_t latent_stride;
    const uint16_t* rope;
    int64_t rope_stride;
    const int32_t* slots;
    int32_t tokens;
    uint8_t* pool;
    int64_t pool_rows, pool_stride;
};

__global__ __launch_bounds__(256) void latent_store_kernel(StoreParams p) {
    const int32_t t = (int32_t)(blockIdx.x * 4 + threadIdx.x / kWave), lane = (int32_t)threadIdx.x % kWave;
    if (t >= p.tokens) return;
    const int32_t slot = p.slots[t];
    const u32x4 x = *reinterpret_cast<const u32x4*>(p.latent + t * p.latent_stride + 8 * lane);
    u32x4 r = {0, 0, 0, 0};
    if (lane < 8) r = *reinterpret_cast<const u32x4*>(p.rope + t * p.rope_stride + 8 * lane);
    if (slot < 0 || slot >= p.pool_rows) return;
    float v[8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(x[i] << 16);
        v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
        amax = fmaxf(amax, fmaxf(finite_abs(v[2 * i]), finite_abs(v[2 * i + 1])));
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, kWave));
    const int e = scale_exponent(amax);
    const float inv = exp2i(-e);  // (e is -126 .. 120)
    uint8_t* row = p.pool + slot * p.pool_stride;
    const u32x2 codes = {codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                         codes4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
    *reinterpret_cast<u32x2*>(row + 8 * lane) = codes;
    if (lane < 8) *reinterpret_cast<u32x4*>(row + kRopeAt + 16 * lane) = r;
    if (lane % 16 == 0) *reinterpret_cast<float*>(row + kScaleAt + lane / 4) = exp2i(e);
}

// --------------------------------------------------------------- absorbed
struct AbsorbedParams {
    const uint16_t* q;
    int64_t q_row, q_head;
    const uint8_t* pool;
    int64_t pool_rows, pool_stride;
    const int32_t* map;  // NULL: ids are rows of the pool
    int64_t map_len, map_stride;
    int32_t map_shift;
    const int32_t* ids;  // NULL: positions 0, 1, ...
    int64_t ids_stride;
    Plan plan;
    int32_t heads, splits, spread;  // splits: work-groups of a row's heads; spread: items on an XCD
    float scale2;
    uint16_t* out;
    int64_t o_row, o_head;
    float* lse;
    Parts parts;
};

// The row of keys that are not attended (their scores are -inf).
__device__ const u32x4 zero_latent[kChunks] = {};

// A tile in LDS: 16-row regions; in a region the rows' chunks of 16 bytes in
// blocks of four, chunk 4j + q of row r at 1024 j + 64 r + 16 (q ^ (r / 4)), then
// the scales, [block][row].  A copy is then 64 bytes of each of 16 rows: its
// address differs from the last one's by a constant (whole rows end to end need
// ten operations a copy for theirs), reads of 16 rows at one place are 1 KB in a
// piece, and the transposing reads of eight rows meet different banks.
constexpr int kRegionRows = 16, kRegion = kRegionRows * kRowBytes, kCopies = 11;
constexpr int kScales = kRegion - kRegionRows * 4 * kScaleBlocks;

template <int HT, int HG>
struct AbsorbedLds {
    static constexpr int kHeads = 16 * HT * HG, kQuarters = 4 / HG;
    uint8_t tile[3][kTileBytes];
    float prob[kHeads][kTileKeys];         // 16-byte chunk n of head h at n ^ (h % 16)
    float scale[kScaleBlocks][kTileKeys];  // of the tile whose probabilities these are
    u32x4 q_rope[HG][HT][2][kWave];        // fragments of the queries' rope numbers
    float hidden[3][kTileKeys];            // 0, or -inf: not attended
    float top[kQuarters][kHeads];
    float keep[kHeads];
    float total[kQuarters][kHeads];
    int32_t ids[4][kWave], pages[4][kWave];
    int32_t seen[4];
};

// (opaque: offsets of the three buffers kept apart for every read of the loop
// take the registers that Q and the sums need)
__device__ __forceinline__ int32_t buffer_of(int32_t t) {
    int32_t b = t % 3;
    asm volatile("" : "+s"(b));
    return b;
}

// Copy j of a tile's region: 16 bytes per lane from `src` + 64 j.  (The
// instruction adds its offset to the address in LDS as well.)
template <int J>
__device__ __forceinline__ void copy_block(uint64_t src, uint32_t region) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%2"
                 :: "v"(src), "s"(__builtin_amdgcn_readfirstlane(region + (1024 - 64) * J)), "n"(64 * J) : "memory", "m0");
}

// A work-group of eight waves attends HB = 16 * HT * HG heads of one row over one
// part of its keys, tile by tile of 64 keys that come memory -> LDS as they are
// stored.  Four waves make the probabilities of tile t while the other four, one
// on each SIMD beside them, multiply those of tile t - 1 with its latents (held in
// registers, so that their buffer is free) and bring in tile t + 2: the products
// keep the matrix cores busy through the others' softmax, and neither kind holds
// both Q and the output (128 registers each at 64 heads; two waves per SIMD have
// 256 each).
//   scores  S^T = K Q^T: wave (hg, kq) takes heads 16 HT hg .. and 16 HG keys;
//           codes become bf16 (exact) as they are read, one accumulator per block
//           of 128 numbers, joined with the block's scales in fp32.
//   softmax the key groups exchange their maxima through LDS; probabilities and
//           their sums stay fp32.
//   output  O^T = C^T P^T: a wave takes a block of 128 columns of all heads: the
//           probabilities times their keys' scale of that block, and its codes
//           transposed by the LDS read (ds_read_b64_tr_b8), exact in bf16.  Up to 32
//           heads the former are two bf16 numbers, which leaves 2^-17 (1 us of 44 for
//           128 rows of 16 heads, 20 of 265 for 1024 rows of 32); 64 heads round them
//           once (2^-8 of each at most, as the output is), since the second products
//           and their 32 registers would cost more than the waves have.
//
// 1024 rows of 128 heads over 2048 chosen rows each: 650-665 us, 834-853 TFLOP/s (an 8192^3
// library product: 1210), bound by the issue of the two waves of a SIMD: a tile of
// 64 heads is 72 products of 16 cycles a wave, and a conversion or fold for every
// third of their cycles; 12 of a work-group's 80 us are its start and end.  128
// rows of 16 heads: 42-50 us with the join, 3.4-4.1 TB/s; in the loop 1.80 us a tile, 6.0
// TB/s (256 rows of 2048 and of 4096 of two million latent rows, 67 and 125 us), where
// copies of random rows to LDS alone reach 6.2.  7 contexts of 5000 to 131072, 64
// heads: 62-70 us, 9 of them the join.  On the way: all eight waves doing both halves, a tile at a time,
// 2786 us for the first; scorers and multipliers apart 1280; products between the
// conversions and the copies 768; tiles by blocks of 16 rows 680.
template <int HT, int HG>
__global__ __launch_bounds__(512, 2) void absorbed_kernel(AbsorbedParams p) {
    constexpr int HB = 16 * HT * HG, KT = HG, KQ = 4 / HG, RPW = kRegionRows, GT = kWave / RPW;
    constexpr int DT = 8, PT = HB / 16;
    constexpr bool TWICE = HB < 64;  // probabilities in two bf16 numbers
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto& lds = *reinterpret_cast<AbsorbedLds<HT, HG>*>(lds_raw);
    const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave) & 3;
    const bool scorer = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave) < 4;
    const int32_t lane = (int32_t)threadIdx.x % kWave;
    int32_t g = lane >> 4, c = lane & 15;  // (opaque in the loops, as buffer_of)

    // Work-groups reach the XCDs in turn: the splits of an item follow each other on one
    // of them, and so do rows of equal capacity, which may choose from one context.
    const int32_t xcd = (int32_t)blockIdx.x % 8, turn = (int32_t)blockIdx.x / 8, split = turn % p.splits;
    const int32_t index = p.plan.chunk > 0 ? xcd * p.spread + turn / p.splits : turn / p.splits * 8 + xcd;
    Item it;
    if (!find_item(p.plan, index, it)) return;
    const int32_t head0 = split * HB, tiles = it.tiles;
    if (p.plan.chunk == 0 && it.part == 0 && split == 0 && threadIdx.x == 0) p.parts.of_row[it.row] = i32x2{index, it.parts};

    if (scorer) {
        const int32_t hg = wave / KQ, kq = wave % KQ;
        // B fragments of Q^T: column c = head c of 16; 64 numbers in two steps: lane
        // group g takes 16g .. 16g + 7 of them, then 16g + 8 .. 16g + 15 (the order in which the codes are read)
        Frag q[HT][16];
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
            const int32_t h = min(head0 + hg * 16 * HT + 16 * ht + c, p.heads - 1);
            const uint16_t* src = p.q + it.row * p.q_row + h * p.q_head;
#pragma unroll
            for (int s = 0; s < 16; ++s)
                q[ht][s].u = *reinterpret_cast<const u32x4*>(src + 64 * (s / 2) + 16 * g + 8 * (s % 2));
            if (kq == 0)  // (read before the first tile's products, behind its barrier)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    lds.q_rope[hg][ht][s][lane] = *reinterpret_cast<const u32x4*>(src + kLatent + 32 * s + 8 * g);
        }
        float mx[HT], total[HT];
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) mx[ht] = -__builtin_inff(), total[ht] = 0.f;

#pragma unroll 1
        for (int32_t t = 0; t < tiles; ++t) {
            asm volatile("" : "+v"(g), "+v"(c));
            lds_barrier();  // tile t has landed; probabilities of tile t - 1 are written
            const int32_t buf = buffer_of(t);
            const uint8_t* const region = lds.tile[buf] + kRegion * KT * kq;
            f32x4 s[KT][HT];  // of keys 16 (KT kq + kt) + 4g + i, heads c
            {
                // Steps of one block of one key tile (the rope numbers are a fifth
                // block, of scale 1, which starts from -inf at the hidden keys).  A
                // step's products are issued between the conversions of the next
                // one's codes, the reads of those after it and the folding of the
                // last one's products: 16 cycles of the matrix core cover three
                // vector operations.
                constexpr int STEPS = KT * 5;
                const uint8_t* const key0 = region + 64 * c + 16 * (g ^ (c >> 2));
                const uint8_t* const scale0 = region + kScales + 16 * g;
                u32x4 raw[2];
                Frag k[4], qr[HT][2];
                f32x4 sc[2], d[2][HT], hidden;
                auto fetch = [&](int n, int half) __attribute__((always_inline)) {
                    if (n < STEPS) raw[half] = *reinterpret_cast<const u32x4*>(key0 + n / 5 * kRegion + 1024 * (2 * (n % 5) + half));
                };
                auto fetch_scale = [&](int n) __attribute__((always_inline)) {
                    if (n < STEPS && n % 5 < kScaleBlocks)
                        sc[n & 1] = *reinterpret_cast<const f32x4*>(scale0 + n / 5 * kRegion + 4 * kRegionRows * (n % 5));
                };
                // quarter m % 4 of step m / 4 (of the rope's step the first two): its fragment, words lo .. hi
                auto convert = [&](int m, int part) __attribute__((always_inline)) {
                    const int n = m / 4, j = m % 4;
                    if (n >= STEPS) return;
                    const u32x4 w = raw[j / 2];
                    if (n % 5 < kScaleBlocks) {
                        k[j].w[2 * part] = codes_pair<0>(w[2 * (j & 1) + part]);
                        k[j].w[2 * part + 1] = codes_pair<1>(w[2 * (j & 1) + part]);
                    } else if (j < 2 && part == 1) {
                        k[j].u = raw[j];
                    }
                    if (part == 1 && (j & 1)) fetch(n + 1, j / 2);
                };
                auto fold = [&](int n, int ht, int i) __attribute__((always_inline)) {
                    if (n < 0) return;
                    const float x = s[n / 5][ht][i], y = d[n & 1][ht][i];
                    s[n / 5][ht][i] = n % 5 == 0 ? sc[n & 1][i] * y : n % 5 < kScaleBlocks ? fmaf(sc[n & 1][i], y, x) : x + y;
                };
#pragma unroll
                for (int half = 0; half < 2; ++half) fetch(0, half);
                fetch_scale(0);
                convert(0, 0), convert(0, 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int m = 0; m < 4 * STEPS; ++m) {
                    const int n = m / 4, b = n % 5, j = m % 4;
                    if (b == kScaleBlocks - 1 && j == 3) {
                        hidden = *reinterpret_cast<const f32x4*>(&lds.hidden[buf][16 * (KT * kq + n / 5) + 4 * g]);
#pragma unroll
                        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                            for (int i = 0; i < 2; ++i) qr[ht][i].u = lds.q_rope[hg][ht][i][16 * g + c];
                    }
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht) {
                        if (j < (b < kScaleBlocks ? 4 : 2))
                            d[n & 1][ht] = mfma16(k[j], b < kScaleBlocks ? q[ht][4 * (b % 4) + j] : qr[ht][j % 2],
                                                  j > 0 ? d[n & 1][ht] : b < kScaleBlocks ? f32x4{0.f, 0.f, 0.f, 0.f} : hidden);
                        if (HT == 1) convert(m + 1, 0);
                        convert(m + 1, HT == 1 ? 1 : ht);
                        fold(n - 1, ht, j);
                        if (ht == HT - 1 && j == 3) fetch_scale(n + 1);  // (after the last use of these registers)
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                    for (int i = 0; i < 4; ++i) fold(STEPS - 1, ht, i);
#pragma unroll
                for (int ht = 0; ht < HT; ++ht) {
                    float top = -__builtin_inff();
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kt][ht][i]);
                    top = fmaxf(top, __shfl_xor(top, 16, kWave));
                    top = fmaxf(top, __shfl_xor(top, 32, kWave));
                    if (g == 0) lds.top[kq][16 * (HT * hg + ht) + c] = top * p.scale2;
                }
            }
            lds_barrier();  // maxima of tile t are there; probabilities of tile t - 1 have been read
            {
                float sub[HT];
                lds.scale[g][16 * wave + c] = *reinterpret_cast<const float*>(lds.tile[buf] + kRegion * wave + kScales + 64 * g + 4 * c);
#pragma unroll
                for (int ht = 0; ht < HT; ++ht) {
                    const int32_t h = 16 * (HT * hg + ht) + c;
                    float top = lds.top[0][h];
#pragma unroll
                    for (int k = 1; k < KQ; ++k) top = fmaxf(top, lds.top[k][h]);
                    float keep = 1.f;
                    if (top > mx[ht] + kLag) {  // (-inf + kLag is -inf)
                        keep = mx[ht] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mx[ht] - top);
                        mx[ht] = top;
                    }
                    sub[ht] = mx[ht] == -__builtin_inff() ? 0.f : mx[ht];
                    total[ht] *= keep;
                    if (kq == 0 && g == 0) lds.keep[h] = keep;
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const int32_t k0 = 16 * (KT * kq + kt);
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht) {
                        const int32_t h = 16 * (HT * hg + ht) + c;
                        f32x4 x;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][ht][i], p.scale2, -sub[ht]));
                            total[ht] += x[i];
                        }
                        *reinterpret_cast<f32x4*>(&lds.prob[h][4 * ((k0 / 4 + g) ^ c)]) = x;
                        __builtin_amdgcn_sched_barrier(0);  // (mixed, the two tiles' values take Q's registers)
                    }
                }
            }
        }
        lds_barrier();  // (the multipliers' last round)
        lds_barrier();
        // totals of the key groups
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
            const int32_t h = 16 * (HT * hg + ht) + c;
            float x = total[ht];
            x += __shfl_xor(x, 16, kWave);
            x += __shfl_xor(x, 32, kWave);
            if (g == 0) lds.total[kq][h] = x;
            if (g == 0 && kq == 0) lds.top[0][h] = mx[ht];
        }
        __syncthreads();
        return;
    }

    // rows of this wave's region of a tile, GT tiles at a time: lane = 16 * tile + row
    const int32_t* ids = p.ids ? p.ids + it.row * p.ids_stride : nullptr;
    const int32_t* map = p.map ? p.map + it.row * p.map_stride : nullptr;
    // Positions and page entries of the groups to come are copied to LDS like the
    // rows: loads into registers would have the compiler wait for every copy in flight.
    auto position = [&](int32_t group) __attribute__((always_inline)) -> int32_t {  // in ids; -1: none
        const int32_t tile = group * GT + g, j = (it.first + tile) * kTileKeys + RPW * wave + c;
        return tile < tiles && j < it.keys ? j : -1;
    };
    auto ask_id = [&](int32_t group) __attribute__((always_inline)) {
        const int32_t j = position(group);
        if (ids) copy4_to_lds(j < 0 ? reinterpret_cast<const int32_t*>(zero_latent) : ids + j, lds_offset(&lds.ids[wave][0]));
    };
    auto take_id = [&](int32_t group) __attribute__((always_inline)) -> int32_t {
        const int32_t j = position(group);
        return j < 0 ? -1 : ids ? lds.ids[wave][16 * g + c] : j;
    };
    auto ask_page = [&](int32_t id) __attribute__((always_inline)) {
        const int64_t e = (int64_t)id >> p.map_shift;
        if (map) copy4_to_lds(id < 0 || e >= p.map_len ? reinterpret_cast<const int32_t*>(zero_latent) : map + e,
                              lds_offset(&lds.pages[wave][0]));
    };
    auto take_row = [&](int32_t id) __attribute__((always_inline)) -> int32_t {
        if (id < 0) return -1;
        int64_t row = id;
        if (map) {
            const int32_t m = lds.pages[wave][16 * g + c];
            if (((int64_t)id >> p.map_shift) >= p.map_len || m < 0) return -1;
            row = ((int64_t)m << p.map_shift) | (id & ((1 << p.map_shift) - 1));
        }
        return row < p.pool_rows ? (int32_t)row : -1;
    };
    const uint64_t nowhere = reinterpret_cast<uint64_t>(zero_latent);
    bool seen = false;  // a key that is attended
    auto address = [&](int32_t row) __attribute__((always_inline)) -> uint64_t {
        seen |= __ballot(row >= 0) != 0;
        return row < 0 ? nowhere : reinterpret_cast<uint64_t>(p.pool) + (uint64_t)((int64_t)row * p.pool_stride);
    };
    ask_id(0);
    wait_copies<0>();
    int32_t id_next = take_id(0);
    wait_copies<0>();
    ask_page(id_next);
    ask_id(1);
    wait_copies<0>();
    uint64_t at_now = address(take_row(id_next));
    id_next = take_id(1);
    wait_copies<0>();
    ask_page(id_next);  // of the next group; its rows are taken, and the group after it asked for, when its first tile begins
    ask_id(2);
    // Copies of tile t into buffer t % 3, asked for in the order of the tiles:
    // lane 4r + q takes chunks 4j + (q ^ (r / 4)) of row r, at last four scales of 16 rows.
    uint64_t from, from_scale;
    uint32_t to;
    auto begin_tile = [&](int32_t t) __attribute__((always_inline)) {
        if (t > 0 && t % GT == 0) {
            at_now = address(take_row(id_next));
            id_next = take_id(t / GT + 1);
            wait_lds();
            ask_page(id_next);
            ask_id(t / GT + 2);
        }
        const int32_t buf = buffer_of(t);
        to = __builtin_amdgcn_readfirstlane(lds_offset(&lds.tile[buf][kRegion * wave]));
        if (g == t % GT) lds.hidden[buf][RPW * wave + c] = at_now == nowhere ? -__builtin_inff() : 0.f;
        auto of_row = [&](int32_t r) __attribute__((always_inline)) -> uint64_t {
            const int at = 4 * (RPW * (t % GT) + r);
            const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)(uint32_t)at_now);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)(at_now >> 32));
            return ((uint64_t)hi << 32) | lo;
        };
        from = of_row(4 * g + (c >> 2)) + (uint32_t)(16 * ((c & 3) ^ g));
        from_scale = of_row(c) + (uint32_t)(kScaleAt + 4 * g);
    };
    auto copy = [&](auto j) __attribute__((always_inline)) {
        if constexpr (j.value < kCopies - 1) copy_block<j.value>(from, to);
        else copy4_to_lds(reinterpret_cast<const void*>(from_scale), to + kScales);
    };
    auto copy_tile = [&](int32_t t) __attribute__((always_inline)) {
        begin_tile(t);
        each_of<kCopies>(copy);
    };
    f32x4 acc[DT][PT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int h = 0; h < PT; ++h) acc[d][h] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (tiles past the last are copies of the row of zeros: no copy is conditional,
    // and the waits count the same for every tile)
    copy_tile(0);
    copy_tile(1);
    i32x2 v[2][DT];  // this wave's codes of the last tile, transposed: its buffer is free for the next copies
    // lanes 2r, 2r + 1 of a group hand in 16 columns of key 8g + r; lane c gets column c of its eight keys
    auto fetch = [&](int32_t t, int ks) __attribute__((always_inline)) {
        const int32_t r = 8 * (g & 1) + (c >> 1);
        const uint32_t at = lds_offset(lds.tile[buffer_of(t)]) + kRegion * (2 * ks + (g >> 1)) + 1024 * 2 * wave + 64 * r +
                            16 * (r >> 2) + 8 * (c & 1);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int d = q; d < DT; d += 4)
                v[ks][d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (__attribute__((address_space(3))) i32x2*)((at ^ (16 * q)) + 1024 * (d / 4)));
    };
    wait_barrier<kCopies>();
    fetch(0, 0);
    copy_tile(2);  // (asked for before, it held the first scores up)
    lds_barrier();
    fetch(0, 1);
#pragma unroll 1
    for (int32_t t = 1; t <= tiles; ++t) {
        asm volatile("" : "+v"(g), "+v"(c));
        wait_barrier<kCopies>();
        begin_tile(t + 2);
        Frag pf[2][PT], rest[2][TWICE ? PT : 1];
        float keep[PT];
        bool any = false;
#pragma unroll
        for (int h = 0; h < PT; ++h) {
            keep[h] = lds.keep[16 * h + c];
            any |= keep[h] != 1.f;
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(&lds.scale[wave][32 * ks + 8 * g]);
            const f32x4 b = *reinterpret_cast<const f32x4*>(&lds.scale[wave][32 * ks + 8 * g + 4]);
#pragma unroll
            for (int h = 0; h < PT; ++h) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(&lds.prob[16 * h + c][4 * ((8 * ks + 2 * g) ^ c)]);
                const f32x4 y = *reinterpret_cast<const f32x4*>(&lds.prob[16 * h + c][4 * ((8 * ks + 2 * g + 1) ^ c)]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p0 = i < 2 ? x[2 * i] * a[2 * i] : y[2 * i - 4] * b[2 * i - 4];
                    const float p1 = i < 2 ? x[2 * i + 1] * a[2 * i + 1] : y[2 * i - 3] * b[2 * i - 3];
                    const uint32_t w = pack_bf16(p0, p1);
                    pf[ks][h].w[i] = w;
                    if constexpr (TWICE) rest[ks][h].w[i] = pack_bf16(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
                }
                asm volatile("" : "+v"(pf[ks][h].u));  // (here, not where they are used)
                if constexpr (TWICE) asm volatile("" : "+v"(rest[ks][h].u));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__ballot(any))
#pragma unroll
            for (int h = 0; h < PT; ++h)
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d][h] *= keep[h];
        // (a copy is held up at the memory's rate: they are spread over the products)
        auto product = [&](auto ks) __attribute__((always_inline)) {
            Frag a[2];
            a[0] = bf16_of_codes((uint32_t)v[ks.value][0][0], (uint32_t)v[ks.value][0][1]);
            each_of<DT>([&](auto d) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < PT; ++h) {
                    acc[d.value][h] = mfma16(a[d.value & 1], pf[ks.value][h], acc[d.value][h]);
                    if constexpr (TWICE) acc[d.value][h] = mfma16(a[d.value & 1], rest[ks.value][h], acc[d.value][h]);
                    if (h == 0 && d.value + 1 < DT)
                        a[(d.value + 1) & 1] = bf16_of_codes((uint32_t)v[ks.value][(d.value + 1) % DT][0],
                                                             (uint32_t)v[ks.value][(d.value + 1) % DT][1]);
                }
                constexpr int j = DT * ks.value + d.value;
                if constexpr (j < kCopies) copy(Number<j>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        product(Number<0>{});
        fetch(t, 0);
        lds_barrier();
        product(Number<1>{});
        fetch(t, 1);
    }
    wait_copies<0>();  // no copy is left in flight
    if (lane == 0) lds.seen[wave] = seen;
    __syncthreads();
    const bool whole = it.parts == 1;
    const bool none = !(lds.seen[0] | lds.seen[1] | lds.seen[2] | lds.seen[3]);  // no key attended
    // The sums leave through the tiles' memory, a head's columns end to end: as they
    // lie in the registers a store would be 16 heads' pieces of 32 or 64 bytes.
    uint8_t* const rows = lds.tile[0] + wave * (HB * 256);
    static_assert(4 * HB * 256 <= 3 * kTileBytes, "a wave's rows of 256 bytes");
    if (whole) {
        float inv[PT];
#pragma unroll
        for (int ht = 0; ht < PT; ++ht) {
            const int32_t h = 16 * ht + c, head = head0 + h;
            float sum = lds.total[0][h];
#pragma unroll
            for (int k = 1; k < KQ; ++k) sum += lds.total[k][h];
            inv[ht] = 1.0f / sum;
            if (p.lse && wave == 0 && g == 0 && head < p.heads)
                p.lse[(int64_t)it.row * p.heads + head] =
                    none ? -__builtin_inff() : (lds.top[0][h] + __builtin_amdgcn_logf(sum)) * kLn2;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                *reinterpret_cast<u32x2*>(rows + 256 * h + 8 * ((4 * d + g) ^ (2 * c))) =
                    none ? u32x2{0, 0} : u32x2{pack_bf16(acc[d][ht][0] * inv[ht], acc[d][ht][1] * inv[ht]),
                                               pack_bf16(acc[d][ht][2] * inv[ht], acc[d][ht][3] * inv[ht])};
        }
        wait_lds();
        uint16_t* out = p.out + it.row * p.o_row + wave * 128 + 4 * (lane & 31);
#pragma unroll
        for (int j = 0; j < HB / 2; ++j) {
            const int32_t h = 2 * j + (lane >> 5);
            const u32x2 x = *reinterpret_cast<const u32x2*>(rows + 256 * h + 8 * ((lane & 31) ^ (2 * (h & 15))));
            if (head0 + h < p.heads) *reinterpret_cast<u32x2*>(out + (head0 + h) * p.o_head) = x;
        }
        return;
    }
    const int64_t at = (int64_t)index * p.heads + head0;
    if (wave == 0 && lane < HB && head0 + lane < p.heads) {
        float sum = lds.total[0][lane];
#pragma unroll
        for (int k = 1; k < KQ; ++k) sum += lds.total[k][lane];
        p.parts.stats[at + lane] = f32x2{none ? -__builtin_inff() : fmaxf(lds.top[0][lane], kLowest), none ? 0.f : sum};
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int ht = 0; ht < PT; ++ht)
#pragma unroll
            for (int d = 0; d < 4; ++d)
                *reinterpret_cast<f32x4*>(rows + 256 * (16 * ht + c) + 16 * ((4 * d + g) ^ c)) =
                    none ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[4 * half + d][ht];
        wait_lds();
#pragma unroll
        for (int j = 0; j < HB / 4; ++j) {
            const int32_t h = 4 * j + g;
            const f32x4 x = *reinterpret_cast<const f32x4*>(rows + 256 * h + 16 * (c ^ (h & 15)));
            if (head0 + h < p.heads)
                *reinterpret_cast<f32x4*>(p.parts.sums + (at + h) * kLatent + wave * 128 + 64 * half + 4 * c) = x;
        }
        wait_lds();
    }
}

// Heads of a work-group: 16, 32 or 64 (more: several work-groups a row).  More heads
// share each key's conversion; fewer start and end sooner.  So the fewest whose
// work-groups all run at once with at most eight tiles a CU.  64 heads, 2048 keys, in
// work-groups of 16 / 32 / 64:
//      8 rows  18.6 / 21.0 / 25.7 us  (4 tiles at 16)
//     32 rows  34.9 / 34.2 / 36.0     (16 at 16, 8 at 32)
//     64 rows  48.4 / 47.3 / 43.9
//    128 rows  95.5 / 73.5 / 63.9
//   1024 rows   754 /  534 /  360
// (Keys are the row's capacity: a call does not wait for the device to know its
// lengths.  8 rows of 64 heads and some 2000 tokens take 21 us in tables of 2048, 29
// in tables of 16384 and more.  So a row's heads, and with them its probabilities' bits,
// depend on the batch.)
inline int32_t absorbed_heads(int32_t rows, int32_t heads, int32_t keys) {
    const int64_t cus = device_cus(), tiles = cdiv(keys, kTileKeys);
    auto few = [&](int32_t of) {
        const int64_t groups = (int64_t)rows * cdiv(heads, of);
        return heads <= of || (groups <= cus && groups * tiles <= 8 * cus);
    };
    return few(16) ? 16 : few(32) ? 32 : 64;
}

// (One work-group a CU.  A part's start is two to four dependent loads, its sums
// are three tiles' bytes at 64 heads and less than one at 16.)
inline Plan absorbed_plan(const int32_t* lens, int32_t rows, int32_t heads, int32_t keys, bool ragged) {
    const int32_t hb = absorbed_heads(rows, heads, keys);
    const int64_t splits = cdiv(heads, hb), tiles = cdiv(keys, kTileKeys), slots = std::max<int64_t>(1, device_cus() / splits);
    Plan p{lens, rows, keys, 0, 0, (int32_t)slots};
    if (ragged && keys > 0 && planned(rows, tiles) && rows < slots) p.target = (int32_t)std::max(slots - rows, (slots + 1) / 2);
    else p.chunk = chunk_for(rows, tiles, slots, 3, hb / 16);
    return p;
}

template <int HT, int HG>
int launch_absorbed(const AbsorbedParams& p, int64_t blocks, hipStream_t st) {
    static OncePerDevice once;
    constexpr size_t bytes = sizeof(AbsorbedLds<HT, HG>);
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    const int rc = allow_lds(once, reinterpret_cast<const void*>(absorbed_kernel<HT, HG>), bytes, "latent_attend: LDS");
    if (rc != V1_OK) return rc;
    hipLaunchKernelGGL((absorbed_kernel<HT, HG>), dim3((uint32_t)blocks), dim3(512), bytes, st, p);
    return V1_LAUNCHED("latent_attend");
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace v1

using namespace v1;

extern "C" int v1_latent_store(const v1_latent_store_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "latent_store: null arguments");
    auto [latent, latent_stride, rope, rope_stride, slots, pool, pool_rows, pool_stride_bytes, tokens] = *a;
    V1_REQUIRE(tokens >= 0 && pool_rows >= 0 && pool_rows < 1ll << 31, "latent_store: bad shape");
    V1_REQUIRE(aligned16(latent) && aligned16(rope) && aligned16(pool) && latent_stride % 8 == 0 && rope_stride % 8 == 0,
               "latent_store: inputs and pool must be 16-byte aligned, strides multiples of 8");
    V1_REQUIRE(pool_stride_bytes % 16 == 0 && pool_stride_bytes >= kRowBytes,
               "latent_store: pool stride must be a multiple of 16 and >= %d", kRowBytes);
    V1_REQUIRE(launchable(cdiv(tokens, 4), 256), "latent_store: too many tokens for a launch");
    if (tokens == 0) return V1_OK;
    StoreParams p{static_cast<const uint16_t*>(latent), latent_stride, static_cast<const uint16_t*>(rope), rope_stride,
                  slots, tokens, static_cast<uint8_t*>(pool), pool_rows, pool_stride_bytes};
    hipLaunchKernelGGL(latent_store_kernel, dim3((uint32_t)cdiv(tokens, 4)), dim3(256), 0, as_stream(stream), p);
    return V1_LAUNCHED("latent_store");
}

extern "C" int64_t v1_latent_attend_workspace(int32_t rows, int32_t heads, int32_t keys, int32_t ragged) {
    if (rows <= 0 || heads <= 0 || keys <= 0) return 0;
    const attn::Plan plan = absorbed_plan(nullptr, rows, heads, keys, ragged != 0);
    const int64_t items = attn::items_at_most(plan);
    return plan.chunk > 0 && items == rows ? 0 : attn::parts_bytes(plan, heads, kLatent);
}

extern "C" int v1_latent_attend(const v1_latent_attend_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "latent_attend: null arguments");
    auto [q, q_row, q_head, pool, pool_rows, pool_stride_bytes, map, map_len, map_stride, ids, ids_stride, lens,
          out, o_row, o_head, lse, workspace, workspace_bytes, map_shift, rows, heads, keys, scale] = *a;
    V1_REQUIRE(rows >= 0 && heads > 0 && keys >= 0 && pool_rows >= 0 && pool_rows < 1ll << 31, "latent_attend: bad shape");
    V1_REQUIRE(heads < 1 << 16, "latent_attend: too many heads");
    V1_REQUIRE(keys <= kMostKeys, "latent_attend: too many keys");
    V1_REQUIRE(scale > 0.f && scale * kLog2e < __builtin_inff(), "latent_attend: scale must be positive and finite");
    V1_REQUIRE(map_shift >= 0 && map_shift < 31 && map_len >= 0, "latent_attend: bad page map");
    V1_REQUIRE(aligned16(q) && aligned16(pool) && reinterpret_cast<uintptr_t>(out) % 8 == 0 && q_row % 8 == 0 &&
                   q_head % 8 == 0 && o_row % 4 == 0 && o_head % 4 == 0,
               "latent_attend: q and pool must be 16-byte aligned, out 8-byte, q strides multiples of 8, out strides of 4");
    V1_REQUIRE(pool_stride_bytes % 16 == 0 && pool_stride_bytes >= kRowBytes,
               "latent_attend: pool stride must be a multiple of 16 and >= %d", kRowBytes);
    if (rows == 0) return V1_OK;
    const Plan plan = absorbed_plan(lens, rows, heads, keys, lens != nullptr);
    const int64_t items = items_at_most(plan), need = v1_latent_attend_workspace(rows, heads, keys, lens != nullptr);
    V1_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr),
               "latent_attend: workspace of %lld bytes needed", (long long)need);
    const int32_t hb = absorbed_heads(rows, heads, keys);
    const int64_t splits = cdiv(heads, hb), spread = cdiv(items, 8), blocks = 8 * spread * splits;
    V1_REQUIRE(launchable(blocks, 512), "latent_attend: too many rows and heads for a launch");
    AbsorbedParams p{static_cast<const uint16_t*>(q), q_row, q_head, static_cast<const uint8_t*>(pool), pool_rows,
                     pool_stride_bytes, map, map_len, map_stride, map_shift, ids, ids_stride, plan, heads,
                     (int32_t)splits, (int32_t)spread, scale * kLog2e, static_cast<uint16_t*>(out), o_row, o_head, lse,
                     parts_at(workspace, plan, heads, kLatent)};
    const hipStream_t st = as_stream(stream);
    const int rc = hb == 16   ? launch_absorbed<1, 1>(p, blocks, st)
                   : hb == 32 ? launch_absorbed<2, 1>(p, blocks, st)
                              : launch_absorbed<2, 2>(p, blocks, st);
    if (rc != V1_OK || need == 0) return rc;
    JoinParams j{plan, p.parts, p.out, o_row, o_head, lse, heads, nullptr, 0, 0, 0, false};
    return launch_join<kLatent>(j, st, "latent_attend: join");
}
