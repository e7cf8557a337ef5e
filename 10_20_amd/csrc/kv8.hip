// K / V pages of 64 tokens in e4m3 codes with one fp32 scale for each page and
// head (K and V their own), their writer, and attention of one query position
// per row over them:
//   S[h, j] = scale * ks[page(j)] * (q[h] . k_j),  O[h] = sum_j softmax_j(S[h, :]) vs[page(j)] v_j.
#include "attn.h"

namespace v1 {
namespace {

using namespace attn;

constexpr int kDim = 128;
constexpr int kMaxGroup = 16;  // query heads of a KV head: the columns of a fragment

// ------------------------------------------------------------------ store
// A work-group appends the tokens of one request that fall into one page, for
// one head of K or V: 16 threads a token, 16 tokens at a time.  The page's scale
// becomes the smallest power of two that holds the new tokens, or stays where it
// is larger and the page holds older tokens; where it grows, the older codes are
// rounded again at the new scale (off by half a step once more for each growth).
// Bound by latency (a page and head is 16 KB at most): the request is found from the
// lengths by every work-group, its page and the scale by two loads more.  128
// requests of a token, 8 heads: 8.8 us; 4096 tokens of three requests: 9.1 us, 25 MB
// at 2.8 TB/s (11 with the tokens asked for behind the page and divided one by one).
struct Kv8StoreParams {
    const uint16_t* x[2];  // k, v
    int64_t x_token[2], x_head[2];
    uint8_t* pool[2];
    int64_t page[2], token[2], head[2];  // strides, bytes
    float* scale[2];
    int64_t s_page[2];
    const int32_t* table;
    int64_t table_stride;
    int32_t table_len;
    const int32_t* starts;
    const int32_t* cu;
    int32_t tokens, requests, heads;
    int64_t pages;
};

__global__ __launch_bounds__(256) void kv8_store_kernel(Kv8StoreParams p) {
    __shared__ float amax_of[4];
    const int32_t lane = (int32_t)threadIdx.x % kWave, wave = (int32_t)threadIdx.x / kWave;
    const int32_t w = (int32_t)blockIdx.y & 1, head = (int32_t)blockIdx.y >> 1;
    // the blockIdx.x-th page that the call writes to
    int32_t left = (int32_t)blockIdx.x, request = -1, lo = 0, n = 0, start = 0;
    for (int32_t r0 = 0; r0 < p.requests; r0 += kWave) {
        const int32_t r = min(r0 + lane, p.requests - 1);
        const int32_t a = min(max(p.cu[r], 0), p.tokens), b = min(max(p.cu[r + 1], a), p.tokens);
        const int32_t s = p.starts[r];
        const bool some = r0 + lane < p.requests && b > a && s >= 0;
        const uint32_t touched = some ? (uint32_t)(((int64_t)s + (b - a) - 1) / kTileKeys - s / kTileKeys + 1) : 0;
        const uint32_t upto = wave_inclusive_sum(touched);
        const uint64_t here = __ballot(touched > 0 && (int32_t)upto > left && (int32_t)(upto - touched) <= left);
        if (here) {
            const int src = __ffsll((unsigned long long)here) - 1;
            request = r0 + src;
            left -= __shfl((int32_t)(upto - touched), src, kWave);
            lo = __shfl(a, src, kWave);
            n = __shfl(b - a, src, kWave);
            start = __shfl(s, src, kWave);
            break;
        }
        left -= __shfl((int32_t)upto, kWave - 1, kWave);
    }
    if (request < 0) return;
    const int32_t entry = start / kTileKeys + left;
    if (entry >= p.table_len) return;
    const int32_t page = p.table[request * p.table_stride + entry];
    const int64_t first = (int64_t)entry * kTileKeys;
    const int32_t a = (int32_t)max((int64_t)start - first, (int64_t)0);  // rows a .. b - 1 of the page are new
    const int32_t b = (int32_t)min((int64_t)start + n - first, (int64_t)kTileKeys);
    const int64_t token0 = lo + (first - start);  // of the page's row 0
    const int32_t row = (int32_t)threadIdx.x / 16, d = 8 * ((int32_t)threadIdx.x % 16);
    u32x4 x[4];  // (asked for beside the page)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t r = row + 16 * i;
        x[i] = u32x4{0, 0, 0, 0};
        if (r >= a && r < b)
            x[i] = *reinterpret_cast<const u32x4*>(p.x[w] + (token0 + r) * p.x_token[w] + head * p.x_head[w] + d);
    }
    if (page < 0 || page >= p.pages) return;
    uint8_t* codes = p.pool[w] + page * p.page[w] + head * p.head[w];
    float* scale_at = p.scale[w] + page * p.s_page[w] + head;
    const float old = a > 0 ? *scale_at : 0.f;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            amax = fmaxf(amax, fmaxf(finite_abs(__uint_as_float(x[i][k] << 16)),
                                     finite_abs(__uint_as_float(x[i][k] & 0xffff0000u))));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, kWave));
    if (lane == 0) amax_of[wave] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(amax_of[0], amax_of[1]), fmaxf(amax_of[2], amax_of[3]));
    const float need = exp2i(scale_exponent(amax));
    const float scale = need > old ? need : old;
    if (threadIdx.x == 0) *scale_at = scale;
    const bool grew = a > 0 && scale > old;
    const float again = old / scale;  // (scale is a power of two where it grew)
    // (a power of two, unless the caller's old one is not: x / scale is x * inv, exactly)
    const bool power = __builtin_amdgcn_readfirstlane((__float_as_uint(scale) & 0x807fffffu) == 0 && scale >= 0x1p-126f && scale <= 0x1p120f);
    const float inv = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t r = row + 16 * i;
        u32x2* at = reinterpret_cast<u32x2*>(codes + r * p.token[w] + d);
        if (r >= a && r < b) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = __uint_as_float(x[i][k] << 16);
                v[2 * k + 1] = __uint_as_float(x[i][k] & 0xffff0000u);
            }
            if (power) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] *= inv;
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] /= scale;
            }
            *at = u32x2{codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7])};
        } else if (grew && r < a) {
            const u32x2 was = *at;
            u32x2 now;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x2 lo2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)was[k], false);
                const f32x2 hi2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)was[k], true);
                now[k] = codes4(lo2[0] * again, lo2[1] * again, hi2[0] * again, hi2[1] * again);
            }
            *at = now;
        }
    }
}

// -------------------------------------------------------------- attention
struct Kv8Params {
    const uint16_t* q;
    int64_t q_row, q_head;
    const uint8_t* pool[2];
    int64_t page[2], token[2], head[2];  // strides, bytes
    const float* scale[2];
    int64_t s_page[2];
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    int32_t table_len;
    const int32_t* ids;  // NULL: positions 0, 1, ...
    int64_t ids_stride;
    Plan plan;
    int32_t kv_heads, group, spread;
    int32_t together;  // KV heads of a work-group: 1, 2 or 4
    float scale2;
    uint16_t* out;
    int64_t o_row, o_head;
    float* lse;
    Parts parts;
};

// The row of keys that are not attended.
__device__ const u32x4 zero_kv8[kDim / 16] = {};

constexpr int kWaves = 4;

struct Kv8Lds {
    union {
        uint8_t value[2][kTileKeys][kDim];
        float out[kMaxGroup][kDim + 4];
    } u[kWaves];
    float ks[kWaves][kTileKeys];  // of a tile's keys: K scale times the softmax scale, V scale
    float vs[kWaves][kTileKeys];
    float top[kWaves][kMaxGroup], total[kWaves][kMaxGroup];
};

// A work-group attends one, two or four KV heads of a row over one part of its
// keys, a wave each; waves of one head take the part's tiles of 64 keys in turn,
// each with its own running maximum, and join through LDS.
//   scores  S^T = K Q^T (v_mfma_f32_16x16x32_bf16): K codes come straight into
//           registers (lane = key % 16, 32 of its 128 codes), exact in bf16; column
//           c is query head c of the group.
//   output  O^T = V^T P^T: V codes go memory -> LDS and come back transposed
//           (ds_read_b64_tr_b8); the lane's own scores are its B fragment's
//           probabilities, times the page's V scale, in two bf16 numbers, which leaves
//           2^-17 of each (one number, 2^-8: 1.33 times the error of a rounded exact
//           result; 200.5 us where two take 201, 60.5 where 62.8 for 600 rows of one KV head and
//           1000-3000 tokens).
//
// Bound by memory: 48 contexts of 4096 to 65536 tokens, 4 KV heads of 8 query heads,
// 202 us for 1.09 GB, 5.4 TB/s (a 1 GiB copy moves 5.2).  8 rows of 2048 chosen tokens, one KV head: 7 us
// and 3 for the join, a chain of four loads (lengths, id, page, key).
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_attend_kernel(Kv8Params p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto& lds = *reinterpret_cast<Kv8Lds*>(lds_raw);
    const int32_t wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave);
    const int32_t lane = (int32_t)threadIdx.x % kWave, g = lane >> 4, c = lane & 15;
    const int32_t xcd = (int32_t)blockIdx.x % 8, turn = (int32_t)blockIdx.x / 8, sets = p.kv_heads / p.together;
    const int32_t set = p.plan.chunk > 0 ? (xcd * p.spread + turn) % sets : turn % sets;
    const int32_t index = p.plan.chunk > 0 ? (xcd * p.spread + turn) / sets : turn / sets * 8 + xcd;
    Item it;
    if (!find_item(p.plan, index, it)) return;
    if (p.plan.chunk == 0 && it.part == 0 && set == 0 && threadIdx.x == 0) p.parts.of_row[it.row] = i32x2{index, it.parts};
    const int32_t streams = kWaves / p.together, stream = wave / p.together, kvh = set * p.together + wave % p.together;
    const int32_t mine = (it.tiles - stream + streams - 1) / streams;  // this wave's tiles: stream, stream + streams, ...
    const int32_t* ids = p.ids ? p.ids + it.row * p.ids_stride : nullptr;
    const int32_t* table = p.table + it.row * p.table_stride;
    const uint8_t* kb = p.pool[0] + kvh * p.head[0];
    const uint8_t* vb = p.pool[1] + kvh * p.head[1];

    // the lane's key of the wave's tile t: its id, then its page
    auto fetch_id = [&](int32_t t) __attribute__((always_inline)) -> int32_t {
        const int32_t j = (it.first + stream + streams * t) * kTileKeys + lane;
        if (t >= mine || j >= it.keys) return -1;
        return ids ? ids[j] : j;
    };
    auto fetch_page = [&](int32_t id) __attribute__((always_inline)) -> int32_t {
        if (id < 0 || id / kTileKeys >= p.table_len) return -1;
        const int32_t page = table[id / kTileKeys];
        return page < p.pages ? page : -1;
    };
    auto key_at = [&](int32_t id, int32_t page) __attribute__((always_inline)) -> const uint8_t* {
        return page < 0 ? reinterpret_cast<const uint8_t*>(zero_kv8) : kb + page * p.page[0] + (id % kTileKeys) * p.token[0];
    };
    auto value_at = [&](int32_t id, int32_t page) __attribute__((always_inline)) -> const uint8_t* {
        return page < 0 ? reinterpret_cast<const uint8_t*>(zero_kv8) : vb + page * p.page[1] + (id % kTileKeys) * p.token[1];
    };
    auto from_lane = [&](const uint8_t* a, int32_t src) __attribute__((always_inline)) -> const uint8_t* {
        const uint64_t x = reinterpret_cast<uint64_t>(a);
        const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, src, kWave), hi = (uint32_t)__shfl((int)(x >> 32), src, kWave);
        return reinterpret_cast<const uint8_t*>(((uint64_t)hi << 32) | lo);
    };
    // A fragments of K: key 16u + c, codes 16g .. 16g + 15 and 64 + 16g ..
    auto load_keys = [&](u32x4 (&k)[4][2], int32_t id, int32_t page) __attribute__((always_inline)) {
        const uint8_t* own = key_at(id, page);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint8_t* a = from_lane(own, 16 * u + c) + 16 * g;
            k[u][0] = *reinterpret_cast<const u32x4*>(a);
            k[u][1] = *reinterpret_cast<const u32x4*>(a + 64);
        }
    };
    // V rows, memory -> LDS, chunk n of row r at n ^ (r % 8)
    auto copy_values = [&](int32_t t, int32_t id, int32_t page) __attribute__((always_inline)) {
        const uint8_t* own = value_at(id, page);
        const uint32_t to = lds_offset(&lds.u[wave].value[t & 1][0][0]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            copy_to_lds(from_lane(own, 8 * j + (lane >> 3)) + 16 * ((lane ^ (lane >> 3)) & 7), to + 1024 * j);
    };

    // B fragments of Q^T: column c = head c of the group, numbers in the order of K's codes
    Frag q[4];
    {
        const uint16_t* src = p.q + it.row * p.q_row + (int64_t)(kvh * p.group + min(c, p.group - 1)) * p.q_head + 16 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) q[s].u = *reinterpret_cast<const u32x4*>(src + 64 * (s / 2) + 8 * (s % 2));
    }
    f32x4 acc[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float mx = -__builtin_inff(), total = 0.f;
    bool some = false;  // a key that is attended

    int32_t id = fetch_id(0), id1 = fetch_id(1), id2 = fetch_id(2);
    int32_t page = fetch_page(id), page1 = fetch_page(id1);
    u32x4 k[4][2];
    float ks = 0.f, vs = 0.f;
    auto fetch_scales = [&](int32_t pg, float& a, float& b) __attribute__((always_inline)) {
        a = p.scale[0][max(pg, 0) * p.s_page[0] + kvh];
        b = p.scale[1][max(pg, 0) * p.s_page[1] + kvh];
    };
    if (mine > 0) {
        load_keys(k, id, page);
        fetch_scales(page, ks, vs);
        copy_values(0, id, page);
    }
#pragma unroll 1
    for (int32_t t = 0; t < mine; ++t) {
        // scales of this tile, by key
        lds.ks[wave][lane] = ks * p.scale2;
        lds.vs[wave][lane] = page < 0 ? 0.f : vs;
        const uint64_t attended = __ballot(page >= 0), seen = attended >> (4 * g);  // bit 16u + i: key 16u + 4g + i is attended
        some |= attended != 0;
        f32x4 d[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            d[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                d[u] = mfma16(bf16_of_codes(k[u][half][0], k[u][half][1]), q[2 * half], d[u]);
                d[u] = mfma16(bf16_of_codes(k[u][half][2], k[u][half][3]), q[2 * half + 1], d[u]);
            }
        }
        // the next tile's keys and scales, then its values
        id = id1, page = page1;
        id1 = id2;
        page1 = fetch_page(id1);
        id2 = fetch_id(t + 3);
        if (t + 1 < mine) {
            load_keys(k, id, page);
            fetch_scales(page, ks, vs);
        }
        float s[4][4], top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.ks[wave][16 * u + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[u][i] = (seen >> (16 * u + i)) & 1 ? d[u][i] * f[i] : -__builtin_inff();
                top = fmaxf(top, s[u][i]);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        if (__ballot(top > mx + kLag)) {
            const float next = top > mx + kLag ? top : mx;
            const float keep = mx == -__builtin_inff() ? (next == mx ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mx - next);
            mx = next;
            total *= keep;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= keep;
        }
        const float sub = mx == -__builtin_inff() ? 0.f : mx;
        Frag pf[2], rest[2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.vs[wave][16 * u + 4 * g]);
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __builtin_amdgcn_exp2f(s[u][i] - sub);
                total += x[i];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float p0 = x[2 * i] * f[2 * i], p1 = x[2 * i + 1] * f[2 * i + 1];
                const uint32_t w = pack_bf16(p0, p1);
                pf[u / 2].w[2 * (u & 1) + i] = w;
                rest[u / 2].w[2 * (u & 1) + i] = pack_bf16(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
            }
        }
        // this tile's values have landed: behind them at least the next tile's 8 loads of keys were issued, if there is one
        if (t + 1 < mine) {
            asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            copy_values(t + 1, id, page);
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        // number j of a lane's eight keys is 32 ks + 16 (j / 4) + 4g + j % 4: lanes 2j, 2j + 1 of a group hand in 16 columns of it
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            const int32_t j = c >> 1, r = 32 * step + 16 * (j >> 2) + 4 * g + (j & 3);
            const uint8_t* v = &lds.u[wave].value[t & 1][r][0];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (__attribute__((address_space(3))) i32x2*)(v + 16 * (i ^ (r & 7)) + 8 * (c & 1)));
                const Frag a = bf16_of_codes((uint32_t)w[0], (uint32_t)w[1]);
                acc[i] = mfma16(a, pf[step], acc[i]);
                acc[i] = mfma16(a, rest[step], acc[i]);
            }
        }
    }
    total += __shfl_xor(total, 16, kWave);
    total += __shfl_xor(total, 32, kWave);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the values' buffers become the sums'
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<f32x4*>(&lds.u[wave].out[c][16 * i + 4 * g]) = acc[i];
    if (g == 0) {
        lds.top[wave][c] = some ? fmaxf(mx, kLowest) : mx;
        lds.total[wave][c] = total;
    }
    __syncthreads();
    for (int32_t i = (int32_t)threadIdx.x; i < p.together * p.group * (kDim / 2); i += 64 * kWaves) {
        const int32_t row = i / (kDim / 2), dim = 2 * (i % (kDim / 2)), sub_head = row / p.group, h = row % p.group;
        const int32_t head = set * p.together * p.group + row;
        float top = -__builtin_inff();
        for (int32_t w = sub_head; w < kWaves; w += p.together) top = fmaxf(top, lds.top[w][h]);
        const float sub = top == -__builtin_inff() ? 0.f : top;
        float sum = 0.f, o0 = 0.f, o1 = 0.f;
        for (int32_t w = sub_head; w < kWaves; w += p.together) {
            const float f = __builtin_amdgcn_exp2f(lds.top[w][h] - sub);
            sum = fmaf(f, lds.total[w][h], sum);
            o0 = fmaf(f, lds.u[w].out[h][dim], o0);
            o1 = fmaf(f, lds.u[w].out[h][dim + 1], o1);
        }
        if (it.parts == 1) {
            const bool none = top == -__builtin_inff() && sum == 0.f;  // no key attended
            const float inv = none ? 0.f : 1.0f / sum;
            *reinterpret_cast<uint32_t*>(p.out + it.row * p.o_row + head * p.o_head + dim) =
                none ? 0u : pack_bf16(o0 * inv, o1 * inv);
            if (p.lse && dim == 0)
                p.lse[(int64_t)it.row * p.kv_heads * p.group + head] =
                    none ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        } else {
            const int64_t at = (int64_t)index * p.kv_heads * p.group + head;
            *reinterpret_cast<f32x2*>(p.parts.sums + at * kDim + dim) = f32x2{o0, o1};
            if (dim == 0) p.parts.stats[at] = f32x2{top, sum};
        }
    }
}

// KV heads of a work-group: as many as divide them.  The rows of a token's heads lie
// side by side, and four heads in step read them in one go: 48 contexts as above, one
// head to a work-group 230 us, two 207, four 202; 8 rows of 8 heads and up to 32768
// tokens 68, 61, 58; 256 contexts of 2000 tokens, 4 heads, 136, 131, 123.
inline int32_t kv8_together(int32_t kv_heads) { return kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1; }

// (Two work-groups a CU, a tile of each wave at a time.)
inline Plan kv8_plan(const int32_t* lens, int32_t rows, int32_t kv_heads, int32_t keys, bool ragged) {
    const int64_t together = kv8_together(kv_heads), streams = kWaves / together, steps = cdiv(cdiv(keys, kTileKeys), streams);
    const int64_t slots = std::max<int64_t>(1, 2 * device_cus() * together / kv_heads);
    Plan p{lens, rows, keys, 0, 0, (int32_t)slots};
    if (ragged && keys > 0 && planned(rows, cdiv(keys, kTileKeys)) && rows < slots)
        p.target = (int32_t)std::max(slots - rows, (slots + 1) / 2);
    else p.chunk = (int32_t)streams * chunk_for(rows, steps, slots, 2, 1);
    return p;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace v1

using namespace v1;

extern "C" int v1_kv8_store(const v1_kv8_store_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "kv8_store: null arguments");
    auto [k, k_token, k_head, v, v_token, v_head, k_pool, kp_page, kp_token, kp_head, v_pool, vp_page, vp_token,
          vp_head, k_scale, ks_page, v_scale, vs_page, pages, table, table_stride, starts, cu_tokens, table_len,
          tokens, requests, kv_heads] = *a;
    V1_REQUIRE(tokens >= 0 && requests >= 0 && kv_heads > 0 && pages >= 0 && table_len >= 0, "kv8_store: bad shape");
    V1_REQUIRE(kv_heads <= 32767, "kv8_store: too many heads");
    V1_REQUIRE(aligned16(k) && aligned16(v) && (k_token | k_head | v_token | v_head) % 8 == 0,
               "kv8_store: k and v must be 16-byte aligned with strides in multiples of 8");
    // (the store's own pieces are of 8 bytes; the attention that reads the pools takes 16)
    V1_REQUIRE(aligned16(k_pool) && aligned16(v_pool) &&
                   (kp_page | kp_token | kp_head | vp_page | vp_token | vp_head) % 16 == 0,
               "kv8_store: pools must be 16-byte aligned with strides in multiples of 16");
    if (tokens == 0 || requests == 0 || table_len == 0 || pages == 0) return V1_OK;
    Kv8StoreParams p{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                     {k_token, v_token}, {k_head, v_head},
                     {static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool)},
                     {kp_page, vp_page}, {kp_token, vp_token}, {kp_head, vp_head},
                     {k_scale, v_scale}, {ks_page, vs_page}, table, table_stride, table_len, starts, cu_tokens, tokens,
                     requests, kv_heads, pages};
    // n tokens of a request touch at most min(n, n / 64 + 2) pages
    const int64_t most = std::min<int64_t>(tokens, (int64_t)tokens / kTileKeys + 2ll * requests);
    V1_REQUIRE(launchable(most, 256), "kv8_store: too many tokens for a launch");
    hipLaunchKernelGGL(kv8_store_kernel, dim3((uint32_t)most, (uint32_t)(2 * kv_heads)), dim3(256), 0, as_stream(stream), p);
    return V1_LAUNCHED("kv8_store");
}

extern "C" int64_t v1_kv8_attend_workspace(int32_t rows, int32_t kv_heads, int32_t group, int32_t keys, int32_t ragged) {
    if (rows <= 0 || kv_heads <= 0 || group <= 0 || keys <= 0) return 0;
    const attn::Plan plan = kv8_plan(nullptr, rows, kv_heads, keys, ragged != 0);
    const int64_t items = attn::items_at_most(plan);
    return plan.chunk > 0 && items == rows ? 0 : attn::parts_bytes(plan, kv_heads * group, kDim);
}

extern "C" int v1_kv8_attend(const v1_kv8_attend_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "kv8_attend: null arguments");
    auto [q, q_row, q_head, k_pool, kp_page, kp_token, kp_head, v_pool, vp_page, vp_token, vp_head, k_scale,
          ks_page, v_scale, vs_page, pages, table, table_stride, ids, ids_stride, lens, out, o_row, o_head, lse,
          workspace, workspace_bytes, table_len, rows, kv_heads, group, keys, scale] = *a;
    V1_REQUIRE(rows >= 0 && kv_heads > 0 && group > 0 && keys >= 0 && pages >= 0 && table_len >= 0 &&
                   (int64_t)kv_heads * group < 1ll << 16,
               "kv8_attend: bad shape");
    V1_REQUIRE(keys <= kMostKeys, "kv8_attend: too many keys");
    V1_REQUIRE(group <= kMaxGroup, "kv8_attend: at most %d query heads per KV head", kMaxGroup);
    V1_REQUIRE(scale > 0.f && scale * kLog2e < __builtin_inff(), "kv8_attend: scale must be positive and finite");
    V1_REQUIRE(aligned16(q) && (q_row | q_head) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0 &&
                   (o_row | o_head) % 4 == 0,
               "kv8_attend: q must be 16-byte aligned with strides in multiples of 8, out 8-byte and 4");
    V1_REQUIRE(aligned16(k_pool) && aligned16(v_pool) &&
                   (kp_page | kp_token | kp_head | vp_page | vp_token | vp_head) % 16 == 0,
               "kv8_attend: pools must be 16-byte aligned with strides in multiples of 16");
    if (rows == 0) return V1_OK;
    if (pages == 0 || table_len == 0) keys = 0;
    const Plan plan = kv8_plan(lens, rows, kv_heads, keys, lens != nullptr);
    const int32_t together = kv8_together(kv_heads);
    const int64_t items = items_at_most(plan), sets = kv_heads / together;
    const int64_t spread = plan.chunk > 0 ? cdiv(items * sets, 8) : cdiv(items, 8) * sets;
    const int64_t need = v1_kv8_attend_workspace(rows, kv_heads, group, keys, lens != nullptr);
    V1_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr),
               "kv8_attend: workspace of %lld bytes needed", (long long)need);
    V1_REQUIRE(launchable(8 * spread, 64 * kWaves), "kv8_attend: too many rows and heads for a launch");
    const int32_t heads = kv_heads * group;
    Kv8Params p{static_cast<const uint16_t*>(q), q_row, q_head,
                {static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool)},
                {kp_page, vp_page}, {kp_token, vp_token}, {kp_head, vp_head},
                {k_scale, v_scale}, {ks_page, vs_page}, pages, table, table_stride, table_len, ids, ids_stride, plan,
                kv_heads, group, (int32_t)spread, together, scale * kLog2e, static_cast<uint16_t*>(out), o_row, o_head, lse,
                parts_at(workspace, plan, heads, kDim)};
    static OncePerDevice once;
    int rc = allow_lds(once, reinterpret_cast<const void*>(kv8_attend_kernel), sizeof(Kv8Lds), "kv8_attend: LDS");
    if (rc != V1_OK) return rc;
    const hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(kv8_attend_kernel, dim3((uint32_t)(8 * spread)), dim3(64 * kWaves), sizeof(Kv8Lds), st, p);
    rc = V1_LAUNCHED("kv8_attend");
    if (rc != V1_OK || need == 0) return rc;
    JoinParams j{plan, p.parts, p.out, o_row, o_head, lse, heads, nullptr, 0, 0, 0, false};
    return launch_join<kDim>(j, st, "kv8_attend: join");
}
