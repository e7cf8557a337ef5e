// K / V pages of 64 tokens of bf16 or fp16 numbers: new tokens written into them,
// keys (and queries beside them) rotated on the way, and accepted drafted tokens
// moved to the end of their context.
#include "paged.h"

namespace v1 {
namespace {

using namespace paged;

// ------------------------------------------------------------------ append
// A wave takes a token and `splits`-th part of its rows (query heads, then key
// heads, then value heads), 16 lanes a row with eight numbers each, four rows at a
// time; the table's row of the token's angles is loaded once for all of them.  Pairs
// (d, d + R/2) meet through a lane permute, neighbours lie in one lane.  Products and
// sums are fp32, rounded to the row's type once.
//
// Bound by memory, or by the call: 14 thousand tokens of 32 query and 8 KV heads 69-70 us, 367
// MB at 5.3 TB/s, a copy's rate, and up to 77 between passes that move other memory.  Loads
// that leave the tokens, which nobody reads again, in the caches take 78 in turn with it, on
// the same inputs again and on five in turn; two, three and six rows in flight 1 us or 3 more.
// 128 requests of a token 4.8 us, a wave for every four rows: offsets, start, page entry one
// after the other.
struct AppendParams {
    const uint16_t* x[3];  // q, k, v
    int64_t x_token[3], x_head[3];
    uint16_t* out;
    int64_t o_token, o_head;
    uint16_t* pool[2];
    int64_t page[2], token[2], head[2];
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* starts;
    const int32_t* cu;
    const float* angles;
    int64_t angle_row, angle_rows;
    const int32_t* positions;
    int32_t table_len, tokens, requests, heads, kv_heads, half, splits;
};

constexpr int kRowsAhead = 4;  // rows of a lane in flight

template <class T, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
    const int32_t lane = (int32_t)threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane((int32_t)threadIdx.x / kWave);
    const int32_t t = (int32_t)blockIdx.x * 4 + wave, split = (int32_t)blockIdx.y;
    if (t >= p.tokens) return;
    const int32_t r = request_of(p.cu, p.requests, t);
    if (r < 0) return;
    const int64_t at = (int64_t)p.starts[r] + (t - p.cu[r]);
    const int64_t angle = p.positions ? (int64_t)p.positions[t] : at;
    if (angle < 0 || angle >= p.angle_rows) return;
    int32_t page = -1;
    if (p.starts[r] >= 0 && at / kTileKeys < p.table_len) page = p.table[r * p.table_stride + at / kTileKeys];
    if (page >= p.pages) page = -1;
    const int32_t ch = lane & 15, half8 = p.half / 8;  // chunks of 8 numbers of half a rotated row
    // the lane's angles: of numbers 8 ch .. (halves), or of the pairs 4 ch .. (neighbours)
    const bool turned = ch < 2 * half8;
    const float* of = p.angles + angle * p.angle_row + (NEIGHBOURS ? 4 * ch : 8 * (ch < half8 ? ch : ch - half8));
    float cs[NEIGHBOURS ? 4 : 8], sn[NEIGHBOURS ? 4 : 8];
#pragma unroll
    for (int i = 0; i < (NEIGHBOURS ? 1 : 2); ++i) {
        f32x4 a = {1.f, 1.f, 1.f, 1.f}, b = {0.f, 0.f, 0.f, 0.f};
        if (turned) {
            a = *reinterpret_cast<const f32x4*>(of + 4 * i);
            b = *reinterpret_cast<const f32x4*>(of + p.half + 4 * i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) cs[4 * i + k] = a[k], sn[4 * i + k] = b[k];
    }
    const int32_t partner = (lane & 48) + (!turned ? ch : ch < half8 ? ch + half8 : ch - half8);
    const float sign = ch < half8 ? -1.f : 1.f;
    const int32_t rows = p.heads + 2 * p.kv_heads;
    for (int32_t first = 4 * split + (lane >> 4); first - (lane >> 4) < rows; first += 4 * kRowsAhead * p.splits) {
        u32x4 x[kRowsAhead];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
            const int32_t row = first + 4 * i * p.splits;
            const int32_t w = row < p.heads ? 0 : row < p.heads + p.kv_heads ? 1 : 2;
            const int32_t h = row - (w == 0 ? 0 : w == 1 ? p.heads : p.heads + p.kv_heads);
            x[i] = u32x4{0, 0, 0, 0};
            if (row < rows) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.x[w] + t * p.x_token[w] + h * p.x_head[w] + 8 * ch));
        }
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
            const int32_t row = first + 4 * i * p.splits;
            const int32_t w = row < p.heads ? 0 : row < p.heads + p.kv_heads ? 1 : 2;
            const int32_t h = row - (w == 0 ? 0 : w == 1 ? p.heads : p.heads + p.kv_heads);
            u32x4 y = x[i];
            u32x4 other = y;
            if constexpr (!NEIGHBOURS) {
#pragma unroll
                for (int k = 0; k < 4; ++k) other[k] = (uint32_t)__shfl((int)x[i][k], partner, kWave);
            }
            if (w < 2 && turned) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x2 a = unpack<T>(x[i][k]);
                    if constexpr (NEIGHBOURS) {
                        y[k] = pack<T>(a[0] * cs[k] - a[1] * sn[k], a[1] * cs[k] + a[0] * sn[k]);
                    } else {
                        const f32x2 b = unpack<T>(other[k]);
                        y[k] = pack<T>(a[0] * cs[2 * k] + sign * (b[0] * sn[2 * k]), a[1] * cs[2 * k + 1] + sign * (b[1] * sn[2 * k + 1]));
                    }
                }
            }
            if (row >= rows) continue;
            if (w == 0) *reinterpret_cast<u32x4*>(p.out + t * p.o_token + h * p.o_head + 8 * ch) = y;
            else if (page >= 0)
                *reinterpret_cast<u32x4*>(p.pool[w - 1] + page * p.page[w - 1] + (at % kTileKeys) * p.token[w - 1] + h * p.head[w - 1] + 8 * ch) = y;
        }
    }
}

// -------------------------------------------------------------------- keep
// A work-group moves a request's rows of one head of K or V, 64 rows at a time: all of
// them are read before any is written.  A row comes from its own index or a later one,
// so that the next 64 were not written to by those before them.  Bound by latency, five
// dependent loads: 8 requests of five rows and a head 3.2 us, 128 of nine and 8 heads 4.9.
struct KeepParams {
    uint16_t* pool[2];
    int64_t page[2], token[2], head[2];
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* starts;
    const int32_t* ids;
    const int32_t* cu;
    int32_t table_len, count, requests;
};

__global__ __launch_bounds__(256) void keep_kernel(KeepParams p) {
    const int32_t r = (int32_t)blockIdx.x, w = (int32_t)blockIdx.y & 1, h = (int32_t)blockIdx.y >> 1;
    const int32_t lo = min(max(p.cu[r], 0), p.count), n = min(max(p.cu[r + 1], lo), p.count) - lo, start = p.starts[r];
    if (start < 0) return;
    const int32_t* table = p.table + r * p.table_stride;
    const int32_t ch = (int32_t)threadIdx.x % 16, row0 = (int32_t)threadIdx.x / 16;
    uint16_t* const base = p.pool[w] + h * p.head[w] + 8 * ch;
    auto at = [&](int64_t position) __attribute__((always_inline)) -> uint16_t* {
        if (position / kTileKeys >= p.table_len) return nullptr;
        const int32_t page = table[position / kTileKeys];
        return page < 0 || page >= p.pages ? nullptr : base + page * p.page[w] + (position % kTileKeys) * p.token[w];
    };
    for (int32_t i0 = 0; i0 < n; i0 += 64) {
        u32x4 x[4];
        uint16_t* to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int32_t i = i0 + row0 + 16 * k, id = i < n ? p.ids[lo + i] : -1;
            to[k] = nullptr;
            x[k] = u32x4{0, 0, 0, 0};
            if (id <= i) continue;  // (there already, or not one to move)
            const uint16_t* from = at((int64_t)start + id);
            to[k] = from ? at((int64_t)start + i) : nullptr;
            if (from) x[k] = *reinterpret_cast<const u32x4*>(from);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (to[k]) *reinterpret_cast<u32x4*>(to[k]) = x[k];
        if (i0 + 64 < n) __syncthreads();
    }
}

template <class T>
void launch_append(const AppendParams& p, bool neighbours, dim3 grid, hipStream_t st) {
    if (neighbours) hipLaunchKernelGGL((append_kernel<T, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((append_kernel<T, false>), grid, dim3(256), 0, st, p);
}

}  // namespace
}  // namespace v1

using namespace v1;

extern "C" int v1_paged_append(const v1_paged_append_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "paged_append: null arguments");
    auto [q, q_token, q_head, k, k_token, k_head, v, v_token, v_head, out, o_token, o_head, k_pool, kp_page, kp_token,
          kp_head, v_pool, vp_page, vp_token, vp_head, pages, table, table_stride, starts, cu_tokens, rotations,
          rotation_row, rotation_rows, positions, table_len, tokens, requests, heads, kv_heads, rotated, interleaved,
          fp16] = *a;
    V1_REQUIRE(tokens >= 0 && requests >= 0 && heads >= 0 && kv_heads > 0 && pages >= 0 && table_len >= 0 && rotation_rows >= 0,
               "paged_append: bad shape");
    V1_REQUIRE(heads < 1 << 16 && kv_heads < 1 << 16, "paged_append: too many heads");
    V1_REQUIRE(rotated > 0 && rotated <= kDim && rotated % 16 == 0, "paged_append: 16, 32, .. 128 numbers are rotated");
    V1_REQUIRE(paged::aligned16(q) && paged::aligned16(k) && paged::aligned16(v) && paged::aligned16(out) &&
                   (q_token | q_head | k_token | k_head | v_token | v_head | o_token | o_head) % 8 == 0,
               "paged_append: q, k, v and out must be 16-byte aligned with strides in multiples of 8");
    V1_REQUIRE(paged::aligned16(k_pool) && paged::aligned16(v_pool) &&
                   (kp_page | kp_token | kp_head | vp_page | vp_token | vp_head) % 8 == 0,
               "paged_append: pools must be 16-byte aligned with strides in multiples of 8");
    V1_REQUIRE(paged::aligned16(rotations) && rotation_row % 4 == 0,
               "paged_append: rotations must be 16-byte aligned with a stride in multiples of 4");
    if (tokens == 0 || requests == 0) return V1_OK;
    if (pages == 0) table_len = 0;
    // A wave for every four rows of a token, unless the tokens alone fill the GPU.
    const int32_t rows = heads + 2 * kv_heads;
    const int32_t splits = (int32_t)std::min<int64_t>(cdiv(rows, 4), std::max<int64_t>(1, 16ll * device_cus() / tokens));
    AppendParams p{{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                   {q_token, k_token, v_token}, {q_head, k_head, v_head}, static_cast<uint16_t*>(out), o_token, o_head,
                   {static_cast<uint16_t*>(k_pool), static_cast<uint16_t*>(v_pool)}, {kp_page, vp_page},
                   {kp_token, vp_token}, {kp_head, vp_head}, pages, table, table_stride, starts, cu_tokens, rotations,
                   rotation_row, rotation_rows, positions, table_len, tokens, requests, heads, kv_heads, rotated / 2, splits};
    V1_REQUIRE(attn::launchable(cdiv(tokens, 4), 256), "paged_append: too many tokens for a launch");
    const dim3 grid((uint32_t)cdiv(tokens, 4), (uint32_t)splits);
    if (fp16) launch_append<_Float16>(p, interleaved != 0, grid, as_stream(stream));
    else launch_append<__bf16>(p, interleaved != 0, grid, as_stream(stream));
    return V1_LAUNCHED("paged_append");
}

extern "C" int v1_paged_keep(const v1_paged_keep_args* a, void* stream) {
    V1_REQUIRE(a != nullptr, "paged_keep: null arguments");
    auto [k_pool, kp_page, kp_token, kp_head, v_pool, vp_page, vp_token, vp_head, pages, table, table_stride, starts, ids,
          cu_ids, table_len, count, requests, kv_heads] = *a;
    V1_REQUIRE(count >= 0 && requests >= 0 && kv_heads > 0 && pages >= 0 && table_len >= 0, "paged_keep: bad shape");
    V1_REQUIRE(kv_heads <= 32767, "paged_keep: too many heads");
    V1_REQUIRE(paged::aligned16(k_pool) && paged::aligned16(v_pool) &&
                   (kp_page | kp_token | kp_head | vp_page | vp_token | vp_head) % 8 == 0,
               "paged_keep: pools must be 16-byte aligned with strides in multiples of 8");
    if (count == 0 || requests == 0 || pages == 0 || table_len == 0) return V1_OK;
    V1_REQUIRE(attn::launchable(requests, 256), "paged_keep: too many requests for a launch");
    KeepParams p{{static_cast<uint16_t*>(k_pool), static_cast<uint16_t*>(v_pool)}, {kp_page, vp_page},
                 {kp_token, vp_token}, {kp_head, vp_head}, pages, table, table_stride, starts, ids, cu_ids, table_len, count, requests};
    hipLaunchKernelGGL(keep_kernel, dim3((uint32_t)requests, (uint32_t)(2 * kv_heads)), dim3(256), 0, as_stream(stream), p);
    return V1_LAUNCHED("paged_keep");
}
