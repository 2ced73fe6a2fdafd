// Keys and values into and out of the paged 8-bit cache (tb_cache_append_q8, tb_cache_read_q8).
//
// A page of one key-value head has one scale s, 0 (all codes 0) or a power of two, and stands for code * s with |code| <= 127.
// Appending rows x to a page whose earlier rows carry s_old: s = max(s_old, 2^e), e the least with max|x| <= 127 * 2^e; earlier
// codes become rne(code * s_old / s), new ones rne(x / s).  With powers of two a code that is requantised is halved (or
// quartered ...), so its error stays under one step however often the page's maximum rises (1/2 + 1/4 + ...), where a scale of
// amax / 127 would round the whole page anew for every new maximum; the price is a step up to twice as wide.  Both quotients are
// exact, so a code has one right value in any arithmetic.
//
// What bounds it: bytes, and for a call of a few tokens the trips to memory one behind the other (slots, rows and the old scale, codes).
// A block takes the runs (consecutive tokens in consecutive slots of one page) that start in its span of 8 to 64 tokens, of one head and
// one of keys and values; it fetches the span's and a page's slots at once and finds the runs in shared memory.  A single run, a
// prompt's, has the whole block, two have four warps each, up to four have two, and more, a decode step's, a warp each: with a block for
// every run 1024 single tokens took 57 us instead of 8, with a warp for every run a page of 128 rows would take them one by one.  Rows are
// fetched for the maximum and, unless the registers hold all of a warp's, once more, from the L1 or L2, for the codes.  A prompt's chunks,
// 6600 tokens of two heads of 256 in f16: 9.4 us to append, 5.9 to read back (40 MB, 6 us at the copy's rate); 64 single tokens 4 us.
#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t WARPS = 8, MOST_PAGE = 128, LEAST_SPAN = 8, MOST_SPAN = 64;

struct RowsArgs {
    int8_t* codes[2];
    float* scale[2];
    void* rows[2];
    unsigned long long token_stride, head_stride;
    const uint32_t* slots;
    uint32_t tokens, kv_heads, shift, slots_end, span, dim;
};

// Values of a row a lane holds: lane, lane + 32 ... in pieces of four (two for heads of 64), as they lie in memory.  ROWS rows at a time:
// more made no call faster, their code takes longer to arrive than the rows do.
template <int D, bool F16>
struct Piece {
    static constexpr int N = D == 64 ? 2 : 4, TURNS = D == 64 ? 1 : D / 128, WORDS = F16 ? N / 2 : N;
    static constexpr int ROWS = TURNS * WORDS <= 2 ? 2 : 1;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const void* base, unsigned long long at) {
        const char* p = static_cast<const char*>(base) + at * (F16 ? 2 : 4);
        if constexpr (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (WORDS == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ float value(int e) const {
        if constexpr (F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e / 2]));
            return e & 1 ? f.y : f.x;
        } else {
            return __uint_as_float(w[e]);
        }
    }
};

// x * inv (inv a power of two, or 0) to a code: what lies outside (infinities alone do) becomes the nearest end, no number 0.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
    const float v = __fmul_rn(x, inv);
    return v == v ? static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f)) & 0xff) : 0u;
}

template <int D, bool F16>
__global__ void __launch_bounds__(WARPS * 32, 4) cache_append_kernel(const RowsArgs a) {
    using P = Piece<D, F16>;
    __shared__ float top[WARPS];
    __shared__ uint32_t s_slot[1 + MOST_SPAN + MOST_PAGE];  // of the token before the span, the span's and a page's more
    __shared__ uint32_t s_start[MOST_SPAN], s_starts;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y, which = blockIdx.z;
    const uint32_t page = 1u << a.shift;
    const void* rows = which ? a.rows[1] : a.rows[0];
    const uint32_t t_first = blockIdx.x * a.span, t_end = min(t_first + a.span, a.tokens);
    pdl_wait();
    for (uint32_t i = threadIdx.x; i < 1 + a.span + page; i += WARPS * 32) {
        const uint32_t t = t_first + i;  // the token after the one this entry is of
        s_slot[i] = t > 0 && t - 1 < a.tokens ? __ldg(a.slots + t - 1) : 0xffffffffu;
    }
    __syncthreads();
    if (warp == 0) {  // the runs that start here
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i0 = 0; i0 < MOST_SPAN; i0 += 32) {
            const uint32_t i = i0 + lane;
            bool start = false;
            if (t_first + i < t_end) {
                const uint32_t slot = s_slot[1 + i];
                start = slot < a.slots_end && ((slot & (page - 1)) == 0 || t_first + i == 0 || s_slot[i] != slot - 1);
            }
            const uint32_t who = __ballot_sync(0xffffffffu, start);
            if (start) s_start[n + __popc(who & ((1u << lane) - 1))] = i;
            n += __popc(who);
        }
        if (lane == 0) s_starts = n;
    }
    __syncthreads();
    const uint32_t starts = s_starts;
    const uint32_t lg = starts <= 1 ? 3 : starts <= 2 ? 2 : starts <= 4 ? 1 : 0, step = 1u << lg;  // warps a run
    const uint32_t team = warp >> lg, row0 = warp & (step - 1);
    for (uint32_t run = team; run < starts; run += WARPS >> lg) {
        const uint32_t* here = s_slot + 1 + s_start[run];
        const uint32_t t = t_first + s_start[run], slot = here[0], id = slot >> a.shift, off = slot & (page - 1);
        float* sp = (which ? a.scale[1] : a.scale[0]) + (size_t)id * a.kv_heads + head;
        const float was = off > 0 ? *sp : 0.0f;
        uint32_t m = 0;  // the run's length, at most to the page's end
        for (uint32_t len = 32; len == 32; m += len) {
            const bool same = off + m + lane < page && t + m + lane < a.tokens && here[m + lane] == slot + m + lane;
            const uint32_t got = __ballot_sync(0xffffffffu, same);
            len = got == 0xffffffffu ? 32u : (uint32_t)__ffs(~got) - 1;
        }
        float big = 0.0f;
        P x[P::ROWS][P::TURNS];
        const bool held = m <= P::ROWS * step;  // the rows stay in registers
        auto fetch = [&](uint32_t i) {
#pragma unroll
            for (int q = 0; q < P::ROWS; q++)
#pragma unroll
                for (int k = 0; k < P::TURNS; k++)
                    if (i + q * step < m) x[q][k].load(rows, (t + i + q * step) * a.token_stride + head * a.head_stride + lane * P::N + k * 128);
        };
#pragma unroll 1
        for (uint32_t i = row0; i < m; i += P::ROWS * step) {
            fetch(i);
#pragma unroll
            for (int q = 0; q < P::ROWS; q++)
#pragma unroll
                for (int k = 0; k < P::TURNS; k++)
#pragma unroll
                    for (int e = 0; e < P::N; e++) {
                        const float v = i + q * step < m ? fabsf(x[q][k].value(e)) : 0.0f;
                        if (v <= 3.402823466e38f) big = fmaxf(big, v);  // infinities and NaN do not set the scale
                    }
        }
        big = warp_max(big);
        if (step > 1) {  // a team has one run at most, so `top` is written once
            if (lane == 0) top[warp] = big;
            named_bar_sync(1 + team, step * 32);
            for (uint32_t w = 0; w < step; w++) big = fmaxf(big, top[team * step + w]);
        }
        // The least power of two with big <= 127 * 2^e, from the bits: big = 2^x * 1.f gives e = x - 6, or x - 5 above 127 / 64.
        float least = 0.0f;
        if (big > 0.0f) {
            const uint32_t b = __float_as_uint(big);
            const int e = (int)(b >> 23) - 127 - 6 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
            least = __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
        }
        const float s = fmaxf(was, least);
        // 1 / s as a power of two: s >= 2^-126, so it is at most 2^126; s is at most 2^121.
        const float inv = s > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(s)) : 0.0f;
        int8_t* codes = (which ? a.codes[1] : a.codes[0]) + ((size_t)id * a.kv_heads + head) * page * D;
        if (off > 0 && s != was) {
            const float ratio = __fmul_rn(was, inv);
            for (uint32_t i = row0 * 32 + lane; i < off * (D / 4); i += step * 32) {
                uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
                const uint32_t old = *w;
                uint32_t now = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) now |= code_of((float)(int8_t)(old >> (8 * e)), ratio) << (8 * e);
                *w = now;
            }
        }
#pragma unroll 1
        for (uint32_t i = row0; i < m; i += P::ROWS * step) {
            if (!held) fetch(i);
#pragma unroll
            for (int q = 0; q < P::ROWS; q++)
#pragma unroll
                for (int k = 0; k < P::TURNS; k++) {
                    if (i + q * step >= m) continue;
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < P::N; e++) w |= code_of(x[q][k].value(e), inv) << (8 * e);
                    int8_t* dst = codes + (off + i + q * step) * D + k * 128 + lane * P::N;
                    if constexpr (P::N == 4) *reinterpret_cast<uint32_t*>(dst) = w;
                    else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
                }
        }
        __syncwarp();  // every lane has read the old scale, and where warps work together, all of them have, before they met
        if (row0 == 0 && lane == 0) *sp = s;
    }
}

// Sixteen codes a thread: one 16-byte load, two (f16) or four (f32) 16-byte stores.
template <bool F16>
__global__ void __launch_bounds__(256) cache_read_kernel(const RowsArgs a) {
    const uint32_t pieces = a.dim / 16;
    const unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
    pdl_wait();
    if (i >= (unsigned long long)a.tokens * a.kv_heads * pieces) return;
    const uint32_t c = (uint32_t)(i % pieces);
    const unsigned long long rh = i / pieces;
    const uint32_t head = (uint32_t)(rh % a.kv_heads), t = (uint32_t)(rh / a.kv_heads);
    const uint32_t slot = __ldg(a.slots + t);
    if (slot >= a.slots_end) return;
    const uint32_t id = slot >> a.shift, off = slot & ((1u << a.shift) - 1);
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const size_t ph = (size_t)id * a.kv_heads + head;
        const float s = a.scale[which][ph];
        const uint4 w = *reinterpret_cast<const uint4*>(a.codes[which] + ((ph << a.shift) + off) * a.dim + c * 16);
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        const unsigned long long at = t * a.token_stride + head * a.head_stride + c * 16;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = __fmul_rn((float)(int8_t)(words[e / 4] >> (8 * (e % 4))), s);
        if constexpr (F16) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.rows[which]) + at);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const __half2 v = __floats2half2_rn(x[8 * q + 2 * e], x[8 * q + 2 * e + 1]);
                    h[e] = *reinterpret_cast<const uint32_t*>(&v);
                }
                dst[q] = make_uint4(h[0], h[1], h[2], h[3]);
            }
        } else {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.rows[which]) + at);
#pragma unroll
            for (int q = 0; q < 4; q++) dst[q] = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        }
    }
}

int check_rows(const tb_cache_rows* p, const std::string& who) {
    if (!p) return fail(OUT_OF_RANGE, who + ": null descriptor");
    TB_TRY(check_pages(p->cache, who, false));
    if (p->dtype != TB_F32 && p->dtype != TB_F16) return fail(OUT_OF_RANGE, who + ": unknown dtype");
    if (p->tokens == 0) return OK;
    if (p->tokens > 0x7fffffffu) return fail(OUT_OF_RANGE, who + ": more than 2^31 - 1 tokens");
    if (!p->k || !p->v || !p->slots) return fail(OUT_OF_RANGE, who + ": null argument");
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->slots, 4) || p->token_stride % 8 != 0 || p->head_stride % 8 != 0)
        return fail(OUT_OF_RANGE, who + ": rows must start at multiples of 16 bytes: strides are multiples of 8 values");
    return OK;
}

RowsArgs rows_args(const tb_cache_rows& p) {
    RowsArgs a{};
    a.codes[0] = p.cache.k, a.codes[1] = p.cache.v, a.scale[0] = p.cache.k_scale, a.scale[1] = p.cache.v_scale;
    a.rows[0] = p.k, a.rows[1] = p.v, a.token_stride = p.token_stride, a.head_stride = p.head_stride, a.slots = p.slots;
    a.tokens = p.tokens, a.kv_heads = p.cache.kv_heads, a.shift = log2_of(p.cache.page), a.slots_end = p.cache.pages * p.cache.page, a.dim = p.cache.head_dim;
    return a;
}

int launch_append(tb_context* ctx, const tb_cache_rows& p) {
    RowsArgs a = rows_args(p);
    const uint64_t each = (uint64_t)p.tokens * p.cache.kv_heads * 2 / ((uint64_t)ctx->sms * 8);  // eight blocks a multiprocessor
    a.span = LEAST_SPAN;
    while (a.span < MOST_SPAN && a.span < each) a.span *= 2;
    const dim3 grid((p.tokens + a.span - 1) / a.span, p.cache.kv_heads, 2), block(WARPS * 32);
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    auto run = [&](auto kernel) { return launch_kernel(ctx, kernel, grid, block, 0, true, a); };
    const bool h = p.dtype == TB_F16;
    cudaError_t e = cudaSuccess;
    switch (p.cache.head_dim) {
        case 64: e = h ? run(cache_append_kernel<64, true>) : run(cache_append_kernel<64, false>); break;
        case 128: e = h ? run(cache_append_kernel<128, true>) : run(cache_append_kernel<128, false>); break;
        case 256: e = h ? run(cache_append_kernel<256, true>) : run(cache_append_kernel<256, false>); break;
        default: e = h ? run(cache_append_kernel<512, true>) : run(cache_append_kernel<512, false>); break;
    }
    TB_CUDA(e);
    return OK;
}

int launch_read(tb_context* ctx, const tb_cache_rows& p) {
    const RowsArgs a = rows_args(p);
    const uint64_t threads = (uint64_t)p.tokens * a.kv_heads * (a.dim / 16), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_cache_read_q8: too many rows for one call");
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    TB_CUDA(launch_kernel(ctx, p.dtype == TB_F16 ? cache_read_kernel<true> : cache_read_kernel<false>, dim3((uint32_t)grid), dim3(256), 0, true, a));
    return OK;
}

}  // namespace

}  // namespace tb

using namespace tb;

extern "C" int tb_cache_append_q8(tb_context* ctx, const tb_cache_rows* args) {
    return entry([&] {
        TB_TRY(check_rows(args, "tb_cache_append_q8"));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        return args->tokens == 0 ? (int)OK : launch_append(ctx, *args);
    });
}

extern "C" int tb_cache_read_q8(tb_context* ctx, const tb_cache_rows* args) {
    return entry([&] {
        TB_TRY(check_rows(args, "tb_cache_read_q8"));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        return args->tokens == 0 ? (int)OK : launch_read(ctx, *args);
    });
}
