// Prefill attention over the paged 8-bit cache on the fifth-generation tensor cores (tb_prefill_paged_q8), heads of 64, 128, 256.
//
// A block takes 128 query rows of one request and key-value head (row = token * ratio + head) and walks their keys in tiles of KT
// positions that start at multiples of KT.  Everything the tensor cores read of the queries' side stays in tensor memory: the
// queries (stored once), the scores S = Q K^T (two buffers), the probabilities (f16, over the scores they came from) and the
// output, so shared memory only carries keys and values: codes turned to f16 on the way in, a byte read where the f16 cache's
// kernel reads two.  Fourteen warps:
//   warps 0-3    a thread a query row: scores out of tensor memory, maximum, exponentials, probabilities back into it; the running
//                maximum moves only when a tile passes it by 2^8, and only then the output is rescaled;
//   warps 4-11   codes to f16: 16 codes a thread and turn, loaded a tile ahead, as 0x6400 | (code + 128) by byte permutes and one packed
//                fused multiply-add (x * f - 1152 f, exact), stored in the 128-byte swizzle; keys K-major, values as they lie in
//                the cache, which is the MN-major form of a B operand;
//   warp 12      one thread issues the products, S of tile i + 1 ahead of P V of tile i;
//   warp 13      looks up the pages of the tiles ahead: page numbers, the pages' factors, which keys have a page at all.
// A page's scales are powers of two.  Keys carry theirs relative to the tile's largest, which multiplies the scores; values theirs
// relative to the largest scale met so far, which multiplies the output at the end (and rescales it when it grows).  Every wait is bounded.
#include "common.cuh"
#include "paged.h"
#include "tc.cuh"

namespace tb {

namespace {

using namespace tc;

constexpr int ROWS = 128, CONVERT_WARPS = 8, THREADS = 14 * 32, AHEAD = 4, MOST_PAGES = 8;

template <int D>
struct Shape {
    static constexpr int KT = D == 256 ? 64 : 128;            // keys a tile
    static constexpr int KCH = KT * 128;                      // a box of 64 dimensions x KT keys
    static constexpr int STAGE = D / 64 * KCH;                // a tile's keys (or values)
    static constexpr int OFF_V = 2 * STAGE, OFF_SUM = 4 * STAGE;
    static constexpr int COL_O = 0, COL_S = D, COL_Q = D + 2 * KT;  // tensor-memory columns
    static constexpr uint32_t UNITS = KT * (D / 16) / (CONVERT_WARPS * 32);  // sixteen codes each, a thread and tile
    // kind::f16, f32 accumulator, A from tensor memory; N >> 3 at bit 17, M >> 4 at bit 24, bit 16: B is MN-major.
    static constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    static constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    static_assert(COL_Q + D / 2 <= 512, "tensor memory has 512 columns");
};

struct Ahead {  // what warp 13 finds out about a tile
    uint32_t id[MOST_PAGES];             // 0xffffffff: no page
    uint32_t kf[MOST_PAGES], vf[MOST_PAGES];  // factors, two f16 each
    uint32_t keys[4];                    // bit c: key c of the tile has a page
    float kref, shrink;                  // multiplies the scores; what the output is multiplied by before this tile
};

struct Shared {
    uint64_t q_full, k_full[2], v_full[2], s_full[2], p_ready[2], pv_done[AHEAD], known[AHEAD], drained;
    uint32_t tmem;
    float vref;
    Ahead ahead[AHEAD];
    uint32_t part[THREADS / 32];
};

struct PrefillArgs {
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    const uint32_t* table;
    const void* q;
    const uint32_t* starts;
    const uint32_t* lengths;
    void* out;
    unsigned long long q_stride, out_stride;
    uint32_t pages, shift, kv_heads, requests, width, tokens, ratio, most, window;
    float scale;  // softmax scale times log2(e)
    int q_f16, out_f16;
};

// D = A B with A in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
        "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Sixteen codes as f16 times a factor: two 16-byte pieces.
__device__ __forceinline__ void convert16(const uint4& w, uint32_t factor, uint4 (&out)[2]) {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    const __half2 f = *reinterpret_cast<const __half2*>(&factor);
    const __half2 off = __hmul2(f, __half2half2(__ushort_as_half(0xe480)));  // -1152 f
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t b = words[i] ^ 0x80808080u, lo = __byte_perm(b, 0x64646464u, 0x4140), hi = __byte_perm(b, 0x64646464u, 0x4342);
        const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&lo), f, off), y = __hfma2(*reinterpret_cast<const __half2*>(&hi), f, off);
        r[2 * i] = *reinterpret_cast<const uint32_t*>(&x), r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
    out[0] = make_uint4(r[0], r[1], r[2], r[3]), out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) paged_prefill_kernel(const PrefillArgs a, uint32_t* status) {
    using S = Shape<D>;
    constexpr int KT = S::KT;
    extern __shared__ uint8_t raw_unaligned[];
    uint8_t* raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_unaligned) + 1023) & ~uintptr_t(1023));
    __shared__ Shared sh;
    uint32_t* s_sum = reinterpret_cast<uint32_t*>(raw + S::OFF_SUM);  // [requests + 1]: row tiles before each request
    const uint32_t th = threadIdx.x, warp = th >> 5, lane = th & 31;
    pdl_wait();

    auto new_tokens = [&](uint32_t r, uint32_t& first) {
        first = a.starts ? __ldg(a.starts + r) : r;
        const uint32_t next = a.starts ? __ldg(a.starts + r + 1) : r + 1;
        return next > first && first < a.tokens ? min(min(next - first, a.most), a.tokens - first) : 0u;
    };
    {  // row tiles before each request
        const uint32_t per = (a.requests + THREADS - 1) / THREADS, r0 = min(th * per, a.requests), r1 = min(r0 + per, a.requests);
        uint32_t mine = 0, first;
        for (uint32_t r = r0; r < r1; r++) mine += (new_tokens(r, first) * a.ratio + ROWS - 1) / ROWS;
        uint32_t x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (lane == 31) sh.part[warp] = x;
        __syncthreads();
        uint32_t at = x - mine;
        for (uint32_t w = 0; w < warp; w++) at += sh.part[w];
        for (uint32_t r = r0; r < r1; r++) {
            s_sum[r] = at;
            at += (new_tokens(r, first) * a.ratio + ROWS - 1) / ROWS;
            if (r + 1 == a.requests) s_sum[a.requests] = at;
        }
        __syncthreads();
    }
    const uint32_t items = s_sum[a.requests];
    if (blockIdx.x >= items * a.kv_heads) return;
    const uint32_t kvh = blockIdx.x % a.kv_heads, item = items - 1 - blockIdx.x / a.kv_heads;  // a chunk's last rows, which see most, first
    uint32_t r = 0;
    {
        uint32_t hi = a.requests;
        while (hi - r > 1) {
            const uint32_t mid = (r + hi) >> 1;
            if (s_sum[mid] <= item) r = mid;
            else hi = mid;
        }
    }
    uint32_t first;
    const uint32_t n = new_tokens(r, first), len = min(__ldg(a.lengths + r), a.width << a.shift), row0 = (item - s_sum[r]) * ROWS;
    const int pos0 = (int)len - (int)n;  // the first new token's position; negative when the lengths cannot be
    const int p_first = pos0 + (int)(row0 / a.ratio), p_last = pos0 + (int)min((row0 + ROWS - 1) / a.ratio, n - 1);
    const int lowest = a.window != 0 && p_first >= (int)a.window ? p_first + 1 - (int)a.window : 0;
    const uint32_t tile0 = (uint32_t)lowest / KT * KT, end = p_last >= 0 ? (uint32_t)p_last + 1 : 0;  // keys end before `end`
    const uint32_t nt = end > tile0 ? (end - tile0 + KT - 1) / KT : 0;

    if (th == 0) {
        mbar_init(&sh.q_full, 4), mbar_init(&sh.drained, 1);
        for (int i = 0; i < 2; i++) mbar_init(&sh.k_full[i], CONVERT_WARPS), mbar_init(&sh.v_full[i], CONVERT_WARPS), mbar_init(&sh.s_full[i], 1), mbar_init(&sh.p_ready[i], 4);
        for (int i = 0; i < AHEAD; i++) mbar_init(&sh.pv_done[i], 1), mbar_init(&sh.known[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    bool ok = true;
    // A wait that runs out is noted, and the thread goes on without waiting for anything else.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity)) {
            ok = false;
            atomicCAS(status, ERR_NONE, ERR_WAIT_FULL);
        }
    };

    if (warp < 4) {
        // ---- queries, softmax, output: this thread has row `row`, tensor-memory lane of the same number -------------------
        const uint32_t row = row0 + th, tok = row / a.ratio, head = kvh * a.ratio + row % a.ratio;
        const bool valid = tok < n;
        const uint32_t lanes = tmem + ((32 * warp) << 16);
        const unsigned long long q_at = (unsigned long long)(first + tok) * a.q_stride + (unsigned long long)head * D;
        // The row is scaled by a power of two so that its largest lies in [1, 2): f16 then loses 2^-11 of it whatever its size.
        float factor = 0.0f;
        if (nt != 0) {
            auto eight = [&](int d, float (&x)[8]) {
                if (!valid) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = 0.0f;
                } else if (a.q_f16) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + q_at + d));
                    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ww[e]));
                        x[2 * e] = f.x, x[2 * e + 1] = f.y;
                    }
                } else {
                    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + q_at + d);
                    const float4 f = __ldg(p), h = __ldg(p + 1);
                    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w, x[4] = h.x, x[5] = h.y, x[6] = h.z, x[7] = h.w;
                }
            };
            float big = 0.0f;
            for (int d = 0; d < D; d += 8) {
                float x[8];
                eight(d, x);
#pragma unroll
                for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[e]));
            }
            const uint32_t expo = min(max(__float_as_uint(big) >> 23, 1u), 253u);
            const float inv = __uint_as_float((254u - expo) << 23);
            factor = a.scale * __uint_as_float(expo << 23);
            for (int c = 0; c < D / 32; c++) {
                uint32_t h[16];
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    float x[8];
                    eight(c * 32 + g * 8, x);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const __half2 v = __floats2half2_rn(x[2 * e] * inv, x[2 * e + 1] * inv);
                        h[g * 4 + e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                }
                tmem_store16(lanes + S::COL_Q + c * 16, h);
            }
            tmem_wait_st();
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full);

        const int p = valid ? pos0 + (int)tok : -1;
        const int oldest = a.window != 0 && p >= (int)a.window ? p + 1 - (int)a.window : 0;
        float m_used = -INFINITY, l_run = 0.0f;
        for (uint32_t i = 0; i < nt; i++) {
            const uint32_t buf = i & 1, sbuf = lanes + S::COL_S + buf * KT;
            const Ahead& info = sh.ahead[i % AHEAD];
            wait(&sh.known[i % AHEAD], (i / AHEAD) & 1);
            wait(&sh.s_full[buf], (i >> 1) & 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float f = info.kref * factor, shrink = info.shrink;
            const int j0 = (int)(tile0 + i * KT);
            float mt = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < KT / 32; c++) {
                uint32_t s[32];
                tmem_load32(sbuf + c * 32, s);
                const int lo = oldest - (j0 + 32 * c), hi = p + 1 - (j0 + 32 * c);
                const uint32_t keys = info.keys[c];
                if (__all_sync(0xffffffffu, lo <= 0 && hi >= 32) && keys == 0xffffffffu) {
#pragma unroll
                    for (int e = 0; e < 32; e++) mt = fmaxf(mt, __uint_as_float(s[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (e >= lo && e < hi && ((keys >> e) & 1u)) mt = fmaxf(mt, __uint_as_float(s[e]));
                }
            }
            mt *= f;
            float corr = shrink;
            if (mt > m_used + 8.0f) {  // also a row's first keys (m_used = -inf)
                corr = ex2(m_used - mt);
                l_run *= corr;
                corr *= shrink;
                m_used = mt;
            }
            const float base = fmaxf(m_used, -1e30f);  // finite: a row that has seen nothing yet gets 2^-inf = 0 and no NaN
            float sum = 0.0f;
#pragma unroll 1
            for (int c = 0; c < KT / 32; c++) {
                uint32_t s[32], h[16];
                tmem_load32(sbuf + c * 32, s);
                const int lo = oldest - (j0 + 32 * c), hi = p + 1 - (j0 + 32 * c);
                const uint32_t keys = info.keys[c];
                if (__all_sync(0xffffffffu, lo <= 0 && hi >= 32) && keys == 0xffffffffu) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float e0 = ex2(fmaf(__uint_as_float(s[2 * e]), f, -base)), e1 = ex2(fmaf(__uint_as_float(s[2 * e + 1]), f, -base));
                        sum += e0 + e1;
                        const __half2 v = __floats2half2_rn(e0, e1);
                        h[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                } else {
                    auto one = [&](int e) { return e >= lo && e < hi && ((keys >> e) & 1u) ? ex2(fmaf(__uint_as_float(s[e]), f, -base)) : 0.0f; };
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float e0 = one(2 * e), e1 = one(2 * e + 1);
                        sum += e0 + e1;
                        const __half2 v = __floats2half2_rn(e0, e1);
                        h[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                }
                tmem_store16(sbuf + c * 16, h);  // over scores this row has done with
            }
            l_run += sum;
            if (i > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {
                wait(&sh.pv_done[(i - 1) % AHEAD], ((i - 1) / AHEAD) & 1);  // the output must be at rest
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
                    tmem_load32(lanes + S::COL_O + c * 32, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tmem_store32(lanes + S::COL_O + c * 32, o);
                }
            }
            tmem_wait_st();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_ready[buf]);
        }
        if (nt != 0) wait(&sh.pv_done[(nt - 1) % AHEAD], ((nt - 1) / AHEAD) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (ok) {
            const float inv = l_run > 0.0f || l_run != l_run ? sh.vref / l_run : 0.0f;
            const unsigned long long out_at = (unsigned long long)(first + tok) * a.out_stride + (unsigned long long)head * D;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                if (nt != 0) tmem_load32(lanes + S::COL_O + c * 32, o);
                if (valid) {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = nt == 0 || inv == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                    if (a.out_f16) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + out_at + c * 32);
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            uint32_t h[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const __half2 v = __floats2half2_rn(__uint_as_float(o[8 * g + 2 * e]), __uint_as_float(o[8 * g + 2 * e + 1]));
                                h[e] = *reinterpret_cast<const uint32_t*>(&v);
                            }
                            dst[g] = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(a.out) + out_at + c * 32);
#pragma unroll
                        for (int g = 0; g < 8; g++) dst[g] = make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp < 4 + CONVERT_WARPS) {
        // ---- codes to f16 ----------------------------------------------------------------------------------------------
        const uint32_t me = th - 128;
        constexpr uint32_t PER_ROW = D / 16, UNITS = S::UNITS;
        uint4 kw[UNITS], vw[UNITS];
        // Unit u of this thread: key (me + 256 u) / PER_ROW of the tile, its codes 16 ((me + 256 u) % PER_ROW) ...
        auto load = [&](const int8_t* codes, const Ahead& info, uint32_t i, uint4 (&w)[UNITS]) {
            const uint32_t j0 = tile0 + i * KT;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) {
                const uint32_t x = me + u * (CONVERT_WARPS * 32), key = x / PER_ROW, c = x % PER_ROW;
                const uint32_t id = info.id[((j0 + key) >> a.shift) - (j0 >> a.shift)];
                w[u] = make_uint4(0, 0, 0, 0);
                if (id != 0xffffffffu) {
                    const int8_t* p = codes + ((((size_t)id * a.kv_heads + kvh) << a.shift) + ((j0 + key) & ((1u << a.shift) - 1))) * D + c * 16;
                    w[u] = __ldg(reinterpret_cast<const uint4*>(p));
                }
            }
        };
        auto store = [&](uint8_t* stage, const Ahead& info, const uint32_t* factors, uint32_t i, const uint4 (&w)[UNITS]) {
            const uint32_t j0 = tile0 + i * KT;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) {
                const uint32_t x = me + u * (CONVERT_WARPS * 32), key = x / PER_ROW, c = x % PER_ROW;
                const uint32_t factor = factors[((j0 + key) >> a.shift) - (j0 >> a.shift)];
                uint4 out[2];
                convert16(w[u], factor, out);
                uint8_t* box = stage + (c >> 2) * S::KCH + key * 128;
                const uint32_t flip = (c >> 2) & 1;  // neighbours four codes' boxes apart start with different halves: no bank twice in a quarter warp
                const uint32_t piece = (c & 3) * 2;
                *reinterpret_cast<uint4*>(box + (((piece + flip) ^ (key & 7)) << 4)) = flip ? out[1] : out[0];
                *reinterpret_cast<uint4*>(box + (((piece + (flip ^ 1)) ^ (key & 7)) << 4)) = flip ? out[0] : out[1];
            }
        };
        if (nt != 0) {
            wait(&sh.known[0], 0);
            load(a.k, sh.ahead[0], 0, kw);
            load(a.v, sh.ahead[0], 0, vw);
        }
        for (uint32_t i = 0; i < nt; i++) {
            const uint32_t buf = i & 1;
            const Ahead& info = sh.ahead[i % AHEAD];
            if (i >= 2) wait(&sh.s_full[buf], ((i - 2) >> 1) & 1);  // S of the tile two before has read this buffer
            store(raw + buf * S::STAGE, info, info.kf, i, kw);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[buf]);
            const bool more = i + 1 < nt;
            if (more) {
                wait(&sh.known[(i + 1) % AHEAD], ((i + 1) / AHEAD) & 1);
                load(a.k, sh.ahead[(i + 1) % AHEAD], i + 1, kw);
            }
            if (i >= 2) wait(&sh.pv_done[(i - 2) % AHEAD], ((i - 2) / AHEAD) & 1);
            store(raw + S::OFF_V + buf * S::STAGE, info, info.vf, i, vw);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[buf]);
            if (more) load(a.v, sh.ahead[(i + 1) % AHEAD], i + 1, vw);
        }
    } else if (warp == 12) {
        // ---- products --------------------------------------------------------------------------------------------------
        if (lane == 0 && nt != 0) {
            const uint32_t ka = smem_addr(raw), va = smem_addr(raw + S::OFF_V);
            auto scores = [&](uint32_t i) {
                wait(&sh.k_full[i & 1], (i >> 1) & 1);
                if (!ok) return;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int k = 0; k < D / 16; k++)
                    mma_ts(tmem + S::COL_S + (i & 1) * KT, tmem + S::COL_Q + k * 8, desc_k_major(ka + (i & 1) * S::STAGE + (k >> 2) * S::KCH + (k & 3) * 32), S::IDESC_S,
                           k > 0 ? 1u : 0u);
                mma_commit(&sh.s_full[i & 1]);
            };
            wait(&sh.q_full, 0);
            scores(0);
            for (uint32_t i = 0; i < nt && ok; i++) {
                if (i + 1 < nt) scores(i + 1);
                wait(&sh.p_ready[i & 1], (i >> 1) & 1);
                wait(&sh.v_full[i & 1], (i >> 1) & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int k = 0; k < KT / 16; k++)
                    mma_ts(tmem + S::COL_O, tmem + S::COL_S + (i & 1) * KT + k * 8, desc_mn_major(va + (i & 1) * S::STAGE + k * 2048, S::KCH), S::IDESC_PV,
                           (i > 0 || k > 0) ? 1u : 0u);
                mma_commit(&sh.pv_done[i % AHEAD]);
            }
            if (!ok) {  // a wait ran out: nothing may still write tensor memory when it is given back
                mma_commit(&sh.drained);
                mbar_wait(&sh.drained, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- the tiles ahead -------------------------------------------------------------------------------------------
        const uint32_t page = 1u << a.shift, count = page < (uint32_t)KT ? KT / page : 1;
        float vref = 0.0f;
        for (uint32_t i = 0; i < nt; i++) {
            if (i >= AHEAD) wait(&sh.pv_done[i % AHEAD], (i / AHEAD - 1) & 1);  // nobody reads the entry's old tile any more
            const uint32_t j0 = tile0 + i * KT, j = j0 + lane * page;
            uint32_t id = 0xffffffffu;
            if (lane < count && (j & ~(page - 1)) < end) id = __ldg(a.table + (size_t)r * a.width + (j >> a.shift));
            if (id >= a.pages) id = 0xffffffffu;
            float ks = 0.0f, vs = 0.0f;
            if (id != 0xffffffffu) ks = __ldg(a.ks + (size_t)id * a.kv_heads + kvh), vs = __ldg(a.vs + (size_t)id * a.kv_heads + kvh);
            const float kref = warp_max(ks), vnew = fmaxf(vref, warp_max(vs));
            Ahead& info = sh.ahead[i % AHEAD];
            if (lane < MOST_PAGES) {
                info.id[lane] = id;
                const __half2 kf = __float2half2_rn(kref > 0.0f ? __fdiv_rn(ks, kref) : 0.0f), vf = __float2half2_rn(vnew > 0.0f ? __fdiv_rn(vs, vnew) : 0.0f);
                info.kf[lane] = *reinterpret_cast<const uint32_t*>(&kf), info.vf[lane] = *reinterpret_cast<const uint32_t*>(&vf);
            }
            const uint32_t has = __ballot_sync(0xffffffffu, id != 0xffffffffu);
            if (lane < 4) {
                uint32_t keys = 0;
                for (uint32_t e = 0; e < 32; e++) {
                    const uint32_t c = lane * 32 + e, pg = page < (uint32_t)KT ? c >> a.shift : 0;
                    if (c < (uint32_t)KT && ((has >> pg) & 1u)) keys |= 1u << e;
                }
                info.keys[lane] = keys;
            }
            if (lane == 0) {
                info.kref = kref;
                info.shrink = vref > 0.0f ? __fdiv_rn(vref, vnew) : 1.0f;
                if (i + 1 == nt) sh.vref = vnew;
            }
            vref = vnew;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.known[i % AHEAD]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D>
int run(tb_context* ctx, const PrefillArgs& a, uint32_t grid) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t bytes = 1024 + Shape<D>::OFF_SUM;
    TB_CUDA(allow_smem(paged_prefill_kernel<D>, bytes + (MAX_REQUESTS + 1) * 4, ctx->gpu, done));
    TB_CUDA(launch_kernel(ctx, paged_prefill_kernel<D>, dim3(grid), dim3(THREADS), bytes + ((size_t)a.requests + 1) * 4, true, a, ctx->status));
    return OK;
}

}  // namespace

bool prefill_paged_supports(const tb_paged_attend& p) { return p.cache.head_dim <= 256; }

int launch_prefill_paged(tb_context* ctx, const tb_paged_attend& p) {
    const tb_pages& c = p.cache;
    PrefillArgs a{};
    a.k = c.k, a.v = c.v, a.ks = c.k_scale, a.vs = c.v_scale, a.table = c.table, a.pages = c.pages, a.shift = log2_of(c.page), a.kv_heads = c.kv_heads;
    a.requests = c.requests, a.width = c.width, a.q = p.q, a.q_stride = p.q_stride, a.q_f16 = p.q_dtype == TB_F16, a.starts = p.starts, a.lengths = p.lengths;
    a.tokens = p.tokens, a.ratio = p.heads / c.kv_heads, a.most = p.most, a.window = p.window > 0x7fffffffu ? 0 : p.window, a.scale = p.scale * 1.4426950408889634f;
    a.out = p.out, a.out_stride = p.out_stride, a.out_f16 = p.out_dtype == TB_F16;
    // Row tiles: at most one a request that is not full, and no request brings more than `most` tokens.
    const uint64_t full = (uint64_t)p.tokens * a.ratio / ROWS + c.requests, each = (((uint64_t)p.most * a.ratio + ROWS - 1) / ROWS) * c.requests;
    const uint64_t grid = (full < each ? full : each) * c.kv_heads;
    if (grid > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_prefill_paged_q8: too many rows for one call");
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    switch (c.head_dim) {
        case 64: return run<64>(ctx, a, (uint32_t)grid);
        case 128: return run<128>(ctx, a, (uint32_t)grid);
        default: return run<256>(ctx, a, (uint32_t)grid);
    }
}

}  // namespace tb
