// Decode attention over the paged 8-bit cache (tb_attend_paged_q8): one or a few new tokens of every request, ragged lengths.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(scale log2(e) q.k_j - m): each visible key and value is read once, one byte a
// number, and that is what bounds it.  The work of all requests is laid out in a line of tiles of 64 positions (request, then
// key-value head, then tile) and cut into equal shares, one a block, whatever the lengths: a prefix sum over the requests, repeated
// by every block, finds a block's place.  A block whose share ends inside a line of keys leaves its maximum, sum and outputs in
// scratch, and the last of that line's blocks to arrive (a counter, nobody waits) adds them up in the order of the positions.
//
// A warp takes 16 positions at a time straight from global memory into the operands of mma.sync.m16n8k16; tcgen05 has no place
// here, a tile of 64 keys against 8 query rows is two orders of magnitude below one of its tiles.  A sum does not mind the order
// of its terms, so the operands' order is chosen for the loads: a thread's four dimensions (or tokens) of an MMA step lie side by
// side in memory, and 16 bytes of a row feed four steps.  A code becomes f16 by byte permutes: 0x6400 | (code + 128) is
// 1152 + code, one packed subtraction leaves the code, exactly.
//   S = Q K^T: rows 0-7 of the A operand hold the queries rounded to f16, rows 8-15 what the rounding left, so the sum of the
//   two halves is the f32 product to 2^-22; the page's scale, a power of two, multiplies the score.
//   O^T = V^T P^T: the scores' accumulator is the B operand's layout as it stands; the weights again go in two f16 parts.  A page's
//   value scale multiplies the weights, relative to the largest scale met so far, so they stay within f16.
// Softmax statistics and sums are f32.
#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t TILE = 64, SLICE = 16;
constexpr int WARPS = 8, THREADS = WARPS * 32;

struct PagedArgs {
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    const uint32_t* table;
    const void* q;
    const uint32_t* starts;   // or null: a token a request
    const uint32_t* lengths;
    void* out;
    float* partial;           // [2 * blocks][16 + 8 * D]
    uint32_t* count;          // [blocks]: of the line that the block begins and does not finish
    unsigned long long q_stride, out_stride;
    uint32_t pages, shift, kv_heads, requests, width, tokens, heads, ratio, most, window, least;
    float scale;              // softmax scale times log2(e)
    int q_f16, out_f16;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes 0, 1 (or 2, 3) of a word of codes + 128 as two f16 codes.
__device__ __forceinline__ uint32_t halves(uint32_t biased, uint32_t select) {
    const uint32_t h = __byte_perm(biased, 0x64646464u, select);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));  // 1152
    return *reinterpret_cast<const uint32_t*>(&v);
}
constexpr uint32_t LOW = 0x4140, HIGH = 0x4342;
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_stream2(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// What a request asks for, from device memory that may hold anything: clamped so that nothing out of range is touched.
struct Request {
    uint32_t first, n;    // its new tokens in the packed rows
    uint32_t len;         // positions in the cache, the new tokens' own included
    uint32_t low, tiles;  // first tile's first position, tiles of keys
    uint32_t groups;      // groups of eight query rows a key-value head
};
__device__ __forceinline__ Request request_of(const PagedArgs& a, uint32_t r) {
    Request q;
    q.first = a.starts ? __ldg(a.starts + r) : r;
    const uint32_t next = a.starts ? __ldg(a.starts + r + 1) : r + 1;
    q.n = next > q.first && q.first < a.tokens ? min(min(next - q.first, a.most), a.tokens - q.first) : 0;
    q.len = min(__ldg(a.lengths + r), a.width << a.shift);
    const uint32_t oldest = q.len > q.n ? q.len - q.n : 0;  // the first new token's position
    q.low = a.window != 0 && oldest >= a.window ? (oldest + 1 - a.window) / TILE * TILE : 0;
    q.tiles = q.n == 0 ? 0 : q.len > q.low ? (q.len - q.low + TILE - 1) / TILE : 1;  // one, so that rows that see nothing are stored
    q.groups = (q.n * a.ratio + 7) / 8;
    return q;
}

template <int D>
constexpr size_t smem_bytes() {
    return (size_t)D * 32 + WARPS * 8 * (size_t)D * 4 + WARPS * 16 * 4 + 64;
}

template <int D>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 2 : 1) paged_attend_kernel(const PagedArgs a) {
    constexpr int MT = D / 16, SEG = D / 64;
    extern __shared__ __align__(16) uint8_t raw[];
    uint4* s_q = reinterpret_cast<uint4*>(raw);                      // [D / 16][32]: the A operand of every step
    float* s_acc = reinterpret_cast<float*>(raw + D * 32);           // [WARPS][8][D]
    float* s_m = s_acc + WARPS * 8 * D;                              // [WARPS][8]
    float* s_l = s_m + WARPS * 8;
    float* s_row = s_l + WARPS * 8;                                  // [8]: a query row's factor
    uint32_t* s_flag = reinterpret_cast<uint32_t*>(s_row + 8);
    uint32_t* s_sum = s_flag + 8;                                    // [requests + 1]: tiles before each request
    __shared__ uint32_t part[WARPS];
    const uint32_t th = threadIdx.x, lane = th & 31, warp = th >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();

    {  // tiles before each request
        const uint32_t per = (a.requests + THREADS - 1) / THREADS, r0 = min(th * per, a.requests), r1 = min(r0 + per, a.requests);
        uint32_t mine = 0;
        for (uint32_t r = r0; r < r1; r++) {
            const Request q = request_of(a, r);
            mine += q.tiles * q.groups * a.kv_heads;
        }
        uint32_t x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (lane == 31) part[warp] = x;
        __syncthreads();
        uint32_t at = x - mine;
        for (uint32_t w = 0; w < warp; w++) at += part[w];
        for (uint32_t r = r0; r < r1; r++) {
            const Request q = request_of(a, r);
            s_sum[r] = at;
            at += q.tiles * q.groups * a.kv_heads;
            if (r + 1 == a.requests) s_sum[a.requests] = at;
        }
        __syncthreads();
    }
    const uint32_t total = s_sum[a.requests];
    if (total == 0) return;
    const uint32_t blocks = min(gridDim.x, (total + a.least - 1) / a.least);
    if (blockIdx.x >= blocks) return;
    const uint32_t my0 = (uint32_t)((unsigned long long)total * blockIdx.x / blocks), my1 = (uint32_t)((unsigned long long)total * (blockIdx.x + 1) / blocks);

    for (uint32_t at = my0; at < my1;) {
        uint32_t lo = 0, hi = a.requests;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (s_sum[mid] <= at) lo = mid;
            else hi = mid;
        }
        // Requests without tiles share their successor's place: `lo` is the last with that sum, the one that has tiles.
        const uint32_t r = lo;
        const Request rq = request_of(a, r);
        const uint32_t line = (at - s_sum[r]) / rq.tiles, tile0 = (at - s_sum[r]) % rq.tiles;
        const uint32_t kvh = line / rq.groups, group = line % rq.groups;
        const uint32_t line0 = s_sum[r] + line * rq.tiles;  // the line's first tile
        const uint32_t tile1 = min(rq.tiles, tile0 + (my1 - at));
        at += tile1 - tile0;

        // The queries of this line: row i is (token i / ratio, head i % ratio) of the group's eight, scaled so that its largest
        // lies in [1, 2), in two f16 parts, in the order the MMA wants them.
        {
            const uint32_t row = group * 8 + warp, tok = row / a.ratio, head = kvh * a.ratio + row % a.ratio;
            const bool real = tok < rq.n;
            float x[D / 32];
            float big = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 32; e++) {
                const unsigned long long p = (unsigned long long)(rq.first + tok) * a.q_stride + (unsigned long long)head * D + e * 32 + lane;
                x[e] = !real ? 0.0f : a.q_f16 ? __half2float(static_cast<const __half*>(a.q)[p]) : static_cast<const float*>(a.q)[p];
                big = fmaxf(big, fabsf(x[e]));
            }
            big = warp_max(big);
            const uint32_t expo = min(max(__float_as_uint(big) >> 23, 1u), 253u);  // infinities stay what they are
            const float inv = __uint_as_float((254u - expo) << 23);
            if (lane == 0) s_row[warp] = a.scale * __uint_as_float(expo << 23);
            __half* dst = reinterpret_cast<__half*>(s_q);
#pragma unroll
            for (int e = 0; e < D / 32; e++) {
                const uint32_t d = e * 32 + lane, step = d / 64 * 4 + d % 16 / 4, owner = warp * 4 + d % 64 / 16, reg = (d & 2), half = d & 1;
                const float y = x[e] * inv;
                const __half h = __float2half_rn(y);
                __half* p = dst + ((step * 32 + owner) * 4 + reg) * 2 + half;
                p[0] = h;
                p[2] = __float2half_rn(y - __half2float(h));
            }
        }
        __syncthreads();

        float acc[MT][4];
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        float m = -INFINITY, l = 0.0f, vref = 0.0f;
        const uint32_t my_row = group * 8 + g, my_tok = my_row / a.ratio;
        const int pos = my_tok < rq.n ? (int)rq.len - (int)rq.n + (int)my_tok : -1;  // negative: this row sees nothing
        const int oldest = a.window != 0 && pos >= (int)a.window ? pos + 1 - (int)a.window : 0;
        const float factor = s_row[g];
        const uint32_t end = min(rq.len, rq.low + tile1 * TILE);
        for (uint32_t j0 = rq.low + tile0 * TILE + warp * SLICE; j0 < end; j0 += WARPS * SLICE) {
            const uint32_t id = __ldg(a.table + (size_t)r * a.width + (j0 >> a.shift));
            if (id >= a.pages) continue;  // no page: nothing to see
            const size_t ph = (size_t)id * a.kv_heads + kvh;
            const size_t row0 = (ph << a.shift) + (j0 & ((1u << a.shift) - 1));
            const int8_t* kp = a.k + row0 * D;
            const int8_t* vp = a.v + row0 * D;
            const float ks = __ldg(a.ks + ph) * factor, vs = __ldg(a.vs + ph);
            // Scores of tokens j0 + 2t, + 1 (c[0]) and j0 + 8 + 2t, + 1 (c[1]) for query row g.
            float c[2][4] = {};
            uint4 kw[2][SEG];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int s = 0; s < SEG; s++) kw[j][s] = load_stream(kp + (j * 8 + g) * D + s * 64 + t * 16);
#pragma unroll
            for (int s = 0; s < SEG; s++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint4 q = s_q[(s * 4 + i) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t w = (i == 0 ? kw[j][s].x : i == 1 ? kw[j][s].y : i == 2 ? kw[j][s].z : kw[j][s].w) ^ 0x80808080u;
                        mma16816(c[j], q.x, q.y, q.z, q.w, halves(w, LOW), halves(w, HIGH));
                    }
                }
            }
            float s[4] = {(c[0][0] + c[0][2]) * ks, (c[0][1] + c[0][3]) * ks, (c[1][0] + c[1][2]) * ks, (c[1][1] + c[1][3]) * ks};
            float top = m;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = (int)j0 + (e >> 1) * 8 + 2 * (int)t + (e & 1);
                if (j > pos || j < oldest) s[e] = -INFINITY;
                top = fmaxf(top, s[e]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float base = top == -INFINITY ? 0.0f : top;
            const float corr = ex2(m - base);  // 0 before the first visible key
            m = top;
            const float vnew = fmaxf(vref, vs);
            const float ratio = vnew > 0.0f ? __fdiv_rn(vs, vnew) : 0.0f, shrink = vnew > 0.0f ? __fdiv_rn(vref, vnew) : 0.0f;
            vref = vnew;
            float w[4];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = ex2(s[e] - base);
                sum += p;
                w[e] = p * ratio;
            }
            l = fmaf(l, corr, sum);
            const float turn = corr * shrink;
            if (__any_sync(0xffffffffu, turn != 1.0f)) {
                const float c0 = __shfl_sync(0xffffffffu, turn, 8 * t), c1 = __shfl_sync(0xffffffffu, turn, 8 * t + 4);  // rows 2t, 2t + 1
#pragma unroll
                for (int i = 0; i < MT; i++) acc[i][0] *= c0, acc[i][1] *= c1, acc[i][2] *= c0, acc[i][3] *= c1;
            }
            const uint32_t h0 = pack(w[0], w[1]), h1 = pack(w[2], w[3]);
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
            const uint32_t l0 = pack(w[0] - f0.x, w[1] - f0.y), l1 = pack(w[2] - f1.x, w[3] - f1.y);
            // Values of tokens 2t, 2t + 1, 2t + 8, 2t + 9; four dimensions of the four tokens make two MMA tiles' A operands.
            auto four = [&](uint32_t wa, uint32_t wb, uint32_t wc, uint32_t wd, float (&even)[4], float (&odd)[4]) {
                wa ^= 0x80808080u, wb ^= 0x80808080u, wc ^= 0x80808080u, wd ^= 0x80808080u;
                const uint32_t ab = __byte_perm(wa, wb, 0x5140), cd = __byte_perm(wc, wd, 0x5140), ab2 = __byte_perm(wa, wb, 0x7362), cd2 = __byte_perm(wc, wd, 0x7362);
                const uint32_t e0 = halves(ab, LOW), e1 = halves(ab, HIGH), e2 = halves(cd, LOW), e3 = halves(cd, HIGH);
                mma16816(even, e0, e1, e2, e3, h0, h1);
                mma16816(even, e0, e1, e2, e3, l0, l1);
                const uint32_t o0 = halves(ab2, LOW), o1 = halves(ab2, HIGH), o2 = halves(cd2, LOW), o3 = halves(cd2, HIGH);
                mma16816(odd, o0, o1, o2, o3, h0, h1);
                mma16816(odd, o0, o1, o2, o3, l0, l1);
            };
            if constexpr (D == 64) {
                const uint2 va = load_stream2(vp + (2 * t) * D + g * 8), vb = load_stream2(vp + (2 * t + 1) * D + g * 8);
                const uint2 vc = load_stream2(vp + (2 * t + 8) * D + g * 8), vd = load_stream2(vp + (2 * t + 9) * D + g * 8);
                four(va.x, vb.x, vc.x, vd.x, acc[0], acc[1]);
                four(va.y, vb.y, vc.y, vd.y, acc[2], acc[3]);
            } else {
#pragma unroll
                for (int sg = 0; sg < D / 128; sg++) {
                    const int8_t* p = vp + sg * 128 + g * 16;
                    const uint4 va = load_stream(p + (2 * t) * D), vb = load_stream(p + (2 * t + 1) * D), vc = load_stream(p + (2 * t + 8) * D),
                                vd = load_stream(p + (2 * t + 9) * D);
                    four(va.x, vb.x, vc.x, vd.x, acc[sg * 8], acc[sg * 8 + 1]);
                    four(va.y, vb.y, vc.y, vd.y, acc[sg * 8 + 2], acc[sg * 8 + 3]);
                    four(va.z, vb.z, vc.z, vd.z, acc[sg * 8 + 4], acc[sg * 8 + 5]);
                    four(va.w, vb.w, vc.w, vd.w, acc[sg * 8 + 6], acc[sg * 8 + 7]);
                }
            }
        }
        // The warps meet: statistics, then outputs in units of the values.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) s_m[warp * 8 + g] = m, s_l[warp * 8 + g] = l;
        {
            float* dst = s_acc + warp * 8 * D;
            constexpr int RUN = D == 64 ? 8 : 16;  // dimensions a lane group holds side by side
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const uint32_t d = i * 2 / RUN * 8 * RUN + g * RUN + i * 2 % RUN;
                *reinterpret_cast<float2*>(dst + (2 * t) * D + d) = make_float2(acc[i][0] * vref, acc[i][2] * vref);
                *reinterpret_cast<float2*>(dst + (2 * t + 1) * D + d) = make_float2(acc[i][1] * vref, acc[i][3] * vref);
            }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == rq.tiles;
        float* slot = a.partial + (size_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * (16 + 8 * D);  // at most one line is begun and not finished, and one finished and not begun
        auto store = [&](uint32_t row, uint32_t d, float v) {
            const uint32_t i = group * 8 + row, tok = i / a.ratio, head = kvh * a.ratio + i % a.ratio;
            if (tok >= rq.n) return;
            const unsigned long long p = (unsigned long long)(rq.first + tok) * a.out_stride + (unsigned long long)head * D + d;
            if (a.out_f16) static_cast<__half*>(a.out)[p] = __float2half_rn(v);
            else static_cast<float*>(a.out)[p] = v;
        };
        for (uint32_t e = th; e < 8 * D; e += THREADS) {
            const uint32_t row = e / D, d = e % D;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_m[w * 8 + row]);
            const float base = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = ex2(s_m[w * 8 + row] - base);
                sum = fmaf(s_l[w * 8 + row], f, sum);
                v = fmaf(s_acc[(w * 8 + row) * D + d], f, v);
            }
            if (whole) {
                store(row, d, sum > 0.0f || sum != sum ? v / sum : 0.0f);
            } else {
                slot[16 + e] = v;
                if (d == 0) slot[row] = top, slot[8 + row] = sum;
            }
        }
        if (!whole) {
            // Which blocks share this line: block b takes the tiles from floor(total b / blocks) on.
            const uint32_t b0 = (uint32_t)(((unsigned long long)(line0 + 1) * blocks - 1) / total);
            const uint32_t b1 = (uint32_t)(((unsigned long long)(line0 + rq.tiles) * blocks - 1) / total);
            __syncthreads();
            if (th == 0) {
                uint32_t* cnt = a.count + b0;  // b0 begins no other line that it leaves unfinished
                __threadfence();
                const bool last = atomicAdd(cnt, 1u) == b1 - b0;
                if (last) *cnt = 0;
                __threadfence();
                *s_flag = last;
            }
            __syncthreads();
            if (*s_flag) {
                for (uint32_t e = th; e < 8 * D; e += THREADS) {
                    const uint32_t row = e / D, d = e % D;
                    float top = -INFINITY, sum = 0.0f, v = 0.0f;
                    for (uint32_t b = b0; b <= b1; b++) {
                        const float* p = a.partial + (size_t)(2 * b + (b == b0 ? 1 : 0)) * (16 + 8 * D);
                        const float mb = __ldcg(p + row), now = fmaxf(top, mb), base = now == -INFINITY ? 0.0f : now;
                        const float f0 = ex2(top - base), f1 = ex2(mb - base);
                        sum = sum * f0 + __ldcg(p + 8 + row) * f1;
                        v = v * f0 + __ldcg(p + 16 + e) * f1;
                        top = now;
                    }
                    store(row, d, sum > 0.0f || sum != sum ? v / sum : 0.0f);
                }
            }
        }
        __syncthreads();  // the next line writes the queries and the warps' results again
    }
}

// Blocks a launch has at most: what is resident at once.
uint32_t most_blocks(const tb_context* ctx, uint32_t head_dim) { return (uint32_t)ctx->sms * (head_dim <= 128 ? 2 : 1); }

int check_attend(const tb_paged_attend* p, const std::string& who, bool few) {
    if (!p) return fail(OUT_OF_RANGE, who + ": null descriptor");
    TB_TRY(check_pages(p->cache, who, true));
    if ((p->q_dtype != TB_F32 && p->q_dtype != TB_F16) || (p->out_dtype != TB_F32 && p->out_dtype != TB_F16)) return fail(OUT_OF_RANGE, who + ": unknown dtype");
    if (p->heads == 0 || p->heads % p->cache.kv_heads != 0) return fail(OUT_OF_RANGE, who + ": query heads must be a multiple of the key-value heads");
    const uint32_t ratio = p->heads / p->cache.kv_heads;
    if (ratio > 64) return fail(UNSUPPORTED, who + ": more than 64 query heads to a key-value head");
    if (p->most == 0 || p->most > 0x7fffffffu / 64 / ratio) return fail(OUT_OF_RANGE, who + ": `most` outside its range");
    if (!p->starts && (p->most != 1 || p->tokens != p->cache.requests)) return fail(OUT_OF_RANGE, who + ": without `starts` every request brings one token");
    if (p->tokens > 0x7fffffffu) return fail(OUT_OF_RANGE, who + ": more than 2^31 - 1 tokens");
    if (!(p->scale > 0.0f) || p->scale > 3e38f) return fail(OUT_OF_RANGE, who + ": the scale must be positive and finite");
    if (p->tokens == 0) return OK;
    if (!p->q || !p->out || !p->lengths) return fail(OUT_OF_RANGE, who + ": null argument");
    if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->lengths, 4) || !aligned(p->starts, 4) || p->q_stride % 8 != 0 || p->out_stride % 8 != 0)
        return fail(OUT_OF_RANGE, who + ": rows must start at multiples of 16 bytes: strides are multiples of 8 values");
    const uint64_t row = (uint64_t)p->heads * p->cache.head_dim;
    if (p->q_stride < row || p->out_stride < row) return fail(OUT_OF_RANGE, who + ": a stride below heads * head_dim");
    if (few && ratio * p->most > 64) return fail(UNSUPPORTED, who + ": more than 64 query rows a request and key-value head: tb_prefill_paged_q8");
    return OK;
}

uint32_t groups_of(uint32_t heads, uint32_t kv_heads, uint32_t most) { return (heads / kv_heads * most + 7) / 8; }
constexpr size_t COUNT_BYTES = 4096;  // counters first, at one place whatever the shape, so that calls of different shapes may share scratch
size_t scratch_bytes(const tb_context* ctx, uint32_t head_dim) { return COUNT_BYTES + (size_t)2 * most_blocks(ctx, head_dim) * (16 + 8 * (size_t)head_dim) * 4; }

template <int D>
cudaError_t run(tb_context* ctx, uint32_t grid, const PagedArgs& a) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(paged_attend_kernel<D>, smem_bytes<D>() + (MAX_REQUESTS + 1) * 4, ctx->gpu, done);
    if (e != cudaSuccess) return e;
    return launch_kernel(ctx, paged_attend_kernel<D>, dim3(grid), dim3(THREADS), smem_bytes<D>() + ((size_t)a.requests + 1) * 4, true, a);
}

int launch_attend_paged(tb_context* ctx, const tb_paged_attend& p) {
    const tb_pages& c = p.cache;
    const uint32_t groups = groups_of(p.heads, c.kv_heads, p.most), grid = most_blocks(ctx, c.head_dim);
    const uint64_t tiles = ((uint64_t)c.width * c.page + TILE - 1) / TILE;
    if (tiles * c.requests > 0xffffffffull / c.kv_heads / groups) return fail(OUT_OF_RANGE, "tb_attend_paged_q8: more than 2^32 tiles of keys");
    const size_t need = scratch_bytes(ctx, c.head_dim);
    if (grid > COUNT_BYTES / 4) return fail(UNSUPPORTED, "tb_attend_paged_q8: a GPU of that many multiprocessors");
    if (!p.scratch || !aligned(p.scratch, 16) || p.scratch_bytes < need)
        return fail(OUT_OF_RANGE, "tb_attend_paged_q8: needs " + std::to_string(need) + " bytes of 16-byte aligned scratch (tb_paged_scratch_bytes)");
    PagedArgs a{};
    a.k = c.k, a.v = c.v, a.ks = c.k_scale, a.vs = c.v_scale, a.table = c.table, a.pages = c.pages, a.shift = log2_of(c.page), a.kv_heads = c.kv_heads;
    a.requests = c.requests, a.width = c.width, a.q = p.q, a.q_stride = p.q_stride, a.q_f16 = p.q_dtype == TB_F16, a.starts = p.starts, a.lengths = p.lengths;
    a.tokens = p.tokens, a.heads = p.heads, a.ratio = p.heads / c.kv_heads, a.most = p.most, a.window = p.window > 0x7fffffffu ? 0 : p.window, a.least = 4;
    a.scale = p.scale * 1.4426950408889634f, a.out = p.out, a.out_stride = p.out_stride, a.out_f16 = p.out_dtype == TB_F16;
    a.count = static_cast<uint32_t*>(p.scratch);
    a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p.scratch) + COUNT_BYTES);
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    switch (c.head_dim) {
        case 64: TB_CUDA(run<64>(ctx, grid, a)); break;
        case 128: TB_CUDA(run<128>(ctx, grid, a)); break;
        case 256: TB_CUDA(run<256>(ctx, grid, a)); break;
        default: TB_CUDA(run<512>(ctx, grid, a)); break;
    }
    return OK;
}

}  // namespace

}  // namespace tb

using namespace tb;

extern "C" size_t tb_paged_scratch_bytes(const tb_context* ctx, uint32_t head_dim) { return ctx ? scratch_bytes(ctx, head_dim) : 0; }

extern "C" int tb_attend_paged_q8(tb_context* ctx, const tb_paged_attend* args) {
    return entry([&] {
        TB_TRY(check_attend(args, "tb_attend_paged_q8", true));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        return args->tokens == 0 ? (int)OK : launch_attend_paged(ctx, *args);
    });
}

extern "C" int tb_prefill_paged_q8(tb_context* ctx, const tb_paged_attend* args) {
    return entry([&] {
        TB_TRY(check_attend(args, "tb_prefill_paged_q8", false));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        if (args->tokens == 0) return (int)OK;
        return prefill_paged_supports(*args) ? launch_prefill_paged(ctx, *args) : launch_attend_paged(ctx, *args);
    });
}
