// Decode attention over the paged 8-bit cache (tb_attend_paged_q8): one or a few new tokens of every request, ragged lengths.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(scale log2(e) q.k_j - m): each visible key and value is read once, one byte a
// number, and that is what bounds it.  The work of all requests is laid out in a line of tiles of 64 positions (request, then
// key-value head, then tile) and cut into equal shares, one a block, whatever the lengths: a prefix sum over the requests, repeated
// by every block, finds a block's place.  A block whose share ends inside a line of keys leaves its maximum, sum and outputs in
// scratch; the last of 32 neighbours to arrive (a counter, nobody waits) adds theirs up, the last of the line's sets of 32 adds up
// those, always in the order of the positions.
//
// A warp takes 16 positions at a time.  It copies their codes into a ring of its own in shared memory (cp.async, a few slices ahead, so
// that no barrier is needed and no register holds what is on its way) and reads them from there as operands of mma.sync.m16n8k16;
// tcgen05 has no place here, a tile of 64 keys against 8 query rows is two orders of magnitude below one of its tiles.  A sum does
// not mind the order of its terms, so the operands' order is chosen for the loads: a thread's four dimensions (or tokens) of an MMA
// step lie side by side, 16 bytes of a row feed four steps, and the 16-byte pieces of a row are permuted so that eight lanes meet no
// bank twice.  A code becomes f16 by byte permutes: 0x6400 | (code + 128) is 1152 + code, one packed subtraction leaves the code.
//   S = Q K^T: rows 0-7 of the A operand hold the queries rounded to f16, rows 8-15 what the rounding left, so the sum of the
//   two halves is the f32 product to 2^-22; the page's scale, a power of two, multiplies the score.
//   O^T = V^T P^T: the scores' accumulator is the B operand's layout as it stands; the weights again go in two f16 parts.  A page's
//   value scale multiplies the weights, relative to the largest scale met so far, so they stay within f16.
// Softmax statistics and sums are f32.
//
// Measured: 96 requests of up to 16384 positions, 32 query heads on 8 of 128, 1.12 GB: 235 us, 4.8 TB/s or 73 % of a copy's rate; 446
// instructions for 16 positions keep the schedulers 59 % busy, the rest is the conversion's latency.  Two requests of up to 131071
// positions, heads of 512: 103 us (3.7 TB/s; registers and rings leave one block a multiprocessor).  One request of 4096 positions 13 us, 33
// with a window of 512 17 us: the trips to the lengths, the page table, the scales and the codes, and code that is met for the first time.
#include <algorithm>

#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t TILE = 64;
constexpr uint32_t CHUNKS = MAX_REQUESTS / 32;  // chunks of 32 requests, a lane each, with a prefix sum over them
constexpr uint32_t SET = 32;          // partial results of a line that one block adds up

template <int D>
struct Shape {
    // Warps as registers allow (D / 4 hold the output), rings as shared memory does: 16 to 32 KiB a warp, a slice in use and the others
    // on their way.
    static constexpr int WARPS = D == 512 ? 6 : 4, THREADS = WARPS * 32, RESIDENT = D == 512 ? 1 : 3;  // blocks a multiprocessor
    static constexpr int SLICE = D <= 128 ? 32 : 16, HALVES = SLICE / 16;  // positions a warp takes at a time; a page holds sixteen at least
    static constexpr int STAGES = D == 64 ? 4 : 2;
    static constexpr int HALF = 16 * D, STAGE = 2 * HALVES * HALF;  // sixteen positions' keys (or values); a slice's keys, then its values
    static constexpr int OFF_RING = D * 32, RING = STAGES * STAGE, BYTES = OFF_RING + WARPS * RING;
    static_assert(RING >= 8 * D * 4, "a warp's outputs go over its ring at the end of a line");
    static_assert(RESIDENT * (BYTES + 4096) <= 228 * 1024, "over what a multiprocessor has");
};

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
    uint32_t* count;          // [512]: of the line that a block begins and does not finish; [512]: of the set that a block is first of
    unsigned long long q_stride, out_stride;
    uint32_t pages, shift, kv_heads, requests, width, tokens, heads, ratio, most, window;
    float scale;              // softmax scale times log2(e)
    int q_f16, out_f16;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Where 16-byte piece c of row r of a slice lies.  Keys are read by eight lanes as four pieces of two neighbouring rows, values as two
// pieces of rows 0, 2, 4, 6 (or 1, 3, 5, 7): no bank twice in either.
template <int D>
__device__ __forceinline__ uint32_t key_at(uint32_t r, uint32_t c) {
    return D == 64 ? r * 64 + c * 16 : r * D + ((c ^ ((r & 1) << 2)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t value_at(uint32_t r, uint32_t c) {
    return D == 64 ? (r >> 1) * 128 + (((r & 1) ^ ((r >> 2) & 1)) << 6) + ((c ^ (r & 2)) << 4) : r * D + ((c ^ (r & 6)) << 4);
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
__global__ void __launch_bounds__(Shape<D>::THREADS, Shape<D>::RESIDENT) paged_attend_kernel(const PagedArgs a) {
    using S = Shape<D>;
    constexpr int MT = D / 16, SEG = D / 64, WARPS = S::WARPS, THREADS = S::THREADS, STAGES = S::STAGES, SLICE = S::SLICE, HALVES = S::HALVES;
    extern __shared__ __align__(128) uint8_t raw[];
    uint4* s_q = reinterpret_cast<uint4*>(raw);                      // [D / 16][32]: the A operand of every step
    __shared__ float s_m[WARPS * 8], s_l[WARPS * 8];
    __shared__ uint32_t s_chunk[CHUNKS + 1];
    __shared__ float s_row[8], s_wt[2][8];
    __shared__ uint32_t s_flag;
    const uint32_t th = threadIdx.x, lane = th & 31, warp = th >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = raw + S::OFF_RING + warp * S::RING;
    pdl_wait();

    // Tiles before each request: a lane a request of one chunk of 32 (`rq`, and `sum` up to and with it).  With more than one chunk the
    // block first adds up all of them.
    Request mine;
    uint32_t chunk = 0, sum;
    auto look = [&](uint32_t c) {
        const uint32_t r = c * 32 + lane;
        mine.tiles = mine.groups = mine.n = 0;
        if (r < a.requests) mine = request_of(a, r);
        uint32_t x = mine.tiles * mine.groups * a.kv_heads;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        return x;
    };
    uint32_t total;
    if (a.requests <= 32) {
        sum = look(0);
        total = __shfl_sync(0xffffffffu, sum, 31);
    } else {
        const uint32_t chunks = (a.requests + 31) / 32;
        for (uint32_t c = warp; c < chunks; c += WARPS) {
            const uint32_t x = look(c);
            if (lane == 31) s_chunk[c] = x;
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t x = 0, v[CHUNKS / 32];
#pragma unroll
            for (uint32_t e = 0; e < CHUNKS / 32; e++) v[e] = x, x += lane * (CHUNKS / 32) + e < chunks ? s_chunk[lane * (CHUNKS / 32) + e] : 0;
            uint32_t y = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= (uint32_t)o) y += z;
            }
#pragma unroll
            for (uint32_t e = 0; e < CHUNKS / 32; e++) s_chunk[lane * (CHUNKS / 32) + e] = y - x + v[e];
            if (lane == 31) s_chunk[CHUNKS] = y;
        }
        __syncthreads();
        total = s_chunk[CHUNKS];
        chunk = 0xffffffffu;
    }
    if (total == 0) return;
    // Equal shares, the first `more` of them a tile larger; the block that has a tile.
    // Two tiles a block at least once there are enough for every other block of a small launch: halves what has to be added up again.
    const uint32_t blocks = min(gridDim.x, total <= 64 ? total : (total + 1) / 2);
    if (blockIdx.x >= blocks) return;
    const uint32_t share = total / blocks, more = total - share * blocks;
    const uint32_t my0 = share * blockIdx.x + min(blockIdx.x, more), my1 = my0 + share + (blockIdx.x < more ? 1 : 0);
    auto block_of = [&](uint32_t x) { return x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share; };

    for (uint32_t at = my0; at < my1;) {
        // The request that tile `at` belongs to: its chunk by bisection (the last one that starts at or before it), then by lane.
        uint32_t offset = 0;
        if (a.requests > 32) {
            uint32_t lo = 0, hi = (a.requests + 31) / 32;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (s_chunk[mid] <= at) lo = mid;
                else hi = mid;
            }
            if (lo != chunk) sum = look(lo);
            chunk = lo;
            offset = s_chunk[lo];
        }
        const uint32_t here = mine.tiles * mine.groups * a.kv_heads;
        const uint32_t who = __ffs(__ballot_sync(0xffffffffu, here != 0 && at < offset + sum)) - 1;
        const uint32_t r = chunk * 32 + who, before = __shfl_sync(0xffffffffu, offset + sum - here, who);
        Request rq;
        rq.first = __shfl_sync(0xffffffffu, mine.first, who), rq.n = __shfl_sync(0xffffffffu, mine.n, who), rq.len = __shfl_sync(0xffffffffu, mine.len, who);
        rq.low = __shfl_sync(0xffffffffu, mine.low, who), rq.tiles = __shfl_sync(0xffffffffu, mine.tiles, who), rq.groups = __shfl_sync(0xffffffffu, mine.groups, who);
        const uint32_t line = (at - before) / rq.tiles, tile0 = (at - before) % rq.tiles;
        const uint32_t kvh = line / rq.groups, group = line % rq.groups;
        const uint32_t line0 = before + line * rq.tiles;  // the line's first tile
        const uint32_t tile1 = min(rq.tiles, tile0 + (my1 - at));
        at += tile1 - tile0;

        // This warp's slices: positions start + SLICE WARPS i on, up to `end`.  A lane looks up the page of the sixteen positions with its
        // number (mod 32), for this batch of 32 and the next.
        const uint32_t start = rq.low + tile0 * TILE + warp * SLICE, end = min(rq.len, rq.low + tile1 * TILE);
        const uint32_t slices = start < end ? (end - start + WARPS * SLICE - 1) / (WARPS * SLICE) : 0;
        auto page_at = [&](uint32_t x) {
            const uint32_t j = start + x / HALVES * (WARPS * SLICE) + x % HALVES * 16;
            const uint32_t id = j < end ? __ldg(a.table + (size_t)r * a.width + (j >> a.shift)) : 0xffffffffu;
            return id < a.pages ? id : 0xffffffffu;
        };
        auto scales_at = [&](uint32_t id) {
            const size_t p = (size_t)id * a.kv_heads + kvh;
            return id != 0xffffffffu ? make_float2(__ldg(a.ks + p), __ldg(a.vs + p)) : make_float2(0.0f, 0.0f);
        };
        uint32_t id = page_at(lane), id1 = page_at(32 + lane);
        // The queries of this line, asked for before anything waits for the pages: row i is (token i / ratio, head i % ratio) of the
        // group's eight, scaled so that its largest lies in [1, 2), in two f16 parts, in the order the MMA wants them.
        constexpr uint32_t QROWS = (8 + WARPS - 1) / WARPS;
        float qx[QROWS][D / 32];
#pragma unroll
        for (uint32_t k = 0; k < QROWS; k++) {
            const uint32_t row = group * 8 + warp + k * WARPS, tok = row / a.ratio, head = kvh * a.ratio + row % a.ratio;
            const unsigned long long p = (unsigned long long)(rq.first + tok) * a.q_stride + (unsigned long long)head * D + lane;
#pragma unroll
            for (int e = 0; e < D / 32; e++)
                qx[k][e] = tok >= rq.n || warp + k * WARPS >= 8 ? 0.0f : a.q_f16 ? __half2float(static_cast<const __half*>(a.q)[p + e * 32]) : static_cast<const float*>(a.q)[p + e * 32];
        }
        float2 sc = scales_at(id), sc1 = make_float2(0.0f, 0.0f);
        const uint32_t inside = (1u << a.shift) - 1;
        uint32_t to = 0;  // the stage that is filled next
        auto fetch = [&](uint32_t i, uint32_t base) {  // slice i into its stage; base: the first sixteen of the batch that `id` is of
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                const uint32_t x = i * HALVES + h, pid = __shfl_sync(0xffffffffu, x < base + 32 ? id : id1, x & 31);
                if (i < slices && pid != 0xffffffffu) {
                    const uint32_t j = start + i * (WARPS * SLICE) + h * 16;
                    const size_t from = ((((size_t)pid * a.kv_heads + kvh) << a.shift) + (j & inside)) * D + lane * 16;
                    uint8_t* stage = ring + to * S::STAGE + h * S::HALF;
#pragma unroll
                    for (int e = 0; e < D / 32; e++) copy16(stage + key_at<D>((e * 32 + lane) / (D / 16), (e * 32 + lane) % (D / 16)), a.k + from + e * 512);
#pragma unroll
                    for (int e = 0; e < D / 32; e++)
                        copy16(stage + HALVES * S::HALF + value_at<D>((e * 32 + lane) / (D / 16), (e * 32 + lane) % (D / 16)), a.v + from + e * 512);
                }
            }
            copy_commit();
            to = to + 1 == STAGES ? 0 : to + 1;
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) fetch(i, 0);

#pragma unroll
        for (uint32_t k = 0; k < QROWS; k++) {
            const uint32_t mine_row = warp + k * WARPS;
            if (mine_row >= 8) break;
            float big = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 32; e++) big = fmaxf(big, fabsf(qx[k][e]));
            big = warp_max(big);
            const uint32_t expo = min(max(__float_as_uint(big) >> 23, 1u), 253u);  // infinities stay what they are
            const float inv = __uint_as_float((254u - expo) << 23);
            if (lane == 0) s_row[mine_row] = a.scale * __uint_as_float(expo << 23);
            __half* dst = reinterpret_cast<__half*>(s_q);
#pragma unroll
            for (int e = 0; e < D / 32; e++) {
                const uint32_t d = e * 32 + lane, step = d / 64 * 4 + d % 16 / 4, owner = mine_row * 4 + d % 64 / 16, reg = (d & 2), half = d & 1;
                const float y = qx[k][e] * inv;
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
        uint32_t at_stage = 0;
        for (uint32_t i = 0; i < slices; i++) {
            const uint32_t x0 = i * HALVES, base = x0 & ~31u;
            if (i != 0 && x0 == base) id = id1, sc = sc1, id1 = page_at(base + 32 + lane);
            if ((x0 & 31) == 16) sc1 = scales_at(id1);
            copy_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of this slice are there, and every lane is done with the stage that is filled next
            fetch(i + STAGES - 1, base);
            float ks[HALVES], vs[HALVES];
            bool real[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                real[h] = __shfl_sync(0xffffffffu, id, (x0 + h) & 31) != 0xffffffffu;  // no page: nothing to see
                ks[h] = __shfl_sync(0xffffffffu, sc.x, (x0 + h) & 31) * factor, vs[h] = __shfl_sync(0xffffffffu, sc.y, (x0 + h) & 31);
            }
            const uint32_t j0 = start + i * (WARPS * SLICE);
            const uint8_t* kp = ring + at_stage * S::STAGE;
            const uint8_t* vp = kp + HALVES * S::HALF;
            at_stage = at_stage + 1 == STAGES ? 0 : at_stage + 1;
            // Scores of tokens 8 j + 2 t, + 1 of the slice (c[j]) for query row g.
            // Four accumulators at least, so that the products need not wait for one another.
            constexpr int SPLIT = HALVES == 1 ? 2 : 1;
            float c[2 * HALVES * SPLIT][4] = {};
#pragma unroll
            for (int s = 0; s < SEG; s++) {
                uint4 k[2 * HALVES];
#pragma unroll
                for (int j = 0; j < 2 * HALVES; j++) k[j] = *reinterpret_cast<const uint4*>(kp + (j >> 1) * S::HALF + key_at<D>((j & 1) * 8 + g, s * 4 + t));
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint4 q = s_q[(s * 4 + e) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 2 * HALVES; j++) {
                        const uint32_t w = (e == 0 ? k[j].x : e == 1 ? k[j].y : e == 2 ? k[j].z : k[j].w) ^ 0x80808080u;
                        mma16816(c[j + (e & (SPLIT - 1)) * 2 * HALVES], q.x, q.y, q.z, q.w, halves(w, LOW), halves(w, HIGH));
                    }
                }
            }
            if constexpr (SPLIT == 2)
#pragma unroll
                for (int j = 0; j < 2 * HALVES; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) c[j][e] += c[j + 2 * HALVES][e];
            float s[2 * HALVES][2];
            float top = m;
#pragma unroll
            for (int j = 0; j < 2 * HALVES; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int at_j = (int)j0 + j * 8 + 2 * (int)t + e;
                    s[j][e] = at_j > pos || at_j < oldest || !real[j >> 1] ? -INFINITY : (c[j][e] + c[j][2 + e]) * ks[j >> 1];
                    top = fmaxf(top, s[j][e]);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float from = top == -INFINITY ? 0.0f : top;
            float turn = ex2(m - from);  // 0 before the first visible key
            m = top;
            float ratio[HALVES];
            float vnew = vref;
#pragma unroll
            for (int h = 0; h < HALVES; h++) ratio[h] = 1.0f, vnew = fmaxf(vnew, vs[h]);
            const float corr = turn;
            if (vnew != vref || vs[0] != vref || vs[HALVES - 1] != vref) {  // the same in every lane
#pragma unroll
                for (int h = 0; h < HALVES; h++) ratio[h] = vnew > 0.0f ? __fdiv_rn(vs[h], vnew) : 0.0f;
                turn *= vnew > 0.0f ? __fdiv_rn(vref, vnew) : 0.0f;
                vref = vnew;
            }
            float sum = 0.0f;
            uint32_t hi[2 * HALVES], lo[2 * HALVES];
#pragma unroll
            for (int j = 0; j < 2 * HALVES; j++) {
                const float p0 = ex2(s[j][0] - from), p1 = ex2(s[j][1] - from);
                sum += p0 + p1;
                const float w0 = p0 * ratio[j >> 1], w1 = p1 * ratio[j >> 1];
                hi[j] = pack(w0, w1);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
                lo[j] = pack(w0 - f.x, w1 - f.y);
            }
            l = fmaf(l, corr, sum);
            if (__any_sync(0xffffffffu, turn != 1.0f)) {
                const float c0 = __shfl_sync(0xffffffffu, turn, 8 * t), c1 = __shfl_sync(0xffffffffu, turn, 8 * t + 4);  // rows 2t, 2t + 1
#pragma unroll
                for (int k = 0; k < MT; k++) acc[k][0] *= c0, acc[k][1] *= c1, acc[k][2] *= c0, acc[k][3] *= c1;
            }
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                const uint8_t* v = vp + h * S::HALF;
                const uint32_t h0 = hi[2 * h], h1 = hi[2 * h + 1], l0 = lo[2 * h], l1 = lo[2 * h + 1];
                // Values of tokens 2t, 2t + 1, 2t + 8, 2t + 9; four dimensions of the four tokens make two MMA tiles' A operands.
                auto four = [&](uint32_t wa, uint32_t wb, uint32_t wc, uint32_t wd, float (&even)[4], float (&odd)[4]) {
                    const uint32_t ab = __byte_perm(wa, wb, 0x5140) ^ 0x80808080u, cd = __byte_perm(wc, wd, 0x5140) ^ 0x80808080u;
                    const uint32_t ab2 = __byte_perm(wa, wb, 0x7362) ^ 0x80808080u, cd2 = __byte_perm(wc, wd, 0x7362) ^ 0x80808080u;
                    const uint32_t e0 = halves(ab, LOW), e1 = halves(ab, HIGH), e2 = halves(cd, LOW), e3 = halves(cd, HIGH);
                    mma16816(even, e0, e1, e2, e3, h0, h1);
                    const uint32_t o0 = halves(ab2, LOW), o1 = halves(ab2, HIGH), o2 = halves(cd2, LOW), o3 = halves(cd2, HIGH);
                    mma16816(odd, o0, o1, o2, o3, h0, h1);
                    mma16816(even, e0, e1, e2, e3, l0, l1);
                    mma16816(odd, o0, o1, o2, o3, l0, l1);
                };
                if constexpr (D == 64) {
                    auto row = [&](uint32_t r2) { return *reinterpret_cast<const uint2*>(v + value_at<D>(r2, g >> 1) + (g & 1) * 8); };
                    const uint2 va = row(2 * t), vb = row(2 * t + 1), vc = row(2 * t + 8), vd = row(2 * t + 9);
                    four(va.x, vb.x, vc.x, vd.x, acc[0], acc[1]);
                    four(va.y, vb.y, vc.y, vd.y, acc[2], acc[3]);
                } else {
#pragma unroll
                    for (int sg = 0; sg < D / 128; sg++) {
                        auto row = [&](uint32_t r2) { return *reinterpret_cast<const uint4*>(v + value_at<D>(r2, sg * 8 + g)); };
                        const uint4 va = row(2 * t), vb = row(2 * t + 1), vc = row(2 * t + 8), vd = row(2 * t + 9);
                        four(va.x, vb.x, vc.x, vd.x, acc[sg * 8], acc[sg * 8 + 1]);
                        four(va.y, vb.y, vc.y, vd.y, acc[sg * 8 + 2], acc[sg * 8 + 3]);
                        four(va.z, vb.z, vc.z, vd.z, acc[sg * 8 + 4], acc[sg * 8 + 5]);
                        four(va.w, vb.w, vc.w, vd.w, acc[sg * 8 + 6], acc[sg * 8 + 7]);
                    }
                }
            }
        }
        copy_wait<0>();
        __syncwarp();  // the ring is free
        // The warps meet: statistics, then outputs in units of the values, over a warp's own ring.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) s_m[warp * 8 + g] = m, s_l[warp * 8 + g] = l;
        {
            float* dst = reinterpret_cast<float*>(ring);
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
        const uint32_t rows = min(8u, rq.n * a.ratio - group * 8);
        constexpr uint32_t SLOT = 16 + 8 * D;
        float* slot = a.partial + (size_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * SLOT;  // at most one line is begun and not finished, and one finished and not begun
        auto store = [&](uint32_t row, uint32_t d, float4 v, float sum) {
            const uint32_t i = group * 8 + row, tok = i / a.ratio, head = kvh * a.ratio + i % a.ratio;
            const unsigned long long p = (unsigned long long)(rq.first + tok) * a.out_stride + (unsigned long long)head * D + d;
            const float f = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            v.x *= f, v.y *= f, v.z *= f, v.w *= f;
            if (a.out_f16) *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + p) = make_uint2(pack(v.x, v.y), pack(v.z, v.w));
            else *reinterpret_cast<float4*>(static_cast<float*>(a.out) + p) = v;
        };
        for (uint32_t e = th * 4; e < rows * D; e += THREADS * 4) {
            const uint32_t row = e / D, d = e % D;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_m[w * 8 + row]);
            const float from = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = ex2(s_m[w * 8 + row] - from);
                const float4 x = *reinterpret_cast<const float4*>(raw + S::OFF_RING + w * S::RING + (row * D + d) * 4);
                sum = fmaf(s_l[w * 8 + row], f, sum);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
            }
            if (whole) {
                store(row, d, v, sum);
            } else {
                *reinterpret_cast<float4*>(slot + 16 + e) = v;
                if (d == 0) slot[row] = top, slot[8 + row] = sum;
            }
        }
        if (!whole) {
            // Which blocks share this line.
            const uint32_t b0 = block_of(line0), b1 = block_of(line0 + rq.tiles - 1);
            auto slot_of = [&](uint32_t b) { return a.partial + (size_t)(2 * b + (b == b0 ? 1 : 0)) * SLOT; };
            auto arrive = [&](uint32_t* cnt, uint32_t of) {  // whether this block is the last of `of`
                __syncthreads();
                if (th == 0) {
                    uint32_t before_me;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before_me) : "l"(cnt) : "memory");
                    s_flag = before_me == of - 1;
                    if (before_me == of - 1) *cnt = 0;
                }
                __syncthreads();
                return s_flag != 0;
            };
            // First the set of neighbours this block belongs to, its sum over the first one's own result; then the sets.  With one set that
            // is all.  A block alone in its set may be the first of another line's set as well, so it takes no counter.
            const uint32_t count = b1 - b0 + 1;
            uint32_t first = b0 + (blockIdx.x - b0) / SET * SET, step = 1, of = min(SET, b1 + 1 - first);
            bool final = count <= SET;
#pragma unroll 1
            for (;;) {
                if (of > 1 && !arrive(final ? a.count + b0 : a.count + 512 + first, of)) break;
                if (of > 1 || final) {
#pragma unroll 1
                    for (uint32_t e = th * 4; e < rows * D; e += THREADS * 4) {
                        const uint32_t row = e / D, d = e % D;
                        float top = -INFINITY, sum = 0.0f;
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                        for (uint32_t k = 0; k < of; k += 16) {  // sixteen on their way at a time
                            float mb[16], lb[16];
                            float4 x[16];
#pragma unroll
                            for (uint32_t u = 0; u < 16; u++) {
                                mb[u] = -INFINITY, lb[u] = 0.0f, x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (k + u < of) {
                                    const float* p = slot_of(first + (k + u) * step);
                                    mb[u] = __ldcg(p + row), lb[u] = __ldcg(p + 8 + row), x[u] = __ldcg(reinterpret_cast<const float4*>(p + 16 + e));
                                }
                            }
                            float now = top;
#pragma unroll
                            for (uint32_t u = 0; u < 16; u++) now = fmaxf(now, mb[u]);
                            const float from = now == -INFINITY ? 0.0f : now, f0 = ex2(top - from);
                            sum *= f0, v.x *= f0, v.y *= f0, v.z *= f0, v.w *= f0;
#pragma unroll
                            for (uint32_t u = 0; u < 16; u++) {
                                const float f = ex2(mb[u] - from);
                                sum = fmaf(lb[u], f, sum);
                                v.x = fmaf(x[u].x, f, v.x), v.y = fmaf(x[u].y, f, v.y), v.z = fmaf(x[u].z, f, v.z), v.w = fmaf(x[u].w, f, v.w);
                            }
                            top = now;
                        }
                        if (final) {
                            store(row, d, v, sum);
                        } else {  // only this thread reads these
                            *reinterpret_cast<float4*>(slot_of(first) + 16 + e) = v;
                            if (d == 0) s_wt[0][row] = top, s_wt[1][row] = sum;
                        }
                    }
                }
                if (final) break;
                __syncthreads();  // the statistics once every thread has read the old ones
                if (of > 1 && th < rows) slot_of(first)[th] = s_wt[0][th], slot_of(first)[8 + th] = s_wt[1][th];
                first = b0, step = SET, of = (count + SET - 1) / SET, final = true;
            }
        }
        __syncthreads();  // the next line writes the queries and the warps' results again
    }
}

// Blocks a launch has at most: what is resident at once.
uint32_t most_blocks(const tb_context* ctx, uint32_t head_dim) { return (uint32_t)ctx->sms * (head_dim == 512 ? Shape<512>::RESIDENT : Shape<64>::RESIDENT); }

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
size_t scratch_bytes(const tb_context* ctx, uint32_t head_dim) { return PAGED_COUNT_BYTES + (size_t)2 * most_blocks(ctx, head_dim) * (16 + 8 * (size_t)head_dim) * 4; }

template <int D>
cudaError_t run(tb_context* ctx, uint32_t grid, const PagedArgs& a) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(paged_attend_kernel<D>, Shape<D>::BYTES, ctx->gpu, done);
    if (e != cudaSuccess) return e;
    return launch_kernel(ctx, paged_attend_kernel<D>, dim3(grid), dim3(Shape<D>::THREADS), Shape<D>::BYTES, true, a);
}

int launch_attend_paged(tb_context* ctx, const tb_paged_attend& p) {
    const tb_pages& c = p.cache;
    const uint32_t groups = groups_of(p.heads, c.kv_heads, p.most), grid = most_blocks(ctx, c.head_dim);
    const uint64_t tiles = ((uint64_t)c.width * c.page + TILE - 1) / TILE;
    if (tiles * c.requests > 0xffffffffull / c.kv_heads / groups) return fail(OUT_OF_RANGE, "tb_attend_paged_q8: more than 2^32 tiles of keys");
    if (grid > PAGED_COUNT_BYTES / 8) return fail(UNSUPPORTED, "tb_attend_paged_q8: a GPU of that many multiprocessors");
    TB_TRY(check_scratch(ctx, p, "tb_attend_paged_q8"));
    PagedArgs a{};
    a.k = c.k, a.v = c.v, a.ks = c.k_scale, a.vs = c.v_scale, a.table = c.table, a.pages = c.pages, a.shift = log2_of(c.page), a.kv_heads = c.kv_heads;
    a.requests = c.requests, a.width = c.width, a.q = p.q, a.q_stride = p.q_stride, a.q_f16 = p.q_dtype == TB_F16, a.starts = p.starts, a.lengths = p.lengths;
    a.tokens = p.tokens, a.heads = p.heads, a.ratio = p.heads / c.kv_heads, a.most = p.most, a.window = p.window > 0x7fffffffu ? 0 : p.window;
    a.scale = p.scale * 1.4426950408889634f, a.out = p.out, a.out_stride = p.out_stride, a.out_f16 = p.out_dtype == TB_F16;
    a.count = static_cast<uint32_t*>(p.scratch);
    a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p.scratch) + PAGED_COUNT_BYTES);
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

size_t paged_scratch_bytes(const tb_context* ctx, uint32_t head_dim) { return std::max(scratch_bytes(ctx, head_dim), prefill_scratch_bytes(ctx, head_dim)); }

int check_scratch(const tb_context* ctx, const tb_paged_attend& p, const std::string& who) {
    const size_t need = paged_scratch_bytes(ctx, p.cache.head_dim);
    if (p.scratch && aligned(p.scratch, 16) && p.scratch_bytes >= need) return OK;
    return fail(OUT_OF_RANGE, who + ": needs " + std::to_string(need) + " bytes of 16-byte aligned scratch (tb_paged_scratch_bytes)");
}

}  // namespace tb

using namespace tb;

extern "C" size_t tb_paged_scratch_bytes(const tb_context* ctx, uint32_t head_dim) { return ctx ? paged_scratch_bytes(ctx, head_dim) : 0; }

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
        return args->tokens == 0 ? (int)OK : launch_prefill_paged(ctx, *args);
    });
}
