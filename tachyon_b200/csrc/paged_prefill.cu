// Prefill attention over the paged 8-bit cache on the fifth-generation tensor cores (tb_prefill_paged_q8).
//
// out = sum_j p_j v_j / sum_j p_j, p_j = 2^(scale log2(e) q.k_j - m): 4 D operations a query row and key.  A row tile is 128 query rows
// of one request and key-value head (row = token * ratio + head); a block walks its keys in tiles of KT positions that start at
// multiples of KT.  Where there are fewer row tiles than multiprocessors the keys are cut into pieces, one a block; a first kernel of
// one block says who does what, a last one adds the pieces up.  Everything the tensor cores read of the queries' side stays in tensor
// memory: the queries (stored once), the scores S = Q K^T (two buffers), the probabilities (f16, over the scores they came from) and
// the output, so shared memory only carries keys and values: codes turned to f16 on the way in, a byte read where an f16 cache takes
// two.  Sixteen warps:
//   warps 0-7    softmax, two threads a query row, half of a tile's keys each: scores out of tensor memory, maximum (the two trade theirs
//                through shared memory), exponentials, probabilities back into it; the running maximum moves only when a tile passes it
//                by 2^8, and only then the output is rescaled;
//   warps 8-13   codes to f16: 16 codes a thread and turn, loaded a tile ahead, as 0x6400 | (code + 128) by byte permutes and one packed
//                fused multiply-add (x * f - 1152 f, exact), stored in the 128-byte swizzle; keys K-major, values as they lie in
//                the cache, which is the MN-major form of a B operand;
//   warp 14      one thread issues the products, S of tile i + 1 ahead of P V of tile i;
//   warp 15      looks up the pages of the tiles ahead: page numbers, the pages' factors, which keys have a page at all.
// A page's scales are powers of two.  Keys carry theirs relative to the tile's largest, which multiplies the scores; values theirs
// relative to the largest scale met so far, which multiplies the output at the end (and rescales it when it grows).  Every wait is bounded.
//
// Measured, 148 row tiles over 7.6 to 10 thousand keys: heads of 256 216 us (793 TFLOP/s, 48 % of the tensor cores' measured 1654), of
// 128 120 us (714), of 64 111 us (387).  What bounds it: with heads of 256 the products' own issue, 2400 clocks a tile of 64 keys of
// which S takes 1000 (a product of 64 columns takes no less than half of one of 256) and P V 520, and the waits between them; with heads
// of 128 and 64 the softmax, 2600 clocks a tile of 128 keys, 1400 of them exponentials and their conversion.  Heads of 512 work S out four
// times, once for each 128 dimensions of the output: 1412 us.  Tried without gain: a third of the exponentials by a polynomial, packed
// multiply-adds, registers moved between the roles, 20 warps (what did not fit the registers cost more), P V ahead of the next S, a
// block that goes on to its next piece (the same work with the loop's registers on top: 5 to 20 % slower).
#include <algorithm>

#include "common.cuh"
#include "paged.h"
#include "tc.cuh"

namespace tb {

namespace {

using namespace tc;

constexpr int ROWS = 128, SOFT_WARPS = 8, CONVERT_WARPS = 6, GROUP_WARPS = 2, GROUPS = CONVERT_WARPS / GROUP_WARPS, MMA_WARP = SOFT_WARPS + CONVERT_WARPS, THREADS = (MMA_WARP + 2) * 32, AHEAD = 8;
constexpr uint32_t FEW = 128;    // requests up to which they are ordered and their row tiles cut: more have row tiles enough
constexpr uint32_t LEAST = 384;  // keys of a piece, at least: with twice as many 100 tokens behind 8092 (heads of 128) took 39 us instead of 30, with half as many 60 behind 8132 (256) 35 instead of 32

// A piece in the scratch: the output [VD / 4][128 rows][4], the rows' maxima, their sums.
template <int VD>
constexpr uint32_t PIECE = (VD + 2) * ROWS;

// Heads of D; a block works out VD of the output's dimensions (all of them, but for heads of 512, whose output, queries and scores
// would take more than the 512 columns: four blocks take 128 each, every one with scores of its own).
template <int D, int VD>
struct Shape {
    static constexpr int KT = D >= 256 ? 64 : 128;            // keys a tile
    static constexpr int KCH = KT * 128;                      // a box of 64 dimensions x KT keys
    static constexpr int K_STAGE = D / 64 * KCH, V_STAGE = VD / 64 * KCH;  // a tile's keys and values
    static constexpr int QC = D <= 256 ? D : 128, Q_ROW = QC * 2 + 16;  // dimensions of the queries in shared memory at once, on their way to tensor memory
    static constexpr int OFF_V = 2 * K_STAGE, OFF_Q = OFF_V + 2 * V_STAGE, BYTES = 1024 + OFF_Q + ROWS * Q_ROW;
    static constexpr int COL_O = 0, COL_S = VD, COL_Q = VD + 2 * KT;  // tensor-memory columns
    // kind::f16, f32 accumulator, A from tensor memory; N >> 3 at bit 17, M >> 4 at bit 24, bit 16: B is MN-major.
    static constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    static constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(VD >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    static_assert(COL_Q + D / 2 <= 512, "tensor memory has 512 columns");
};

struct Row {  // a request, in the order the blocks take them
    uint32_t r, first, n, len, parts;  // its first row of q, its new tokens, its length, the pieces its row tiles are cut into
    uint32_t unused[3];
};

struct Split {  // what the second kernel reads of a piece: those of a row tile follow one another, the first says how many there are
    uint32_t parts, row0, kvh, first, n;
};

struct Ahead {  // what the last warp finds out about a tile, for every sixteen of its keys: no page is smaller
    unsigned long long at[8];  // where their first code lies (in page 0 where there is no page: its factors are 0)
    uint2 kf[8], vf[8];        // their page's factor f and -1152 f, two f16 each
    uint32_t keys[4];          // bit c: key c of the tile has a page
    float kref, shrink;        // multiplies the scores; what the output is multiplied by before this tile
};

struct Shared {
    uint64_t q_full, k_full[2], v_full[2], s_full[2], p_ready[2], pv_done[AHEAD], known[AHEAD], drained;
    uint32_t tmem;
    float vref;
    Ahead ahead[AHEAD];
    Row row;           // the block's request
    uint32_t place;    // which of its pieces
    unsigned long long q_at[ROWS];  // where a row's queries lie, all bits set: nowhere
    float q_inv[ROWS];              // what they are multiplied by
    float xch[2][2][ROWS];  // [tile's parity][half][row]: what a row's two threads trade: each tile their maxima, at the end their sums
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
    uint32_t shares, blocks;  // blocks that run at once; that are launched
    uint32_t* head;   // how many blocks have a piece of a row tile that was cut, how many have one at all
    uint32_t* before; // [requests]: pieces of a key-value head before each request, in the order of `rows`
    Row* rows;        // [requests]
    Split* splits;    // [2 shares]
    float* partial;   // [2 shares][D / VD] pieces
};

// D = A B with A in tensor memory, and the commit of what was issued; the whole warp calls them, the thread with `leader` issues.  A
// product of 128 rows takes 62 clocks with 64 columns, 71 with 128 and 128 with 256.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_commit_by(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
        "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 32 columns of this thread's lane, there when the statement is done.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
        "%26, %27, %28, %29, %30, %31"
        "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// 64 columns of this thread's lane, there when the statement is done.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
        "%26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, "
        "%50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63"
        "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
          "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]),
          "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]),
          "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Past the L1, which shares its memory with the tiles: with lines kept there a tile of the benchmark's shape took 1.59 us, so 1.39.
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Eight codes as f16 times a factor (f, -1152 f): a 16-byte piece.
__device__ __forceinline__ uint4 convert8(uint32_t a, uint32_t b, const uint2& factor) {
    const __half2 f = *reinterpret_cast<const __half2*>(&factor.x), off = *reinterpret_cast<const __half2*>(&factor.y);
    uint4 out;
    uint32_t* r = &out.x;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t w = (i ? b : a) ^ 0x80808080u, lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&lo), f, off), y = __hfma2(*reinterpret_cast<const __half2*>(&hi), f, off);
        r[2 * i] = *reinterpret_cast<const uint32_t*>(&x), r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
    return out;
}

// The tiles of keys that a row tile sees: from position `from`, to before position `to`.
template <int KT>
__device__ __forceinline__ uint32_t keys_of(const PrefillArgs& a, uint32_t row0, uint32_t n, int pos0, uint32_t& from, uint32_t& to) {
    const int p_first = pos0 + (int)(row0 / a.ratio), p_last = pos0 + (int)min((row0 + ROWS - 1) / a.ratio, n - 1);
    const int lowest = a.window != 0 && p_first >= (int)a.window ? p_first + 1 - (int)a.window : 0;
    from = (uint32_t)lowest / KT * KT, to = p_last >= 0 ? (uint32_t)p_last + 1 : 0;
    return to > from ? (to - from + KT - 1) / KT : 0u;
}

// What each block will do.  Up to FEW requests are taken longest first, so that the last blocks to start are short ones, and their row
// tiles are cut along the keys: into pieces of an even share of all the work, and where that leaves more pieces than run at once although
// there are fewer row tiles, into the longest pieces that do not.  (By every block for itself this took 7 us a block.)
template <int KT>
__global__ void __launch_bounds__(THREADS) paged_prefill_plan_kernel(const PrefillArgs a) {
    __shared__ uint32_t part[THREADS / 32], order[FEW], seen[FEW], sum;
    __shared__ unsigned long long work;
    const uint32_t th = threadIdx.x, lane = th & 31;
    pdl_wait();
    auto row_of = [&](uint32_t r) {
        Row x{r, a.starts ? __ldg(a.starts + r) : r, 0, min(__ldg(a.lengths + r), a.width << a.shift), 1, {0, 0, 0}};
        const uint32_t next = a.starts ? __ldg(a.starts + r + 1) : r + 1;
        if (next > x.first && x.first < a.tokens) x.n = min(min(next - x.first, a.most), a.tokens - x.first);
        return x;
    };
    auto tiles_of = [&](const Row& x) { return (x.n * a.ratio + ROWS - 1) / ROWS; };
    auto total = [&](uint32_t x) {  // over the block
        for (int o = 16; o != 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (th == 0) sum = 0;
        __syncthreads();
        if (lane == 0 && x != 0) atomicAdd(&sum, x);
        __syncthreads();
        x = sum;
        __syncthreads();
        return x;
    };
    const bool few = a.requests <= FEW;
    uint32_t most = 0xffffffffu;  // tiles of keys of a piece
    if (few) {
        if (th == 0) work = 0;
        __syncthreads();
        unsigned long long product = 0;
        uint32_t mine = 0, tiles = 0;  // tiles of keys of a request's last row tile, which sees most; its row tiles
        if (th < a.requests) {
            uint32_t from, to;
            const Row x = row_of(th);
            tiles = tiles_of(x);
            if (tiles != 0) {
                mine = keys_of<KT>(a, (tiles - 1) * ROWS, x.n, (int)x.len - (int)x.n, from, to);
                product = (unsigned long long)mine * tiles * a.kv_heads;
            }
            seen[th] = mine;
        }
        for (int o = 16; o != 0; o >>= 1) product += __shfl_xor_sync(0xffffffffu, product, o);  // by lanes each for itself: 64-bit atomics on one word, 6 us
        if (lane == 0 && product != 0) atomicAdd(&work, product);
        __syncthreads();
        if (th < a.requests) {
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t o = 0; o < a.requests; o++) {
                const uint32_t other = seen[o];
                rank += other > mine || (other == mine && o < th);
            }
            order[rank] = th;
        }
        most = (uint32_t)min(max((unsigned long long)(LEAST / KT), (work + a.shares - 1) / a.shares), 0x7fffffffull);
        if (total(tiles) * (unsigned long long)a.kv_heads <= a.shares)
            while (total(tiles * max(1u, (mine + most - 1) / most)) * (unsigned long long)a.kv_heads > a.shares) most += (most + 15) / 16;
    }
    auto row_at = [&](uint32_t i) {
        Row x = row_of(few ? order[i] : i);
        if (few) x.parts = max(1u, (seen[x.r] + most - 1) / most);
        return x;
    };
    const uint32_t per = (a.requests + THREADS - 1) / THREADS, r0 = min(th * per, a.requests), r1 = min(r0 + per, a.requests);
    uint32_t mine = 0;
    for (uint32_t i = r0; i < r1; i++) {
        const Row x = row_at(i);
        mine += tiles_of(x) * x.parts;
    }
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    if (lane == 31) part[th >> 5] = x;
    __syncthreads();
    uint32_t at = x - mine, cut = 0;
    for (uint32_t w = 0; w < th >> 5; w++) at += part[w];
    for (uint32_t i = r0; i < r1; i++) {
        const Row y = row_at(i);
        a.rows[i] = y, a.before[i] = at;
        at += tiles_of(y) * y.parts;
        if (y.parts > 1) cut = at;  // those come first
        if (i + 1 == a.requests) a.head[1] = at * a.kv_heads;
    }
    if (few) {  // a request a thread
        if (th == 0) sum = 0;
        __syncthreads();
        if (cut != 0) atomicMax(&sum, cut);
        __syncthreads();
        if (th == 0) a.head[0] = min(sum * a.kv_heads, a.blocks);
    }
}

template <int D, int VD>
__global__ void __launch_bounds__(THREADS, 1) paged_prefill_kernel(const PrefillArgs a, uint32_t* status) {
    using S = Shape<D, VD>;
    constexpr int KT = S::KT;
    extern __shared__ uint8_t raw_unaligned[];
    uint8_t* raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_unaligned) + 1023) & ~uintptr_t(1023));
    __shared__ Shared sh;
    const uint32_t th = threadIdx.x, warp = th >> 5, lane = th & 31;
    pdl_wait();

    if (blockIdx.x >= a.head[1]) return;
    if (warp == MMA_WARP + 1) {  // the block's request: 32 places at once
        const uint32_t item = blockIdx.x / a.kv_heads;
        uint32_t lo = 0, start = 0;
        for (uint32_t step = (a.requests + 31) / 32;; step = (step + 31) / 32) {
            const uint32_t at = lo + lane * step, before = at < a.requests ? a.before[at] : 0xffffffffu;
            const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, before <= item));
            lo += last * step, start = __shfl_sync(0xffffffffu, before, last);
            if (step == 1) break;
        }
        if (lane == 0) sh.row = a.rows[lo], sh.place = item - start;
    }
    if (th == 0) {
        mbar_init(&sh.q_full, SOFT_WARPS), mbar_init(&sh.drained, 1);
        for (int i = 0; i < 2; i++) mbar_init(&sh.k_full[i], GROUP_WARPS), mbar_init(&sh.v_full[i], GROUP_WARPS), mbar_init(&sh.s_full[i], 1), mbar_init(&sh.p_ready[i], SOFT_WARPS);
        for (int i = 0; i < AHEAD; i++) mbar_init(&sh.pv_done[i], 1), mbar_init(&sh.known[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    // A request's last rows, which see most, first; a row tile's pieces behind one another.
    const uint32_t r = sh.row.r, kvh = blockIdx.x % a.kv_heads, parts = sh.row.parts, first = sh.row.first, n = sh.row.n, part = sh.place % parts;
    const uint32_t row0 = ((n * a.ratio + ROWS - 1) / ROWS - 1 - sh.place / parts) * ROWS;
    const int pos0 = (int)sh.row.len - (int)n;  // the first new token's position; negative when the lengths cannot be
    uint32_t tile0, end, nt = keys_of<KT>(a, row0, n, pos0, tile0, end);
    if (parts > 1) {
        const uint32_t each = (nt + parts - 1) / parts, t0 = min(part * each, nt);
        nt = min(each, nt - t0), tile0 += t0 * KT;
        if (th == 0 && blockIdx.y == 0) a.splits[blockIdx.x] = Split{part == 0 ? parts : 0, row0, kvh, first, n};
    }
    bool ok = true;
    // A wait that runs out is noted, and the thread goes on without waiting for anything else.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity)) {
            ok = false;
            atomicCAS(status, ERR_NONE, ERR_WAIT_FULL);
        }
    };

    if (warp < SOFT_WARPS) {
        // ---- queries, softmax, output: a query row's two threads (warps w and w + 4, tensor-memory lane = row) take half of a tile's
        // keys and half of the dimensions each ---------------------------------------------------------------------------
        constexpr int HK = KT / 2, HV = VD / 2;  // half of the keys, of the output's dimensions
        const uint32_t quarter = warp & 3, half = warp >> 2, me = 32 * quarter + lane;
        const uint32_t row = row0 + me, tok = row / a.ratio, head = kvh * a.ratio + row % a.ratio;
        const bool valid = tok < n;
        const uint32_t lanes = tmem + ((32 * quarter) << 16);
        const unsigned long long q_at = (unsigned long long)(first + tok) * a.q_stride + (unsigned long long)head * D;
        auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + (int)quarter) : "memory"); };  // the row's two warps
        // Queries, from the q tensor to tensor memory: a row's two warps fetch their 32 rows, neighbouring lanes neighbouring pieces, and
        // pass them through shared memory as f16.  (A thread that reads its own row touches a line of its own with every load.)
        float factor = a.scale;
        if (nt != 0) {
            constexpr int QC = S::QC, UNITS = QC / 16, PARTS = QC / 8, HQ = QC / 2;
            const uint32_t me64 = half * 32 + lane;
            uint8_t* q_rows = raw + S::OFF_Q + 32 * quarter * S::Q_ROW;
            sh.q_at[me] = valid ? q_at : ~0ull;
            meet();
            if (!a.q_f16) {  // rows are scaled by a power of two so that their largest lies in [1, 2): f16 then loses 2^-11 of it whatever its size
#pragma unroll 2
                for (uint32_t x = half; x < 32; x += 2) {
                    const unsigned long long at = sh.q_at[32 * quarter + x];
                    float big = 0.0f;
#pragma unroll
                    for (int d = 0; d < D; d += 64) {
                        const float2 v = at != ~0ull ? __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(a.q) + at + d) + lane) : make_float2(0.0f, 0.0f);
                        big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
                    }
#pragma unroll
                    for (int o = 16; o != 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    const uint32_t expo = min(max(__float_as_uint(big) >> 23, 1u), 253u);
                    if (lane == 0) sh.q_inv[32 * quarter + x] = __uint_as_float((254u - expo) << 23);
                }
                meet();
                factor *= __uint_as_float((254u << 23) - __float_as_uint(sh.q_inv[me]));
            }
#pragma unroll 1
            for (int c = 0; c < D; c += QC) {
                if (c != 0) meet();
                if (a.q_f16) {
                    uint4 w[UNITS];
#pragma unroll
                    for (int u = 0; u < UNITS; u++) {
                        const unsigned long long at = sh.q_at[32 * quarter + (u * 64 + me64) / PARTS];
                        w[u] = at != ~0ull ? __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + at + c + me64 % PARTS * 8)) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int u = 0; u < UNITS; u++) *reinterpret_cast<uint4*>(q_rows + (u * 64 + me64) / PARTS * S::Q_ROW + me64 % PARTS * 16) = w[u];
                } else {
#pragma unroll 4
                    for (int u = 0; u < UNITS; u++) {
                        const uint32_t x = (u * 64 + me64) / PARTS;
                        const unsigned long long at = sh.q_at[32 * quarter + x];
                        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + c + me64 % PARTS * 8);
                        const float4 v = at != ~0ull ? __ldg(p) : make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = at != ~0ull ? __ldg(p + 1) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        const float inv = sh.q_inv[32 * quarter + x];
                        const __half2 h[4] = {__floats2half2_rn(v.x * inv, v.y * inv), __floats2half2_rn(v.z * inv, v.w * inv), __floats2half2_rn(y.x * inv, y.y * inv),
                                              __floats2half2_rn(y.z * inv, y.w * inv)};
                        *reinterpret_cast<uint4*>(q_rows + x * S::Q_ROW + me64 % PARTS * 16) = *reinterpret_cast<const uint4*>(h);
                    }
                }
                meet();
                const uint8_t* from = raw + S::OFF_Q + me * S::Q_ROW + half * QC;
#pragma unroll 1
                for (int e = 0; e < HQ / 8; e += 4) {
                    uint32_t h[16];
#pragma unroll
                    for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(h + 4 * k) = *reinterpret_cast<const uint4*>(from + (e + k) * 16);
                    tmem_store16(lanes + S::COL_Q + c / 2 + half * (HQ / 2) + e * 4, h);
                }
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
            const float f = info.kref * factor, shrink = info.shrink;
            // Key j0 + c is seen when lo <= c < hi and it has a page.
            const int j0 = (int)(tile0 + i * KT + half * HK), lo = oldest - j0, hi = p + 1 - j0;
            bool all = lo <= 0 && hi >= HK;
            uint32_t keys[HK / 32];
#pragma unroll
            for (int c = 0; c < HK / 32; c++) keys[c] = info.keys[half * (HK / 32) + c], all = all && keys[c] == 0xffffffffu;
            all = __all_sync(0xffffffffu, all);
            wait(&sh.s_full[buf], (i >> 1) & 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t s[HK];
            tmem_load(sbuf + half * HK, s);
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (!all) {
#pragma unroll
                for (int c = 0; c < HK / 32; c++)
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!(32 * c + e >= lo && 32 * c + e < hi && ((keys[c] >> e) & 1u))) s[32 * c + e] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int e = 0; e < HK; e++) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(s[e]));
            float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            sh.xch[buf][half][me] = mt;
            meet();  // also: both have read their scores, so the probabilities may go over them
            mt = fmaxf(mt, sh.xch[buf][half ^ 1][me]);
            mt = mt == -INFINITY ? mt : mt * f;  // f may be 0
            float corr = shrink;
            if (mt > m_used + 8.0f) {  // also a row's first keys (m_used = -inf)
                const float turn = ex2(m_used - mt);
                l_run *= turn;
                corr *= turn;
                m_used = mt;
            }
            const float base = fmaxf(m_used, -1e30f);  // finite: a row that has seen nothing yet gets 2^-inf = 0 and no NaN
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < HK / 32; c++) {
                uint32_t h[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float e0 = ex2(fmaf(__uint_as_float(s[32 * c + 2 * e]), f, -base)), e1 = ex2(fmaf(__uint_as_float(s[32 * c + 2 * e + 1]), f, -base));
                    if (!all && f == 0.0f) e0 = s[32 * c + 2 * e] == 0xff800000u ? 0.0f : e0, e1 = s[32 * c + 2 * e + 1] == 0xff800000u ? 0.0f : e1;  // -inf * 0
                    sum[e & 3] += e0 + e1;
                    const __half2 v = __floats2half2_rn(e0, e1);
                    h[e] = *reinterpret_cast<const uint32_t*>(&v);
                }
                tmem_store16(sbuf + (half * (HK / 32) + c) * 16, h);
            }
            l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (i > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {
                wait(&sh.pv_done[(i - 1) % AHEAD], ((i - 1) / AHEAD) & 1);  // the output must be at rest
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int c = 0; c < HV / 32; c++) {
                    uint32_t o[32];
                    const uint32_t at = lanes + S::COL_O + half * HV + c * 32;
                    tmem_load(at, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tmem_store32(at, o);
                }
            }
            tmem_wait_st();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_ready[buf]);
        }
        if (nt != 0) wait(&sh.pv_done[(nt - 1) % AHEAD], ((nt - 1) / AHEAD) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        sh.xch[nt & 1][half][me] = l_run;  // not the slots of the last tile, which the other warp may still read
        meet();
        l_run += sh.xch[nt & 1][half ^ 1][me];
        if (ok && parts > 1) {  // sums and maximum for the second kernel, the output in columns of four
            float* dst = a.partial + ((size_t)blockIdx.x * (D / VD) + blockIdx.y) * PIECE<VD>;
            if (valid && half == 0) dst[VD * ROWS + me] = m_used, dst[(VD + 1) * ROWS + me] = l_run;
            const float vref = sh.vref;
#pragma unroll 1
            for (int c = 0; c < HV / 32 && nt != 0; c++) {
                uint32_t o[32];
                tmem_load(lanes + S::COL_O + half * HV + c * 32, o);
                if (valid) {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * vref);
#pragma unroll
                    for (int e = 0; e < 8; e++) reinterpret_cast<uint4*>(dst)[(half * (HV / 4) + c * 8 + e) * ROWS + me] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
                __syncwarp();
            }
        } else if (ok) {
            const float inv = l_run > 0.0f || l_run != l_run ? sh.vref / l_run : 0.0f;
            const unsigned long long out_at = (unsigned long long)(first + tok) * a.out_stride + (unsigned long long)head * D + blockIdx.y * VD + half * HV;
#pragma unroll 1
            for (int c = 0; c < HV / 32; c++) {
                uint32_t o[32];
                if (nt != 0) tmem_load(lanes + S::COL_O + half * HV + c * 32, o);
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
    } else if (warp < MMA_WARP) {
        // ---- codes to f16 ----------------------------------------------------------------------------------------------
        // Three groups of two warps take tasks in turn: task 2 i is tile i's keys, 2 i + 1 its values.  The fence in front of the tensor cores
        // waits for a warp's loads in flight as well, so a warp asks for its next task behind it and the groups cover each other's trips to
        // the L2.  (Sixteen warps in all: with more, a thread has 96 registers, and what did not fit cost more than the warps brought.)
        const uint32_t group = (warp - SOFT_WARPS) / GROUP_WARPS, me = (th - SOFT_WARPS * 32) % (GROUP_WARPS * 32);
        // A unit of a thread: sixteen codes 64 box + 16 part ... of key key0 + STEP u.  Eight neighbouring lanes take four parts of two keys, so
        // their 16-byte pieces meet no bank twice.  Keys and values go through the same instructions (heads of 512: keys in four blocks of
        // columns): with code of their own each the instruction cache, which all the roles share, cost more than the work.
        constexpr uint32_t BOXES = VD / 64, STEP = GROUP_WARPS * 32 * 16 / VD, UNITS = KT / STEP;
        static_assert(STEP <= 16, "a unit's keys lie within sixteen");
        const uint32_t part = me & 3, box = (me >> 3) & (BOXES - 1), key0 = (me >> 3) / BOXES * 2 + ((me >> 2) & 1);
        const uint32_t from = key0 * D + box * 64 + part * 16, at = box * S::KCH + key0 * 128;
        const uint32_t to0 = ((part * 2) ^ (key0 & 7)) << 4, to1 = ((part * 2 + 1) ^ (key0 & 7)) << 4;
        uint4 w[UNITS];
        auto load = [&](uint32_t task, uint32_t c) {
            const Ahead& info = sh.ahead[(task >> 1) % AHEAD];
            const int8_t* codes = (task & 1 ? a.v + blockIdx.y * VD : a.k + c * VD) + from;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) w[u] = load_once(codes + info.at[u * STEP / 16] + u * STEP % 16 * D);
        };
        if (group >> 1 < nt) wait(&sh.known[(group >> 1) % AHEAD], 0), load(group, 0);
        for (uint32_t task = group; task >> 1 < nt; task += GROUPS) {
            const uint32_t i = task >> 1, values = task & 1, odd = i & 1;
            // S (or P V) of the tile two before has read this buffer.
            if (i >= 2) wait(values ? &sh.pv_done[(i - 2) % AHEAD] : &sh.s_full[odd], values ? ((i - 2) / AHEAD) & 1 : ((i - 2) >> 1) & 1);
            const uint2* factors = values ? sh.ahead[i % AHEAD].vf : sh.ahead[i % AHEAD].kf;
            uint8_t* stage = raw + (values ? S::OFF_V + odd * S::V_STAGE : odd * S::K_STAGE) + at;
            for (uint32_t c = 0; c < (D == VD || values ? 1 : D / VD); c++) {
                if (c != 0) load(task, c);
#pragma unroll
                for (uint32_t u = 0; u < UNITS; u++) {
                    const uint2 f = factors[u * STEP / 16];
                    const uint32_t flip = (STEP * u & 7) << 4;  // the keys of a thread's units differ in the swizzle's upper bits only
                    uint8_t* to = stage + c * (BOXES * S::KCH) + u * STEP * 128;
                    *reinterpret_cast<uint4*>(to + (to0 ^ flip)) = convert8(w[u].x, w[u].y, f);
                    *reinterpret_cast<uint4*>(to + (to1 ^ flip)) = convert8(w[u].z, w[u].w, f);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive((values ? sh.v_full : sh.k_full) + odd);
            const uint32_t next = task + GROUPS;
            if (next >> 1 < nt) wait(&sh.known[(next >> 1) % AHEAD], ((next >> 1) / AHEAD) & 1), load(next, 0);
        }
    } else if (warp == MMA_WARP) {
        // ---- products --------------------------------------------------------------------------------------------------
        if (nt != 0) {
            const uint32_t leader = lane == 0, tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t k_desc = desc_k_major(smem_addr(raw)), v_desc = desc_mn_major(smem_addr(raw + S::OFF_V), S::KCH);  // addresses count in 16 bytes
            auto all_wait = [&](uint64_t* bar, uint32_t parity) {
                wait(bar, parity);
                ok = __all_sync(0xffffffffu, ok);
            };
            auto scores = [&](uint32_t i) {
                all_wait(&sh.k_full[i & 1], (i >> 1) & 1);
                if (!ok) return;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t desc = k_desc + (i & 1) * (S::K_STAGE >> 4);
                const uint32_t d = tm + S::COL_S + (i & 1) * KT;
#pragma unroll
                for (int k = 0; k < D / 16; k++) mma_ts(d, tm + S::COL_Q + k * 8, desc + (((k >> 2) * S::KCH + (k & 3) * 32) >> 4), S::IDESC_S, k > 0 ? 1u : 0u, leader);
                mma_commit_by(&sh.s_full[i & 1], leader);
            };
            all_wait(&sh.q_full, 0);
            scores(0);
            for (uint32_t i = 0; i < nt && ok; i++) {
                if (i + 1 < nt) scores(i + 1);
                all_wait(&sh.p_ready[i & 1], (i >> 1) & 1);
                all_wait(&sh.v_full[i & 1], (i >> 1) & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t desc = v_desc + (i & 1) * (S::V_STAGE >> 4);
                const uint32_t p = tm + S::COL_S + (i & 1) * KT;
#pragma unroll
                for (int k = 0; k < KT / 16; k++) mma_ts(tm + S::COL_O, p + k * 8, desc + (k * 2048 >> 4), S::IDESC_PV, k > 0 ? 1u : i > 0 ? 1u : 0u, leader);
                mma_commit_by(&sh.pv_done[i % AHEAD], leader);
            }
            if (!ok) {  // a wait ran out: nothing may still write tensor memory when it is given back
                mma_commit_by(&sh.drained, leader);
                mbar_wait(&sh.drained, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- the tiles ahead -------------------------------------------------------------------------------------------
        // A lane sixteen keys, as many tiles at once as that makes; page numbers are asked for two such batches ahead, scales one: looked
        // up tile by tile, the two trips to the L2 behind one another took longer than everything else about a tile.
        constexpr uint32_t count = KT / 16, tiles = 32 / count;
        const uint32_t page = 1u << a.shift;
        auto first_key = [&](uint32_t b) { return tile0 + (b + lane / count) * KT + lane % count * 16; };
        auto page_at = [&](uint32_t b) {  // the page of this lane's keys in the batch of tiles that starts with tile b
            const uint32_t j = first_key(b), id = j < end ? __ldg(a.table + (size_t)r * a.width + (j >> a.shift)) : 0xffffffffu;
            return id < a.pages ? id : 0xffffffffu;
        };
        auto scales_at = [&](uint32_t id) {
            const size_t at = (size_t)id * a.kv_heads + kvh;
            return id != 0xffffffffu ? make_float2(__ldg(a.ks + at), __ldg(a.vs + at)) : make_float2(0.0f, 0.0f);
        };
        auto pair = [](float f) {
            const __half2 h = __float2half2_rn(f), o = __hmul2(h, __half2half2(__ushort_as_half(0xe480)));  // -1152
            return make_uint2(*reinterpret_cast<const uint32_t*>(&h), *reinterpret_cast<const uint32_t*>(&o));
        };
        uint32_t id = 0xffffffffu, id1 = 0xffffffffu;
        float2 sc = make_float2(0.0f, 0.0f);
        if (nt != 0) id = page_at(0), id1 = page_at(tiles), sc = scales_at(id);
        float vref = 0.0f;
        for (uint32_t b = 0; b < nt; b += tiles) {
            const float2 sc1 = scales_at(id1);
            const uint32_t id2 = page_at(b + 2 * tiles);
            const uint32_t has = __ballot_sync(0xffffffffu, id != 0xffffffffu);
            float km = sc.x, vm = sc.y;  // the tile's largest
            for (uint32_t o = 1; o < count; o <<= 1) km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, o)), vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
            const uint2 kf = pair(km > 0.0f ? __fdiv_rn(sc.x, km) : 0.0f);
            for (uint32_t t = 0; t < tiles && b + t < nt; t++) {
                const uint32_t i = b + t;
                const float vnew = fmaxf(vref, __shfl_sync(0xffffffffu, vm, t * count));
                if (i >= AHEAD) wait(&sh.pv_done[i % AHEAD], (i / AHEAD - 1) & 1);  // nobody reads the entry's old tile any more
                Ahead& info = sh.ahead[i % AHEAD];
                if (lane / count == t) {
                    const uint32_t k = lane % count;
                    info.at[k] = ((((unsigned long long)(id != 0xffffffffu ? id : 0) * a.kv_heads + kvh) << a.shift) + (first_key(b) & (page - 1))) * D;
                    info.kf[k] = kf, info.vf[k] = pair(vnew > 0.0f ? __fdiv_rn(sc.y, vnew) : 0.0f);
                    if (k == 0) {
                        info.kref = km, info.shrink = vref > 0.0f ? __fdiv_rn(vref, vnew) : 1.0f;
                        if (i + 1 == nt) sh.vref = vnew;
                    }
                }
                if (lane < KT / 32) {
                    const uint32_t mine = has >> (t * count + 2 * lane);
                    const uint32_t keys = (mine & 1u ? 0xffffu : 0u) | (mine & 2u ? 0xffff0000u : 0u);
                    info.keys[lane] = keys;
                }
                vref = vnew;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.known[i % AHEAD]);
            }
            id = id1, id1 = id2, sc = sc1;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Row tiles that were cut: a block adds up the pieces of one of them, always in the order of the keys, a thread a row and sixteen of
// its columns.
template <int D, int VD>
__global__ void __launch_bounds__(ROWS) paged_prefill_join_kernel(const PrefillArgs a) {
    const uint32_t row = threadIdx.x, col = blockIdx.y * 16;
    pdl_wait();
    const uint32_t cut = a.head[0];
    for (uint32_t b = blockIdx.x; b < cut; b += gridDim.x) {
        const Split s = a.splits[b];
        const uint32_t at = s.row0 + row, tok = at / a.ratio, head = s.kvh * a.ratio + at % a.ratio;
        if (s.parts == 0 || tok >= s.n) continue;
        float m = -INFINITY, l = 0.0f;
        float4 o[4] = {};
#pragma unroll 4
        for (uint32_t i = 0; i < s.parts; i++) {
            const float* src = a.partial + ((size_t)(b + i * a.kv_heads) * (D / VD) + blockIdx.z) * PIECE<VD>;
            const float mi = src[VD * ROWS + row], li = src[(VD + 1) * ROWS + row];
            float4 x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = reinterpret_cast<const float4*>(src)[(col / 4 + e) * ROWS + row];
            const float top = fmaxf(m, mi);
            const bool none = mi == -INFINITY;  // then its output was perhaps not written
            const float was = top == -INFINITY ? 1.0f : ex2(m - top), is = none ? 0.0f : ex2(mi - top);
            m = top, l = l * was + li * is;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (none) x[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                o[e].x = o[e].x * was + x[e].x * is, o[e].y = o[e].y * was + x[e].y * is;
                o[e].z = o[e].z * was + x[e].z * is, o[e].w = o[e].w * was + x[e].w * is;
            }
        }
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const unsigned long long to = (unsigned long long)(s.first + tok) * a.out_stride + (unsigned long long)head * D + blockIdx.z * VD + col;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (inv == 0.0f) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            o[e].x *= inv, o[e].y *= inv, o[e].z *= inv, o[e].w *= inv;
        }
        if (a.out_f16) {
            __half2 h[8];
#pragma unroll
            for (int e = 0; e < 4; e++) h[2 * e] = __floats2half2_rn(o[e].x, o[e].y), h[2 * e + 1] = __floats2half2_rn(o[e].z, o[e].w);
            uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + to);
            dst[0] = *reinterpret_cast<uint4*>(h), dst[1] = *reinterpret_cast<uint4*>(h + 4);
        } else {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + to);
#pragma unroll
            for (int e = 0; e < 4; e++) dst[e] = o[e];
        }
    }
}

uint32_t shares_of(const tb_context* ctx, uint32_t head_dim) { return std::max((uint32_t)ctx->sms / (head_dim == 512 ? 4 : 1), 1u); }

template <int D, int VD>
int run(tb_context* ctx, const PrefillArgs& a, uint32_t grid) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t bytes = Shape<D, VD>::BYTES;
    static_assert(bytes + sizeof(Shared) <= 232448, "over what a block may use");
    TB_CUDA(allow_smem(paged_prefill_kernel<D, VD>, bytes, ctx->gpu, done));
    TB_CUDA(launch_kernel(ctx, paged_prefill_plan_kernel<Shape<D, VD>::KT>, dim3(1), dim3(THREADS), 0, true, a));
    TB_CUDA(launch_kernel(ctx, paged_prefill_kernel<D, VD>, dim3(grid, D / VD), dim3(THREADS), bytes, true, a, ctx->status));
    if (a.requests <= FEW) TB_CUDA(launch_kernel(ctx, paged_prefill_join_kernel<D, VD>, dim3(a.shares, VD / 16, D / VD), dim3(ROWS), 0, true, a));
    return OK;
}

// The scratch: the decode kernel's counters, which stay zero; `head`, `before`, `rows`, `splits`; the pieces.
constexpr size_t BEFORE_AT = PAGED_COUNT_BYTES + 16, ROWS_AT = BEFORE_AT + MAX_REQUESTS * 4, SPLITS_AT = ROWS_AT + MAX_REQUESTS * sizeof(Row);
size_t partial_at(uint32_t shares) { return SPLITS_AT + ((size_t)2 * shares * sizeof(Split) + 15) / 16 * 16; }

}  // namespace

size_t prefill_scratch_bytes(const tb_context* ctx, uint32_t head_dim) {
    const uint32_t shares = shares_of(ctx, head_dim), parts = head_dim == 512 ? 4 : 1;
    return partial_at(shares) + (size_t)2 * shares * (head_dim + 2 * parts) * ROWS * 4;
}

int launch_prefill_paged(tb_context* ctx, const tb_paged_attend& p) {
    const tb_pages& c = p.cache;
    PrefillArgs a{};
    a.k = c.k, a.v = c.v, a.ks = c.k_scale, a.vs = c.v_scale, a.table = c.table, a.pages = c.pages, a.shift = log2_of(c.page), a.kv_heads = c.kv_heads;
    a.requests = c.requests, a.width = c.width, a.q = p.q, a.q_stride = p.q_stride, a.q_f16 = p.q_dtype == TB_F16, a.starts = p.starts, a.lengths = p.lengths;
    a.tokens = p.tokens, a.ratio = p.heads / c.kv_heads, a.most = p.most, a.window = p.window > 0x7fffffffu ? 0 : p.window, a.scale = p.scale * 1.4426950408889634f;
    a.out = p.out, a.out_stride = p.out_stride, a.out_f16 = p.out_dtype == TB_F16;
    if ((uint64_t)p.tokens * p.heads > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_prefill_paged_q8: too many rows for one call");
    // Row tiles: at most one a request that is not full, and no request brings more than `most` tokens.
    const uint64_t full = (uint64_t)p.tokens * a.ratio / ROWS + c.requests, each = (((uint64_t)p.most * a.ratio + ROWS - 1) / ROWS) * c.requests;
    a.shares = shares_of(ctx, c.head_dim);
    const uint64_t grid = (full < each ? full : each) * c.kv_heads + (c.requests <= FEW ? a.shares : 0);  // cutting makes at most as many more
    a.blocks = (uint32_t)grid;
    if (grid > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_prefill_paged_q8: too many rows for one call");
    TB_TRY(check_scratch(ctx, p, "tb_prefill_paged_q8"));
    uint8_t* scratch = static_cast<uint8_t*>(p.scratch);
    a.head = reinterpret_cast<uint32_t*>(scratch + PAGED_COUNT_BYTES), a.before = reinterpret_cast<uint32_t*>(scratch + BEFORE_AT);
    a.rows = reinterpret_cast<Row*>(scratch + ROWS_AT), a.splits = reinterpret_cast<Split*>(scratch + SPLITS_AT);
    a.partial = reinterpret_cast<float*>(scratch + partial_at(a.shares));
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    switch (c.head_dim) {
        case 64: return run<64, 64>(ctx, a, (uint32_t)grid);
        case 128: return run<128, 128>(ctx, a, (uint32_t)grid);
        case 256: return run<256, 256>(ctx, a, (uint32_t)grid);
        default: return run<512, 128>(ctx, a, (uint32_t)grid);
    }
}

}  // namespace tb
