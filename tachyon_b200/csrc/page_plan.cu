// Page tables and slot maps on the GPU (tb_page_plan): the host need not know the lengths of the requests it serves.
//
// With have = ceil(length / page) pages and `fresh` new tokens, a request needs ceil((length + fresh) / page) - have more; one
// that ends gives `have` back.  The pages to give are the stack S = free[0 .. count) followed by the pages given back, and new
// page k (in the order of the requests) is S[|S| - 1 - k]: one prefix sum over the requests fixes every answer, so the result
// does not depend on which block writes it.  Nothing is read that the launch writes: new pages go to table entries behind the
// ones a request has, given-back pages are read from requests that get none, and the free list is only written from `count`
// on.  Lengths and the count may be updated in place, so the last block to finish stores them.
//
// Every block repeats the prefix sum (8 bytes a request from the L2) and takes its share of the tokens and pages, finding a
// token's request by bisection in shared memory; a second launch behind a scan of one block would cost more than the repeats.
// What bounds it: trips to memory one behind the other (lengths, table entries).  64 single tokens 5 us, an empty launch being 2.5; 1000
// requests that bring up to 257 tokens each 8.7 us (with 4096 tokens a block instead of 1024: 15.5).
#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t THREADS = 512;
constexpr uint32_t SHARE = 1024;  // tokens a block takes at least; two a thread, each a bisection and two trips to the L2
constexpr uint32_t ENDS = 0xffffffffu;

struct PlanArgs {
    tb_plan p;
    uint32_t shift;  // log2(page)
};

// The last i in [0, n) with at[i] <= x (at[0] = 0, rising).
__device__ __forceinline__ uint32_t owner(const uint32_t* at, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(THREADS) page_plan_kernel(const PlanArgs a) {
    extern __shared__ uint32_t sums[];  // three prefix sums over the requests (new tokens, new pages, pages given back) and their lengths
    __shared__ unsigned long long part[3][THREADS / 32];
    __shared__ uint32_t last;
    const tb_plan& p = a.p;
    const uint32_t n = p.requests, th = threadIdx.x, lane = th & 31, warp = th >> 5;
    uint32_t* s_tok = sums;
    uint32_t* s_need = sums + n;
    uint32_t* s_back = sums + 2 * n;
    uint32_t* s_len = sums + 3 * n;
    const unsigned long long most = (unsigned long long)p.width << a.shift;  // positions a request can have
    pdl_wait();

    // Sums of a thread's consecutive requests, then over the block, in 64 bits: lengths are the caller's and may be anything.
    const uint32_t per = (n + THREADS - 1) / THREADS, r0 = min(th * per, n), r1 = min(r0 + per, n);
    unsigned long long tok = 0, need = 0, back = 0;
    uint32_t bad = 0;
    for (uint32_t r = r0; r < r1; r++) {
        const uint32_t len = __ldcg(p.lengths + r), f = __ldcg(p.fresh + r), add = f == ENDS ? 0 : f;
        if ((unsigned long long)len + add > most) bad |= TB_PLAN_LENGTH;
        const unsigned long long have = ((unsigned long long)len + p.page - 1) >> a.shift;
        tok += add;
        if (f == ENDS) back += have;
        else need += (((unsigned long long)len + add + p.page - 1) >> a.shift) - have;
    }
    unsigned long long v[3] = {tok, need, back}, before[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        unsigned long long x = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        before[k] = x - v[k];
        if (lane == 31) part[k][warp] = x;
    }
    bad = __syncthreads_or((int)bad) ? TB_PLAN_LENGTH : 0u;
    unsigned long long total[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        unsigned long long sum = 0;
        for (uint32_t w = 0; w < THREADS / 32; w++) {
            if (w == warp) before[k] += sum;
            sum += part[k][w];
        }
        total[k] = sum;
    }
    const uint32_t count = __ldcg(p.free_count);
    if (count > p.pages || count + total[2] > p.pages) bad |= TB_PLAN_FREE_LIST;
    if (total[1] > count + total[2]) bad |= TB_PLAN_PAGES;
    if (total[0] > p.max_tokens) bad |= TB_PLAN_TOKENS;
    if (bad == 0) {
        uint32_t t = (uint32_t)before[0], q = (uint32_t)before[1], b = (uint32_t)before[2];
        for (uint32_t r = r0; r < r1; r++) {
            const uint32_t len = __ldcg(p.lengths + r), f = __ldcg(p.fresh + r), add = f == ENDS ? 0 : f, have = (len + p.page - 1) >> a.shift;
            s_tok[r] = t, s_need[r] = q, s_back[r] = b, s_len[r] = len;
            if (blockIdx.x == 0) p.starts[r] = t;
            t += add;
            if (f == ENDS) b += have;
            else q += ((len + add + p.page - 1) >> a.shift) - have;
        }
        if (blockIdx.x == 0 && th == 0) p.starts[n] = (uint32_t)total[0];
    } else if (blockIdx.x == 0) {
        for (uint32_t r = th; r <= n; r += THREADS) p.starts[r] = 0;
    }
    __syncthreads();

    if (bad == 0) {
        const uint32_t tokens = (uint32_t)total[0], pages = (uint32_t)total[1], top = count + (uint32_t)total[2];
        auto given = [&](uint32_t q) {  // page q of those given back
            const uint32_t r = owner(s_back, n, q);
            return __ldcg(p.table + (size_t)r * p.width + (q - s_back[r]));
        };
        auto page_of = [&](uint32_t k) {  // new page k
            const uint32_t at = top - 1 - k;
            return at < count ? __ldcg(p.free_pages + at) : given(at - count);
        };
        const uint32_t first = blockIdx.x * THREADS + th, step = gridDim.x * THREADS;
        for (uint32_t t = first; t < tokens; t += step) {
            const uint32_t r = owner(s_tok, n, t), len = s_len[r], pos = len + (t - s_tok[r]), at = pos >> a.shift, have = (len + p.page - 1) >> a.shift;
            const uint32_t id = at < have ? __ldcg(p.table + (size_t)r * p.width + at) : page_of(s_need[r] + at - have);
            p.slots[t] = id < p.pages ? (id << a.shift) + (pos & (p.page - 1)) : 0xffffffffu;
            if (p.positions) p.positions[t] = pos;
        }
        for (uint32_t k = first; k < pages; k += step) {
            const uint32_t r = owner(s_need, n, k), have = (s_len[r] + p.page - 1) >> a.shift;
            p.table[(size_t)r * p.width + have + (k - s_need[r])] = page_of(k);
        }
        for (uint32_t q = count + first; q + pages < top; q += step) p.free_pages[q] = given(q - count);  // given back and not given out
    }
    // Lengths and the count last: they may lie where they were read from.
    if (gridDim.x > 1) {
        __syncthreads();
        if (th == 0) {
            __threadfence();
            last = atomicAdd(p.scratch, 1u) == gridDim.x - 1;
            if (last) *p.scratch = 0;
        }
        __syncthreads();
        if (!last) return;
    } else {
        __syncthreads();
    }
    for (uint32_t r = th; r < n; r += THREADS) {
        const uint32_t len = __ldcg(p.lengths + r), f = __ldcg(p.fresh + r);
        p.lengths_out[r] = bad ? len : f == ENDS ? 0 : len + f;
    }
    if (th == 0) {
        *p.free_count_out = bad ? count : count + (uint32_t)total[2] - (uint32_t)total[1];
        *p.refused = bad;
    }
}

int check_plan(const tb_plan* p) {
    if (!p) return fail(OUT_OF_RANGE, "tb_page_plan: null descriptor");
    if (!p->lengths || !p->fresh || !p->lengths_out || !p->table || !p->free_pages || !p->free_count || !p->free_count_out || !p->starts || !p->refused || !p->scratch ||
        (!p->slots && p->max_tokens))
        return fail(OUT_OF_RANGE, "tb_page_plan: null argument");
    if (p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128) return fail(OUT_OF_RANGE, "tb_page_plan: pages of 16, 32, 64 or 128 tokens");
    if (p->requests == 0 || p->requests > MAX_REQUESTS) return fail(OUT_OF_RANGE, "tb_page_plan: 1 to 8192 requests");
    if (p->width == 0 || (uint64_t)p->width * p->page > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_page_plan: a page table of no width, or positions past 31 bits");
    if (p->pages == 0 || (uint64_t)p->pages * p->page > 0xfffffffeull) return fail(OUT_OF_RANGE, "tb_page_plan: no pages, or slots past 32 bits");
    if (p->max_tokens > 0x7fffffffu) return fail(OUT_OF_RANGE, "tb_page_plan: more than 2^31 - 1 tokens");
    const void* all[] = {p->lengths, p->fresh, p->lengths_out, p->table, p->free_pages, p->free_count, p->free_count_out, p->starts, p->slots, p->positions, p->refused, p->scratch};
    for (const void* q : all)
        if (!aligned(q, 4)) return fail(OUT_OF_RANGE, "tb_page_plan: buffers must be 4-byte aligned");
    return OK;
}

int launch_plan(tb_context* ctx, const tb_plan& p) {
    static std::atomic<uint64_t> done{0};
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    TB_CUDA(allow_smem(page_plan_kernel, 4 * MAX_REQUESTS * sizeof(uint32_t), ctx->gpu, done));
    const PlanArgs a{p, log2_of(p.page)};
    uint32_t grid = (p.max_tokens + SHARE - 1) / SHARE;
    if (grid < 1) grid = 1;
    if (grid > (uint32_t)ctx->sms) grid = (uint32_t)ctx->sms;
    TB_CUDA(launch_kernel(ctx, page_plan_kernel, dim3(grid), dim3(THREADS), 4 * (size_t)p.requests * sizeof(uint32_t), true, a));
    return OK;
}

}  // namespace

}  // namespace tb

using namespace tb;

extern "C" int tb_page_plan(tb_context* ctx, const tb_plan* args) {
    return entry([&] {
        TB_TRY(check_plan(args));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        return launch_plan(ctx, *args);
    });
}
