// What the operators on the paged 8-bit cache share (page_plan.cu, cache_q8.cu, paged_attend.cu, paged_prefill.cu): checks of
// the cache's descriptor, which need no GPU, and the guard every entry point runs its launch under.
#pragma once

#include <atomic>
#include <new>
#include <string>

#include "../../include/tachyon_b200.h"
#include "internal.h"

namespace tb {

constexpr uint32_t MAX_REQUESTS = 8192;  // a block keeps a prefix sum over the requests in shared memory

inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline uint32_t log2_of(uint32_t x) { return 31u - (uint32_t)__builtin_clz(x); }

inline int check_pages(const tb_pages& c, const std::string& who, bool table) {
    if (!c.k || !c.v || !c.k_scale || !c.v_scale) return fail(OUT_OF_RANGE, who + ": null cache");
    if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128) return fail(OUT_OF_RANGE, who + ": pages of 16, 32, 64 or 128 tokens");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256 && c.head_dim != 512) return fail(UNSUPPORTED, who + ": heads of 64, 128, 256 or 512");
    if (c.pages == 0 || c.kv_heads == 0 || c.kv_heads > 1024) return fail(OUT_OF_RANGE, who + ": no pages, or a number of key-value heads outside 1..1024");
    if ((uint64_t)c.pages * c.page > 0xfffffffeull) return fail(OUT_OF_RANGE, who + ": slots pass 32 bits");
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 4) || !aligned(c.v_scale, 4)) return fail(OUT_OF_RANGE, who + ": the cache must be 16-byte aligned");
    if (table) {
        if (!c.table || !aligned(c.table, 4)) return fail(OUT_OF_RANGE, who + ": null or misaligned page table");
        if (c.requests == 0 || c.requests > MAX_REQUESTS) return fail(OUT_OF_RANGE, who + ": 1 to 8192 requests");
        if (c.width == 0 || (uint64_t)c.width * c.page > 0x7fffffffull) return fail(OUT_OF_RANGE, who + ": a page table of no width, or positions past 31 bits");
    }
    return OK;
}

// Attention's scratch begins with the decode kernel's counters, zero between calls; calls of every shape may share it.
constexpr size_t PAGED_COUNT_BYTES = 4096;

// Prefill attention on tcgen05 (paged_prefill.cu); the caller has checked the descriptor, not the scratch.
int launch_prefill_paged(tb_context* ctx, const tb_paged_attend& p);
size_t prefill_scratch_bytes(const tb_context* ctx, uint32_t head_dim);

// What both take of it (paged_attend.cu), and the check that a call brings it.
size_t paged_scratch_bytes(const tb_context* ctx, uint32_t head_dim);
int check_scratch(const tb_context* ctx, const tb_paged_attend& p, const std::string& who);

// Makes a context's GPU the current one for a launch and puts the caller's back.
class DeviceScope {
  public:
    explicit DeviceScope(int gpu) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = gpu;
        if (before_ != gpu) error_ = cudaSetDevice(gpu);
        else before_ = -1;
    }
    ~DeviceScope() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    cudaError_t error() const { return error_; }

  private:
    int before_ = -1;
    cudaError_t error_ = cudaSuccess;
};

// Runs an entry point's body: no C++ exception leaves it.
template <typename F>
inline int entry(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return OUT_OF_MEMORY;
    } catch (...) {
        return CUDA;
    }
}

// Raises a kernel's dynamic shared memory limit, once for each GPU; `done` has a bit for each.
template <typename K>
inline cudaError_t allow_smem(K kernel, size_t bytes, int gpu, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (gpu & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace tb
