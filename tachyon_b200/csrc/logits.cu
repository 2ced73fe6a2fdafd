// Penalties, biases and masks on a batch of logits (tb_logits_adjust), in front of a sampler.
//
//   y = x / repetition (x > 0) or x * repetition, for tokens in the row's history (prompt or generated)
//   y -= frequency * c + presence * (c > 0), c the token's count among the generated ones
//   y += the token's biases, added up in the order of the list
//   y = -inf where the row's mask lets the token not through
//
// What bounds it: the logits, read and written once.  A block takes one range of one row's vocabulary.  It counts the history's
// tokens that fall into its range in shared memory (whole numbers, so the order of the atomics does not matter; bit 31 marks a
// prompt token), adds the biases up in one warp in the list's order, then streams its logits.  Every block of a row walks the
// row's whole history from the L2: with ranges of 8192 tokens a history of 8000 costs a block the bytes of its f32 logits again,
// in L2 traffic alone; smaller ranges would multiply that, larger ones leave too few blocks for a small batch.
#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t THREADS = 512, MOST_RANGE = 8192, LEAST_RANGE = 1024, PROMPT = 0x80000000u;

struct LogitsArgs {
    tb_logits p;
    uint32_t range, ranges;
};

template <bool F16>
__device__ __forceinline__ float get(const void* p, unsigned long long i) {
    if constexpr (F16) return __half2float(static_cast<const __half*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
template <bool F16>
__device__ __forceinline__ void put(void* p, unsigned long long i, float v) {
    if constexpr (F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<float*>(p)[i] = v;
}

// VEC: 16 bytes a thread and turn; rows and ranges then start at multiples of 16 bytes.
template <bool F16, bool VEC>
__global__ void __launch_bounds__(THREADS) logits_adjust_kernel(const LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t s_count[];  // [range] counts, then [range] biases, as far as there are any
    constexpr uint32_t N = !VEC ? 1 : F16 ? 8 : 4;
    const tb_logits& p = a.p;
    const uint32_t th = threadIdx.x, row = blockIdx.x / a.ranges, first = blockIdx.x % a.ranges * a.range, n = min(a.range, p.vocab - first);
    const bool history = p.history != nullptr, biased = p.bias_token != nullptr;
    float* s_bias = reinterpret_cast<float*>(s_count + (history ? a.range : 0));
    pdl_wait();
    if (history || biased) {
        const uint32_t words = (history ? a.range : 0) + (biased ? a.range : 0);
        for (uint32_t i = th; i < words / 4; i += THREADS) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (biased && th < 32) {
            const uint32_t* token = p.bias_token + (size_t)row * p.bias_stride;
            const float* bias = p.bias + (size_t)row * p.bias_stride;
            const uint32_t count = min(__ldg(p.bias_count + row), p.bias_stride);
            for (uint32_t i = 0; i < count; i += 32) {
                const uint32_t at = i + th < count ? __ldg(token + i + th) - first : 0xffffffffu;
                const float b = at < n ? __ldg(bias + i + th) : 0.0f;
                const uint32_t key = at < n ? at : 0x80000000u | th;  // a key of its own for what lies elsewhere
                const uint32_t same = __match_any_sync(0xffffffffu, key);
                float sum = b;
                if (__any_sync(0xffffffffu, (same & (same - 1)) != 0)) {  // a token more than once: its first lane adds them up in order
                    sum = at < n ? s_bias[at] : 0.0f;
                    for (uint32_t k = 0; k < 32; k++) {
                        const float other = __shfl_sync(0xffffffffu, b, k);
                        if ((same >> k) & 1u) sum += other;
                    }
                    if (at < n && (uint32_t)__ffs(same) - 1 == th) s_bias[at] = sum;
                } else if (at < n) {
                    s_bias[at] += b;
                }
                __syncwarp();
            }
        }
        if (history) {
            const uint32_t* token = p.history + (size_t)row * p.history_stride;
            const uint32_t total = min(__ldg(p.total + row), p.history_stride), prompt = min(__ldg(p.prompt + row), total);
#pragma unroll 4
            for (uint32_t i = th; i < total; i += THREADS) {
                const uint32_t at = __ldg(token + i) - first;
                if (at < n) {
                    if (i < prompt) atomicOr(s_count + at, PROMPT);
                    else atomicAdd(s_count + at, 1u);
                }
            }
        }
        __syncthreads();
    }
    const float rep = history && p.repetition ? __ldg(p.repetition + row) : 1.0f;
    const float freq = history && p.frequency ? __ldg(p.frequency + row) : 0.0f, pres = history && p.presence ? __ldg(p.presence + row) : 0.0f;
    const uint32_t* allowed = nullptr;
    if (p.allowed) {
        const uint32_t m = p.mask_of ? __ldg(p.mask_of + row) : row;
        if (m < p.masks) allowed = p.allowed + (size_t)m * p.allowed_stride;
    }
    auto value = [&](float x, uint32_t i, uint32_t bits) {
        if (history) {
            const uint32_t c = s_count[i], said = c & ~PROMPT;
            if (c != 0) x = x > 0.0f ? __fdiv_rn(x, rep) : x * rep;
            if (said != 0) x -= fmaf(freq, (float)said, pres);
        }
        if (biased) x += s_bias[i];
        return (bits >> ((first + i) & 31)) & 1u ? x : -INFINITY;
    };
    const unsigned long long src = (unsigned long long)row * p.stride + first, dst = (unsigned long long)row * p.out_stride + first;
    for (uint32_t i = th * N; i < n; i += THREADS * N) {
        const uint32_t bits = allowed ? __ldg(allowed + ((first + i) >> 5)) : 0xffffffffu;
        if (VEC && i + N <= n) {
            float x[N];
            if constexpr (F16 && VEC) {
                uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.logits) + src + i);
                uint32_t* ww = &w.x;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float2 f = __half22float2(*reinterpret_cast<const __half2*>(ww + e));
                    const __half2 h = __floats2half2_rn(value(f.x, i + 2 * e, bits), value(f.y, i + 2 * e + 1, bits));
                    ww[e] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + dst + i) = w;
            } else if constexpr (VEC) {
                float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + src + i);
                f.x = value(f.x, i, bits), f.y = value(f.y, i + 1, bits), f.z = value(f.z, i + 2, bits), f.w = value(f.w, i + 3, bits);
                *reinterpret_cast<float4*>(static_cast<float*>(p.out) + dst + i) = f;
            }
            (void)x;
        } else {
            for (uint32_t e = 0; e < N && i + e < n; e++) put<F16>(p.out, dst + i + e, value(get<F16>(p.logits, src + i + e), i + e, bits));
        }
    }
}

int check_logits(const tb_logits* p) {
    if (!p) return fail(OUT_OF_RANGE, "tb_logits_adjust: null descriptor");
    if (p->dtype != TB_F32 && p->dtype != TB_F16) return fail(OUT_OF_RANGE, "tb_logits_adjust: unknown dtype");
    if (p->vocab == 0 || p->vocab > 0x7fffffffu) return fail(OUT_OF_RANGE, "tb_logits_adjust: a vocabulary of 1 to 2^31 - 1 tokens");
    if (p->rows == 0) return OK;
    if (!p->logits || !p->out) return fail(OUT_OF_RANGE, "tb_logits_adjust: null logits");
    const size_t size = p->dtype == TB_F16 ? 2 : 4;
    if (!aligned(p->logits, size) || !aligned(p->out, size)) return fail(OUT_OF_RANGE, "tb_logits_adjust: misaligned logits");
    if (p->rows > 1 && (p->stride < p->vocab || p->out_stride < p->vocab)) return fail(OUT_OF_RANGE, "tb_logits_adjust: a stride below the vocabulary");
    if (p->out == p->logits && p->rows > 1 && p->out_stride != p->stride) return fail(OUT_OF_RANGE, "tb_logits_adjust: in place the strides are the same");
    if (p->history && (!p->total || !p->prompt)) return fail(OUT_OF_RANGE, "tb_logits_adjust: a history without its lengths");
    if (!p->history && (p->repetition || p->frequency || p->presence)) return fail(OUT_OF_RANGE, "tb_logits_adjust: penalties without a history");
    if (p->bias_token && (!p->bias || !p->bias_count)) return fail(OUT_OF_RANGE, "tb_logits_adjust: biases without values or counts");
    if (p->allowed && (p->masks == 0 || (uint64_t)p->allowed_stride * 32 < p->vocab)) return fail(OUT_OF_RANGE, "tb_logits_adjust: no masks, or masks shorter than the vocabulary");
    const void* words[] = {p->history, p->prompt, p->total, p->repetition, p->frequency, p->presence, p->bias_token, p->bias, p->bias_count, p->allowed, p->mask_of};
    for (const void* w : words)
        if (!aligned(w, 4)) return fail(OUT_OF_RANGE, "tb_logits_adjust: buffers must be 4-byte aligned");
    return OK;
}

int launch_logits(tb_context* ctx, const tb_logits& p) {
    const bool f16 = p.dtype == TB_F16;
    const size_t size = f16 ? 2 : 4;
    const bool vec = aligned(p.logits, 16) && aligned(p.out, 16) && (p.rows == 1 || (p.stride * size % 16 == 0 && p.out_stride * size % 16 == 0));
    LogitsArgs a{p, MOST_RANGE, 0};
    // Two blocks a multiprocessor, as far as ranges of 1024 tokens give them.
    while (a.range > LEAST_RANGE && (uint64_t)p.rows * ((p.vocab + a.range - 1) / a.range) < 2ull * ctx->sms) a.range /= 2;
    a.ranges = (p.vocab + a.range - 1) / a.range;
    if ((uint64_t)p.rows * a.ranges > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_logits_adjust: too many rows for one call");
    const size_t smem = (size_t)a.range * 4 * ((p.history ? 1 : 0) + (p.bias_token ? 1 : 0));
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    auto run = [&](auto kernel, std::atomic<uint64_t>& done) {
        const cudaError_t e = allow_smem(kernel, MOST_RANGE * 8, ctx->gpu, done);
        return e != cudaSuccess ? e : launch_kernel(ctx, kernel, dim3(p.rows * a.ranges), dim3(THREADS), smem, true, a);
    };
    static std::atomic<uint64_t> done[4];
    TB_CUDA(f16 ? vec ? run(logits_adjust_kernel<true, true>, done[0]) : run(logits_adjust_kernel<true, false>, done[1])
                : vec ? run(logits_adjust_kernel<false, true>, done[2]) : run(logits_adjust_kernel<false, false>, done[3]));
    return OK;
}

}  // namespace

}  // namespace tb

using namespace tb;

extern "C" int tb_logits_adjust(tb_context* ctx, const tb_logits* args) {
    return entry([&] {
        TB_TRY(check_logits(args));
        if (!ctx) return fail(OUT_OF_RANGE, "null context");
        return args->rows == 0 ? (int)OK : launch_logits(ctx, *args);
    });
}
