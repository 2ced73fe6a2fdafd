// Penalties, biases and masks on a batch of logits (tb_logits_adjust), in front of a sampler.
//
//   y = x / repetition (x > 0) or x * repetition, for tokens in the row's history (prompt or generated)
//   y -= frequency * c + presence * (c > 0), c the token's count among the generated ones
//   y += the token's biases, added up in the order of the list
//   y = -inf where the row's mask lets the token not through
//
// What bounds it: the logits, read and written once, and the history's walk.  A block takes one range of one row's vocabulary.  It counts
// the history's tokens that fall into the range in shared memory (whole numbers, so the order of the atomics does not matter; the
// start of the lists is asked for before anything else), notes the biases that do, and streams its logits.  A token's word: bit 31 it is
// in the prompt, bits 20-30 which of the noted biases its own are summed in (in the list's order), the rest its occurrences.  A thread none of
// whose tokens has a word only masks them.  Every block of a row walks all of its history, so ranges are as long as leaves three blocks a
// multiprocessor, for a small batch shorter.  Measured slower: clusters that share the walk and count in each other's shared memory;
// the few tokens with words worked out one by one; a kernel of their own for those with hashed tables (64 rows of 262144 in f16 with 8000
// tokens of history: 53 us, 13 of them the stream; this one 33, and 3.3 for one row in f32 with 2000).
#include "common.cuh"
#include "paged.h"

namespace tb {

namespace {

constexpr uint32_t THREADS = 512, MOST_RANGE = 16384, LEAST_RANGE = 1024;
constexpr uint32_t NONE = 0xffffffffu, PROMPT = 0x80000000u, MOST_BIASES = 1024, MOST_HISTORY = (1u << 20) - 1;

struct LogitsArgs {
    tb_logits p;
    uint32_t range, ranges;  // tokens of a range, ranges of a row
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
// VEC: 16 bytes at a time; a row of logits and of outputs then lie alike within 16 bytes, and places count from the 16-byte boundary
// at or below the row's start (`skew` values in front of it).  Otherwise a value at a time.
template <bool F16, bool VEC>
__global__ void __launch_bounds__(THREADS, 3) logits_adjust_kernel(const LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t s_word[];  // [range], when there is a history or a bias
    uint32_t* s_place = s_word + a.range;               // [bias_stride] biases in this range, in no order: their token's place,
    uint32_t* s_which = s_place + a.p.bias_stride;      // their number in the list,
    float* s_bias = reinterpret_cast<float*>(s_which + a.p.bias_stride);  // the bias,
    float* s_sum = s_bias + a.p.bias_stride;            // the sum of the token's (with its first)
    __shared__ uint32_t s_noted, s_again;
    constexpr uint32_t SIZE = F16 ? 2 : 4, N = !VEC ? 1 : 16 / SIZE, AT_ONCE = 8;
    const tb_logits& p = a.p;
    const uint32_t th = threadIdx.x, row = blockIdx.x / a.ranges;
    const bool history = p.history != nullptr, biased = p.bias_token != nullptr, words = history || biased;
    const char* src = static_cast<const char*>(p.logits) + (unsigned long long)row * p.stride * SIZE;
    char* dst = static_cast<char*>(p.out) + (unsigned long long)row * p.out_stride * SIZE;
    const int skew = VEC ? (int)((reinterpret_cast<uintptr_t>(src) & 15) / SIZE) : 0;
    // Place i stands for token from + i; the first place and the one behind the last that stand for any.
    const int from = (int)(blockIdx.x % a.ranges * a.range) - skew, vocab = (int)p.vocab;
    const uint32_t first = from < 0 ? (uint32_t)-from : 0, end = vocab > from ? (uint32_t)min((int)a.range, vocab - from) : 0;
    if (end <= first) return;
    const uint32_t base = (uint32_t)(from + (int)first), count = end - first;  // the range's tokens: base .. base + count - 1
    pdl_wait();

    const uint32_t* allowed = nullptr;
    if (p.allowed) {
        const uint32_t m = p.mask_of ? __ldg(p.mask_of + row) : row;
        if (m < p.masks) allowed = p.allowed + (size_t)m * p.allowed_stride;
    }
    float rep = 1.0f, inv_rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (words) {
        const uint32_t* said = p.history + (size_t)row * p.history_stride;
        const uint32_t* bias_token = p.bias_token + (size_t)row * p.bias_stride;
        const float* bias = p.bias + (size_t)row * p.bias_stride;
        uint32_t at[AT_ONCE], total = 0, prompt = 0, biases = 0, b_at = NONE;
        float b = 0.0f;
        if (history) {
#pragma unroll
            for (uint32_t u = 0; u < AT_ONCE; u++) at[u] = th + u * THREADS < p.history_stride ? __ldg(said + th + u * THREADS) - base : NONE;
            total = min(__ldg(p.total + row), p.history_stride), prompt = min(__ldg(p.prompt + row), total);
            if (p.repetition) rep = __ldg(p.repetition + row);
            if (p.frequency) freq = __ldg(p.frequency + row);
            if (p.presence) pres = __ldg(p.presence + row);
        }
        if (biased) {
            if (th < p.bias_stride) b_at = __ldg(bias_token + th) - base, b = __ldg(bias + th);
            biases = min(__ldg(p.bias_count + row), p.bias_stride);
        }
        for (uint32_t i = th; i < a.range / 4; i += THREADS) reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0, 0, 0, 0);
        if (th == 0) s_noted = 0, s_again = 0;
        __syncthreads();
        for (uint32_t i = th; i < biases; i += THREADS) {
            if (i != th) b_at = __ldg(bias_token + i) - base, b = __ldg(bias + i);
            if (b_at >= count) continue;
            const uint32_t k = atomicAdd(&s_noted, 1u), place = first + b_at;
            s_place[k] = place, s_which[k] = i, s_bias[k] = b, s_sum[k] = b;
            if (atomicOr(s_word + place, (k + 1) << 20) >> 20 & 0x7ffu) s_again = 1;  // more than one on this token
        }
        if (history)
            for (uint32_t i = th;;) {  // eight tokens a thread and turn
#pragma unroll
                for (uint32_t u = 0; u < AT_ONCE; u++) {
                    const uint32_t k = i + u * THREADS;
                    if (at[u] < count && k < total) {
                        if (k < prompt) atomicOr(s_word + first + at[u], PROMPT);
                        else atomicAdd(s_word + first + at[u], 1u);
                    }
                }
                i += AT_ONCE * THREADS;
                if (i - th >= total) break;
#pragma unroll
                for (uint32_t u = 0; u < AT_ONCE; u++) at[u] = i + u * THREADS < total ? __ldg(said + i + u * THREADS) - base : NONE;
            }
        __syncthreads();
        if (s_again) {  // a token's first bias adds them up, one after the other
            const uint32_t noted = s_noted;
            for (uint32_t k = th; k < noted; k += THREADS) {
                const uint32_t place = s_place[k], which = s_which[k];
                float sum = s_bias[k];
                bool owner = true;
                for (uint32_t after = which;;) {
                    uint32_t next = NONE, next_k = 0;
                    for (uint32_t o = 0; o < noted; o++)
                        if (s_place[o] == place) {
                            if (s_which[o] < which) owner = false;
                            if (s_which[o] > after && s_which[o] < next) next = s_which[o], next_k = o;
                        }
                    if (!owner || next == NONE) break;
                    sum += s_bias[next_k];
                    after = next;
                }
                if (owner) s_sum[k] = sum, s_word[place] = (s_word[place] & ~(0x7ffu << 20)) | (k + 1) << 20;
            }
            __syncthreads();
        }
        inv_rep = __fdiv_rn(1.0f, rep);
    }
    auto value = [&](float x, uint32_t c) {  // before the mask; c 0: x
        const uint32_t n = c & MOST_HISTORY, biased_by = (c >> 20) & 0x7ffu;
        const float factor = (c & (PROMPT | MOST_HISTORY)) == 0 ? 1.0f : x > 0.0f ? inv_rep : rep, less = n == 0 ? 0.0f : fmaf(freq, (float)n, pres);
        float y = fmaf(x, factor, -less);
        if (biased_by != 0) y += s_sum[biased_by - 1];
        return y;
    };
#pragma unroll 2
    for (uint32_t i = th * N; i < end; i += THREADS * N) {
        if (i + N <= first) continue;
        const int t = from + (int)i;  // negative in the piece that the row starts in
        const bool whole = VEC && i >= first && i + N <= end;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (whole) raw = *reinterpret_cast<const uint4*>(src + (long long)t * SIZE);
        uint32_t bits = 0xffffffffu;
        if (allowed) {  // bits of tokens t ... t + N - 1, from one word or two
            const int w = t >> 5;
            const uint32_t lo = t >= 0 ? __ldg(allowed + w) : 0u, hi = (t + (int)N - 1) >> 5 != w && (w + 1) * 32 < vocab ? __ldg(allowed + w + 1) : 0u;
            bits = __funnelshift_r(lo, hi, t & 31);
        }
        if constexpr (VEC) {
            uint32_t c[N] = {}, any = 0;
            if (words) {
#pragma unroll
                for (uint32_t e = 0; e < N / 4; e++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(s_word + i + 4 * e);
                    c[4 * e] = v.x, c[4 * e + 1] = v.y, c[4 * e + 2] = v.z, c[4 * e + 3] = v.w;
                    any |= v.x | v.y | v.z | v.w;
                }
            }
            if (whole) {
                uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                if (any != 0) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) {
                        if constexpr (F16) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                            const __half2 h = __floats2half2_rn(value(f.x, c[2 * e]), value(f.y, c[2 * e + 1]));
                            w[e] = *reinterpret_cast<const uint32_t*>(&h);
                        } else {
                            w[e] = __float_as_uint(value(__uint_as_float(w[e]), c[e]));
                        }
                    }
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    if constexpr (F16) {  // a bit for each half: bytes 0x00 or 0xff by a byte permute
                        const uint32_t b = bits >> (2 * e), keep = __byte_perm(0x0000ff00u, 0u, (b & 1u) * 0x11u + (b & 2u) * 0x880u);
                        w[e] = (w[e] & keep) | (0xfc00fc00u & ~keep);  // -inf
                    } else {
                        w[e] = (bits >> e) & 1u ? w[e] : 0xff800000u;
                    }
                }
                *reinterpret_cast<uint4*>(dst + (long long)t * SIZE) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {  // the row's first or last piece
                for (uint32_t e = 0; e < N; e++)
                    if (i + e >= first && i + e < end) put<F16>(dst, t + (int)e, (bits >> e) & 1u ? value(get<F16>(src, t + (int)e), words ? s_word[i + e] : 0) : -INFINITY);
            }
        } else {
            put<F16>(dst, t, bits & 1u ? value(get<F16>(src, t), words ? s_word[i] : 0) : -INFINITY);
        }
    }
}

int check_logits(const tb_logits* p) {
    if (!p) return fail(OUT_OF_RANGE, "tb_logits_adjust: null descriptor");
    if (p->dtype != TB_F32 && p->dtype != TB_F16) return fail(OUT_OF_RANGE, "tb_logits_adjust: unknown dtype");
    if (p->vocab == 0 || p->vocab > 0x40000000u) return fail(OUT_OF_RANGE, "tb_logits_adjust: a vocabulary of 1 to 2^30 tokens");
    if (p->rows == 0) return OK;
    if (!p->logits || !p->out) return fail(OUT_OF_RANGE, "tb_logits_adjust: null logits");
    const size_t size = p->dtype == TB_F16 ? 2 : 4;
    if (!aligned(p->logits, size) || !aligned(p->out, size)) return fail(OUT_OF_RANGE, "tb_logits_adjust: misaligned logits");
    if (p->rows > 1 && (p->stride < p->vocab || p->out_stride < p->vocab)) return fail(OUT_OF_RANGE, "tb_logits_adjust: a stride below the vocabulary");
    if (p->out == p->logits && p->rows > 1 && p->out_stride != p->stride) return fail(OUT_OF_RANGE, "tb_logits_adjust: in place the strides are the same");
    if (p->history && (!p->total || !p->prompt)) return fail(OUT_OF_RANGE, "tb_logits_adjust: a history without its lengths");
    if (!p->history && (p->repetition || p->frequency || p->presence)) return fail(OUT_OF_RANGE, "tb_logits_adjust: penalties without a history");
    if (p->bias_token && (!p->bias || !p->bias_count)) return fail(OUT_OF_RANGE, "tb_logits_adjust: biases without values or counts");
    if (p->history && p->history_stride > MOST_HISTORY) return fail(OUT_OF_RANGE, "tb_logits_adjust: at most 2^20 - 1 tokens of history");
    if (p->bias_token && p->bias_stride > MOST_BIASES) return fail(OUT_OF_RANGE, "tb_logits_adjust: at most 1024 biases a row");
    if (p->allowed && (p->masks == 0 || (uint64_t)p->allowed_stride * 32 < p->vocab)) return fail(OUT_OF_RANGE, "tb_logits_adjust: no masks, or masks shorter than the vocabulary");
    const void* words[] = {p->history, p->prompt, p->total, p->repetition, p->frequency, p->presence, p->bias_token, p->bias, p->bias_count, p->allowed, p->mask_of};
    for (const void* w : words)
        if (!aligned(w, 4)) return fail(OUT_OF_RANGE, "tb_logits_adjust: buffers must be 4-byte aligned");
    return OK;
}

int launch_logits(tb_context* ctx, const tb_logits& p) {
    const bool f16 = p.dtype == TB_F16;
    const size_t size = f16 ? 2 : 4;
    // 16 bytes at a time where a row of logits and of outputs lie alike within 16 bytes.
    const bool vec = ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 && (p.rows == 1 || (p.stride - p.out_stride) * size % 16 == 0);
    LogitsArgs a{p, MOST_RANGE, 0};
    if (!p.bias_token) a.p.bias_stride = 0;
    const uint32_t places = p.vocab + (vec ? 15 / (uint32_t)size : 0);  // in front of a row's first token up to 15 bytes
    // Two blocks a multiprocessor, as far as ranges of 1024 tokens give them; with a long history, which every range walks again, one
    // (16 rows of 128000 with 32000 tokens: ranges of 4096 22 us, of 8192 14.5 us).
    const uint64_t wish = (uint64_t)ctx->sms * (p.history && p.history_stride > 4096 ? 1 : 2);
    while (a.range > LEAST_RANGE && (uint64_t)p.rows * ((places + a.range - 1) / a.range) < wish) a.range /= 2;
    a.ranges = (places + a.range - 1) / a.range;
    if ((uint64_t)p.rows * a.ranges > 0x7fffffffull) return fail(OUT_OF_RANGE, "tb_logits_adjust: too many rows for one call");
    const size_t smem = p.history || p.bias_token ? ((size_t)a.range + 4 * (size_t)a.p.bias_stride) * 4 : 0;
    DeviceScope scope(ctx->gpu);
    TB_CUDA(scope.error());
    auto run = [&](auto kernel, std::atomic<uint64_t>& done) {
        const cudaError_t e = allow_smem(kernel, (MOST_RANGE + 4 * MOST_BIASES) * 4, ctx->gpu, done);
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
