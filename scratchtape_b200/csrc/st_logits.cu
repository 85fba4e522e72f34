// st_logits.cu -- logits adjusted before a token is drawn from them.
//
// Row r, token v, with n_all and n_said the number of times v occurs in the
// row's history and in the part of it after the prompt:
//     x <- n_all > 0 ? (x > 0 ? x / repetition : x * repetition) : x
//     x <- x - frequency * n_said - (n_said > 0 ? presence : 0)
//     x <- x + the sum of the row's bias entries for v, in the list's order
//     x <- -inf where the row's mask has a 0 for v (whatever x is, NaN too)
// in f32, each operation rounded, and once more to the output's type.
#include <type_traits>

#include "st_kv4.cuh"

namespace {

using namespace st;

struct LogitsArgs {
    const void *in;
    void *out;
    int64_t ld, out_ld, rows;
    int vocab;
    const int32_t *tokens, *starts, *prompt;
    const float *repetition, *presence, *frequency;
    const int32_t *bias_tokens, *bias_starts;
    const float *bias_values;
    const int32_t *mask, *mask_rows;
    int64_t masks;
    int words, vec;
    int *status;
};

constexpr int CHUNK = 16384, THREADS = 512, HOLD = 8, LIST = 4096;

// Four words of logits, -inf where their mask bits are 0.
template <typename T>
__device__ __forceinline__ void mask_words(uint32_t (&w)[4], uint32_t bits) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (sizeof(T) == 4) {
            if (!(bits >> k & 1u)) w[k] = 0xff800000u;
        } else {
            const uint32_t keep = (bits >> (2 * k) & 1u) * 0xffffu | (bits >> (2 * k + 1) & 1u) * 0xffff0000u;
            const uint32_t none = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
            w[k] = (w[k] & keep) | (none & ~keep);
        }
    }
}

// One block per (piece of a row, row).  A piece is CHUNK tokens from a 16-byte
// boundary of the row's memory on; `shift` elements of the first one lie
// before the row.  Few tokens of a piece occur in the history, so the block
// looks through the history while the piece's logits are on their way to
// registers: each token that occurs (or has a bias) is listed once and its
// count cleared, then they are counted, and a thread for each listed token
// computes its new logit.  The piece itself is only masked and stored; the
// listed tokens' logits follow it.
template <typename T>
__global__ void __launch_bounds__(THREADS) k_logits_adjust(const LogitsArgs a) {
    constexpr int VEC = 16 / sizeof(T), EACH = CHUNK / VEC / THREADS;
    extern __shared__ uint32_t cnt[];  // [CHUNK]: 2 n_said + (once in the prompt), in the end the new logit's bits
    __shared__ uint32_t touched[CHUNK / 32], biased[CHUNK / 32];
    __shared__ uint16_t list[LIST];
    __shared__ int listed;
    grid_dep_wait();
    const int64_t r = blockIdx.y;
    const T *in = static_cast<const T *>(a.in) + r * a.ld;
    T *out = static_cast<T *>(a.out) + r * a.out_ld;
    const int shift = a.vec ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % VEC) : 0;
    const int v0 = static_cast<int>(blockIdx.x) * CHUNK - shift;  // the token of the piece's first element
    if (v0 >= a.vocab) return;
    const int s = a.tokens ? a.starts[r] : 0, e = a.tokens ? a.starts[r + 1] : 0;
    const int bs = a.bias_tokens ? a.bias_starts[r] : 0, be = a.bias_tokens ? a.bias_starts[r + 1] : 0;
    const int said = s + (a.prompt ? a.prompt[r] : 0);
    int64_t mr = -1;
    if (a.mask) {
        mr = a.mask_rows ? a.mask_rows[r] : r;
        if (mr >= a.masks) {
            if (threadIdx.x == 0) set_status(a.status, DEV_BAD_ARG);
            mr = -1;
        }
    }
    const uint32_t *mask = mr >= 0 ? reinterpret_cast<const uint32_t *>(a.mask) + mr * a.words : nullptr;
    uint32_t x[EACH][4];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int v = v0 + (i * THREADS + static_cast<int>(threadIdx.x)) * VEC;
        if (a.vec && v >= 0 && v + VEC <= a.vocab) {
            const uint4 w = *reinterpret_cast<const uint4 *>(in + v);
            x[i][0] = w.x, x[i][1] = w.y, x[i][2] = w.z, x[i][3] = w.w;
        }
    }
    const int low = max(v0, 0);
    const uint32_t here = min(v0 + CHUNK, a.vocab) - low;
    const auto place = [&](int token) {  // in the piece, or -1
        return static_cast<uint32_t>(token - low) < here ? token - v0 : -1;
    };
    int held[HOLD];  // the history's first tokens, for both looks
#pragma unroll
    for (int k = 0; k < HOLD; k++) {
        const int i = s + k * THREADS + static_cast<int>(threadIdx.x);
        held[k] = i < e ? a.tokens[i] : -1;
    }
    if (threadIdx.x == 0) listed = 0;
    for (int i = threadIdx.x; i < CHUNK / 32; i += THREADS) touched[i] = biased[i] = 0;
    __syncthreads();
    const auto touch = [&](int p) {
        const uint32_t bit = 1u << (p & 31);
        if (p >= 0 && !(atomicOr(&touched[p / 32], bit) & bit)) {
            cnt[p] = 0;
            const int at = atomicAdd(&listed, 1);
            if (at < LIST) list[at] = static_cast<uint16_t>(p);
        }
    };
#pragma unroll
    for (int k = 0; k < HOLD; k++) touch(held[k] = place(held[k]));
    for (int i = s + HOLD * THREADS + threadIdx.x; i < e; i += THREADS) touch(place(a.tokens[i]));
    for (int i = bs + threadIdx.x; i < be; i += THREADS) {
        const int p = place(a.bias_tokens[i]);
        touch(p);
        if (p >= 0) atomicOr(&biased[p / 32], 1u << (p % 32));
    }
    __syncthreads();
    const auto count = [&](int p, int i) {
        if (p >= 0) {
            if (i >= said)
                atomicAdd(&cnt[p], 2u);
            else
                atomicOr(&cnt[p], 1u);
        }
    };
#pragma unroll
    for (int k = 0; k < HOLD; k++) count(held[k], s + k * THREADS + static_cast<int>(threadIdx.x));
    for (int i = s + HOLD * THREADS + threadIdx.x; i < e; i += THREADS) count(place(a.tokens[i]), i);
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.0f, pres = a.presence ? a.presence[r] : 0.0f,
                freq = a.frequency ? a.frequency[r] : 0.0f;
    // every listed token, or where they are more than the list holds, every bit
    const bool whole = listed <= LIST;
    const int many = whole ? listed : CHUNK;
    const auto token_of = [&](int i) { return whole ? list[i] : touched[i / 32] >> (i % 32) & 1u ? i : -1; };
    for (int i = threadIdx.x; i < many; i += THREADS) {
        const int p = token_of(i);
        if (p < 0) continue;
        float y = to_f32(in[v0 + p]);
        const uint32_t n = cnt[p];
        if (n) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
        if (n > 1) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n >> 1))), pres);
        if (biased[p / 32] >> (p % 32) & 1u) {
            float sum = 0.0f;
            for (int j = bs; j < be; j++)
                if (a.bias_tokens[j] == v0 + p) sum = __fadd_rn(sum, a.bias_values[j]);
            y = __fadd_rn(y, sum);
        }
        if (mask && !(mask[(v0 + p) / 32] >> ((v0 + p) % 32) & 1u)) y = -INFINITY;
        cnt[p] = __float_as_uint(y);
    }
    __syncthreads();  // all of the piece is read before any of it is written: out may be in
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int v = v0 + (i * THREADS + static_cast<int>(threadIdx.x)) * VEC;
        if (a.vec && v >= 0 && v + VEC <= a.vocab) {
            if (mask) mask_words<T>(x[i], __funnelshift_r(mask[v / 32], mask[(v + VEC - 1) / 32], v % 32));
            *reinterpret_cast<uint4 *>(out + v) = make_uint4(x[i][0], x[i][1], x[i][2], x[i][3]);
        } else {
#pragma unroll 1
            for (int k = max(0, -v); k < VEC && v + k < a.vocab; k++)
                out[v + k] = mask && !(mask[(v + k) / 32] >> ((v + k) % 32) & 1u) ? from_f32<T>(-INFINITY) : in[v + k];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < many; i += THREADS)
        if (const int p = token_of(i); p >= 0) out[v0 + p] = from_f32<T>(__uint_as_float(cnt[p]));
}

template <typename T>
st_status launch(st_handle *h, const LogitsArgs &a) {
    constexpr int VEC = 16 / sizeof(T);
    const dim3 grid(static_cast<unsigned>((a.vocab + (a.vec ? VEC - 1 : 0) + CHUNK - 1) / CHUNK),
                    static_cast<unsigned>(a.rows));
    const size_t smem = sizeof(uint32_t) * CHUNK;
    ST_CHECK_CUDA(h, cudaFuncSetAttribute(k_logits_adjust<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          static_cast<int>(smem)));
    ST_CHECK_CUDA(h, st_launch_dependent(h, k_logits_adjust<T>, grid, dim3(THREADS), smem, a));
    return st_after_launch(h, "k_logits_adjust");
}

}  // namespace

extern "C" st_status st_logits_adjust(st_handle *h, const void *logits, int64_t ld, void *out, int64_t out_ld,
                                      int64_t rows, int64_t vocab, const int32_t *tokens, const int32_t *starts,
                                      const int32_t *prompt, const float *repetition, const float *presence,
                                      const float *frequency, const int32_t *bias_tokens, const float *bias_values,
                                      const int32_t *bias_starts, const int32_t *mask, int64_t masks,
                                      const int32_t *mask_rows, int32_t dtype) {
    if (!h) return ST_INVALID_ARG;
    if (rows < 0 || vocab < 1 || ld < vocab || out_ld < vocab || dtype < ST_F32 || dtype > ST_BF16)
        return h->fail(ST_INVALID_ARG, "st_logits_adjust: bad arguments");
    if (rows > 65535 || vocab > (1 << 30))
        return h->fail(ST_UNSUPPORTED_SHAPE, "st_logits_adjust: at most 65535 rows and 2^30 tokens");
    if (rows == 0) return ST_OK;
    if (!logits || !out) return h->fail(ST_INVALID_ARG, "st_logits_adjust: null logits or out");
    if (tokens && !starts) return h->fail(ST_INVALID_ARG, "st_logits_adjust: a history needs its starts");
    if (bias_tokens && (!bias_values || !bias_starts))
        return h->fail(ST_INVALID_ARG, "st_logits_adjust: a bias needs its values and starts");
    if (mask && (masks < 1 || (!mask_rows && masks < rows)))
        return h->fail(ST_INVALID_ARG, "st_logits_adjust: %lld masks for %lld rows", static_cast<long long>(masks),
                       static_cast<long long>(rows));
    cudaSetDevice(h->device);
    // 16-byte accesses where a row of logits and of out start at the same place between 16-byte boundaries
    const int size = dtype == ST_F32 ? 4 : 2;
    const uintptr_t in0 = reinterpret_cast<uintptr_t>(logits), out0 = reinterpret_cast<uintptr_t>(out);
    const int vec = (in0 - out0) % 16 == 0 && (rows == 1 || (ld - out_ld) * size % 16 == 0) && in0 % size == 0;
    const LogitsArgs a = {logits, out, ld, out_ld, rows, static_cast<int>(vocab), tokens, starts, prompt, repetition,
                          presence, frequency, bias_tokens, bias_starts, bias_values, mask, mask_rows, masks,
                          static_cast<int>((vocab + 31) / 32), vec, h->d_status};
    return dtype == ST_F32 ? launch<float>(h, a) : dtype == ST_F16 ? launch<__half>(h, a) : launch<__nv_bfloat16>(h, a);
}
