// st_logits.cu -- logits adjusted before a token is drawn from them.
//
// Row r, token v, with n_all and n_said the number of times v occurs in the
// row's history and in the part of it after the prompt:
//     x <- n_all > 0 ? (x > 0 ? x / repetition : x * repetition) : x
//     x <- x - frequency * n_said - (n_said > 0 ? presence : 0)
//     x <- x + the sum of the row's bias entries for v, in the list's order
//     x <- -inf where the row's mask has a 0 for v (whatever x is, NaN too)
// in f32, each operation rounded, and once more to the output's type.
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
    int words;
    int *status;
};

constexpr int CHUNK = 8192;  // tokens of one block's piece of a row: 32 KB of counts in shared memory

// One block per (piece of a row, row).  cnt[v] = 2 n_said + (n_all > 0).
template <typename T>
__global__ void k_logits_adjust(const LogitsArgs a) {
    extern __shared__ uint32_t cnt[];
    float *bias = reinterpret_cast<float *>(cnt + CHUNK);
    const int64_t r = blockIdx.y;
    const int v0 = blockIdx.x * CHUNK, nv = min(CHUNK, a.vocab - v0);
    for (int v = threadIdx.x; v < nv; v += blockDim.x) {
        cnt[v] = 0;
        if (a.bias_tokens) bias[v] = 0.0f;
    }
    __syncthreads();
    if (a.tokens) {
        const int s = a.starts[r], e = a.starts[r + 1], said = s + (a.prompt ? a.prompt[r] : 0);
        for (int i = s + threadIdx.x; i < e; i += blockDim.x) {
            const uint32_t v = static_cast<uint32_t>(a.tokens[i]) - static_cast<uint32_t>(v0);
            if (v < static_cast<uint32_t>(nv)) {
                atomicOr(&cnt[v], 1u);
                if (i >= said) atomicAdd(&cnt[v], 2u);
            }
        }
    }
    if (a.bias_tokens && threadIdx.x == 0) {
        for (int i = a.bias_starts[r]; i < a.bias_starts[r + 1]; i++) {
            const uint32_t v = static_cast<uint32_t>(a.bias_tokens[i]) - static_cast<uint32_t>(v0);
            if (v < static_cast<uint32_t>(nv)) bias[v] = __fadd_rn(bias[v], a.bias_values[i]);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.0f, pres = a.presence ? a.presence[r] : 0.0f,
                freq = a.frequency ? a.frequency[r] : 0.0f;
    int64_t mr = -1;
    if (a.mask) {
        mr = a.mask_rows ? a.mask_rows[r] : r;
        if (mr >= a.masks) {
            if (threadIdx.x == 0) set_status(a.status, DEV_BAD_ARG);
            mr = -1;
        }
    }
    const T *in = static_cast<const T *>(a.in) + r * a.ld + v0;
    T *out = static_cast<T *>(a.out) + r * a.out_ld + v0;
    for (int v = threadIdx.x; v < nv; v += blockDim.x) {
        float x = to_f32(in[v]);
        const uint32_t n = cnt[v];
        if (n) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (n > 1) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(n >> 1))), pres);
        if (a.bias_tokens) x = __fadd_rn(x, bias[v]);
        if (mr >= 0) {
            const uint32_t word = static_cast<uint32_t>(a.mask[mr * a.words + (v0 + v) / 32]);
            if (!(word >> ((v0 + v) & 31) & 1u)) x = -INFINITY;
        }
        out[v] = from_f32<T>(x);
    }
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
    const LogitsArgs a = {logits, out, ld, out_ld, rows, static_cast<int>(vocab), tokens, starts, prompt, repetition,
                          presence, frequency, bias_tokens, bias_starts, bias_values, mask, mask_rows, masks,
                          static_cast<int>((vocab + 31) / 32), h->d_status};
    const dim3 grid(static_cast<unsigned>((vocab + CHUNK - 1) / CHUNK), static_cast<unsigned>(rows));
    const size_t smem = sizeof(uint32_t) * CHUNK * (bias_tokens ? 2 : 1);
    auto kern = dtype == ST_F32 ? k_logits_adjust<float>
                                : dtype == ST_F16 ? k_logits_adjust<__half> : k_logits_adjust<__nv_bfloat16>;
    ST_CHECK_CUDA(h, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 4 * CHUNK));
    kern<<<grid, 256, smem, h->stream>>>(a);
    return st_after_launch(h, "k_logits_adjust");
}
