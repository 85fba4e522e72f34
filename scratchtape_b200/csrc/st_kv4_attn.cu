// st_kv4_attn.cu -- attention over the 4-bit paged cache (layout: st_kv4.cuh).
//
// Row i (a query of sequence b at position p = len - queries + index) sees key
// j < len with j <= p (causal) and j > p - window (window > 0):
//     x_j = scale q . k_j,  o = sum_j e^{x_j - m} v_j / (sum_j e^{x_j - m} [+ e^{-m}])
// A row that sees nothing gives o = 0 and lse = -inf (softmax1: lse = 0).
#include "st_kv4.cuh"

namespace {

using namespace st;

struct AttnArgs {
    const void *q;
    int64_t q_token, q_head;
    void *o;
    float *lse;
    const uint8_t *data;
    int64_t n_pages;
    int page, heads, kv_heads;
    const int32_t *pages;
    int64_t max_pages;
    const int32_t *kv_len, *q_start;
    int64_t batch, rows;
    int max_q;
    float scale;
    int causal, one, window;
    int *status;
};

// One warp per (row, head), one key at a time.
template <typename T, int D, int G>
__global__ void k_kv4_attn_rows(const AttnArgs a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x * static_cast<int64_t>(blockDim.x / 32) + threadIdx.x / 32;
    if (w >= a.rows * a.heads) return;
    const int64_t row = w / a.heads;
    const int head = static_cast<int>(w % a.heads), kv_head = head / (a.heads / a.kv_heads), c = lane * E;
    int64_t b = row, first = row, count = 1;
    if (a.q_start) {
        int64_t lo = 0, hi = a.batch;  // the last b with q_start[b] <= row
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            (a.q_start[mid] <= row ? lo : hi) = mid;
        }
        b = lo;
        first = a.q_start[b];
        count = a.q_start[b + 1] - first;
        if (first > row || row >= first + count || count > a.max_q) {
            if (lane == 0) set_status(a.status, DEV_BAD_ARG);
            return;
        }
    }
    int64_t len = a.kv_len[b];
    if (len < 0 || len > a.max_pages * a.page) {
        if (lane == 0) set_status(a.status, DEV_BAD_ARG);
        len = len < 0 ? 0 : a.max_pages * a.page;
    }
    const int64_t pos = len - count + (row - first);
    const int64_t end = a.causal ? (pos + 1 < len ? pos + 1 : len) : len;
    const int64_t begin = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const T *q = static_cast<const T *>(a.q) + row * a.q_token + head * a.q_head + c;
    float qf[E], o[E], m = a.one ? 0.0f : -INFINITY, l = a.one ? 1.0f : 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        qf[e] = to_f32(q[e]);
        o[e] = 0.0f;
    }
    for (int64_t j = begin; j < end; j++) {
        const int64_t p = a.pages[b * a.max_pages + j / a.page];
        if (p < 0 || p >= a.n_pages) {
            if (lane == 0) set_status(a.status, DEV_BAD_ARG);
            continue;
        }
        const int off = static_cast<int>(j % a.page), r = off & 15;
        const uint8_t *t =
            a.data + ((p * a.kv_heads + kv_head) * (a.page / 16) + off / 16) * kv4_tile_bytes(D, G);
        const float2 km =
            __half22float2(*reinterpret_cast<const __half2 *>(t + kv4_kmeta(D) + ((c / G) * 16 + r) * 4));
        const float2 vm =
            __half22float2(*reinterpret_cast<const __half2 *>(t + kv4_vmeta(D, G) + ((c / G) * 16 + r) * 4));
        const uint8_t *kr = t + (c / G) * 8 * G + r * (G / 2) + (c % G) / 2;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++)
            x += qf[e] * fmaf(static_cast<float>(kr[e / 2] >> (e % 2 * 4) & 15), km.x, km.y);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        x *= a.scale;
        const float m2 = fmaxf(m, x), f = expf(m - m2), pr = expf(x - m2);
        m = m2;
        l = l * f + pr;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t vb = t[kv4_val(D) + (c + e) / 2 * 16 + kv4_col(r)];
            o[e] = o[e] * f + pr * fmaf(static_cast<float>(vb >> (e % 2 * 4) & 15), vm.x, vm.y);
        }
    }
    T *out = static_cast<T *>(a.o) + w * D + c;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) out[e] = from_f32<T>(o[e] * inv);
    if (a.lse && lane == 0) a.lse[w] = l > 0.0f ? m + logf(l) : -INFINITY;
}

template <typename T, int D, int G>
st_status launch(st_handle *h, const AttnArgs &a) {
    const int64_t blocks = (a.rows * a.heads + 3) / 4;
    if (blocks > 0x7fffffff) return h->fail(ST_UNSUPPORTED_SHAPE, "st_kv4_attn: too many rows");
    k_kv4_attn_rows<T, D, G><<<static_cast<unsigned>(blocks), 128, 0, h->stream>>>(a);
    return st_after_launch(h, "k_kv4_attn_rows");
}

}  // namespace

extern "C" st_status st_kv4_attn_workspace(st_handle *h, int64_t batch, int64_t rows, int64_t max_q, int32_t heads,
                                           int32_t kv_heads, int32_t d, int64_t *bytes) {
    if (!h) return ST_INVALID_ARG;
    if (!bytes) return h->fail(ST_INVALID_ARG, "st_kv4_attn_workspace: null bytes");
    *bytes = 0;
    return ST_OK;
}

extern "C" st_status st_kv4_attn(st_handle *h, const void *q, int64_t q_token, int64_t q_head, void *o, float *lse,
                                 const void *data, int64_t n_pages, int32_t page, int32_t heads, int32_t kv_heads,
                                 int32_t d, int32_t group, const int32_t *pages, int64_t max_pages,
                                 const int32_t *kv_len, const int32_t *q_start, int64_t batch, int64_t rows,
                                 int64_t max_q, float scale, int32_t causal, int32_t one, int32_t window,
                                 int32_t dtype, void *workspace, int64_t workspace_bytes) {
    if (!h) return ST_INVALID_ARG;
    if (st_status s = kv4_check(h, "st_kv4_attn", data, n_pages, page, kv_heads, d, group); s != ST_OK) return s;
    if (batch < 0 || rows < 0 || max_pages < 0 || max_q < 1 || window < 0 || dtype < ST_F32 || dtype > ST_BF16)
        return h->fail(ST_INVALID_ARG, "st_kv4_attn: bad arguments");
    if (heads < kv_heads || heads % kv_heads != 0)
        return h->fail(ST_INVALID_ARG, "st_kv4_attn: %d heads do not share %d", heads, kv_heads);
    if (max_pages * page > 0x7fffffff || rows > 0x7fffffff || max_q > 0x7fffffff || batch > 0x7fffffff)
        return h->fail(ST_UNSUPPORTED_SHAPE, "st_kv4_attn: over 2^31 - 1 rows or keys");
    if (!q_start && rows != batch)
        return h->fail(ST_INVALID_ARG, "st_kv4_attn: without q_start there is one row per sequence");
    if (rows == 0 || batch == 0) return ST_OK;
    if (!q || !o || (!pages && max_pages > 0) || !kv_len) return h->fail(ST_INVALID_ARG, "st_kv4_attn: null argument");
    (void)workspace;
    (void)workspace_bytes;
    cudaSetDevice(h->device);
    const AttnArgs a = {q, q_token, q_head, o, lse, static_cast<const uint8_t *>(data), n_pages, page, heads,
                        kv_heads, pages, max_pages, kv_len, q_start, batch, rows, static_cast<int>(max_q), scale,
                        causal, one, window, h->d_status};
#define KV4_CASE(D_, G_)                                                       \
    if (d == D_ && group == G_) {                                              \
        if (dtype == ST_F32) return launch<float, D_, G_>(h, a);               \
        if (dtype == ST_F16) return launch<__half, D_, G_>(h, a);              \
        return launch<__nv_bfloat16, D_, G_>(h, a);                            \
    }
    KV4_CASE(64, 32)
    KV4_CASE(64, 64)
    KV4_CASE(128, 32)
    KV4_CASE(128, 64)
    KV4_CASE(128, 128)
#undef KV4_CASE
    return ST_UNSUPPORTED_SHAPE;
}
