// st_kv4.cu -- writing and reading the 4-bit paged cache (layout: st_kv4.cuh).
//
// Append, for each new token with a slot: keys are rotated by the token's
// position, (a, b) -> (a cos - b sin, b cos + a sin) for each pair of channels,
// each product and sum rounded to f32; then keys and values are quantised by
// groups of G channels,
//     zero = f16(min x), scale = f16((max x - zero) * (1/15)),
//     code = clamp(rint((x - zero) * (1 / scale)), 0, 15)   (scale 0: code 0),
// with x clamped to the f16 range and NaN taken as 0, so the cache never
// holds a non-finite value.  Queries are rotated in the same launch.
#include "st_kv4.cuh"

namespace {

using namespace st;

struct AppendArgs {
    uint8_t *data;
    int64_t n_pages, n;
    int page, kv_heads, heads, rotary, interleaved;
    const void *k, *v, *q;
    void *q_out;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head;
    const float *cos, *sin;
    const int32_t *positions;
    int64_t n_positions;
    const int64_t *slots;
    int *status;
};

// Channels c .. c + E of x, rotated by the position whose cos / sin rows are
// given (rows of rotary / 2).
template <typename T, int E>
__device__ __forceinline__ void load_rotated(const T *x, int c, const float *cs, const float *sn, int rotary,
                                             int interleaved, float (&out)[E]) {
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int ch = c + e;
        const float own = to_f32(x[ch]);
        out[e] = own;
        if (ch < rotary) {
            const int half = rotary / 2;
            const bool first = interleaved ? (ch & 1) == 0 : ch < half;
            const int i = interleaved ? ch >> 1 : (first ? ch : ch - half);
            const float other = to_f32(x[interleaved ? ch ^ 1 : (first ? ch + half : ch - half)]);
            const float p = __fmul_rn(own, cs[i]), r = __fmul_rn(other, sn[i]);
            out[e] = first ? __fsub_rn(p, r) : __fadd_rn(p, r);
        }
    }
}

// Quantises a warp's d = 32 E channels (lane's E consecutive ones in x) by
// groups of G; the lane's codes go to code[], its group's pair to meta.
template <int E, int G>
__device__ __forceinline__ void quantise(float (&x)[E], uint32_t (&code)[E], __half2 &meta) {
    float lo = 65504.0f, hi = -65504.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -65504.0f), 65504.0f);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
#pragma unroll
    for (int o = G / E / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const __half zero = __float2half_rn(lo);
    const float z = __half2float(zero);
    const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f));
    const float s = __half2float(scale);
    const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++)
        code[e] = static_cast<uint32_t>(fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[e], z), inv)), 0.0f), 15.0f));
    meta = __halves2half2(scale, zero);
}

// One warp per (token, head) of the keys, the values and (when rotated) the
// queries.
template <typename T, int D, int G>
__global__ void k_kv4_append(const AppendArgs a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x * static_cast<int64_t>(blockDim.x / 32) + threadIdx.x / 32;
    const int64_t per = 2 * a.kv_heads + (a.q ? a.heads : 0);
    if (w >= a.n * per) return;
    const int64_t i = w / per;
    const int j = static_cast<int>(w % per);
    const int c = lane * E;
    int64_t pos = 0;
    if (a.rotary) {
        pos = a.positions[i];
        if (pos < 0 || pos >= a.n_positions) {
            if (lane == 0) set_status(a.status, DEV_BAD_ARG);
            return;
        }
    }
    const float *cs = a.cos + pos * (a.rotary / 2), *sn = a.sin + pos * (a.rotary / 2);
    float x[E];
    if (j >= 2 * a.kv_heads) {
        const int64_t head = j - 2 * a.kv_heads;
        load_rotated<T, E>(static_cast<const T *>(a.q) + i * a.q_token + head * a.q_head, c, cs, sn, a.rotary,
                           a.interleaved, x);
        T *out = static_cast<T *>(a.q_out) + (i * a.heads + head) * D + c;
#pragma unroll
        for (int e = 0; e < E; e++) out[e] = from_f32<T>(x[e]);
        return;
    }
    const int64_t slot = a.slots[i];
    if (slot < 0) return;
    if (slot >= a.n_pages * a.page) {
        if (lane == 0) set_status(a.status, DEV_BAD_ARG);
        return;
    }
    const bool value = j >= a.kv_heads;
    const int head = value ? j - a.kv_heads : j;
    if (value)
        load_rotated<T, E>(static_cast<const T *>(a.v) + i * a.v_token + head * a.v_head, c, cs, sn, 0, 0, x);
    else
        load_rotated<T, E>(static_cast<const T *>(a.k) + i * a.k_token + head * a.k_head, c, cs, sn, a.rotary,
                           a.interleaved, x);
    uint32_t code[E];
    __half2 meta;
    quantise<E, G>(x, code, meta);
    const int off = static_cast<int>(slot % a.page), r = off & 15;
    const int64_t tile = ((slot / a.page) * a.kv_heads + head) * (a.page / 16) + off / 16;
    uint8_t *t = a.data + tile * kv4_tile_bytes(D, G);
    if (value) {
#pragma unroll
        for (int e = 0; e < E; e += 2)
            t[kv4_val(D) + (c + e) / 2 * 16 + kv4_col(r)] = static_cast<uint8_t>(code[e] | code[e + 1] << 4);
    } else {
        uint8_t *row = t + (c / G) * 8 * G + r * (G / 2) + (c % G) / 2;
#pragma unroll
        for (int e = 0; e < E; e += 2) row[e / 2] = static_cast<uint8_t>(code[e] | code[e + 1] << 4);
    }
    if (c % G == 0)
        *reinterpret_cast<__half2 *>(t + (value ? kv4_vmeta(D, G) : kv4_kmeta(D)) + ((c / G) * 16 + r) * 4) = meta;
}

// One warp per (slot, head): the lane's E channels of the key and the value.
template <typename T, int D, int G>
__global__ void k_kv4_read(const uint8_t *data, int64_t n_pages, int page, int kv_heads, const int64_t *slots,
                           int64_t n, T *k, T *v, int *status) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x * static_cast<int64_t>(blockDim.x / 32) + threadIdx.x / 32;
    if (w >= n * kv_heads) return;
    const int64_t i = w / kv_heads;
    const int head = static_cast<int>(w % kv_heads), c = lane * E;
    int64_t slot = slots[i];
    if (slot >= n_pages * page) {
        if (lane == 0) set_status(status, DEV_BAD_ARG);
        slot = -1;
    }
    T *ko = k + w * D + c, *vo = v + w * D + c;
    if (slot < 0) {
#pragma unroll
        for (int e = 0; e < E; e++) ko[e] = vo[e] = from_f32<T>(0.0f);
        return;
    }
    const int off = static_cast<int>(slot % page), r = off & 15;
    const int64_t tile = ((slot / page) * kv_heads + head) * (page / 16) + off / 16;
    const uint8_t *t = data + tile * kv4_tile_bytes(D, G);
    const float2 km = __half22float2(*reinterpret_cast<const __half2 *>(t + kv4_kmeta(D) + ((c / G) * 16 + r) * 4));
    const float2 vm = __half22float2(*reinterpret_cast<const __half2 *>(t + kv4_vmeta(D, G) + ((c / G) * 16 + r) * 4));
    const uint8_t *kr = t + (c / G) * 8 * G + r * (G / 2) + (c % G) / 2;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const uint32_t kb = kr[e / 2], vb = t[kv4_val(D) + (c + e) / 2 * 16 + kv4_col(r)];
        ko[e] = from_f32<T>(fmaf(static_cast<float>(kb & 15), km.x, km.y));
        ko[e + 1] = from_f32<T>(fmaf(static_cast<float>(kb >> 4), km.x, km.y));
        vo[e] = from_f32<T>(fmaf(static_cast<float>(vb & 15), vm.x, vm.y));
        vo[e + 1] = from_f32<T>(fmaf(static_cast<float>(vb >> 4), vm.x, vm.y));
    }
}

// Calls f with the instantiation for (dtype, d, group).
template <template <typename, int, int> class F, typename... Args>
st_status by_shape(int dtype, int d, int group, Args &&...args) {
#define KV4_CASE(D_, G_)                                                                \
    if (d == D_ && group == G_) {                                                       \
        if (dtype == ST_F32) return F<float, D_, G_>::run(args...);                     \
        if (dtype == ST_F16) return F<__half, D_, G_>::run(args...);                    \
        return F<__nv_bfloat16, D_, G_>::run(args...);                                  \
    }
    KV4_CASE(64, 32)
    KV4_CASE(64, 64)
    KV4_CASE(128, 32)
    KV4_CASE(128, 64)
    KV4_CASE(128, 128)
#undef KV4_CASE
    return ST_UNSUPPORTED_SHAPE;
}

template <typename T, int D, int G>
struct AppendLaunch {
    static st_status run(st_handle *h, const AppendArgs &a) {
        const int64_t warps = a.n * (2 * a.kv_heads + (a.q ? a.heads : 0));
        const int64_t blocks = (warps + 3) / 4;
        if (blocks > 0x7fffffff) return h->fail(ST_UNSUPPORTED_SHAPE, "st_kv4_append: too many tokens");
        k_kv4_append<T, D, G><<<static_cast<unsigned>(blocks), 128, 0, h->stream>>>(a);
        return st_after_launch(h, "k_kv4_append");
    }
};

template <typename T, int D, int G>
struct ReadLaunch {
    static st_status run(st_handle *h, const uint8_t *data, int64_t n_pages, int page, int kv_heads,
                         const int64_t *slots, int64_t n, void *k, void *v) {
        const int64_t blocks = (n * kv_heads + 3) / 4;
        if (blocks > 0x7fffffff) return h->fail(ST_UNSUPPORTED_SHAPE, "st_kv4_read: too many tokens");
        k_kv4_read<T, D, G><<<static_cast<unsigned>(blocks), 128, 0, h->stream>>>(
            data, n_pages, page, kv_heads, slots, n, static_cast<T *>(k), static_cast<T *>(v), h->d_status);
        return st_after_launch(h, "k_kv4_read");
    }
};

}  // namespace

extern "C" st_status st_kv4_append(st_handle *h, void *data, int64_t n_pages, int32_t page, int32_t kv_heads,
                                   int32_t d, int32_t group, const void *k, int64_t k_token, int64_t k_head,
                                   const void *v, int64_t v_token, int64_t v_head, const int64_t *slots, int64_t n,
                                   const void *q, int64_t q_token, int64_t q_head, void *q_out, int32_t heads,
                                   const float *cos, const float *sin, const int32_t *positions, int64_t n_positions,
                                   int32_t rotary, int32_t interleaved, int32_t dtype) {
    if (!h) return ST_INVALID_ARG;
    if (st_status s = kv4_check(h, "st_kv4_append", data, n_pages, page, kv_heads, d, group); s != ST_OK) return s;
    if (n < 0 || dtype < ST_F32 || dtype > ST_BF16)
        return h->fail(ST_INVALID_ARG, "st_kv4_append: bad token count or dtype");
    if (rotary < 0 || rotary > d || rotary % 2 != 0)
        return h->fail(ST_INVALID_ARG, "st_kv4_append: rotary = %d (even, at most d)", rotary);
    if (n == 0) return ST_OK;
    if (!k || !v || !slots) return h->fail(ST_INVALID_ARG, "st_kv4_append: null keys, values or slots");
    if (rotary > 0 && (!cos || !sin || !positions || n_positions < 1))
        return h->fail(ST_INVALID_ARG, "st_kv4_append: a rotation needs cos, sin and positions");
    if (q && (!q_out || heads < 1 || rotary == 0))
        return h->fail(ST_INVALID_ARG, "st_kv4_append: queries are only rotated: they need q_out and a rotation");
    cudaSetDevice(h->device);
    const AppendArgs a = {static_cast<uint8_t *>(data), n_pages, n, page, kv_heads, heads, rotary, interleaved, k, v,
                          q, q_out, k_token, k_head, v_token, v_head, q_token, q_head, cos, sin, positions,
                          n_positions, slots, h->d_status};
    return by_shape<AppendLaunch>(dtype, d, group, h, a);
}

extern "C" st_status st_kv4_read(st_handle *h, const void *data, int64_t n_pages, int32_t page, int32_t kv_heads,
                                 int32_t d, int32_t group, const int64_t *slots, int64_t n, void *k, void *v,
                                 int32_t dtype) {
    if (!h) return ST_INVALID_ARG;
    if (st_status s = kv4_check(h, "st_kv4_read", data, n_pages, page, kv_heads, d, group); s != ST_OK) return s;
    if (n < 0 || dtype < ST_F32 || dtype > ST_BF16)
        return h->fail(ST_INVALID_ARG, "st_kv4_read: bad token count or dtype");
    if (n == 0) return ST_OK;
    if (!k || !v || !slots) return h->fail(ST_INVALID_ARG, "st_kv4_read: null keys, values or slots");
    cudaSetDevice(h->device);
    return by_shape<ReadLaunch>(dtype, d, group, h, static_cast<const uint8_t *>(data), n_pages, page, kv_heads,
                                slots, n, k, v);
}
