// Attention over a KV cache held in 4 bits (MXFP4: e2m1 nibbles, an e8m0 byte per 32 values), for a batch of sequences.
//
//   append   rows of every sequence behind the positions it holds; K and V per kv head as MXFP4, an optional K tail of `rope`
//            values shared by the heads (taken from head 0) as bfloat16
//   to_f32   the values the cache stands for
//   attn     s_j = scale * (q . k_j), softmax over the positions a row may see, o = sum p_j v_j; query heads nh / nkv to a kv head
//
// Quantization of a block: e = the smallest exponent with 6 * 2^e >= max|x|, clamped to [-127, 125]; the nearest level, upwards at
// a midpoint (the rule of the MXFP4 codec); NaN becomes 0 and what lies beyond 6 * 2^125 saturates, so that the cache holds
// finite values only: a position that a row may not see has weight 0, and 0 times a finite value is 0.
#include "mk_mixer.h"

namespace {

// ------------------------------------------------------------------------------------------------------------ append

// One wave: 64 items of a row of the call.  An item is 8 values: nkv * dk / 8 of K, nkv * dv / 8 of V, rope / 8 of the K tail.
// dk and dv are multiples of 32, so a block of 32 values is an aligned quad of lanes.
template <typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(MkKv4 c, MkSeqs s, const T *__restrict__ k_rows, size_t k_stride, const T *__restrict__ v_rows,
                                                         size_t v_stride, int fresh, int waves_per_row) {
    const int w = (int)(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int t = w / waves_per_row;
    if (t >= s.T) return;
    const int b = s.of_row(t);
    if (b < 0) return;
    const int pos = (fresh ? 0 : c.lens[b]) + (t - s.at(b));
    if (pos < 0 || pos >= c.cap) return;
    const int item = (w - t * waves_per_row) * 64 + (threadIdx.x & 63);
    const int nk = c.nkv * c.dk / 8, nv = c.nkv * c.dv / 8;
    float v[8];
    if (item < nk + nv) {
        const bool is_v = item >= nk;
        const int width = is_v ? c.dv : c.dk, e = (is_v ? item - nk : item) * 8;
        const int h = e / width, d = e - h * width;
        if (is_v) mk_load8(v_rows + (size_t)t * v_stride + (size_t)h * c.dv + d, v);
        else mk_load8(k_rows + (size_t)t * k_stride + (size_t)h * (c.dk + c.rope) + d, v);
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
        m = fmaxf(m, mk_dpp<0xB1>(m));
        m = fmaxf(m, mk_dpp<0x4E>(m));
        const uint32_t bits = __float_as_uint(m);
        int ex = (int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) > 0x400000u ? 1 : 2);
        ex = max(-127, min(125, ex));
        const float inv = mk_scale_from_byte((uint32_t)(127 - ex));
        uint32_t code = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float a = fabsf(v[i]) * inv;
            const uint32_t lev = (a >= 0.25f) + (a >= 0.75f) + (a >= 1.25f) + (a >= 1.75f) + (a >= 2.5f) + (a >= 3.5f) + (a >= 5.0f);
            code |= (lev | (v[i] < 0.0f ? 8u : 0u)) << (4 * i);
        }
        const size_t row = ((size_t)b * c.nkv + h) * c.cap + pos;
        uint8_t *q = is_v ? c.vq : c.kq, *sc = is_v ? c.vs : c.ks;
        *(uint32_t *)(q + row * (width / 2) + d / 2) = code;
        if ((item & 3) == 0) sc[row * (width / 32) + d / 32] = (uint8_t)(ex + 127);
    } else if (item < nk + nv + c.rope / 8) {
        const int d = (item - nk - nv) * 8;
        mk_load8(k_rows + (size_t)t * k_stride + c.dk + d, v);
        mk_b8 o;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = (__bf16)v[i];
        *(mk_b8 *)(c.kr + ((size_t)b * c.cap + pos) * c.rope + d) = o;
    }
}

__global__ __launch_bounds__(256) void kv4_advance_kernel(MkKv4 c, MkSeqs s, int fresh) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < c.B) c.lens[b] = (fresh ? 0 : c.lens[b]) + max(s.at(b + 1) - s.at(b), 0);
}

// ------------------------------------------------------------------------------------------------------------ to_f32

// One thread: 8 values of K or V of (sequence, position, head); positions a sequence does not hold are zero.
__global__ __launch_bounds__(256) void kv4_to_f32_kernel(MkKv4 c, int n, float *__restrict__ k, float *__restrict__ v, int items, size_t total) {
    const size_t idx = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= total) return;
    const int item = (int)(idx % items);
    const size_t row = idx / items;  // (b * n + pos) * nkv + h
    const int h = (int)(row % c.nkv);
    const size_t bp = row / c.nkv;
    const int pos = (int)(bp % n), b = (int)(bp / n);
    const bool held = pos < c.lens[b];
    const int nk = c.dk / 8, nr = c.rope / 8;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = 0.0f;
    float *dst;
    const size_t at = ((size_t)b * c.nkv + h) * c.cap + pos;
    if (item >= nk && item < nk + nr) {
        const int d = (item - nk) * 8;
        dst = k + row * (c.dk + c.rope) + c.dk + d;
        if (held) mk_load8((const __bf16 *)(c.kr + ((size_t)b * c.cap + pos) * c.rope + d), o);
    } else {
        const bool is_v = item >= nk + nr;
        const int d = (is_v ? item - nk - nr : item) * 8, width = is_v ? c.dv : c.dk;
        dst = is_v ? v + row * c.dv + d : k + row * (c.dk + c.rope) + d;
        if (held) {
            const uint32_t code = *(const uint32_t *)((is_v ? c.vq : c.kq) + at * (width / 2) + d / 2);
            const float sc = mk_scale_from_byte((is_v ? c.vs : c.ks)[at * (width / 32) + d / 32]);
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = mk_e2m1((code >> (4 * i)) & 15u) * sc;
        }
    }
    *(mk_f4 *)dst = mk_f4{o[0], o[1], o[2], o[3]};
    *(mk_f4 *)(dst + 4) = mk_f4{o[4], o[5], o[6], o[7]};
}

}  // namespace

extern "C" int mk_dev_kv4_append(const mk_kv4_cache *c, int dtype, const void *k_rows, size_t k_stride, const void *v_rows, size_t v_stride, size_t T,
                                 const int32_t *cu, int fresh, void *stream) {
    int st = mk_kv4_check(c);
    if (st != MK_OK || (st = mk_kv4_check_rows(c, dtype, T, cu)) != MK_OK) return st;
    MK_REQUIRE(T == 0 || (k_rows && v_rows), "null pointer");
    MK_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0 && mk_aligned16(k_rows) && mk_aligned16(v_rows), "rows must be 16-byte aligned, their strides multiples of 8 values");
    MK_REQUIRE(T <= 1 || (k_stride >= c->nkv * (c->dk + c->rope) && v_stride >= c->nkv * c->dv), "a row stride is shorter than a row");
    const MkSeqs s{cu, (int)T, (int)c->B};
    const MkKv4 v = mk_kv4_view(c);
    const size_t items = c->nkv * (c->dk + c->dv) / 8 + c->rope / 8, wpr = (items + 63) / 64;
    MK_REQUIRE(T * wpr <= 0x7FFFFFFFull / 64, "too many rows in one call");
    if (T) {
        const unsigned grid = (unsigned)((T * wpr + 3) / 4);
        if (dtype == MK_F32)
            hipLaunchKernelGGL(kv4_append_kernel<float>, dim3(grid), dim3(256), 0, (hipStream_t)stream, v, s, (const float *)k_rows, k_stride, (const float *)v_rows,
                               v_stride, fresh, (int)wpr);
        else
            hipLaunchKernelGGL(kv4_append_kernel<__bf16>, dim3(grid), dim3(256), 0, (hipStream_t)stream, v, s, (const __bf16 *)k_rows, k_stride,
                               (const __bf16 *)v_rows, v_stride, fresh, (int)wpr);
        if ((st = mk_launch_status("kv4_append")) != MK_OK) return st;
    }
    hipLaunchKernelGGL(kv4_advance_kernel, dim3((unsigned)((c->B + 255) / 256)), dim3(256), 0, (hipStream_t)stream, v, s, fresh);
    return mk_launch_status("kv4_advance");
}

extern "C" int mk_dev_kv4_to_f32(const mk_kv4_cache *c, size_t n, float *k, float *v, void *stream) {
    int st = mk_kv4_check(c);
    if (st != MK_OK) return st;
    MK_REQUIRE(n <= c->cap, "more positions than the cache holds");
    if (n == 0) return MK_OK;
    MK_REQUIRE(k && v && mk_aligned16(k) && mk_aligned16(v), "outputs must be 16-byte aligned");
    const size_t items = (c->dk + c->rope + c->dv) / 8, total = c->B * n * c->nkv * items;
    MK_REQUIRE((total + 255) / 256 <= 0x7FFFFFFFull, "too many values in one call");
    hipLaunchKernelGGL(kv4_to_f32_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream, mk_kv4_view(c), (int)n, k, v, (int)items, total);
    return mk_launch_status("kv4_to_f32");
}
