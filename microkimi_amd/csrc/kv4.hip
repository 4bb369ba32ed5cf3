// A KV cache held in 4 bits (MXFP4: e2m1 nibbles, an e8m0 byte per 32 values), for a batch of sequences (attention: kv4_attn.hip).
//
//   append   rows of every sequence behind the positions it holds; K and V per kv head as MXFP4, an optional K tail of `rope`
//            values shared by the heads (taken from head 0) as bfloat16
//   to_f32   the values the cache stands for
//
// Quantization of a block: e = the smallest exponent with 6 * 2^e >= max|x|, clamped to [-127, 125]; the nearest level, upwards at
// a midpoint (the rule of the MXFP4 codec); NaN becomes 0 and what lies beyond 6 * 2^125 saturates, so that the cache holds
// finite values only: a position that a row may not see has weight 0, and 0 times a finite value is 0.
#include "mk_mixer.h"

namespace {

// ------------------------------------------------------------------------------------------------------------ append

// Positions held after the rows [first, last) of a call; far beyond every capacity the count stays where it is.
__device__ __forceinline__ int advanced(int held, int n) { return (int)min((int64_t)held + max(n, 0), (int64_t)1 << 30); }

// Two rows a wave: 6340 rows of 2048 values 12.3 us (four rows the same, one row 14.8), 16 rows of one token 5.0 us (four rows 6.8, one 3.8).
// A push of 16 tokens with the launch that advances lens: 5.3 us in a graph.
constexpr int APPEND_ROWS = 2;

// One wave: 64 items of ROWS rows of the call.  An item is 8 values: nkv * dk / 8 of K, nkv * dv / 8 of V, rope / 8 of the K tail.
// dk and dv are multiples of 32, so a block of 32 values is an aligned quad of lanes.  Levels come from v_cvt_scalef32_pk_fp4_f32,
// which rounds a midpoint to the even code: half of the midpoints go down.  With the lowest mantissa bit set first a midpoint is just
// above itself, and no other value reaches or passes one (their lowest bit is clear), so every midpoint goes up.
// When `fresh`, no row reads lens, and the last workgroup writes them; otherwise kv4_advance_kernel does behind this one.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void kv4_append_kernel(MkKv4 c, MkSeqs s, const T *__restrict__ k_rows, size_t k_stride, const T *__restrict__ v_rows,
                                                         size_t v_stride, int fresh, int waves_per_row) {
    if (fresh && blockIdx.x == gridDim.x - 1) {
        for (int b = threadIdx.x; b < c.B; b += 256) c.lens[b] = advanced(0, s.at(b + 1) - s.at(b));
        return;
    }
    const int w = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int t0 = w / waves_per_row * ROWS;
    if (t0 >= s.T) return;
    const int item = (w % waves_per_row) * 64 + (threadIdx.x & 63);
    const int nk = c.nkv * c.dk / 8, nv = c.nkv * c.dv / 8;
    const bool coded = item < nk + nv, is_v = coded && item >= nk, tail = !coded && item < nk + nv + c.rope / 8;
    const int width = is_v ? c.dv : c.dk, e = (is_v ? item - nk : item) * 8;
    const int h = coded ? e / width : 0, d = coded ? e - h * width : (item - nk - nv) * 8;
    const T *src = is_v ? v_rows + (size_t)h * c.dv + d : k_rows + (coded ? (size_t)h * (c.dk + c.rope) + d : (size_t)c.dk + d);
    const size_t stride = is_v ? v_stride : k_stride;
    float v[ROWS][8];  // every row is asked for before the first sequence is looked up
    if (coded || tail) {
#pragma unroll
        for (int r = 0; r < ROWS; r++) mk_load8(src + (size_t)min(t0 + r, s.T - 1) * stride, v[r]);
    }
    int b = -1, first = 0, next = 0, held = 0;
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int t = t0 + r;
        if (b < 0 || t >= next) {
            b = t < s.T ? s.of_row(t) : -1;
            if (b >= 0) first = s.at(b), next = s.at(b + 1), held = fresh ? 0 : min(c.lens[b], 1 << 30);
        }
        const int pos = held + t - first;
        if (b >= 0 && pos >= 0 && pos < c.cap) {
            if (coded) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[r][i]));
                m = fmaxf(m, mk_dpp<0xB1>(m));
                m = fmaxf(m, mk_dpp<0x4E>(m));
                const uint32_t bits = __float_as_uint(m);
                int ex = (int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) > 0x400000u ? 1 : 2);
                ex = max(-127, min(125, ex));
                const float inv = mk_scale_from_byte((uint32_t)(127 - ex));
                float a[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = v[r][i] == v[r][i] ? (v[r][i] + 0.0f) * inv : 0.0f;  // (-0 becomes 0; a negative value that underflows keeps its sign)
                    a[i] = __uint_as_float(__float_as_uint(x) | 1u);
                }
                uint32_t code = 0;
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, a[0], a[1], 1.0f, 0);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, a[2], a[3], 1.0f, 1);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, a[4], a[5], 1.0f, 2);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, a[6], a[7], 1.0f, 3);
                const size_t row = ((size_t)b * c.nkv + h) * c.cap + pos;
                uint8_t *q = is_v ? c.vq : c.kq, *sc = is_v ? c.vs : c.ks;
                *(uint32_t *)(q + row * (width / 2) + d / 2) = code;
                if ((item & 3) == 0) sc[row * (width / 32) + d / 32] = (uint8_t)(ex + 127);
            } else if (tail) {
                mk_b8 o;
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = (__bf16)v[r][i];
                *(mk_b8 *)(c.kr + ((size_t)b * c.cap + pos) * c.rope + d) = o;
            }
        }
    }
}

__global__ __launch_bounds__(256) void kv4_advance_kernel(MkKv4 c, MkSeqs s, int fresh) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < c.B) c.lens[b] = advanced(fresh ? 0 : c.lens[b], s.at(b + 1) - s.at(b));
}

// ------------------------------------------------------------------------------------------------------------ to_f32

// A thread: 4 values (an item of a position's K or V rows) of SNAP positions of a sequence, so that a wave stores 1 KiB in a row; positions
// a sequence does not hold are zero.  HBM-bound: 1500 positions of 96 heads of 192 + 128 (184 MB written) 32 us, 5.8 TB/s (with two and
// four items a thread 34.5 and 37.4 us); four sequences of 2048 positions of 8 heads of 128 + 128 13.0 us.
constexpr int SNAP = 4;

__global__ __launch_bounds__(256) void kv4_to_f32_kernel(MkKv4 c, int n, int parts, float *__restrict__ k, float *__restrict__ v) {
    const int b = blockIdx.y, p0 = blockIdx.x / parts * SNAP, item = blockIdx.x % parts * 256 + threadIdx.x;
    const int len = c.lens[b], wk = c.dk + c.rope, nk = c.nkv * wk / 4, nv = c.nkv * c.dv / 4;
    if (item >= nk + nv) return;
    const bool is_v = item >= nk;
    const int e = (is_v ? item - nk : item) * 4, across = is_v ? c.dv : wk, h = e / across, d = e - h * across;
    const bool tail = !is_v && d >= c.dk;
    const int width = is_v ? c.dv : c.dk;
    const size_t at = ((size_t)b * c.nkv + h) * c.cap + p0;
    const uint8_t *codes = (is_v ? c.vq : c.kq) + at * (width / 2) + d / 2, *scales = (is_v ? c.vs : c.ks) + at * (width / 32) + d / 32;
    float *dst = (is_v ? v : k) + ((size_t)b * n + p0) * c.nkv * across + e;
    mk_f4 o[SNAP];
    if (tail) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int p = 0; p < SNAP; p++) {
            o[p] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (p0 + p < min(len, n)) {
                const b4 x = *(const b4 *)(c.kr + ((size_t)b * c.cap + p0 + p) * c.rope + d - c.dk);
                o[p] = mk_f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
            }
        }
    } else {
        uint32_t code[SNAP], byte[SNAP];
#pragma unroll
        for (int p = 0; p < SNAP; p++) {
            code[p] = byte[p] = 0;
            if (p0 + p < min(len, n)) code[p] = *(const uint16_t *)(codes + (size_t)p * (width / 2)), byte[p] = scales[(size_t)p * (width / 32)];
        }
#pragma unroll
        for (int p = 0; p < SNAP; p++) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            const float sc = mk_scale_from_byte(byte[p]);
            const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[p], 1.0f, 0), y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[p], 1.0f, 1);
            o[p] = mk_f4{x[0] * sc, x[1] * sc, y[0] * sc, y[1] * sc};
        }
    }
#pragma unroll
    for (int p = 0; p < SNAP; p++) {
        if (p0 + p < n) __builtin_nontemporal_store(o[p], (mk_f4 *)(dst + (size_t)p * c.nkv * across));
    }
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
        const size_t grid = ((T + APPEND_ROWS - 1) / APPEND_ROWS * wpr + 3) / 4 + (fresh ? 1 : 0);
        if (dtype == MK_F32)
            hipLaunchKernelGGL((kv4_append_kernel<float, APPEND_ROWS>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, v, s, (const float *)k_rows, k_stride,
                               (const float *)v_rows, v_stride, fresh, (int)wpr);
        else
            hipLaunchKernelGGL((kv4_append_kernel<__bf16, APPEND_ROWS>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, v, s, (const __bf16 *)k_rows,
                               k_stride, (const __bf16 *)v_rows, v_stride, fresh, (int)wpr);
        if ((st = mk_launch_status("kv4_append")) != MK_OK || fresh) return st;
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
    const size_t parts = (c->nkv * (c->dk + c->rope + c->dv) / 4 + 255) / 256, grid = (n + SNAP - 1) / SNAP * parts;
    MK_REQUIRE(grid <= MAX_GROUPS, "too many values in one call");
    hipLaunchKernelGGL(kv4_to_f32_kernel, dim3((unsigned)grid, (unsigned)c->B), dim3(256), 0, (hipStream_t)stream, mk_kv4_view(c), (int)n, (int)parts, k, v);
    return mk_launch_status("kv4_to_f32");
}
