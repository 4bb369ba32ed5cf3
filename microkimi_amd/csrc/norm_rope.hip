// RMS norm of every query and key head with the rotation of its position, one pass over the rows.
//
//   r = x / sqrt(mean(x^2) + eps) * w        per head row of hd values (w: one row of weights for the queries, one for the keys)
//   (a, b) -> (a c - b s, a s + b c)         on the rot values from rot_at on; (a, b) = (2 i, 2 i + 1) or (i, i + rot / 2),
//                                            c, s = table row of the token's position, entry i
//
// Everything between the load and the store is f32; a bfloat16 result is rounded once.  A row of hd values lies in LPR
// lanes, 8 values (one or two 16-byte loads) each: the sum of squares is log2(LPR) exchanges, a pair (i, i + rot / 2) one
// exchange per value.  A group of LPR lanes keeps the token's table values and the weights in registers and walks its heads.
// HBM-bound from some hundred tokens on (8192 tokens of 64 + 8 bfloat16 heads of 128: 62 us, 4.9 TB/s, a large copy 5.1); a
// single token is the launch (3.7 us).
#include "mk_mixer.h"

namespace {

__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    *(mk_f4 *)p = mk_f4{v[0], v[1], v[2], v[3]};
    *(mk_f4 *)(p + 4) = mk_f4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(__bf16 *p, const float (&v)[8]) {
    mk_b8 a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (__bf16)v[i];
    *(mk_b8 *)p = a;
}

struct NormRopeArgs {
    const void *q, *k;
    void *qo, *ko;
    size_t qs, ks, qos, kos;  // values from one token's row to the next
    const float *wq, *wk, *cos, *sin;
    const int32_t *pos;
    int n_pos, nh, nkv, hd, rot, rot_at, norm, parts, apart;  // apart: the shares of the queries and those of the keys are workgroups of their own
    float eps;
};

// One workgroup: a token, or one of `parts` equal shares of its query heads and of its key heads.
template <typename T, int LPR, bool HALVES>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
    constexpr int GROUPS = 256 / LPR;
    const int per_token = a.apart ? 2 * a.parts : a.parts, t = blockIdx.x / per_token, share = blockIdx.x - t * per_token;
    const int part = share % a.parts;
    const int l = threadIdx.x % LPR, e0 = l * 8, grp = threadIdx.x / LPR;
    const bool live = e0 < a.hd;
    const int p = a.pos ? a.pos[t] : 0;
    float c[8], s[8];
    const int ri = e0 - a.rot_at;
    const bool turned = a.rot && live && ri >= 0 && ri < a.rot, upper = HALVES && ri >= a.rot / 2;
    const int me = threadIdx.x & 63, mate = HALVES && turned ? me + (upper ? -(a.rot / 16) : a.rot / 16) : me;
    bool have = false;
    auto side = [&](const T *src, T *dst, const float *wp, int heads) {
        const int per = (heads + a.parts - 1) / a.parts, h1 = min(heads, (part + 1) * per);
        for (int h0 = part * per; h0 < h1; h0 += GROUPS) {
            const int h = h0 + grp;
            float x[8];
            if (live && h < h1) {
                mk_load8(src + (size_t)h * a.hd + e0, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = 0.0f;
            }
            if (!have) {  // (behind the first rows' loads: the position, and with it the table, is a chain of two)
                have = true;
#pragma unroll
                for (int i = 0; i < 8; i++) c[i] = 1.0f, s[i] = 0.0f;
                if (turned && p >= 0) {
                    if (p < a.n_pos) {
                        const size_t row = (size_t)p * (a.rot / 2);
                        if (HALVES) {
                            const int i0 = upper ? ri - a.rot / 2 : ri;
                            mk_load8(a.cos + row + i0, c);
                            mk_load8(a.sin + row + i0, s);
                        } else {
                            const mk_f4 cv = *(const mk_f4 *)(a.cos + row + ri / 2), sv = *(const mk_f4 *)(a.sin + row + ri / 2);
#pragma unroll
                            for (int i = 0; i < 4; i++) c[i] = cv[i], s[i] = sv[i];
                        }
                    } else {  // the table has no such position: the rotated values are NaN
#pragma unroll
                        for (int i = 0; i < 8; i++) c[i] = __builtin_nanf(""), s[i] = __builtin_nanf("");
                    }
                    if (HALVES && !upper) {  // lower half: mine * c - partner * s; upper half: mine * c + partner * s
#pragma unroll
                        for (int i = 0; i < 8; i++) s[i] = -s[i];
                    }
                }
            }
            if (p < 0) return;  // a padding row
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = 1.0f;
            if (live && wp) mk_load8(wp + e0, w);
            float f = 1.0f;
            if (a.norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                for (int off = 1; off < LPR; off <<= 1) ss += __shfl_xor(ss, off, MK_WAVE);
                f = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
            }
            float y[8], o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x[i] * f * w[i];
            if (HALVES && a.rot) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float other = __shfl(y[i], mate, MK_WAVE);
                    o[i] = turned ? fmaf(y[i], c[i], other * s[i]) : y[i];
                }
            } else if (!HALVES && turned) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    o[2 * i] = fmaf(y[2 * i], c[i], -(y[2 * i + 1] * s[i]));
                    o[2 * i + 1] = fmaf(y[2 * i], s[i], y[2 * i + 1] * c[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = y[i];
            }
            if (live && h < h1) store8(dst + (size_t)h * a.hd + e0, o);
        }
    };
    if (!a.apart || share < a.parts) side((const T *)a.q + (size_t)t * a.qs, (T *)a.qo + (size_t)t * a.qos, a.wq, a.nh);
    if (!a.apart || share >= a.parts) side((const T *)a.k + (size_t)t * a.ks, (T *)a.ko + (size_t)t * a.kos, a.wk, a.nkv);
}

template <typename T, int LPR>
int launch(NormRopeArgs a, size_t n_tok, int halves, hipStream_t st) {
    constexpr int GROUPS = 256 / LPR;
    // From 1024 tokens on a token is one workgroup: its heads share the table's row and the weights, and the device is full (8192 tokens of
    // 64 + 8 bfloat16 heads of 128: 62 us, with one head a group of lanes 77 us).  Below, every group of lanes gets one head (777
    // tokens of 96 + 96 f32 heads of 192: 52 us, as one workgroup a token 59 us).  Nothing between the two was measured.
    a.apart = n_tok < 1024;
    a.parts = a.apart ? ((a.nh > a.nkv ? a.nh : a.nkv) + GROUPS - 1) / GROUPS : 1;
    const size_t grid = n_tok * (size_t)a.parts * (a.apart ? 2 : 1);
    MK_REQUIRE(grid <= MAX_GROUPS, "too many rows in one call");
    if (halves)
        hipLaunchKernelGGL((norm_rope_kernel<T, LPR, true>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((norm_rope_kernel<T, LPR, false>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return mk_launch_status("norm_rope");
}

template <typename T>
int launch_width(const NormRopeArgs &a, size_t n_tok, int halves, hipStream_t st) {
    if (a.hd <= 64) return launch<T, 8>(a, n_tok, halves, st);
    if (a.hd <= 128) return launch<T, 16>(a, n_tok, halves, st);
    if (a.hd <= 256) return launch<T, 32>(a, n_tok, halves, st);
    return launch<T, 64>(a, n_tok, halves, st);
}

}  // namespace

extern "C" int mk_dev_qk_norm_rope(int dtype, const void *q, size_t q_stride, size_t nh, const void *k, size_t k_stride, size_t nkv, size_t T,
                                   size_t hd, int norm, const float *wq, const float *wk, float eps, const float *cos, const float *sin,
                                   size_t n_pos, const int32_t *pos, size_t rot, size_t rot_at, int halves, void *q_out, size_t q_out_stride,
                                   void *k_out, size_t k_out_stride, void *stream) {
    MK_REQUIRE(dtype == MK_F32 || dtype == MK_BF16, "dtype must be MK_F32 or MK_BF16");
    MK_REQUIRE(T == 0 || ((nh == 0 || (q && q_out)) && (nkv == 0 || (k && k_out))), "null pointer");
    MK_REQUIRE(nh <= 65535 && nkv <= 65535 && T <= 0x7FFFFFFFull && n_pos <= 0x7FFFFFFFull, "size out of range");
    MK_REQUIRE(hd >= 8 && hd <= 512 && hd % 8 == 0, "head width must be a multiple of 8 up to 512");
    MK_REQUIRE(rot % 16 == 0 && rot_at % 8 == 0 && rot_at <= hd && rot <= hd - rot_at, "rot must be a multiple of 16, rot_at of 8, both inside the head");
    MK_REQUIRE(T == 0 || rot == 0 || (cos && sin && pos), "a rotation needs the tables and the positions");
    MK_REQUIRE(q_stride % 8 == 0 && k_stride % 8 == 0 && q_out_stride % 8 == 0 && k_out_stride % 8 == 0, "token strides must be multiples of 8 values");
    MK_REQUIRE((nh == 0 || T <= 1 || (q_stride >= nh * hd && q_out_stride >= nh * hd)) &&
                   (nkv == 0 || T <= 1 || (k_stride >= nkv * hd && k_out_stride >= nkv * hd)),
               "a token stride is shorter than a token's heads");
    MK_REQUIRE(mk_aligned16(q) && mk_aligned16(k) && mk_aligned16(q_out) && mk_aligned16(k_out) && mk_aligned16(wq) && mk_aligned16(wk) && mk_aligned16(cos) && mk_aligned16(sin),
               "pointers must be 16-byte aligned");
    if (T == 0 || nh + nkv == 0) return MK_OK;
    NormRopeArgs a;
    a.q = q, a.k = k, a.qo = q_out, a.ko = k_out;
    a.qs = q_stride, a.ks = k_stride, a.qos = q_out_stride, a.kos = k_out_stride;
    a.wq = wq, a.wk = wk, a.cos = cos, a.sin = sin, a.pos = pos;
    a.n_pos = (int)n_pos, a.nh = (int)nh, a.nkv = (int)nkv, a.hd = (int)hd, a.rot = (int)rot, a.rot_at = (int)rot_at, a.norm = norm ? 1 : 0, a.eps = eps;
    return dtype == MK_F32 ? launch_width<float>(a, T, halves, (hipStream_t)stream) : launch_width<__bf16>(a, T, halves, (hipStream_t)stream);
}
