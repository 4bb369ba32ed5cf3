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
#include "mk_common.h"

namespace {

typedef __bf16 mk_b8 __attribute__((ext_vector_type(8)));
constexpr int MAX_SPLITS = 64;

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const mk_f4 a = *(const mk_f4 *)p, b = *(const mk_f4 *)(p + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
    } else {
        const mk_b8 a = *(const mk_b8 *)p;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)a[i];
    }
}

// Rows t of the call and the sequences they belong to.  cu [B + 1] (or null: T / B rows each); entries are taken within [0, T].
struct Seqs {
    const int32_t *cu;
    int T, B;
    __device__ __forceinline__ int at(int b) const { return cu ? min(max(cu[b], 0), T) : (int)((int64_t)T / B * b); }
    // sequence of row t, or -1: the last b with at(b) <= t, if t < at(b + 1)
    __device__ __forceinline__ int of_row(int t) const {
        if (!cu) return t / (T / B);
        int lo = 0, hi = B;  // at(lo) <= t < at(hi), once both hold
        if (t < at(0) || t >= at(B)) return -1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (at(mid) <= t) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

struct Kv4 {
    uint8_t *kq, *ks, *vq, *vs;
    uint16_t *kr;
    int32_t *lens;
    int B, nkv, dk, rope, dv, cap;
};

// ------------------------------------------------------------------------------------------------------------ append

// One wave: 64 items of a row of the call.  An item is 8 values: nkv * dk / 8 of K, nkv * dv / 8 of V, rope / 8 of the K tail.
// dk and dv are multiples of 32, so a block of 32 values is an aligned quad of lanes.
template <typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 c, Seqs s, const T *__restrict__ k_rows, size_t k_stride, const T *__restrict__ v_rows,
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
        if (is_v) load8(v_rows + (size_t)t * v_stride + (size_t)h * c.dv + d, v);
        else load8(k_rows + (size_t)t * k_stride + (size_t)h * (c.dk + c.rope) + d, v);
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
        load8(k_rows + (size_t)t * k_stride + c.dk + d, v);
        mk_b8 o;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = (__bf16)v[i];
        *(mk_b8 *)(c.kr + ((size_t)b * c.cap + pos) * c.rope + d) = o;
    }
}

__global__ __launch_bounds__(256) void kv4_advance_kernel(Kv4 c, Seqs s, int fresh) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < c.B) c.lens[b] = (fresh ? 0 : c.lens[b]) + max(s.at(b + 1) - s.at(b), 0);
}

// ------------------------------------------------------------------------------------------------------------ to_f32

// One thread: 8 values of K or V of (sequence, position, head); positions a sequence does not hold are zero.
__global__ __launch_bounds__(256) void kv4_to_f32_kernel(Kv4 c, int n, float *__restrict__ k, float *__restrict__ v, int items, size_t total) {
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
        if (held) load8((const __bf16 *)(c.kr + ((size_t)b * c.cap + pos) * c.rope + d), o);
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

// --------------------------------------------------------------------------------------------------- attention: any width

struct AttnArgs {
    const void *q;
    size_t q_stride;
    void *out;        // [T][nh][dv]
    float *po;        // partial sums [split][T * nh][dv], unnormalized
    float *pm, *pl;   // their maxima (of s * log2 e) and sums [split][T * nh]
    int nh, n_splits;
    float scale_log2; // scale * log2(e)
};

// positions a row may see: 0 ..= the returned one; -1: none; cap and beyond: the cache does not hold them all
__device__ __forceinline__ int64_t row_limit(const Kv4 &c, const Seqs &s, int b, int t) { return (int64_t)c.lens[b] - (s.at(b + 1) - t); }

template <typename T> __device__ __forceinline__ void store1(void *out, size_t i, float v) {
    if constexpr (sizeof(T) == 4) ((float *)out)[i] = v;
    else ((__bf16 *)out)[i] = (__bf16)v;
}

constexpr int GT = 256;  // positions of a tile: one a thread

// One workgroup: (row, query head, split).  Scores: a thread takes a position of the tile.  Output: a thread takes 8 values (one
// dword) of V for every (256 / (dv / 8))-th position of the tile.  Every cache byte is read once per query head, so this is the
// form for widths that the matrix kernels below do not take.
template <typename T>
__global__ __launch_bounds__(256) void kv4_attn_any_kernel(Kv4 c, Seqs s, AttnArgs a) {
    __shared__ float q_l[512 + 64], p_l[GT], red_l[8], acc_l[256 * 9];
    const int t = blockIdx.x, h = blockIdx.y, split = blockIdx.z, tid = threadIdx.x;
    const int b = s.of_row(t);
    if (b < 0) return;
    const int hk = h / (a.nh / c.nkv), qw = c.dk + c.rope;
    const int64_t lim64 = row_limit(c, s, b, t);
    const bool beyond = lim64 >= c.cap;
    const int n = beyond ? 0 : (int)max(lim64 + 1, (int64_t)0);
    for (int i = tid; i < qw; i += 256) q_l[i] = (float)((const T *)a.q)[(size_t)t * a.q_stride + (size_t)h * qw + i];
    const int tiles = (n + GT - 1) / GT, per = (tiles + a.n_splits - 1) / a.n_splits;
    const int j0 = split * per * GT, j1 = min(n, j0 + per * GT);
    const size_t base = ((size_t)b * c.nkv + hk) * c.cap;
    const int cols = c.dv / 8, groups = 256 / cols, col = tid % cols, grp = tid / cols;
    float m = -INFINITY, l = 0.0f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = 0.0f;
    __syncthreads();
    for (int jt = j0; jt < j1; jt += GT) {
        const int j = jt + tid;
        float sc = -INFINITY;
        if (j < j1) {
            const uint8_t *kp = c.kq + (base + j) * (c.dk / 2), *ksp = c.ks + (base + j) * (c.dk / 32);
            float sum = 0.0f;
            for (int g = 0; g < c.dk / 32; g++) {
                float blk = 0.0f;
                for (int w = 0; w < 4; w++) {
                    const uint32_t code = *(const uint32_t *)(kp + g * 16 + w * 4);
#pragma unroll
                    for (int i = 0; i < 8; i++) blk = fmaf(mk_e2m1((code >> (4 * i)) & 15u), q_l[g * 32 + w * 8 + i], blk);
                }
                sum = fmaf(blk, mk_scale_from_byte(ksp[g]), sum);
            }
            for (int i = 0; i < c.rope; i++) sum = fmaf(__uint_as_float((uint32_t)c.kr[((size_t)b * c.cap + j) * c.rope + i] << 16), q_l[c.dk + i], sum);
            sc = sum * a.scale_log2;
        }
        float mx = mk_wave_max(sc);
        if ((tid & 63) == 0) red_l[tid >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(fmaxf(red_l[0], red_l[1]), fmaxf(red_l[2], red_l[3])), m);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float corr = exp2f(m - ref), p = j < j1 ? exp2f(sc - ref) : 0.0f;
        p_l[tid] = p;
        const float sum = mk_wave_sum(p);
        if ((tid & 63) == 0) red_l[4 + (tid >> 6)] = sum;
        __syncthreads();
        l = l * corr + ((red_l[4] + red_l[5]) + (red_l[6] + red_l[7]));
        m = mx;
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] *= corr;
        if (grp < groups) {
            const int nj = min(GT, j1 - jt);
            for (int i = grp; i < nj; i += groups) {
                const size_t row = base + jt + i;
                const uint32_t code = *(const uint32_t *)(c.vq + row * (c.dv / 2) + col * 4);
                const float w = p_l[i] * mk_scale_from_byte(c.vs[row * (c.dv / 32) + col / 4]);
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] = fmaf(mk_e2m1((code >> (4 * e)) & 15u), w, acc[e]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; i++) acc_l[tid * 9 + i] = acc[i];
    __syncthreads();
    for (int d = tid; d < c.dv; d += 256) {
        float o = 0.0f;
        for (int g = 0; g < groups; g++) o += acc_l[(g * cols + d / 8) * 9 + d % 8];
        const size_t row = (size_t)t * a.nh + h;
        if (a.n_splits > 1) a.po[((size_t)split * s.T * a.nh + row) * c.dv + d] = o;
        else store1<T>(a.out, row * c.dv + d, beyond ? __builtin_nanf("") : n == 0 || l == 0.0f ? 0.0f : o / l);
    }
    if (a.n_splits > 1 && tid == 0) {
        a.pm[(size_t)split * s.T * a.nh + (size_t)t * a.nh + h] = m;
        a.pl[(size_t)split * s.T * a.nh + (size_t)t * a.nh + h] = beyond ? __builtin_nanf("") : l;
    }
}

// The splits' partial results of one (row, head): weights 2^(m_s - max), one division.
template <typename T>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Seqs s, AttnArgs a, int dv) {
    const size_t rows = (size_t)s.T * a.nh, row = blockIdx.x;
    if (s.of_row((int)(row / a.nh)) < 0) return;
    float mx = -INFINITY, den = 0.0f;
    for (int i = 0; i < a.n_splits; i++) mx = fmaxf(mx, a.pm[i * rows + row]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    for (int i = 0; i < a.n_splits; i++) den += a.pl[i * rows + row] * exp2f(a.pm[i * rows + row] - ref);
    for (int d = threadIdx.x; d < dv; d += 256) {
        float num = 0.0f;
        for (int i = 0; i < a.n_splits; i++) num += a.po[(i * rows + row) * dv + d] * exp2f(a.pm[i * rows + row] - ref);
        store1<T>(a.out, row * dv + d, den == 0.0f ? 0.0f : num / den);
    }
}

int splits_for(size_t T, size_t nh, size_t cap) {
    const size_t tiles = (cap + GT - 1) / GT, have = T * nh;
    size_t n = (1024 + have - 1) / have;
    n = n < tiles ? n : tiles;
    n = n < MAX_SPLITS ? n : MAX_SPLITS;
    return (int)(n ? n : 1);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_cache(const mk_kv4_cache *c) {
    MK_REQUIRE(c && c->kq && c->ks && c->vq && c->vs && c->lens && (c->kr || c->rope == 0), "null pointer");
    MK_REQUIRE(c->B >= 1 && c->B <= 65535 && c->nkv >= 1 && c->nkv <= 65535, "bad sequence or head count");
    MK_REQUIRE(c->dk >= 32 && c->dk <= 512 && c->dk % 32 == 0 && c->dv >= 32 && c->dv <= 512 && c->dv % 32 == 0, "K and V widths must be multiples of 32 up to 512");
    MK_REQUIRE(c->rope % 8 == 0 && c->rope <= 64, "the shared K tail must be a multiple of 8 up to 64");
    MK_REQUIRE(c->cap >= 1 && c->cap <= 0x7FFFFFull, "capacity out of range (at most 8388607 positions)");
    MK_REQUIRE(aligned16(c->kq) && aligned16(c->vq) && aligned16(c->kr) && aligned16(c->ks) && aligned16(c->vs), "cache arrays must be 16-byte aligned");
    return MK_OK;
}
Kv4 view(const mk_kv4_cache *c) {
    return Kv4{c->kq, c->ks, c->vq, c->vs, c->kr, c->lens, (int)c->B, (int)c->nkv, (int)c->dk, (int)c->rope, (int)c->dv, (int)c->cap};
}
int check_rows(const mk_kv4_cache *c, int dtype, size_t T, const int32_t *cu) {
    MK_REQUIRE(dtype == MK_F32 || dtype == MK_BF16, "dtype must be MK_F32 or MK_BF16");
    MK_REQUIRE(T <= 0x3FFFFF, "at most 4194303 rows per call");
    MK_REQUIRE(cu || T % c->B == 0, "without cu every sequence has the same number of rows");
    return MK_OK;
}

}  // namespace

extern "C" int mk_dev_kv4_append(const mk_kv4_cache *c, int dtype, const void *k_rows, size_t k_stride, const void *v_rows, size_t v_stride, size_t T,
                                 const int32_t *cu, int fresh, void *stream) {
    int st = check_cache(c);
    if (st != MK_OK || (st = check_rows(c, dtype, T, cu)) != MK_OK) return st;
    MK_REQUIRE(T == 0 || (k_rows && v_rows), "null pointer");
    MK_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0 && aligned16(k_rows) && aligned16(v_rows), "rows must be 16-byte aligned, their strides multiples of 8 values");
    MK_REQUIRE(T <= 1 || (k_stride >= c->nkv * (c->dk + c->rope) && v_stride >= c->nkv * c->dv), "a row stride is shorter than a row");
    const Seqs s{cu, (int)T, (int)c->B};
    const Kv4 v = view(c);
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
    int st = check_cache(c);
    if (st != MK_OK) return st;
    MK_REQUIRE(n <= c->cap, "more positions than the cache holds");
    if (n == 0) return MK_OK;
    MK_REQUIRE(k && v && aligned16(k) && aligned16(v), "outputs must be 16-byte aligned");
    const size_t items = (c->dk + c->rope + c->dv) / 8, total = c->B * n * c->nkv * items;
    MK_REQUIRE((total + 255) / 256 <= 0x7FFFFFFFull, "too many values in one call");
    hipLaunchKernelGGL(kv4_to_f32_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream, view(c), (int)n, k, v, (int)items, total);
    return mk_launch_status("kv4_to_f32");
}

extern "C" size_t mk_kv4_attn_workspace_bytes(const mk_kv4_cache *c, size_t T, size_t nh) {
    if (!c || !T || !nh) return 256;
    const size_t n = splits_for(T, nh, c->cap);
    return n <= 1 ? 256 : align_up(n * T * nh * c->dv * 4, 256) + 2 * align_up(n * T * nh * 4, 256);
}

extern "C" int mk_dev_kv4_attn(const mk_kv4_cache *c, int dtype, const void *q, size_t q_stride, size_t T, const int32_t *cu, size_t nh, float scale,
                               size_t max_len, void *workspace, void *out, void *stream) {
    int st = check_cache(c);
    if (st != MK_OK || (st = check_rows(c, dtype, T, cu)) != MK_OK) return st;
    MK_REQUIRE(nh >= 1 && nh <= 65535 && nh % c->nkv == 0, "the query heads must be a multiple of the kv heads");
    if (T == 0) return MK_OK;
    MK_REQUIRE(q && out && workspace, "null pointer");
    MK_REQUIRE(q_stride % 8 == 0 && aligned16(q) && aligned16(out) && ((uintptr_t)workspace & 255) == 0,
               "q and out must be 16-byte, the workspace 256-byte aligned, the query stride a multiple of 8 values");
    MK_REQUIRE(T == 1 || q_stride >= nh * (c->dk + c->rope), "the query stride is shorter than a token's heads");
    MK_REQUIRE(T * nh <= 0x7FFFFFFFull, "too many query rows in one call");
    (void)max_len;
    AttnArgs a;
    a.q = q, a.q_stride = q_stride, a.out = out, a.nh = (int)nh, a.scale_log2 = scale * 1.44269504088896340736f;
    a.n_splits = splits_for(T, nh, c->cap);
    uint8_t *w = (uint8_t *)workspace;
    a.po = (float *)w;
    w += align_up((size_t)a.n_splits * T * nh * c->dv * 4, 256);
    a.pm = (float *)w;
    w += align_up((size_t)a.n_splits * T * nh * 4, 256);
    a.pl = (float *)w;
    const Seqs s{cu, (int)T, (int)c->B};
    const Kv4 v = view(c);
    hipStream_t hs = (hipStream_t)stream;
    const dim3 grid((unsigned)T, (unsigned)nh, (unsigned)a.n_splits);
    if (dtype == MK_F32) hipLaunchKernelGGL(kv4_attn_any_kernel<float>, grid, dim3(256), 0, hs, v, s, a);
    else hipLaunchKernelGGL(kv4_attn_any_kernel<__bf16>, grid, dim3(256), 0, hs, v, s, a);
    if ((st = mk_launch_status("kv4_attn_any")) != MK_OK) return st;
    if (a.n_splits > 1) {
        if (dtype == MK_F32) hipLaunchKernelGGL(kv4_merge_kernel<float>, dim3((unsigned)(T * nh)), dim3(256), 0, hs, s, a, (int)c->dv);
        else hipLaunchKernelGGL(kv4_merge_kernel<__bf16>, dim3((unsigned)(T * nh)), dim3(256), 0, hs, s, a, (int)c->dv);
        return mk_launch_status("kv4_merge");
    }
    return MK_OK;
}
