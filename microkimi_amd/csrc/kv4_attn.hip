// Attention over the 4-bit KV cache (kv4.hip writes it).
#include "mk_mixer.h"

namespace {

constexpr int MAX_SPLITS = 64;

// --------------------------------------------------------------------------------------------------- attention: any width

struct AttnArgs {
    const void *q;
    size_t q_stride;
    void *out;        // [T][nh][dv]
    float *po;        // partial sums [split][T * nh][dv], unnormalized
    float *pm, *pl;   // their maxima (of s * log2 e) and sums [split][T * nh]
    int nh, n_splits, chunk;  // chunk: positions of a split (the last one takes what is left)
    float scale_log2; // |scale| * log2(e)
    float sign;       // the scale's sign, taken by the query
};

// positions a row may see: 0 ..= the returned one; -1: none; cap and beyond: the cache does not hold them all
__device__ __forceinline__ int64_t row_limit(const MkKv4 &c, const MkSeqs &s, int b, int t) { return (int64_t)c.lens[b] - (s.at(b + 1) - t); }

// the end of a split's positions when there are n in all
__device__ __forceinline__ int chunk_end(const AttnArgs &a, int split, int n) { return split + 1 == a.n_splits ? n : min(n, (split + 1) * a.chunk); }

template <typename T> __device__ __forceinline__ void store1(void *out, size_t i, float v) {
    if constexpr (sizeof(T) == 4) ((float *)out)[i] = v;
    else ((__bf16 *)out)[i] = (__bf16)v;
}

constexpr int GT = 256;  // positions of a tile: one a thread

// One workgroup: (row, query head, split).  Scores: a thread takes a position of the tile.  Output: a thread takes 8 values (one
// dword) of V for every (256 / (dv / 8))-th position of the tile.  Every cache byte is read once per query head, so this is the
// form for widths that the matrix kernels below do not take (one token over 4096 positions, 16 heads to 2 kv heads, bfloat16: 42 us at 96 | 96, 63 at
// 192 | 128, 203 at 512 + 64 | 512; 64 rows 0.87, 1.41 and 4.49 ms).
template <typename T>
__global__ __launch_bounds__(256) void kv4_attn_any_kernel(MkKv4 c, MkSeqs s, AttnArgs a) {
    __shared__ float q_l[512 + 64], p_l[GT], red_l[8], acc_l[256 * 9];
    const int t = blockIdx.x, h = blockIdx.y, split = blockIdx.z, tid = threadIdx.x;
    const int b = s.of_row(t);
    if (b < 0) return;
    const int hk = h / (a.nh / c.nkv), qw = c.dk + c.rope;
    const int64_t lim64 = row_limit(c, s, b, t);
    const bool beyond = lim64 >= c.cap;
    const int n = beyond ? 0 : (int)max(lim64 + 1, (int64_t)0);
    for (int i = tid; i < qw; i += 256) q_l[i] = (float)((const T *)a.q)[(size_t)t * a.q_stride + (size_t)h * qw + i];
    const int j0 = split * a.chunk, j1 = chunk_end(a, split, n);
    if (a.n_splits > 1 && j0 >= j1) return;
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
            sc = sum * (a.sign * a.scale_log2);
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
        else store1<T>(a.out, row * c.dv + d, beyond ? __builtin_nanf("") : n == 0 ? 0.0f : o / l);
    }
    if (a.n_splits > 1 && tid == 0) {
        a.pm[(size_t)split * s.T * a.nh + (size_t)t * a.nh + h] = m;
        a.pl[(size_t)split * s.T * a.nh + (size_t)t * a.nh + h] = l;
    }
}

// ------------------------------------------------------------------------------- attention on the matrix cores, pieces
//
// Both kernels below compute S^T = K Q^T and O^T = V^T P^T: a query column (row of the call x head of the kv head's group) is a
// column n = lane % 16 of every tile, so its running maximum and sum live in that lane, and the scores of a tile, as the
// instruction returns them (rows 4 g + j, g = lane / 16), ARE the second product's operand once the positions of a 32-step are
// taken in the order {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3}: a sum over positions has no order of its own.  In the same way
// the sum over the K width takes the values (DK / 4) g .. of lane group g: a lane reads DK / 8 consecutive bytes of one
// position, which is one block (one scale byte) at DK = 128.
//
// 4-bit values become bfloat16 exactly (two significant bits, and the exponent of an f32), so the products are exact in f32.
// f32 queries enter as three bfloat16 terms (24 bits: every bit of the value).  A weight p of the softmax enters as P terms: three for
// f32 results, two for bfloat16 ones (17 bits, so that the result's own rounding, 2^-8 of it at most, is the only one that counts).  One term
// would cost a second whole rounding: a result with values of both signs shrinks with the sum of its weights' errors, which is why these
// do not average out (2.3e-3 against 1.7e-3 over 4096 positions).  With few columns the second term costs no time (bound by memory: one term 59.7, two 59.8
// us at 96 heads x 16384 positions), with many it does (512 rows behind 3584 positions: one term 165, two 200 us).
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float FAR = 1048576.0f;  // 2^20: weights up to this above the reference point are summed as they are

template <typename T> struct Terms;
template <> struct Terms<float> { static constexpr int Q = 3, P = 3; };
template <> struct Terms<__bf16> { static constexpr int Q = 1, P = 2; };

__device__ __forceinline__ mk_f4 mfma(mk_b8 a, mk_b8 b, mk_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// x as the sum of N bfloat16 terms, largest first
template <int N> __device__ __forceinline__ void split8(const float (&x)[8], mk_b8 (&t)[N]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int k = 0; k < N; k++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const __bf16 h = (__bf16)r[i];
            t[k][i] = h;
            if (k + 1 < N) r[i] -= (float)h;
        }
    }
}

// eight 4-bit values of a block with scale sc -> bfloat16
__device__ __forceinline__ mk_b8 fp4x8(uint32_t w, float sc) {
    const mk_b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1);
    const mk_b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3);
    return mk_b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The work of a workgroup: number `idx` in the list of (tile of CT columns, chunk of the context) of all sequences (a sequence with m rows
// and group G has m * G columns, and the chunks that its positions fill: what is not there takes no place in the list, so that the
// workgroups without work come last: between the others they took a third of the time of 32 ragged sequences).  Every wave finds it for itself.  false: past the end of the list.
__device__ __forceinline__ bool find_work(const MkKv4 &c, const MkSeqs &s, const AttnArgs &a, int G, int CT, int idx, int &b, int &tile, int &split) {
    if (s.B == 1) {
        b = 0;
        tile = idx / a.n_splits;
        split = idx - tile * a.n_splits;
        return tile < ((s.at(1) - s.at(0)) * G + CT - 1) / CT;
    }
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < s.B; b0 += 64) {
        const int mine = b0 + lane;
        int chunks = 1, n = 0;
        if (mine < s.B) {
            if (a.n_splits > 1) chunks = min((int)((min(max(c.lens[mine], 0), c.cap) + (int64_t)a.chunk - 1) / a.chunk), a.n_splits);
            n = (max(s.at(mine + 1) - s.at(mine), 0) * G + CT - 1) / CT * chunks;
        }
        int sum = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(sum, off, MK_WAVE);
            if (lane >= off) sum += o;
        }
        const int total = __shfl(sum, 63, MK_WAVE);
        if (idx < total) {
            const int l = __builtin_ctzll(__ballot(sum > idx));
            b = b0 + l;
            const int r = idx - __shfl(sum - n, l, MK_WAVE);
            chunks = max(__shfl(chunks, l, MK_WAVE), 1);
            tile = r / chunks;
            split = r - tile * chunks;
            return r >= 0 && r < __shfl(n, l, MK_WAVE);  // (sequences that overlap, which no cu should say, may pass 31 bits together)
        }
        idx -= total;
    }
    return false;
}

// A query column.
struct Column {
    int t, h, lim;  // row of the call, query head, last position it may see (-1: none)
    bool live, beyond;
};
__device__ __forceinline__ Column column(const MkKv4 &c, const MkSeqs &s, int G, int hk, int b, int idx) {
    Column o;
    const int first = s.at(b), m = max(s.at(b + 1) - first, 0), i = idx / G;
    o.live = i < m;
    o.t = first + i;
    o.h = hk * G + idx - i * G;
    const int64_t lim = (int64_t)c.lens[b] - m + i;
    o.beyond = o.live && lim >= c.cap;
    o.lim = o.live && !o.beyond && lim >= 0 ? (int)lim : -1;
    return o;
}
__device__ __forceinline__ int columns_max(int v) {  // over the 16 columns of the wave
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) v = max(v, __shfl_xor(v, off, MK_WAVE));
    return v;
}
__device__ __forceinline__ int columns_min(int v) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) v = min(v, __shfl_xor(v, off, MK_WAVE));
    return v;
}

// The query operand: step st of lane group g is values (DK / 4) g + 8 st .. of the K width, then (R / 4) g + 8 (st - NS) .. of the tail.
template <typename T, int DK, int R>
__device__ __forceinline__ void load_query(const AttnArgs &a, const Column &o, int g, mk_b8 (&qf)[DK / 32 + R / 32][Terms<T>::Q]) {
    constexpr int N = DK / 32 + R / 32;
    // (a column without a row reads row 0 and drops it: all loads are in flight together)
    const T *row = (const T *)a.q + (o.live ? (size_t)o.t * a.q_stride + (size_t)o.h * (DK + R) : 0);
    float x[N][8];
#pragma unroll
    for (int st = 0; st < N; st++) mk_load8(row + (st < DK / 32 ? DK / 4 * g + 8 * st : DK + R / 4 * g + 8 * (st - DK / 32)), x[st]);
#pragma unroll
    for (int st = 0; st < N; st++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[st][i] = o.live ? x[st][i] * a.sign : 0.0f;
        split8<Terms<T>::Q>(x[st], qf[st]);
    }
}

// ------------------------------------------------------------------------- few query columns: every wave its own positions
//
// Bound by memory: 96 heads over 16384 positions of 128 + 64 | 128, bfloat16 queries (216 MB): 48 us, 4.5 TB/s, and 4.8 us for the merge; 32
// sequences of 1 .. 16384 positions, 8 kv heads (99.7 MB) 24.4 + 4.4 us; 1024 positions of 96 heads 12.6 us, the rate of 96 compute
// units (eight waves instead of four: 11.6 us for 10.6).
//
// One workgroup: (tile of 16 query columns, kv head, chunk of the context), the heads fastest: neighbours in the grid, which go to
// the eight XCDs in turn, then have the same length (with the sequences fastest a long one's workgroups all met on one XCD:
// 75 us instead of 35 for 32 ragged sequences).  Its four waves take the chunk's steps of 32 positions
// in turn, straight from global memory into registers (no LDS, no barrier); at the end the four partial results meet in LDS.
//   K  lane (n, g): position n of 16, DK / 8 bytes from (DK / 4) g on: one load; a wave's load is 16 whole rows
//   V  lane (n, g): the DV / 16 values from (DV / 16) n on of its 8 positions; the values of one dimension at 8 positions are put
//      together with byte permutes and are the first operand of tile j = dimension (DV / 16) n + j
// A step's K registers are asked for again (for the next step) as soon as the scores are formed, its V registers as soon as they
// are converted: the loads fly over the other half of the step and no register is copied.  Addresses are a scalar base (the
// step) plus a lane offset that never changes.  A chunk's last step that is not whole is moved back to end with it; the
// positions it then sees twice, or that lie behind the sequence, are masked.
template <int BYTES> struct Raw;
template <> struct Raw<2> { typedef uint16_t type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<8> { typedef mk_u2 type; };
template <> struct Raw<16> { typedef mk_v4u type; };

template <typename V> __device__ __forceinline__ V ldg(const uint8_t *base, uint32_t off) {
    const MK_GLOBAL uint8_t *b = (const MK_GLOBAL uint8_t *)base;
    return *(const MK_GLOBAL V *)(b + off);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
template <typename P> __device__ __forceinline__ const uint8_t *uniform(const P *p) { return mk_uniform_ptr((const uint8_t *)p); }

template <int DK, int R> struct KStep {
    static constexpr int KL = DK == 256 ? 2 : 1;  // 16-byte loads
    typedef typename Raw<DK == 256 ? 16 : DK / 8>::type KT;
    KT k[2][KL];
    uint32_t ks[2];
    mk_b8 kr[2][R ? R / 32 : 1];
    // 32 positions from j on; kq, ks, kr: the rows of the head's position 0
    __device__ __forceinline__ void load(const uint8_t *kqp, const uint8_t *ksp, const uint8_t *krp, int j, int n, int g) {
        const uint8_t *kj = kqp + (size_t)j * (DK / 2), *sj = ksp + (size_t)j * (DK / 32), *rj = krp + (size_t)j * (R * 2);
        const uint32_t ko = n * (DK / 2) + g * (DK / 8), so = n * (DK / 32) + (DK == 256 ? 2 * g : DK == 128 ? g : g / 2), ro = n * (R * 2) + g * (R / 2);
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int i = 0; i < KL; i++) k[s][i] = ldg<KT>(kj, ko + (8 * DK * s + 16 * i));
            if constexpr (DK == 256) ks[s] = ldg<uint16_t>(sj, so + DK / 2 * s);
            else ks[s] = ldg<uint8_t>(sj, so + DK / 2 * s);
#pragma unroll
            for (int i = 0; i < R / 32; i++) kr[s][i] = ldg<mk_b8>(rj, ro + (32 * R * s + 16 * i));
        }
    }
    __device__ __forceinline__ uint32_t word(int s, int i) const {
        if constexpr (DK == 256) return k[s][i / 4][i % 4];
        else return k[s][0][i];
    }
    __device__ __forceinline__ float scale(int s, int st) const {
        if constexpr (DK == 256) return scale_of(st < 4 ? ks[s] & 255u : ks[s] >> 8);
        else return scale_of(ks[s]);
    }
};

template <int DV> struct VStep {
    typedef typename Raw<DV / 32>::type VT;
    typedef typename Raw<DV == 64 ? 4 : DV / 32>::type VL;
    VL v[8];
    uint32_t vs[8];  // (whole registers: a byte of a packed one would be waited for at its load)
    __device__ __forceinline__ void load(const uint8_t *vqp, const uint8_t *vsp, int j, int n, int g) {
        const uint8_t *vj = vqp + (size_t)j * (DV / 2), *sj = vsp + (size_t)j * (DV / 32);
        const uint32_t vo = 4 * g * (DV / 2) + n * (DV / 32), so = 4 * g * (DV / 32) + n / (512 / DV);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int p = (i & 3) + 16 * (i >> 2);
            v[i] = ldg<VT>(vj, vo + p * (DV / 2));
            vs[i] = ldg<uint8_t>(sj, so + p * (DV / 32));
        }
    }
    __device__ __forceinline__ uint32_t word(int i, int w) const {
        if constexpr (DV == 256) return v[i][w];
        else return v[i];
    }
    // first operand of V^T for tile j: element i = value (DV / 16) n + j at the lane's position i
    __device__ __forceinline__ void tiles(mk_b8 (&vt)[DV / 16]) const {
        constexpr int W = DV / 32;  // pairs of values of a position
        uint32_t pr[8][W];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float sc = scale_of(vs[i]);
#pragma unroll
            for (int w = 0; w < (W + 3) / 4; w++) {
                const uint32_t d = word(i, w);
                pr[i][4 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 0));
                pr[i][4 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 1));
                if constexpr (W >= 4) {
                    pr[i][4 * w + 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 2));
                    pr[i][4 * w + 3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 3));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < DV / 16; j++) {
            mk_v4u o;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_amdgcn_perm(pr[2 * i + 1][j / 2], pr[2 * i][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
            vt[j] = __builtin_bit_cast(mk_b8, o);
        }
    }
};

template <typename T, int DK, int R, int DV>
__global__ __launch_bounds__(256, DK == 256 && sizeof(T) == 4 ? 1 : 2) void kv4_attn_few_kernel(MkKv4 c, MkSeqs s, AttnArgs a) {
    constexpr int NS = DK / 32, NR = R / 32, NT = DV / 16, QT = Terms<T>::Q, PT = Terms<T>::P, LD = DV + 4;
    __shared__ float o_l[4][16][LD], m_l[4][16], l_l[4][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % c.nkv, G = a.nh / c.nkv;
    int b, tile, split;
    if (!find_work(c, s, a, G, 16, blockIdx.x / c.nkv, b, tile, split)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    split = __builtin_amdgcn_readfirstlane(split);
    const Column col = column(c, s, G, hk, b, tile * 16 + n);
    const int top = __builtin_amdgcn_readfirstlane(columns_max(col.lim));
    const int low = __builtin_amdgcn_readfirstlane(columns_min(col.live ? col.lim : 0x7FFFFFFF));
    const int j0 = split * a.chunk, j1 = chunk_end(a, split, top + 1);
    if (a.n_splits > 1 && j0 >= j1) return;  // nothing here: the merge knows which chunks a row has

    float m = -INFINITY, l = 0.0f;
    mk_f4 o[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) o[j] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
    int j = j0 + 32 * wave;
    if (j < j1) {
        const size_t row0 = ((size_t)b * c.nkv + hk) * c.cap, kr0 = (size_t)b * c.cap;
        const uint8_t *kqp = uniform(c.kq + row0 * (DK / 2)), *ksp = uniform(c.ks + row0 * (DK / 32)), *vqp = uniform(c.vq + row0 * (DV / 2)),
                      *vsp = uniform(c.vs + row0 * (DV / 32)), *krp = R ? uniform(c.kr + kr0 * R) : nullptr;
        mk_b8 qf[NS + NR][QT];
        KStep<DK, R> ks;
        VStep<DV> vs;
        int at = max(min(j, j1 - 32), 0);  // (a cache has room for 32 positions at least)
        load_query<T, DK, R>(a, col, g, qf);
        ks.load(kqp, ksp, krp, at, n, g);
        vs.load(vqp, vsp, at, n, g);
        while (true) {
            const int nj = j + 128, nat = max(min(nj, j1 - 32), 0);
            // scores
            float sc[8];
#pragma unroll
            for (int ss = 0; ss < 2; ss++) {
                mk_f4 acc = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    const mk_b8 kf = fp4x8(ks.word(ss, st), ks.scale(ss, st));
#pragma unroll
                    for (int t = 0; t < QT; t++) acc = mfma(kf, qf[st][t], acc);
                }
#pragma unroll
                for (int st = 0; st < NR; st++)
#pragma unroll
                    for (int t = 0; t < QT; t++) acc = mfma(ks.kr[ss][st], qf[NS + st][t], acc);
#pragma unroll
                for (int i = 0; i < 4; i++) sc[4 * ss + i] = acc[i];
            }
            ks.load(kqp, ksp, krp, nat, n, g);  // (past the last step: that step again, so that the loads in flight are always the same)
            if (at < j || at + 31 > low) {  // positions seen before, or that some column does not see
                const int last = min(col.lim, j1 - 1);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int p = at + 4 * g + (i & 3) + 16 * (i >> 2);
                    if (p < j || p > last) sc[i] = -INFINITY;
                }
                if (at + 32 > j1) {  // a sequence shorter than a step: what lies behind it may hold any scale byte
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (at + 4 * g + (i & 3) + 16 * (i >> 2) >= j1) vs.vs[i] = 0;
                }
            }
            // weights against the reference point of the steps before; only where one of them is far above it (or there is none
            // yet) is the maximum looked for and what has been summed rescaled
            float p[8], sum;
            auto weigh = [&](float ref) {
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], a.scale_log2, -ref));
                sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            };
            weigh(m);
            if (__any(!(sum < FAR))) {
                float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
                mx = fmaxf(mk_rows_max(mx) * a.scale_log2, m);
                const float corr = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
                m = mx;
                l *= corr;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[t][i] *= corr;
                weigh(mx == -INFINITY ? 0.0f : mx);
            }
            l += sum;
            mk_b8 pf[PT], vt[NT];
            split8<PT>(p, pf);
            vs.tiles(vt);
            vs.load(vqp, vsp, nat, n, g);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < PT; k++) o[t] = mfma(vt[t], pf[k], o[t]);
            if (nj >= j1) break;
            at = nat;
            j = nj;
        }
        l = mk_rows_sum(l);
    }
    // the waves' partial results: lane (n, g) holds values NT (4 g + i) + t of column n
    if (g == 0) m_l[wave][n] = m, l_l[wave][n] = l;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < NT; t += 4) *(mk_f4 *)&o_l[wave][n][NT * (4 * g + i) + t] = mk_f4{o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]};
    __syncthreads();
    const int oc = threadIdx.x >> 4, od = (threadIdx.x & 15) * (DV / 16);  // 16 threads a column
    const Column out = column(c, s, G, hk, b, tile * 16 + oc);
    if (!out.live) return;
    float mw[4], mx = -INFINITY, den = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mx = fmaxf(mx, m_l[w][oc]);
    // (a query that is not finite gives NaN sums, whatever the maximum says)
    const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int w = 0; w < 4; w++) mw[w] = __builtin_amdgcn_exp2f(m_l[w][oc] - ref), den = fmaf(l_l[w][oc], mw[w], den);
    float r[DV / 16];
#pragma unroll
    for (int i = 0; i < DV / 16; i++) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) v = fmaf(o_l[w][oc][od + i], mw[w], v);
        r[i] = v;
    }
    const size_t row = (size_t)out.t * a.nh + out.h;
    if (a.n_splits > 1) {
        const size_t at = (size_t)split * s.T * a.nh + row;
        float *po = a.po + at * DV + od;
#pragma unroll
        for (int i = 0; i < DV / 16; i += 4) *(mk_f4 *)(po + i) = mk_f4{r[i], r[i + 1], r[i + 2], r[i + 3]};
        if (od == 0) a.pm[at] = mx, a.pl[at] = den;
    } else {
        const float inv = out.beyond ? __builtin_nanf("") : out.lim < 0 ? 0.0f : 1.0f / den;
#pragma unroll
        for (int i = 0; i < DV / 16; i++) store1<T>(a.out, row * DV + od + i, r[i] * inv);
    }
}

// ----------------------------------------------------------------------- many query columns: the workgroup shares K and V
//
// 512 rows behind 3584 positions, 96 heads of 128 + 64 | 128 in bfloat16 (121 GFLOP): 200 us, 605 TFLOP/s (a large library product:
// 1085); 244 us in a row of calls without pauses, when the card lowers its clock.  Operand reads from LDS (80 KB a step and workgroup) alone take
// 96 us, vector issue 95, the matrix cores 68 (49 without the weights' second term).  32 columns a wave would halve the reads, but 128 columns a
// workgroup leave 384 of them to 512 places.
//
// One workgroup: (tile of 64 query columns, 16 a wave; kv head; chunk of the context), 32 positions a step.  Waves 0 and 1 turn the K
// rows of 16 positions each into bfloat16 operands in LDS, waves 2 and 3 the V rows (as in the kernel above, so no transposed read
// is needed); every wave multiplies all of them with its columns.  Software pipeline of step h, one barrier a step:
//   scores of step h + 1 on the matrix cores, beside them the weights of step h on the vector units
//   O += V P of step h, beside it the operands of K of step h + 2 and of V of step h + 1; the bytes of the step after are asked for
// The statements stand in the order in which they are to be issued (sched_barrier keeps it): a matrix instruction runs for 16 cycles,
// in which the wave can issue what does not wait for it; operands are read from LDS three (scores) or two (outputs) of them ahead.
// A wave's share of a step: the K, or the V rows of 16 positions.  Positions past `last` are read as `last`.
template <int DK, int R> struct KQuarter {
    static constexpr int KL = DK == 256 ? 2 : 1;
    typedef typename Raw<DK == 256 ? 16 : DK / 8>::type KT;
    KT k[KL];
    uint32_t ks;
    mk_b8 kr[R ? R / 32 : 1];
    __device__ __forceinline__ void load(const uint8_t *kqp, const uint8_t *ksp, const uint8_t *krp, int j, int last, int n, int g) {
        const uint32_t p = min(j + n, last);
#pragma unroll
        for (int i = 0; i < KL; i++) k[i] = ldg<KT>(kqp, p * (DK / 2) + (g * (DK / 8) + 16 * i));
        if constexpr (DK == 256) ks = ldg<uint16_t>(ksp, p * (DK / 32) + 2 * g);
        else ks = ldg<uint8_t>(ksp, p * (DK / 32) + (DK == 128 ? g : g / 2));
#pragma unroll
        for (int i = 0; i < R / 32; i++) kr[i] = ldg<mk_b8>(krp, p * (R * 2) + (g * (R / 2) + 16 * i));
    }
    static constexpr int SLICES = DK / 32 + R / 32;
    __device__ __forceinline__ void store(mk_b8 (*dst)[64], int st, int lane) const {  // operand st of the position's row
        if (st < DK / 32) {
            uint32_t w;
            if constexpr (DK == 256) w = k[st / 4][st % 4];
            else w = k[0][st];
            dst[st][lane] = fp4x8(w, scale_of(DK == 256 ? (st < 4 ? ks & 255u : ks >> 8) : ks));
        } else {
            dst[st][lane] = kr[R ? st - DK / 32 : 0];
        }
    }
};
template <int DV> struct VQuarter {
    typedef typename Raw<DV / 32>::type VT;
    typedef typename Raw<DV == 64 ? 4 : DV / 32>::type VL;
    VL v[4];
    uint32_t vs[4];
    __device__ __forceinline__ void load(const uint8_t *vqp, const uint8_t *vsp, int j, int last, int n, int g) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t p = min(j + 4 * g + i, last);
            v[i] = ldg<VT>(vqp, p * (DV / 2) + n * (DV / 32));
            vs[i] = ldg<uint8_t>(vsp, p * (DV / 32) + n / (512 / DV));
        }
    }
    // its half (hi: positions 16 .. 31 of the 32) of the operands of the tiles 2 w and 2 w + 1
    static constexpr int SLICES = DV / 32;
    __device__ __forceinline__ void store(mk_b8 (*dst)[64], int w, int hi, int lane) const {
        uint32_t pr[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float sc = scale_of(vs[i]);
            uint32_t d;
            if constexpr (DV == 256) d = v[i][w / 4];
            else d = v[i];
            const mk_b2 x = w % 4 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 0) : w % 4 == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 1)
                          : w % 4 == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 2) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, sc, 3);
            pr[i] = __builtin_bit_cast(uint32_t, x);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            mk_u2 o;
#pragma unroll
            for (int i = 0; i < 2; i++) o[i] = __builtin_amdgcn_perm(pr[2 * i + 1], pr[2 * i], t & 1 ? 0x07060302u : 0x05040100u);
            ((mk_u2 *)&dst[2 * w + t][lane])[hi] = o;
        }
    }
};

// N consecutive values to the output
template <typename T, int N> __device__ __forceinline__ void store_run(void *out, size_t at, const float (&r)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *(mk_f4 *)((float *)out + at + i) = mk_f4{r[i], r[i + 1], r[i + 2], r[i + 3]};
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < N; i += 4) *(b4 *)((__bf16 *)out + at + i) = b4{(__bf16)r[i], (__bf16)r[i + 1], (__bf16)r[i + 2], (__bf16)r[i + 3]};
    }
}

// Workgroups of the kernel below that a compute unit holds (registers; at width 256 two instead of one: 512 rows at 4096 positions, 16 heads,
// 73 us instead of 113 with one-term weights, 76 us with two).
constexpr int many_per_cu(size_t elem, size_t dk) { return dk == 256 ? (elem == 4 ? 1 : 2) : elem == 4 ? 2 : 3; }

template <typename T, int DK, int R, int DV>
__global__ __launch_bounds__(256, many_per_cu(sizeof(T), DK)) void kv4_attn_many_kernel(MkKv4 c, MkSeqs s, AttnArgs a) {
    constexpr int NS = DK / 32, NR = R / 32, NF = NS + NR, NK = 2 * NF, NT = DV / 16, QT = Terms<T>::Q, PT = Terms<T>::P;
    __shared__ mk_b8 k_l[2][2][NF][64], v_l[2][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % c.nkv, G = a.nh / c.nkv;
    int b, tile, split;
    if (!find_work(c, s, a, G, 64, blockIdx.x / c.nkv, b, tile, split)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    split = __builtin_amdgcn_readfirstlane(split);
    const Column col = column(c, s, G, hk, b, tile * 64 + wave * 16 + n);
    const int low = __builtin_amdgcn_readfirstlane(columns_min(col.live ? col.lim : 0x7FFFFFFF));
    // the last position that a column of the workgroup sees (limits grow with the column; one beyond the capacity sees nothing)
    const int first = s.at(b), m_rows = max(s.at(b + 1) - first, 0), c_last = min(tile * 64 + 64, m_rows * G) - 1;
    const int top = __builtin_amdgcn_readfirstlane((int)min((int64_t)c.lens[b] - m_rows + c_last / G, (int64_t)c.cap - 1));
    const int j0 = split * a.chunk, j1 = chunk_end(a, split, top + 1);
    if (a.n_splits > 1 && j0 >= j1) return;

    mk_b8 qf[NF][QT];
    load_query<T, DK, R>(a, col, g, qf);
    float m = -INFINITY, l = 0.0f;
    mk_f4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (j0 < j1) {
        const size_t row0 = ((size_t)b * c.nkv + hk) * c.cap, kr0 = (size_t)b * c.cap;
        const uint8_t *kqp = uniform(c.kq + row0 * (DK / 2)), *ksp = uniform(c.ks + row0 * (DK / 32)), *vqp = uniform(c.vq + row0 * (DV / 2)),
                      *vsp = uniform(c.vs + row0 * (DV / 32)), *krp = R ? uniform(c.kr + kr0 * R) : nullptr;
        const bool k_wave = wave < 2;
        const int half = wave & 1;
        KQuarter<DK, R> kx;
        VQuarter<DV> vx;
        auto fetch_k = [&](int j) { kx.load(kqp, ksp, krp, j + 16 * half, j1 - 1, n, g); };
        auto fetch_v = [&](int j) { vx.load(vqp, vsp, j + 16 * half, j1 - 1, n, g); };
        auto store_k = [&](int buf) {
#pragma unroll
            for (int i = 0; i < NF; i++) kx.store(k_l[buf][half], i, lane);
        };
        mk_f4 sc[2], nx[2];  // scores of this step and of the next
        if (k_wave) {
            fetch_k(j0);
            store_k(0);
            fetch_k(j0 + 32);
            store_k(1);
            fetch_k(j0 + 64);
        } else {
            fetch_v(j0);
#pragma unroll
            for (int i = 0; i < NT / 2; i++) vx.store(v_l[0], i, half, lane);
            fetch_v(j0 + 32);
        }
        mk_wg_barrier();
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const mk_b8 kf = k_l[0][k / NF][k % NF][lane];
#pragma unroll
            for (int t = 0; t < QT; t++) sc[k / NF] = mfma(kf, qf[k % NF][t], k % NF || t ? sc[k / NF] : mk_f4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        mk_wg_barrier();  // (the first step stores into K's first buffer)
        for (int j = j0, buf = 0; j < j1; j += 32, buf ^= 1) {
            if (j + 31 > low || j + 32 > j1) {
                const int last = min(col.lim, j1 - 1) - j - 4 * g;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (16 * u + e > last) sc[u][e] = -INFINITY;
            }
            float p[8], sum;
            const mk_b8 (*kn)[NF][64] = k_l[buf ^ 1];
            mk_b8 ring[4];
#pragma unroll
            for (int k = 0; k < 3; k++) ring[k] = kn[k % 2][k / 2][lane];
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const int u = k % 2, st = k / 2;  // two sums in turn: one waits for itself longer than an instruction runs
                if (k + 3 < NK) ring[(k + 3) & 3] = kn[(k + 3) % 2][(k + 3) / 2][lane];
#pragma unroll
                for (int t = 0; t < QT; t++) nx[u] = mfma(ring[k & 3], qf[st][t], st || t ? nx[u] : mk_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int e = 8 * k / NK; e < 8 * (k + 1) / NK; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e / 4][e % 4], a.scale_log2, -m));
                __builtin_amdgcn_sched_barrier(0);
            }
            auto add = [&]() { sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])); };
            add();
            // only where a weight is far above the reference point of the steps before (or there is none yet) is the maximum looked
            // for and what has been summed rescaled
            if (__any(!(sum < FAR))) {
                float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])), fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
                mx = fmaxf(mk_rows_max(mx) * a.scale_log2, m);
                const float corr = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx), ref = mx == -INFINITY ? 0.0f : mx;
                m = mx;
                l *= corr;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[t][e] *= corr;
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], a.scale_log2, -ref));
                add();
            }
            l += sum;
#pragma unroll
            for (int k = 0; k < 2; k++) ring[k] = v_l[buf][k][lane];
            mk_b8 pf[PT];
            split8<PT>(p, pf);
            __builtin_amdgcn_sched_barrier(0);
            // (two sums in turn, as above)
            auto out_tiles = [&](int t) {
#pragma unroll
                for (int i = 2; i < 4; i++)
                    if (t + i < NT) ring[(t + i) & 3] = v_l[buf][t + i][lane];
#pragma unroll
                for (int k = 0; k < PT; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) o[t + i] = mfma(ring[(t + i) & 3], pf[k], o[t + i]);
            };
            if (k_wave) {
#pragma unroll
                for (int t = 0; t < NT; t += 2) {
                    out_tiles(t);
#pragma unroll
                    for (int e = NF * t / NT; e < NF * (t + 2) / NT; e++) kx.store(k_l[buf][half], e, lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                fetch_k(j + 96);
            } else {
#pragma unroll
                for (int t = 0; t < NT; t += 2) {
                    out_tiles(t);
                    vx.store(v_l[buf ^ 1], t / 2, half, lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                fetch_v(j + 64);
            }
            sc[0] = nx[0], sc[1] = nx[1];
            mk_wg_barrier();
        }
    }
    const float den = mk_rows_sum(l);
    if (!col.live) return;
    const size_t row = (size_t)col.t * a.nh + col.h;
    if (a.n_splits > 1) {
        const size_t at = (size_t)split * s.T * a.nh + row;
        if (g == 0) a.pm[at] = m, a.pl[at] = den;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < NT; t += 4) *(mk_f4 *)(a.po + at * DV + NT * (4 * g + e) + t) = mk_f4{o[t][e], o[t + 1][e], o[t + 2][e], o[t + 3][e]};
    } else {
        const float inv = col.beyond ? __builtin_nanf("") : col.lim < 0 ? 0.0f : 1.0f / den;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float r[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) r[t] = o[t][e] * inv;
            store_run<T, NT>(a.out, row * DV + NT * (4 * g + e), r);
        }
    }
}

// ------------------------------------------------------------------------------------------- the chunks' results together

// One wave: (row, head).  Lane i has the statistics of chunk i: weights 2^(m_i - max), one division.
template <typename T>
__global__ __launch_bounds__(256) void kv4_merge_kernel(MkKv4 c, MkSeqs s, AttnArgs a) {
    static_assert(MAX_SPLITS <= MK_WAVE, "one lane a chunk");
    const size_t rows = (size_t)s.T * a.nh, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63, t = (int)(row / a.nh), b = s.of_row(t);
    if (b < 0) return;
    const int64_t lim = row_limit(c, s, b, t);
    const int used = lim < 0 || lim >= c.cap ? 0 : min((int)lim / a.chunk + 1, a.n_splits);
    const float empty = lim < 0 ? 0.0f : __builtin_nanf("");
    const float m = lane < used ? a.pm[lane * rows + row] : -INFINITY, l = lane < used ? a.pl[lane * rows + row] : 0.0f;
    const float mx = mk_wave_max(m), ref = mx == -INFINITY ? 0.0f : mx;
    const float w = __builtin_amdgcn_exp2f(m - ref), den = mk_wave_sum(l * w);
    for (int d = 4 * lane; d < c.dv; d += 4 * MK_WAVE) {
        mk_f4 num = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < used; i0 += 8) {  // eight loads in flight
            mk_f4 o[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i0 + i < used) o[i] = *(const mk_f4 *)(a.po + ((size_t)(i0 + i) * rows + row) * c.dv + d);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i0 + i < used) {
                    const float wi = mk_readlane(w, i0 + i);
#pragma unroll
                    for (int k = 0; k < 4; k++) num[k] = fmaf(o[i][k], wi, num[k]);
                }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) store1<T>(a.out, row * c.dv + d + k, used ? num[k] / den : empty);
    }
}

// Prompts of widths that have no matrix kernel: enough workgroups without a cut, whose results would be as large as the rows.
bool uncut(int columns, size_t T, size_t B, size_t pairs) { return columns == 1 && T > B && pairs >= 1024; }

// the widths the matrix kernels are built for: (K, tail, V)
bool matrix_widths(const mk_kv4_cache *c) {
    return c->dk == c->dv ? (c->dk == 64 || c->dk == 128 || c->dk == 256) && (c->rope == 0 || c->rope == 64) : false;
}

// Which kernel a call takes, by the query columns a sequence has on average: a wave's 16 are all there is, or the workgroup shares K and V.
// (The kernel for 16 reads 32 positions at a time and a cache has to hold them; the other reads none past the last.)
enum Form { FEW = 16, MANY = 64, ANY = 1 };  // the value: query columns of a workgroup
Form form_of(const mk_kv4_cache *c, size_t T, size_t group) {
    if (!matrix_widths(c)) return ANY;
    return T * group <= FEW * c->B && c->cap >= 32 ? FEW : MANY;
}

// Chunks that a context is cut into when `pairs` (column tile, kv head) walk `len` positions each.  `len` is max_len or the capacity, for the host does not
// read lens: in a cache with much room the chunks are longer than what is held asks for (8 kv heads of 128 | 128, one row over 2048 positions:
// capacity 2048 10.9, 16384 11.8, 131072 16.9 us; 64 rows over 4096: capacity 4096 39, 32768 73, 131072 100 us; with max_len as with the tight cache).
//
// Few columns: about 1024 chunks fill the 256 compute units; below 256 positions (two steps a wave) a chunk is start and end only,
// above 1024 one long sequence among short ones is a tail (32 ragged sequences of up to 16384 positions: 30.2 / 24.2 / 27.0 us in chunks of
// 512 / 1024 / 2048).  Up to 1024 positions are one chunk: the second launch costs what the split saves (96 heads, 1024
// positions: 13.2 us, in four chunks 10.3 + 4.0 us).
void plan_few(AttnArgs &a, size_t pairs, size_t len) {
    size_t chunk = (pairs * len / 1024 + 127) / 128 * 128;
    chunk = len <= 1024 ? len : chunk < 256 ? 256 : chunk > 1024 ? 1024 : chunk;
    const size_t least = (len + MAX_SPLITS - 1) / MAX_SPLITS;
    if (chunk < least) chunk = (least + 127) / 128 * 128;
    a.chunk = (int)chunk;
    a.n_splits = (int)((len + chunk - 1) / chunk);
}
// The most chunks that it makes for `pairs` or more and any length up to cap: chunks of 256 until pairs * len reaches 1024 * 256, then
// at most 1024 / pairs (and one that is not whole) of them, from chunks of 1024 on len / 1024.
size_t most_few(size_t pairs, size_t cap) {
    if (cap <= 1024) return 1;
    size_t n = (1024 + pairs - 1) / pairs + 1;
    const size_t by_len = (cap + 1023) / 1024;
    n = n < by_len ? by_len : n;
    n = n < (cap + 255) / 256 ? n : (cap + 255) / 256;
    return n < MAX_SPLITS ? n : MAX_SPLITS;
}

// Many columns: the number of chunks with the least estimated time, of those that make no more than about 1024 workgroups.  A step of 32
// positions takes 0.38 + 0.62 us for every 256 values of K and V (f32: 1.5 times that); a second workgroup on a compute unit costs 5 %, a third
// 20 % more; a merge takes 8 us and its results' way to memory and back.  (96 heads over 4096 positions: 192 rows 142 us uncut, 118 in two
// chunks, 300 rows 145 and 185; 200 rows of 48 heads over 16000: 277 us in two chunks, 206 in four, 227 in six.)
size_t most_many(size_t pairs, size_t cap) {
    size_t n = (1024 + pairs - 1) / pairs;
    n = n < cap / 256 ? n : cap / 256;
    n = n < MAX_SPLITS ? n : MAX_SPLITS;
    return n < 1 ? 1 : n;
}
void plan_many(AttnArgs &a, size_t pairs, size_t len, size_t rows, size_t elem, const mk_kv4_cache *c) {
    const size_t at_once = many_per_cu(elem, c->dk);
    const double share[4] = {0.0, 1.0, 1.05, 1.25};  // time of 0 .. 3 workgroups on a compute unit
    const double step = (0.38 + 0.62 * (c->dk + c->rope + c->dv) / 256) * (elem == 4 ? 1.5 : 1.0);
    double best = 0.0;
    a.chunk = (int)len, a.n_splits = 1;
    for (size_t n = 1; n <= most_many(pairs, len); n++) {
        const size_t chunk = n == 1 ? len : ((len + n - 1) / n + 127) / 128 * 128, splits = (len + chunk - 1) / chunk;
        const size_t on_cu = (pairs * splits + 255) / 256;
        double t = chunk / 32.0 * step * (on_cu / at_once * share[at_once] + share[on_cu % at_once]);
        if (splits > 1) t += 8.0 + splits * rows * c->dv * 8 / 3e6;
        if (n > 1 && t >= best) continue;
        best = t, a.chunk = (int)chunk, a.n_splits = (int)splits;
    }
}

// results of n chunks
size_t piece_bytes(size_t n, size_t rows, size_t dv) { return mk_align_up(n * rows * dv * 4, 256) + 2 * mk_align_up(n * rows * 4, 256); }

size_t column_tiles(const mk_kv4_cache *c, size_t T, const int32_t *cu, size_t group, size_t ct) {
    return cu ? T * group / ct + c->B : c->B * ((T / c->B * group + ct - 1) / ct);
}

template <typename T, int D, int R>
void launch_matrix(Form form, const dim3 &grid, hipStream_t st, const MkKv4 &v, const MkSeqs &s, const AttnArgs &a) {
    if (form == FEW) hipLaunchKernelGGL((kv4_attn_few_kernel<T, D, R, D>), grid, dim3(256), 0, st, v, s, a);
    else hipLaunchKernelGGL((kv4_attn_many_kernel<T, D, R, D>), grid, dim3(256), 0, st, v, s, a);
}
template <typename T, int D>
void launch_matrix(Form form, const dim3 &grid, hipStream_t st, const MkKv4 &v, const MkSeqs &s, const AttnArgs &a) {
    if (v.rope) launch_matrix<T, D, 64>(form, grid, st, v, s, a);
    else launch_matrix<T, D, 0>(form, grid, st, v, s, a);
}
template <typename T>
void launch_matrix(Form form, const dim3 &grid, hipStream_t st, const MkKv4 &v, const MkSeqs &s, const AttnArgs &a) {
    if (v.dk == 64) launch_matrix<T, 64>(form, grid, st, v, s, a);
    else if (v.dk == 128) launch_matrix<T, 128>(form, grid, st, v, s, a);
    else launch_matrix<T, 256>(form, grid, st, v, s, a);
}

}  // namespace

extern "C" size_t mk_kv4_attn_workspace_bytes(const mk_kv4_cache *c, size_t T, size_t nh) {
    if (!c || !T || !nh || !c->nkv || !c->cap) return 0;
    // (column tile, kv head) pairs: no fewer than this, wherever the sequences begin
    const size_t group = nh / c->nkv ? nh / c->nkv : 1, cols = T * group;
    const Form form = form_of(c, T, group);
    const size_t pairs = c->nkv * (cols / form ? cols / form : 1);
    const size_t n = form == MANY ? most_many(pairs, c->cap) : uncut(form, T, c->B, pairs) ? 1 : most_few(pairs, c->cap);
    return n <= 1 ? 0 : piece_bytes(n, T * nh, c->dv);
}

extern "C" int mk_dev_kv4_attn(const mk_kv4_cache *c, int dtype, const void *q, size_t q_stride, size_t T, const int32_t *cu, size_t nh, float scale,
                               size_t max_len, void *workspace, void *out, void *stream) {
    int st = mk_kv4_check(c);
    if (st != MK_OK || (st = mk_kv4_check_rows(c, dtype, T, cu)) != MK_OK) return st;
    MK_REQUIRE(nh >= 1 && nh <= 65535 && nh % c->nkv == 0, "the query heads must be a multiple of the kv heads");
    if (T == 0) return MK_OK;
    MK_REQUIRE(q && out && (workspace || mk_kv4_attn_workspace_bytes(c, T, nh) == 0), "null pointer");
    MK_REQUIRE(q_stride % 8 == 0 && mk_aligned16(q) && mk_aligned16(out) && ((uintptr_t)workspace & 255) == 0,
               "q and out must be 16-byte, the workspace 256-byte aligned, the query stride a multiple of 8 values");
    MK_REQUIRE(T == 1 || q_stride >= nh * (c->dk + c->rope), "the query stride is shorter than a token's heads");
    MK_REQUIRE(T * nh <= 0x7FFFFF00ull, "too many query rows in one call");
    AttnArgs a;
    a.q = q, a.q_stride = q_stride, a.out = out, a.nh = (int)nh, a.scale_log2 = fabsf(scale) * LOG2E, a.sign = scale < 0.0f ? -1.0f : 1.0f;
    if (scale == 0.0f) a.sign = 0.0f, a.scale_log2 = 1.0f;  // (a hidden position's -inf times 0 would be NaN)
    const size_t len = max_len && max_len < c->cap ? max_len : c->cap, group = nh / c->nkv;
    const Form form = form_of(c, T, group);
    const size_t tiles = form == ANY ? T * group : column_tiles(c, T, cu, group, form), pairs = tiles * c->nkv;
    if (form == MANY) plan_many(a, pairs, len, T * nh, dtype == MK_F32 ? 4 : 2, c);
    else if (uncut(form, T, c->B, pairs)) a.chunk = (int)len, a.n_splits = 1;
    else plan_few(a, pairs, len);
    MK_REQUIRE(a.n_splits == 1 || (T * nh + 3) / 4 <= MAX_GROUPS, "too many query rows in one call");
    MK_REQUIRE(a.n_splits == 1 || piece_bytes(a.n_splits, T * nh, c->dv) <= mk_kv4_attn_workspace_bytes(c, T, nh), "chunks beyond the workspace");
    uint8_t *w = (uint8_t *)workspace;
    a.po = (float *)w;
    w += mk_align_up((size_t)a.n_splits * T * nh * c->dv * 4, 256);
    a.pm = (float *)w;
    w += mk_align_up((size_t)a.n_splits * T * nh * 4, 256);
    a.pl = (float *)w;
    const MkSeqs s{cu, (int)T, (int)c->B};
    const MkKv4 v = mk_kv4_view(c);
    hipStream_t hs = (hipStream_t)stream;
    if (form != ANY) {
        MK_REQUIRE(pairs * a.n_splits <= MAX_GROUPS, "too many query rows in one call");
        const dim3 grid((unsigned)(pairs * a.n_splits));
        if (dtype == MK_F32) launch_matrix<float>(form, grid, hs, v, s, a);
        else launch_matrix<__bf16>(form, grid, hs, v, s, a);
    } else {
        const dim3 grid((unsigned)T, (unsigned)nh, (unsigned)a.n_splits);
        if (dtype == MK_F32) hipLaunchKernelGGL(kv4_attn_any_kernel<float>, grid, dim3(256), 0, hs, v, s, a);
        else hipLaunchKernelGGL(kv4_attn_any_kernel<__bf16>, grid, dim3(256), 0, hs, v, s, a);
    }
    if ((st = mk_launch_status("kv4_attn")) != MK_OK) return st;
    if (a.n_splits > 1) {
        const unsigned blocks = (unsigned)((T * nh + 3) / 4);
        if (dtype == MK_F32) hipLaunchKernelGGL(kv4_merge_kernel<float>, dim3(blocks), dim3(256), 0, hs, v, s, a);
        else hipLaunchKernelGGL(kv4_merge_kernel<__bf16>, dim3(blocks), dim3(256), 0, hs, v, s, a);
        return mk_launch_status("kv4_merge");
    }
    return MK_OK;
}
