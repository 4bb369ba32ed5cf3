// Linear attention with a decay for each head, and its recurrent state:
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T        S [dk][dv] per value head, f32
//   o_t = scale * S_t^T q_t
//
// g_t is a log decay per token and head, or one constant per head; g = -inf empties the state.  Query / key heads may be fewer
// than value heads (head h reads key head h / (nh / nkh)).  Sequences of a batch lie one behind the other.
#include "mk_mixer.h"

namespace {

struct LinArgs {
    const void *q, *k, *v;
    size_t qs, ks, vs;      // values from one token's row to the next
    const float *g;
    size_t gs;              // 0: one constant per head
    const int32_t *cu;
    int T, B, nh, nkh, dk, dv;
    float scale;
    const float *state;     // may be null: zeros
    float *state_out;
    void *out;              // [T][nh][dv]
    int slices;             // workgroups that share out a head's columns of dv
    __device__ __forceinline__ int at(int b) const { return cu ? min(max(cu[b], 0), T) : (int)((int64_t)T / B * b); }
};

// ------------------------------------------------------------------------------------------------ token by token
//
// One workgroup: (64 columns of dv, value head, sequence).  Thread (rg, cg) = (tid / 16, tid % 16) holds rows rg + 16 i,
// columns 4 cg .. 4 cg + 3 of the slice in registers: the state is read and written once, in runs of 256 bytes.  The tokens'
// rows go through LDS, STAGE at a time.  For widths that the blocks below do not take; bound by two barriers a token (1024 tokens of 16
// bfloat16 heads of 96 x 96: 0.80 ms, of 256 x 256 1.24 ms).
constexpr int COLS = 64, STAGE = 8;

template <typename T> __device__ __forceinline__ float ldf(const T *p) { return (float)*p; }

template <typename T, int NR>
__global__ __launch_bounds__(256) void linear_token_kernel(LinArgs a) {
    __shared__ float q_l[STAGE][NR * 16], k_l[STAGE][NR * 16], v_l[STAGE][COLS], e_l[STAGE], o_l[4][COLS];
    const int b = blockIdx.z, h = blockIdx.y, c0 = blockIdx.x * COLS, tid = threadIdx.x;
    const int rg = tid >> 4, cg = tid & 15, col = c0 + cg * 4;
    const int hk = h / (a.nh / a.nkh);
    const int t0 = a.at(b), t1 = a.at(b + 1);
    const size_t sbase = ((size_t)b * a.nh + h) * a.dk * a.dv;
    mk_f4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int r = rg + 16 * i;
        S[i] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (a.state && r < a.dk && col < a.dv) S[i] = *(const mk_f4 *)(a.state + sbase + (size_t)r * a.dv + col);
    }
    for (int ts = t0; ts < t1; ts += STAGE) {
        const int n = min(STAGE, t1 - ts);
        __syncthreads();
        for (int i = tid; i < n * NR * 16; i += 256) {
            const int t = i / (NR * 16), d = i - t * (NR * 16);
            q_l[t][d] = d < a.dk ? ldf((const T *)a.q + (size_t)(ts + t) * a.qs + (size_t)hk * a.dk + d) * a.scale : 0.0f;
            k_l[t][d] = d < a.dk ? ldf((const T *)a.k + (size_t)(ts + t) * a.ks + (size_t)hk * a.dk + d) : 0.0f;
        }
        for (int i = tid; i < n * COLS; i += 256) {
            const int t = i / COLS, d = i - t * COLS;
            v_l[t][d] = c0 + d < a.dv ? ldf((const T *)a.v + (size_t)(ts + t) * a.vs + (size_t)h * a.dv + c0 + d) : 0.0f;
        }
        if (tid < n) e_l[tid] = expf(a.g[a.gs ? (size_t)(ts + tid) * a.gs + h : h]);
        __syncthreads();
        for (int t = 0; t < n; t++) {
            const float e = e_l[t];
            const mk_f4 v = *(const mk_f4 *)&v_l[t][cg * 4];
            mk_f4 o = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const float k = k_l[t][rg + 16 * i], q = q_l[t][rg + 16 * i];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    S[i][j] = fmaf(e, S[i][j], k * v[j]);
                    o[j] = fmaf(q, S[i][j], o[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = mk_rows_sum(o[j]);
            if ((tid & 63) < 16) *(mk_f4 *)&o_l[tid >> 6][cg * 4] = o;
            __syncthreads();
            if (tid < COLS && c0 + tid < a.dv) {
                const float r = (o_l[0][tid] + o_l[1][tid]) + (o_l[2][tid] + o_l[3][tid]);
                const size_t at = ((size_t)(ts + t) * a.nh + h) * a.dv + c0 + tid;
                if constexpr (sizeof(T) == 4) ((float *)a.out)[at] = r;
                else ((__bf16 *)a.out)[at] = (__bf16)r;
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int r = rg + 16 * i;
        if (r < a.dk && col < a.dv) *(mk_f4 *)(a.state_out + sbase + (size_t)r * a.dv + col) = S[i];
    }
}

// ------------------------------------------------------------------------------------------------ one token
//
// The state goes through once, as a copy does: a thread's rows are all asked for, then row by row updated, written back and added to the
// output, so that a workgroup reads and writes at the same time.  CG threads of 4 columns make a row of the slice, 256 / CG rows at
// a time.  HBM-bound: 64 sequences x 32 heads x 128 x 128 (270 MB) 48 us, 5.6 TB/s (a large copy: 5.1); with the whole slice held
// until its last row is updated 78 us, without the non-temporal hints 51 us; rows of 128 or 512 bytes a slice: 52 and 51 us.
template <typename T, int NR, int CG>
__global__ __launch_bounds__(256) void linear_step_kernel(LinArgs a) {
    constexpr int GROUPS = 256 / CG;
    __shared__ float q_l[NR * GROUPS], k_l[NR * GROUPS];
    __shared__ mk_f4 o_l[GROUPS][CG];
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, rg = tid / CG, cg = tid % CG, col = blockIdx.x * (4 * CG) + 4 * cg;
    const int hk = h / (a.nh / a.nkh);
    const size_t sbase = ((size_t)b * a.nh + h) * a.dk * a.dv + col;
    const T *q = (const T *)a.q + (size_t)b * a.qs + (size_t)hk * a.dk, *k = (const T *)a.k + (size_t)b * a.ks + (size_t)hk * a.dk;
    const bool live = col < a.dv;
    float qr[(NR * GROUPS + 255) / 256], kr[(NR * GROUPS + 255) / 256], v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < (NR * GROUPS + 255) / 256; i++) {
        const int d = min(tid + 256 * i, a.dk - 1);
        qr[i] = (float)q[d];
        kr[i] = (float)k[d];
    }
    if (live) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)((const T *)a.v)[(size_t)b * a.vs + (size_t)h * a.dv + col + j];
    }
    const float e = expf(a.g[a.gs ? (size_t)b * a.gs + h : h]);
    mk_f4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int r = rg + GROUPS * i;
        S[i] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (a.state && live && r < a.dk) S[i] = __builtin_nontemporal_load((const mk_f4 *)(a.state + sbase + (size_t)r * a.dv));
    }
#pragma unroll
    for (int i = 0; i < (NR * GROUPS + 255) / 256; i++) {
        const int d = tid + 256 * i;
        if (d < NR * GROUPS) {
            q_l[d] = d < a.dk ? qr[i] * a.scale : 0.0f;
            k_l[d] = d < a.dk ? kr[i] : 0.0f;
        }
    }
    mk_wg_barrier();
    mk_f4 o = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int r = rg + GROUPS * i;
        const float kk = k_l[r], qq = q_l[r];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            S[i][j] = fmaf(e, S[i][j], kk * v[j]);
            o[j] = fmaf(qq, S[i][j], o[j]);
        }
        if (live && r < a.dk) __builtin_nontemporal_store(S[i], (mk_f4 *)(a.state_out + sbase + (size_t)r * a.dv));
    }
    o_l[rg][cg] = o;
    mk_wg_barrier();
    if (tid < 4 * CG && blockIdx.x * (4 * CG) + tid < a.dv) {
        float r = 0.0f;
#pragma unroll
        for (int i = 0; i < GROUPS; i++) r += ((const float *)o_l[i])[tid];
        const size_t at = ((size_t)b * a.nh + h) * a.dv + blockIdx.x * (4 * CG) + tid;
        if constexpr (sizeof(T) == 4) ((float *)a.out)[at] = r;
        else ((__bf16 *)a.out)[at] = (__bf16)r;
    }
}

template <typename T, int CG>
int launch_step(const LinArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.dv + 4 * CG - 1) / (4 * CG)), (unsigned)a.nh, (unsigned)a.B);
    constexpr int G = 256 / CG;
    if (a.dk <= 64) hipLaunchKernelGGL((linear_step_kernel<T, 64 / G, CG>), grid, dim3(256), 0, st, a);
    else if (a.dk <= 128) hipLaunchKernelGGL((linear_step_kernel<T, 128 / G, CG>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((linear_step_kernel<T, 256 / G, CG>), grid, dim3(256), 0, st, a);
    return mk_launch_status("linear_step");
}

template <typename T>
int launch_token(const LinArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.dv + COLS - 1) / COLS), (unsigned)a.nh, (unsigned)a.B);
    if (a.dk <= 64) hipLaunchKernelGGL((linear_token_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else if (a.dk <= 128) hipLaunchKernelGGL((linear_token_kernel<T, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((linear_token_kernel<T, 16>), grid, dim3(256), 0, st, a);
    return mk_launch_status("linear_token");
}

// ------------------------------------------------------------------------------------------------ blocks of 64 tokens
//
// With b_i the sum of the log decays of a block up to its token i (S: the state before the block, m: its last token):
//   o_i = scale * ( e^{b_i} S^T q_i + sum_{j <= i} e^{b_i - b_j} (q_i . k_j) v_j )
//   S'  = e^{b_m} S + sum_j (e^{b_m - b_j} v_j) k_j^T
// which is all matrix products, and every exponent of the decays is a difference of sums of the same block: formed in 64 bits, so that
// no large sum cancels, it is never positive for log decays that are not (a log decay below -200 counts as -200: e^-200 is 0).
//
// One workgroup: a run of blocks of (value head, sequence), one wave for every 16 or 32 columns of dv.  The state stays in registers across the
// blocks, as the matrix instruction returns it: tile kt of S = rows 16 kt + 4 g + j, column n of 16 (lane = 16 g + n).  Two such
// tiles ARE an operand of the next product once the sum over dk takes its terms in the order {4 g .. , 16 + 4 g ..}; the same
// holds for the block's scores and the sum over its tokens.  So the waves exchange only the scores, through LDS in operand order:
//   scores   A = K rows, B = Q rows               -> (key, query), weighted by the decay, masked, to LDS (six operands, shared out)
//   out      A = S^T, B = Q^T; times e^{b_i}; A = V^T, B = scores     -> (dv, token)
//   state    A = K^T, B = weighted V^T            -> (dk, dv)
// bfloat16 rows: S and the weighted scores enter the products of the output as two bfloat16 terms each (17 bits, so that the result is rounded
// once; as one term, whose rounding is as large as the result's own, the error against 64 bits is 2.3e-3 instead of 1.7e-3);
// the state itself is f32 through and through, so its weighted values enter in three bfloat16 terms (24 bits).
// f32 rows: the same on the f32 matrix instruction (in three bfloat16 terms, six products: 128 x 128 heads 100 -> 95 us, but 64 x 128 heads 40 -> 46
// us, whose terms take the LDS of the second workgroup).
//
// 8192 tokens of 32 bfloat16 heads of 128 x 128: 130 us, of which local states 38 (168 MB), the states before each segment 12 (67 MB), outputs 78
// (301 MB, 22 % of the matrix cores' time; with one-term operands 69).  The first two move their bytes at the rate of a large copy (5.1 TB/s), the
// outputs at 4.0; reading K and V twice is what the split over the device costs.  Five ragged f32 sequences (1683 tokens, 16 heads of
// 64 x 128): 40 us, bound by the f32 matrix instruction and three launches.
constexpr int CH = 64;

typedef float mk_f8v __attribute__((ext_vector_type(8)));
template <typename T> struct Op;
template <> struct Op<__bf16> {
    typedef mk_b8 F;
    // values a row of K and V (read down the columns: eight rows of 4 + 4 words side by side) and of Q (read along the rows) is padded by
    static constexpr int PAD = 16, QPAD = 8, TERMS = 3, OUT_TERMS = 2;
    static __device__ __forceinline__ mk_f4 mma(F a, F b, mk_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ bool finite(const mk_v4u &r) {  // of a 16-byte piece of a row
        bool ok = true;
#pragma unroll
        for (int i = 0; i < 4; i++) ok &= (r[i] & 0x7F80u) != 0x7F80u && (r[i] & 0x7F800000u) != 0x7F800000u;
        return ok;
    }
};
template <> struct Op<float> {
    typedef mk_f8v F;
    static constexpr int PAD = 4, QPAD = 4, TERMS = 1, OUT_TERMS = 1;
    static __device__ __forceinline__ mk_f4 mma(F a, F b, mk_f4 c) {
#pragma unroll
        for (int i = 0; i < 8; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ bool finite(const mk_v4u &r) {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < 4; i++) ok &= (r[i] & 0x7F800000u) != 0x7F800000u;
        return ok;
    }
};
// two result tiles (or any 8 values) as an operand, the sum of N terms, largest first
template <typename T, int N> __device__ __forceinline__ void operand(const mk_f4 &lo, const mk_f4 &hi, typename Op<T>::F (&f)[N]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = lo[i], r[4 + i] = hi[i];
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f[k][i] = (T)r[i];
            if (k + 1 < N) r[i] -= (float)f[k][i];
        }
}
// values 8 consecutive of a row
__device__ __forceinline__ mk_b8 row8(const __bf16 *p) { return *(const mk_b8 *)p; }
__device__ __forceinline__ mk_f8v row8(const float *p) {
    const mk_f4 a = *(const mk_f4 *)p, b = *(const mk_f4 *)(p + 4);
    return mk_f8v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// values 4 + 4 of a row, 16 apart
typedef __bf16 mk_b4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ mk_b8 row44(const __bf16 *p) {
    const mk_b4 a = *(const mk_b4 *)p, b = *(const mk_b4 *)(p + 16);
    return mk_b8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ mk_f8v row44(const float *p) {
    const mk_f4 a = *(const mk_f4 *)p, b = *(const mk_f4 *)(p + 16);
    return mk_f8v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// A 16-byte piece of a query row (values d ..) into its LDS row, whose 32-value groups hold the values in operand order: lane group g's {4 g .. ,
// 16 + 4 g ..} side by side, so that the operand is one read.
__device__ __forceinline__ void store_q(__bf16 *row, int d, const mk_v4u &x) {
    __bf16 *p = row + (d & ~31) + 8 * ((d & 15) >> 2) + 4 * ((d & 31) >> 4);
    *(mk_u2 *)p = mk_u2{x[0], x[1]};
    *(mk_u2 *)(p + 8) = mk_u2{x[2], x[3]};
}
__device__ __forceinline__ void store_q(float *row, int d, const mk_v4u &x) { *(mk_v4u *)(row + (d & ~31) + 8 * ((d & 15) >> 2) + 4 * ((d & 31) >> 4)) = x; }
// a transposed operand of a tile in LDS [token][LD]: lane (g, n) gets column cols + n of the tokens 32 ks + 4 g .. + 3 and 16 further
template <int LD> __device__ __forceinline__ mk_b8 column8(const __bf16 *tile, int ks, int cols, int g, int n) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    const __bf16 *p = tile + (32 * ks + 4 * g + (n >> 2)) * LD + cols + 4 * (n & 3);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(p + 16 * LD));
    typedef short s8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(mk_b8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}
template <int LD> __device__ __forceinline__ mk_f8v column8(const float *tile, int ks, int cols, int g, int n) {
    mk_f8v f;
    const float *p = tile + (32 * ks + 4 * g) * LD + cols + n;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = p[((i & 3) + 16 * (i >> 2)) * LD];
    return f;
}

template <int N> struct Int { static constexpr int value = N; };

// A sequence is cut into segments of `per` blocks, each a slot of the workspace and a workgroup per head; sequence b has the slots from
// at(b) / (64 per) + b on: never fewer than its segments (some stay empty, those before the first sequence's too), T / (64 per) + B in all,
// whatever the lengths are.
struct LinSeg {
    int per;        // 0: a sequence is one workgroup per head, without a workspace
    mk_f4 *local;   // [slot][h][DK / 16][4 DV]: local states, then the states before each segment
    float *decay;   // [slot][h]: e^{sum of the segment's log decays}
    __device__ __forceinline__ int first(const LinArgs &a, int b) const { return a.at(b) / (CH * per) + b; }
};
// 2^x for the decays: x is a difference of 64-bit sums of log2 decays, rounded once
__device__ __forceinline__ float pow2(double x) { return __builtin_amdgcn_exp2f((float)x); }

// inclusive sum over the wave in 64 bits: within rows of 16 lanes by shifts, then the row before and the half before (all lanes active)
template <int CTRL, int ROWS> __device__ __forceinline__ double shifted(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
    v += shifted<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += shifted<0x112, 0xF>(v);
    v += shifted<0x114, 0xF>(v);
    v += shifted<0x118, 0xF>(v);
    v += shifted<0x142, 0xA>(v);  // lane 15 of the row before, into rows 1 and 3
    v += shifted<0x143, 0xC>(v);  // lane 31, into rows 2 and 3
    return v;
}
__device__ __forceinline__ double last_lane(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

enum Mode { LOCAL, OUTPUT, BOTH };  // local states of the segments; outputs from the states before them; one segment: outputs and state
// NT: tiles of 16 columns a wave.  Two (a wave's operands of Q, K and the scores, read from LDS, serve both) where the reads bound it: with one, 16
// waves a compute unit read 16 KB of queries each block.  One for the local states, whose four waves a SIMD hide more.
template <typename T, int DK, int DV, Mode MODE> constexpr int tiles() { return MODE != LOCAL && sizeof(T) == 2 && DV == 128 ? 2 : 1; }
template <typename T, int DK, int DV, Mode MODE>
__global__ __launch_bounds__((DV * 4 / tiles<T, DK, DV, MODE>()), MODE == LOCAL ? (sizeof(T) == 2 ? 4 : 2) : sizeof(T) == 4 && DK > DV ? 1 : 2) void linear_block_kernel(LinArgs a, LinSeg sg) {
    typedef typename Op<T>::F F;
    constexpr bool OUT = MODE != LOCAL;
    // the state that only leads to the next outputs takes its updates as two terms, as it enters them (2^-16 of a value at most)
    constexpr int TERMS = MODE == OUTPUT && Op<T>::TERMS > 2 ? 2 : Op<T>::TERMS, OT = Op<T>::OUT_TERMS;
    constexpr int NT = tiles<T, DK, DV, MODE>(), NW = DV / 16 / NT, TH = 64 * NW, KT = DK / 16, KS = DK / 32, LK = DK + Op<T>::PAD, LV = DV + Op<T>::PAD, LQ = DK + Op<T>::QPAD;
    constexpr int E = 16 / sizeof(T), KP = CH * DK / E / TH, VP = CH * DV / E / TH;  // values of a 16-byte piece; pieces a thread moves
    __shared__ __attribute__((aligned(16))) T k_l[CH * LK], v_l[CH * LV], q_l[OUT ? CH * LQ : 8];
    __shared__ F p_l[OT][OUT ? 6 : 1][64];              // scores: query tiles 0 .. 3 with keys 0 .. 31, query tiles 2, 3 with keys 32 .. 63
    __shared__ double b_l[2][CH];                       // sums of the log2 decays of a block and of the next
    __shared__ float w_l[2][CH], e_l[2][CH], last_l[2];  // 2^(b_m - b_i), scale * 2^(b_i), 2^(b_m)
    __shared__ int bad_l;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int slices = MODE == BOTH ? a.slices : 1, dv = MODE == BOTH ? a.dv : DV;
    const int hs = blockIdx.x % (a.nh * slices), h = hs / slices, col0 = (hs - h * slices) * DV, slot = blockIdx.x / (a.nh * slices), hk = h / (a.nh / a.nkh);
    int b = slot, c0 = 0;
    if (MODE != BOTH) {  // the last sequence whose slots begin at this one or before
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sg.first(a, mid) <= slot) lo = mid;
            else hi = mid;
        }
        b = lo;
        c0 = slot - sg.first(a, b);
        if (c0 < 0) return;  // a slot of the rows before the first sequence
        c0 *= sg.per;
    }
    const int t0 = a.at(b), len = max(a.at(b + 1) - t0, 0), nch = (len + CH - 1) / CH, c1 = MODE == BOTH ? nch : min(c0 + sg.per, nch);
    if (MODE != BOTH && c0 >= c1) return;
    const size_t sh = (size_t)slot * a.nh + h, sbase = ((size_t)b * a.nh + h) * DK * dv + col0 + 16 * NT * wave + n;
    mk_f4 S[KT][NT];
    mk_f4 *mine = sg.local + sh * KT * (DV * 4) + 64 * NT * wave + lane;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            S[kt][t] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (MODE == OUTPUT) {
                S[kt][t] = mine[kt * (DV * 4) + 64 * t];
            } else if (MODE == BOTH && a.state) {
#pragma unroll
                for (int j = 0; j < 4; j++) S[kt][t][j] = a.state[sbase + 16 * t + (size_t)(16 * kt + 4 * g + j) * dv];
            }
        }
    const T *qp = (const T *)a.q + (size_t)hk * DK, *kp = (const T *)a.k + (size_t)hk * DK, *vp = (const T *)a.v + (size_t)h * dv + col0;
    mk_v4u kr[KP], vr[VP], qr[OUT ? KP : 1];
    float gr;
    // A block's rows into registers: a scalar base, a lane offset that never changes, and a scalar step from piece to piece.  Rows behind the
    // sequence are read as its last one (and dropped at the store).
    auto rows = [&](mk_v4u *dst, const T *base, size_t stride, int first, int r0, int d0, auto pieces, auto step) {
        const T *p = base + (size_t)(t0 + first) * stride;
        if (first + CH <= len) {
            const uint32_t off = (uint32_t)(r0 * (uint32_t)stride + d0) * sizeof(T);
#pragma unroll
            for (int i = 0; i < decltype(pieces)::value; i++) dst[i] = *(const MK_GLOBAL mk_v4u *)((const MK_GLOBAL uint8_t *)(p + i * (decltype(step)::value * stride)) + off);
        } else {
#pragma unroll
            for (int i = 0; i < decltype(pieces)::value; i++) dst[i] = *(const mk_v4u *)(p + (size_t)min(r0 + i * decltype(step)::value, len - 1 - first) * stride + d0);
        }
    };
    auto fetch = [&](int c, int tid) {
        const int rk = tid / (DK / E), rv = tid / (DV / E), dk0 = tid % (DK / E) * E, dv0 = tid % (DV / E) * E;
        rows(kr, kp, a.ks, c * CH, rk, dk0, Int<KP>(), Int<CH / KP>());
        if constexpr (OUT) rows(qr, qp, a.qs, c * CH, rk, dk0, Int<KP>(), Int<CH / KP>());
        rows(vr, vp, a.vs, c * CH, rv, dv0, Int<VP>(), Int<CH / VP>());
    };
    auto decays = [&](int c) { return a.g[a.gs ? (size_t)(t0 + min(c * CH + lane, len - 1)) * a.gs + h : h]; };
    double total = 0.0;
    auto scan = [&](int c, float gr) {  // one wave: the sums of block c
        const int u = c & 1;
        const double s = wave_scan(c * CH + lane < len ? (double)(gr < -200.0f ? -200.0f : gr) * 1.4426950408889634 : 0.0), end = last_lane(s);
        b_l[u][lane] = s;
        w_l[u][lane] = pow2(end - s);
        e_l[u][lane] = pow2(s) * a.scale;
        if (lane == 0) last_l[u] = pow2(end);
        total += end;
    };
    if (c0 < c1) {
        fetch(c0, threadIdx.x);
        if (wave == NW - 1) {
            scan(c0, decays(c0));
            gr = decays(c0 + 1);
        }
    }
    if (threadIdx.x == 0) bad_l = 0;
    for (int c = c0; c < c1; c++) {
        mk_wg_barrier();
        // (addresses are formed anew in every block: held across it they would not fit the registers)
        int n = lane & 15, g = lane >> 4, tid = threadIdx.x;
        asm volatile("" : "+v"(n), "+v"(g), "+v"(tid));
        const int rk = tid / (DK / E), rv = tid / (DV / E), dk0 = tid % (DK / E) * E, dv0 = tid % (DV / E) * E;
        bool ok = true;
        const int left = len - c * CH;  // tokens from this block on: behind them zeros, and no decay
        const mk_v4u zero = mk_v4u{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const int r = rk + i * (CH / KP);
            *(mk_v4u *)&k_l[r * LK + dk0] = r < left ? kr[i] : zero;
            if constexpr (OUT) store_q(&q_l[r * LQ], dk0, r < left ? qr[i] : zero);
        }
#pragma unroll
        for (int i = 0; i < VP; i++) {
            const int r = rv + i * (CH / VP);
            const mk_v4u x = r < left ? vr[i] : zero;
            *(mk_v4u *)&v_l[r * LV + dv0] = x;
            ok &= Op<T>::finite(x);
        }
        if (OUT && !ok) bad_l = c + 1;
        mk_wg_barrier();
        const int u = c & 1;
        if constexpr (OUT) {
            // scores: operand f = (query tile j, 32 keys from 32 s2 on); the masked half of a diagonal one is not computed
            for (int i = wave; i < 6; i += NW) {
                const int f = NW == 4 ? (0x405321 >> (4 * i)) & 15 : i;  // (of four waves: 1 + 0, 2 + 4, 3, 5)
                const int j = f < 4 ? f : f - 2, s2 = f < 4 ? 0 : 1;
                const double bq = b_l[u][16 * j + n];
                F qf[KS];
#pragma unroll
                for (int s = 0; s < KS; s++) qf[s] = row8(&q_l[(16 * j + n) * LQ + 32 * s + 8 * g]);
                mk_f4 pt[2];
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int i = 2 * s2 + v;
                    pt[v] = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (i <= j) {
#pragma unroll
                        for (int s = 0; s < KS; s++) pt[v] = Op<T>::mma(row44(&k_l[(16 * i + n) * LK + 32 * s + 4 * g]), qf[s], pt[v]);
#pragma unroll
                        for (int e = 0; e < 4; e++) pt[v][e] *= pow2(bq - b_l[u][16 * i + 4 * g + e]) * a.scale;
                        if (i == j) {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (4 * g + e > n) pt[v][e] = 0.0f;
                        }
                    }
                }
                F pf[OT];
                operand<T>(pt[0], pt[1], pf);
#pragma unroll
                for (int k = 0; k < OT; k++) p_l[k][f][lane] = pf[k];
            }
        }
        // (a wave with few or no scores forms the next block's sums)
        if (wave == NW - 1 && c + 1 < c1) scan(c + 1, gr), gr = decays(c + 2);
        if constexpr (OUT) mk_wg_barrier();
        __builtin_amdgcn_sched_barrier(0);
        F vt[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) vt[t][ks] = column8<LV>(v_l, ks, 16 * (NT * wave + t), g, n);
        if constexpr (OUT) {
            const bool plain = bad_l == c + 1;  // a value that is not finite: 0 times it must not reach earlier tokens
            mk_f4 o[NT][4];
#pragma unroll
            for (int s = 0; s < KS; s++) {
                F sf[NT][OT], qb[4];
#pragma unroll
                for (int t = 0; t < NT; t++) operand<T>(S[2 * s][t], S[2 * s + 1][t], sf[t]);
#pragma unroll
                for (int j = 0; j < 4; j++) qb[j] = row8(&q_l[(16 * j + n) * LQ + 32 * s + 8 * g]);
#pragma unroll
                for (int k = 0; k < OT; k++)  // several sums in turn
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int t = 0; t < NT; t++) o[t][j] = Op<T>::mma(sf[t][k], qb[j], s || k ? o[t][j] : mk_f4{0.0f, 0.0f, 0.0f, 0.0f});
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float e = e_l[u][16 * j + n];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[t][j][i] *= e;
            }
            if (!plain) {
#pragma unroll
                for (int k = 0; k < OT; k++)
#pragma unroll
                    for (int f = 0; f < 6; f++) {
                        const F pb = p_l[k][f][lane];
#pragma unroll
                        for (int t = 0; t < NT; t++) o[t][f < 4 ? f : f - 2] = Op<T>::mma(vt[t][f < 4 ? 0 : 1], pb, o[t][f < 4 ? f : f - 2]);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    for (int key = 0; key <= 16 * j + n; key++) {
                        const int r = key & 31;
                        float p = 0.0f;
#pragma unroll
                        for (int k = 0; k < OT; k++) p += (float)p_l[k][key < 32 ? j : 2 + j][16 * ((r & 15) >> 2) + n][4 * (r >> 4) + (r & 3)];
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) o[t][j][i] = fmaf(p, (float)v_l[key * LV + 16 * (NT * wave + t) + 4 * g + i], o[t][j][i]);
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int tok = c * CH + 16 * j + n;
                if (tok < len) {
                    T *dst = (T *)a.out + ((size_t)(t0 + tok) * a.nh + h) * dv + col0 + 16 * NT * wave + 4 * g;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const mk_f4 x = o[t][j];
                        if constexpr (sizeof(T) == 4) *(mk_f4 *)(dst + 16 * t) = x;
                        else *(mk_b4 *)(dst + 16 * t) = mk_b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (the phases' registers do not add up)
        if (c + 1 < c1) {
            int tid = threadIdx.x;
            asm volatile("" : "+v"(tid));
            fetch(c + 1, tid);
        }
        // the state behind the block
        if (MODE != OUTPUT || c + 1 < c1) {
            const float end = last_l[u];
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) S[kt][t][j] *= end;
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                F wv[NT][TERMS];
                float w[8];
                *(mk_f4 *)&w[0] = *(const mk_f4 *)&w_l[u][32 * ks + 4 * g];
                *(mk_f4 *)&w[4] = *(const mk_f4 *)&w_l[u][32 * ks + 16 + 4 * g];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float r[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) r[i] = (float)vt[t][ks][i] * w[i];
#pragma unroll
                    for (int k = 0; k < TERMS; k++)
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            wv[t][k][i] = (T)r[i];
                            r[i] -= (float)wv[t][k][i];
                        }
                }
#pragma unroll
                for (int kt = 0; kt < KT; kt += 2) {  // several sums in turn
                    F kf[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) kf[i] = column8<LK>(k_l, ks, 16 * (kt + i), g, n);
#pragma unroll
                    for (int k = 0; k < TERMS; k++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int t = 0; t < NT; t++) S[kt + i][t] = Op<T>::mma(kf[i], wv[t][k], S[kt + i][t]);
                }
            }
        }
    }
    if (MODE == OUTPUT) return;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (MODE == BOTH) {
#pragma unroll
                for (int j = 0; j < 4; j++) a.state_out[sbase + 16 * t + (size_t)(16 * kt + 4 * g + j) * dv] = S[kt][t][j];
            } else {
                mine[kt * (DV * 4) + 64 * t] = S[kt][t];
            }
        }
    if (MODE == LOCAL && threadIdx.x == TH - 1) sg.decay[sh] = pow2(total);
}

// Between the two passes over the segments: local states -> the states before each segment, and the state behind the last.  One
// workgroup: a tile of 16 rows of the state of (head, sequence).
template <int DK, int DV>
__global__ __launch_bounds__(DV * 4) void linear_carry_kernel(LinArgs a, LinSeg sg) {
    constexpr int KT = DK / 16, TH = DV * 4;
    const int kt = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const size_t bh = (size_t)b * a.nh + h, at = bh * DK * DV + (size_t)(16 * kt + 4 * g) * DV + 16 * wave + n;
    const int len = max(a.at(b + 1) - a.at(b), 0);
    mk_f4 S = mk_f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (a.state) {
#pragma unroll
        for (int j = 0; j < 4; j++) S[j] = a.state[at + (size_t)j * DV];
    }
    const size_t sh = (size_t)sg.first(a, b) * a.nh + h, step = (size_t)a.nh * KT * TH;
    mk_f4 *p = sg.local + (sh * KT + kt) * TH + threadIdx.x;
    const float *decay = sg.decay + sh;
    const int used = (len + CH * sg.per - 1) / (CH * sg.per);
    for (int s0 = 0; s0 < used; s0 += 8) {
        mk_f4 L[8];
        float E[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (s0 + i < used) L[i] = p[(s0 + i) * step], E[i] = decay[(size_t)(s0 + i) * a.nh];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (s0 + i < used) {
                p[(s0 + i) * step] = S;
#pragma unroll
                for (int j = 0; j < 4; j++) S[j] = fmaf(E[i], S[j], L[i][j]);
            }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) a.state_out[at + (size_t)j * DV] = S[j];
}

size_t least_segment(size_t T, size_t nh) {  // no call takes shorter ones: the workspace is measured by this
    const size_t per = ((T + CH - 1) / CH * nh + 511) / 512;
    return per < 2 ? 2 : per;
}
size_t slots(size_t T, size_t B, size_t per) { return T / (CH * per) + B; }
size_t segment_bytes(size_t n, size_t dk, size_t dv) { return n * dk * dv * 4 + mk_align_up(n * 4, 256); }  // of n (slot, head) pairs

// Blocks of a segment, 0: no segments.  Without them a (sequence, head) is one workgroup; with them the keys and values are read twice
// (local states first, then the outputs from the right states), and a long sequence beside short ones spreads over the device.
// As many as two workgroups a compute unit ask for (8192 tokens of 32 heads, with one-term operands: 118 us, as 768 or 1024 workgroups 132 and
// 136 us).  Equal lengths (no cu) are better off without from 192 heads on (bfloat16, 128 x 128; without / with): 192 heads of 1500 tokens 154 / 176 us,
// 176 heads 150 / 164, 160 heads 145 / 124, 128 heads 106 / 98; of 400 tokens 52 / 67, 48 / 64, 48 / 62 and 37 / 51 us, for which the bound is high.
// What cu holds is not known here: up to 256 heads it is taken for ragged (8 sequences of 24 heads, 1 .. 6000 tokens long: 340 us without, 137 with).
// A sequence needs four blocks on average, six of 128 bfloat16 columns, which two workgroups share when they are few (32 heads of 128 x 128
// without / with: 256 tokens 21 / 27 us, 400 tokens 33 / 31 us; in f32 256 tokens 44 / 46 us, 320 tokens 54 / 48 us).
// f32 heads wider than 64 x 64 leave room for one workgroup a compute unit: longer segments of equal sequences, so that all of them run at
// once (2048 tokens of 32 heads of 128 x 128: 91 us, in segments of two blocks 100; 3241 of 24 heads 123 and 132 us).  From 129 heads on that
// would be one segment a sequence, which is the work of the segments without their workgroups: none then (160 heads of 400 tokens without / one
// segment 99 / 140 us, of 4096 tokens 859 / 1167 us; 5 sequences of 32 heads of 1024 tokens 220 / 360 us).
int segment_blocks(size_t T, size_t B, size_t nh, size_t dk, size_t dv, bool bf16, bool ragged) {
    const size_t blocks = (T + CH - 1) / CH;
    if (B * nh > (ragged ? 256 : 191) || blocks < (bf16 && dv == 128 ? 6 : 4) * B) return 0;
    size_t per = least_segment(T, nh);
    if (!ragged && !bf16 && dk + dv > 128) {
        const size_t each = (T / B + CH - 1) / CH, most = 256 / (B * nh), even = (each + most - 1) / most;
        per = even > per ? even : per;
        if (per >= each) return 0;
    }
    return (int)per;
}
constexpr size_t SLICED = 128;
bool block_widths(size_t dk, size_t dv) { return (dk == 64 || dk == 128) && (dv == 64 || dv == 128); }

template <typename T, int DK, int DV>
int launch_blocks(const LinArgs &a, const LinSeg &sg, hipStream_t st) {
    const dim3 grid((unsigned)(a.nh * (sg.per ? slots(a.T, a.B, sg.per) : (size_t)a.B * a.slices)));
    int e;
    if (sg.per == 0) {
        hipLaunchKernelGGL((linear_block_kernel<T, DK, DV, BOTH>), grid, dim3(DV * 4 / tiles<T, DK, DV, BOTH>()), 0, st, a, sg);
        return mk_launch_status("linear_block");
    }
    hipLaunchKernelGGL((linear_block_kernel<T, DK, DV, LOCAL>), grid, dim3(DV * 4 / tiles<T, DK, DV, LOCAL>()), 0, st, a, sg);
    if ((e = mk_launch_status("linear_block")) != MK_OK) return e;
    hipLaunchKernelGGL((linear_carry_kernel<DK, DV>), dim3(DK / 16, (unsigned)a.nh, (unsigned)a.B), dim3(DV * 4), 0, st, a, sg);
    if ((e = mk_launch_status("linear_carry")) != MK_OK) return e;
    hipLaunchKernelGGL((linear_block_kernel<T, DK, DV, OUTPUT>), grid, dim3(DV * 4 / tiles<T, DK, DV, OUTPUT>()), 0, st, a, sg);
    return mk_launch_status("linear_block");
}
template <typename T>
int launch_blocks(LinArgs a, const LinSeg &sg, hipStream_t st) {
    // While heads leave compute units free, two workgroups share a head of 128 columns (128 x 128, one workgroup / two: 32 heads of 70 tokens f32 30 / 23,
    // bfloat16 15.6 / 12.1 us; 128 heads of 100 tokens 32 / 28 and 16.5 / 13.6 us; 192 heads 34 / 52 and 18 / 19 us)
    if (sg.per == 0 && a.dv == 128 && (size_t)a.B * a.nh <= SLICED) {
        a.slices = 2;
        return a.dk == 64 ? launch_blocks<T, 64, 64>(a, sg, st) : launch_blocks<T, 128, 64>(a, sg, st);
    }
    if (a.dk == 64) return a.dv == 64 ? launch_blocks<T, 64, 64>(a, sg, st) : launch_blocks<T, 64, 128>(a, sg, st);
    return a.dv == 64 ? launch_blocks<T, 128, 64>(a, sg, st) : launch_blocks<T, 128, 128>(a, sg, st);
}

int check_linear(int dtype, const void *q, size_t qs, const void *k, size_t ks, const void *v, size_t vs, const float *g, size_t gs, size_t T, size_t B,
                 size_t nh, size_t nkh, size_t dk, size_t dv, const float *state, const float *state_out, const void *out) {
    MK_REQUIRE(dtype == MK_F32 || dtype == MK_BF16, "dtype must be MK_F32 or MK_BF16");
    MK_REQUIRE(B >= 1 && B <= 65535 && T <= 0x3FFFFFFF, "bad token or sequence count");
    MK_REQUIRE(nh >= 1 && nh <= 65535 && nkh >= 1 && nh % nkh == 0, "the value heads must be a multiple of the key heads");
    MK_REQUIRE(dk >= 8 && dk <= 256 && dk % 8 == 0 && dv >= 8 && dv <= 256 && dv % 8 == 0, "head widths must be multiples of 8 up to 256");
    MK_REQUIRE(state_out && (T == 0 || (q && k && v && g && out)), "null pointer");
    MK_REQUIRE(qs % 8 == 0 && ks % 8 == 0 && vs % 8 == 0, "token strides must be multiples of 8 values");
    MK_REQUIRE(qs <= 0x7FFFFF && ks <= 0x7FFFFF && vs <= 0x7FFFFF, "a token stride is out of range");
    MK_REQUIRE(T <= 1 || (qs >= nkh * dk && ks >= nkh * dk && vs >= nh * dv && (gs == 0 || gs >= nh)), "a token stride is shorter than a token's heads");
    MK_REQUIRE(mk_aligned16(q) && mk_aligned16(k) && mk_aligned16(v) && mk_aligned16(out) && mk_aligned16(state) && mk_aligned16(state_out), "pointers must be 16-byte aligned");
    return MK_OK;
}

}  // namespace

extern "C" size_t mk_linear_attn_workspace_bytes(size_t T, size_t B, size_t nh, size_t dk, size_t dv) {
    if (!B || !nh || !block_widths(dk, dv)) return 0;
    const size_t n = B * nh <= 256 && (T + CH - 1) / CH >= 4 * B ? slots(T, B, least_segment(T, nh)) * nh : 0;
    return n ? segment_bytes(n, dk, dv) : 0;
}

extern "C" int mk_dev_linear_attn(int dtype, const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v, size_t v_stride, const float *g,
                                  size_t g_stride, size_t T, const int32_t *cu, size_t B, size_t nh, size_t nkh, size_t dk, size_t dv, float scale,
                                  const float *state, float *state_out, void *workspace, void *out, void *stream) {
    int st = check_linear(dtype, q, q_stride, k, k_stride, v, v_stride, g, g_stride, T, B, nh, nkh, dk, dv, state, state_out, out);
    if (st != MK_OK) return st;
    MK_REQUIRE(cu || T % B == 0, "without cu every sequence has the same number of tokens");
    MK_REQUIRE((workspace || mk_linear_attn_workspace_bytes(T, B, nh, dk, dv) == 0) && ((uintptr_t)workspace & 255) == 0, "the workspace must be 256-byte aligned");
    const LinArgs a{q, k, v, q_stride, k_stride, v_stride, g, g_stride, cu, (int)T, (int)B, (int)nh, (int)nkh, (int)dk, (int)dv, scale, state, state_out, out, 1};
    hipStream_t hs = (hipStream_t)stream;
    if (!block_widths(dk, dv)) return dtype == MK_F32 ? launch_token<float>(a, hs) : launch_token<__bf16>(a, hs);
    LinSeg sg{segment_blocks(T, B, nh, dk, dv, dtype == MK_BF16, cu != nullptr), (mk_f4 *)workspace, nullptr};
    const size_t n = (sg.per ? slots(T, B, sg.per) : B) * nh;
    sg.decay = sg.per ? (float *)((uint8_t *)workspace + n * dk * dv * 4) : nullptr;
    MK_REQUIRE(n <= MAX_GROUPS / 2, "too many heads and sequences in one call");
    MK_REQUIRE(sg.per == 0 || segment_bytes(n, dk, dv) <= mk_linear_attn_workspace_bytes(T, B, nh, dk, dv), "segments beyond the workspace");
    return dtype == MK_F32 ? launch_blocks<float>(a, sg, hs) : launch_blocks<__bf16>(a, sg, hs);
}

extern "C" int mk_dev_linear_attn_step(int dtype, const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v, size_t v_stride,
                                       const float *g, size_t g_stride, size_t B, size_t nh, size_t nkh, size_t dk, size_t dv, float scale,
                                       const float *state, float *state_out, void *out, void *stream) {
    int st = check_linear(dtype, q, q_stride, k, k_stride, v, v_stride, g, g_stride, B, B, nh, nkh, dk, dv, state, state_out, out);
    if (st != MK_OK) return st;
    const LinArgs a{q, k, v, q_stride, k_stride, v_stride, g, g_stride, nullptr, (int)B, (int)B, (int)nh, (int)nkh, (int)dk, (int)dv, scale, state, state_out, out, 1};
    return dtype == MK_F32 ? launch_step<float, 16>(a, (hipStream_t)stream) : launch_step<__bf16, 16>(a, (hipStream_t)stream);
}
