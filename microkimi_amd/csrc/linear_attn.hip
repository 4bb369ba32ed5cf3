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
    __device__ __forceinline__ int at(int b) const { return cu ? min(max(cu[b], 0), T) : (int)((int64_t)T / B * b); }
};

// ------------------------------------------------------------------------------------------------ token by token
//
// One workgroup: (64 columns of dv, value head, sequence).  Thread (rg, cg) = (tid / 16, tid % 16) holds rows rg + 16 i,
// columns 4 cg .. 4 cg + 3 of the slice in registers: the state is read and written once, in runs of 256 bytes.  The tokens'
// rows go through LDS, STAGE at a time.
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

template <typename T>
int launch_token(const LinArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.dv + COLS - 1) / COLS), (unsigned)a.nh, (unsigned)a.B);
    if (a.dk <= 64) hipLaunchKernelGGL((linear_token_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else if (a.dk <= 128) hipLaunchKernelGGL((linear_token_kernel<T, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((linear_token_kernel<T, 16>), grid, dim3(256), 0, st, a);
    return mk_launch_status("linear_token");
}


int check_linear(int dtype, const void *q, size_t qs, const void *k, size_t ks, const void *v, size_t vs, const float *g, size_t gs, size_t T, size_t B,
                 size_t nh, size_t nkh, size_t dk, size_t dv, const float *state, const float *state_out, const void *out) {
    MK_REQUIRE(dtype == MK_F32 || dtype == MK_BF16, "dtype must be MK_F32 or MK_BF16");
    MK_REQUIRE(B >= 1 && B <= 65535 && T <= 0x3FFFFFFF, "bad token or sequence count");
    MK_REQUIRE(nh >= 1 && nh <= 65535 && nkh >= 1 && nh % nkh == 0, "the value heads must be a multiple of the key heads");
    MK_REQUIRE(dk >= 8 && dk <= 256 && dk % 8 == 0 && dv >= 8 && dv <= 256 && dv % 8 == 0, "head widths must be multiples of 8 up to 256");
    MK_REQUIRE(g && state_out && (T == 0 || (q && k && v && out)), "null pointer");
    MK_REQUIRE(qs % 8 == 0 && ks % 8 == 0 && vs % 8 == 0, "token strides must be multiples of 8 values");
    MK_REQUIRE(T <= 1 || (qs >= nkh * dk && ks >= nkh * dk && vs >= nh * dv && (gs == 0 || gs >= nh)), "a token stride is shorter than a token's heads");
    MK_REQUIRE(mk_aligned16(q) && mk_aligned16(k) && mk_aligned16(v) && mk_aligned16(out) && mk_aligned16(state) && mk_aligned16(state_out), "pointers must be 16-byte aligned");
    return MK_OK;
}

}  // namespace

extern "C" size_t mk_linear_attn_workspace_bytes(size_t T, size_t B, size_t nh, size_t dk, size_t dv) {
    (void)T, (void)B, (void)nh, (void)dk, (void)dv;
    return 256;
}

extern "C" int mk_dev_linear_attn(int dtype, const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v, size_t v_stride, const float *g,
                                  size_t g_stride, size_t T, const int32_t *cu, size_t B, size_t nh, size_t nkh, size_t dk, size_t dv, float scale,
                                  const float *state, float *state_out, void *workspace, void *out, void *stream) {
    int st = check_linear(dtype, q, q_stride, k, k_stride, v, v_stride, g, g_stride, T, B, nh, nkh, dk, dv, state, state_out, out);
    if (st != MK_OK) return st;
    MK_REQUIRE(cu || T % B == 0, "without cu every sequence has the same number of tokens");
    MK_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "the workspace must be 256-byte aligned");
    const LinArgs a{q, k, v, q_stride, k_stride, v_stride, g, g_stride, cu, (int)T, (int)B, (int)nh, (int)nkh, (int)dk, (int)dv, scale, state, state_out, out};
    return dtype == MK_F32 ? launch_token<float>(a, (hipStream_t)stream) : launch_token<__bf16>(a, (hipStream_t)stream);
}

extern "C" int mk_dev_linear_attn_step(int dtype, const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v, size_t v_stride,
                                       const float *g, size_t g_stride, size_t B, size_t nh, size_t nkh, size_t dk, size_t dv, float scale,
                                       const float *state, float *state_out, void *out, void *stream) {
    int st = check_linear(dtype, q, q_stride, k, k_stride, v, v_stride, g, g_stride, B, B, nh, nkh, dk, dv, state, state_out, out);
    if (st != MK_OK) return st;
    const LinArgs a{q, k, v, q_stride, k_stride, v_stride, g, g_stride, nullptr, (int)B, (int)B, (int)nh, (int)nkh, (int)dk, (int)dv, scale, state, state_out, out};
    return dtype == MK_F32 ? launch_token<float>(a, (hipStream_t)stream) : launch_token<__bf16>(a, (hipStream_t)stream);
}
