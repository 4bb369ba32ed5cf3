// Shared by the token-mixer kernels: row loads, the sequences of a call, the 4-bit cache as the kernels see it.
#pragma once
#include "mk_common.h"

typedef __bf16 mk_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 mk_b2 __attribute__((ext_vector_type(2)));

constexpr size_t MAX_GROUPS = 0xFFFFFF;  // workgroups of 256 threads in one dimension of a grid, which has 2^32 threads

static inline size_t mk_align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
static inline bool mk_aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Workgroup barrier that waits for this wave's LDS traffic only: __syncthreads() waits for the global loads in flight too, which would put
// the latency of the next step's prefetch into every barrier.
__device__ __forceinline__ void mk_wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename T> __device__ __forceinline__ void mk_load8(const T *p, float (&v)[8]) {
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
struct MkSeqs {
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

struct MkKv4 {
    uint8_t *kq, *ks, *vq, *vs;
    uint16_t *kr;
    int32_t *lens;
    int B, nkv, dk, rope, dv, cap;
};

static inline int mk_kv4_check(const mk_kv4_cache *c) {
    MK_REQUIRE(c && c->kq && c->ks && c->vq && c->vs && c->lens && (c->kr || c->rope == 0), "null pointer");
    MK_REQUIRE(c->B >= 1 && c->B <= 65535 && c->nkv >= 1 && c->nkv <= 65535, "bad sequence or head count");
    MK_REQUIRE(c->dk >= 32 && c->dk <= 512 && c->dk % 32 == 0 && c->dv >= 32 && c->dv <= 512 && c->dv % 32 == 0, "K and V widths must be multiples of 32 up to 512");
    MK_REQUIRE(c->rope % 8 == 0 && c->rope <= 64, "the shared K tail must be a multiple of 8 up to 64");
    MK_REQUIRE(c->cap >= 1 && c->cap <= 0x7FFFFFull, "capacity out of range (at most 8388607 positions)");
    MK_REQUIRE(mk_aligned16(c->kq) && mk_aligned16(c->vq) && mk_aligned16(c->kr) && mk_aligned16(c->ks) && mk_aligned16(c->vs), "cache arrays must be 16-byte aligned");
    return MK_OK;
}
static inline MkKv4 mk_kv4_view(const mk_kv4_cache *c) {
    return MkKv4{c->kq, c->ks, c->vq, c->vs, c->kr, c->lens, (int)c->B, (int)c->nkv, (int)c->dk, (int)c->rope, (int)c->dv, (int)c->cap};
}
static inline int mk_kv4_check_rows(const mk_kv4_cache *c, int dtype, size_t T, const int32_t *cu) {
    MK_REQUIRE(dtype == MK_F32 || dtype == MK_BF16, "dtype must be MK_F32 or MK_BF16");
    MK_REQUIRE(T <= 0x3FFFFF, "at most 4194303 rows per call");
    MK_REQUIRE(cu || T % c->B == 0, "without cu every sequence has the same number of rows");
    return MK_OK;
}
