// The shared projection for few rows (scs_lowrank.hip): one new token of each request, a mini-batch of the dense head.
//
// Reading W once is the work: a workgroup of eight waves owns 16 MT rows x 64 columns, the contraction is dealt over its waves (and, where the
// tiles alone do not fill the card, over `splits` workgroups), and every wave runs its share from global memory straight into the matrix
// cores.  A lane loads four consecutive columns of a row of W (8 or 16 bytes; a wave: whole 128- or 256-byte lines); column 4 c + t of the tile
// is row c of matrix product t, so that no element changes lanes: 16-bit operands take their eight contraction values from eight such loads by
// byte permutes.  A lane ends with 16 consecutive columns of one row.
// The adapters' directions are dealt over the waves the same way: each adds scale_s H[row][j] P_s[j][..] for its j to its own sums, row by row
// with the row's own adapter.  The waves join through LDS, the workgroups through f32 partial sums and a ticket: the last one adds them
// up in their order, so the result does not depend on which one that is.
#pragma once
#include "scs_ops.h"
#include "lowrank_mfma16.h"

namespace scs {
namespace {

// what a coherent store has written is visible to every XCD once it is acknowledged: no cache has to be written back for it
__device__ __forceinline__ void coherent_store(float* p, const f32x4& v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) __hip_atomic_store(p + i, v[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 coherent_load(const float* p) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return v;
}
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

constexpr int kFewWaves = 8;

// one step of the contraction: 32 (16-bit) or 16 (f32) values, four products of sixteen columns
template <class T, int MT, bool TRANS> struct FewStep;
template <class T, int MT, bool TRANS> struct FewStep16 {
    static constexpr int K = 32;
    typedef typename Frag<T>::v8 v8;
    u32x4 x[MT];
    u32x2 w[TRANS ? 1 : 8];
    u32x4 wt[TRANS ? 4 : 1];
    __device__ __forceinline__ void load(const ProjectArgs<T>& g, int m0, int n, int k0, int lr, int kq) {
        const int k = k0 + 8 * kq;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = m0 + 16 * i + lr;
            x[i] = load8(g.x + (int64_t)m * g.ldx + k, m < g.r.rows ? g.K - k : 0);
        }
        if constexpr (TRANS) {
#pragma unroll
            for (int t = 0; t < 4; ++t) wt[t] = load8(g.w + (int64_t)(n + t) * g.ldw + k, n + t < g.N ? g.K - k : 0);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) raw_load<T>(w[i], g.w + (int64_t)(k + i) * g.ldw + n, k + i < g.K ? g.N - n : 0);
        }
    }
    __device__ __forceinline__ void run(f32x4 (&acc)[MT][4]) const {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            u32x4 a;
            if constexpr (TRANS) a = wt[t];
            else
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    a[p] = __builtin_amdgcn_perm(w[2 * p + 1][t >> 1], w[2 * p][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            v8 av, bv;
            __builtin_memcpy(&av, &a, 16);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                __builtin_memcpy(&bv, &x[i], 16);
                acc[i][t] = mfma16(av, bv, acc[i][t]);
            }
        }
    }
};
template <int MT, bool TRANS> struct FewStep<__bf16, MT, TRANS> : FewStep16<__bf16, MT, TRANS> {};
template <int MT, bool TRANS> struct FewStep<_Float16, MT, TRANS> : FewStep16<_Float16, MT, TRANS> {};
template <int MT, bool TRANS> struct FewStep<float, MT, TRANS> {
    static constexpr int K = 16;
    f32x4 x[MT], w[4];
    __device__ __forceinline__ void load(const ProjectArgs<float>& g, int m0, int n, int k0, int lr, int kq) {
        const int k = k0 + 4 * kq;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = m0 + 16 * i + lr;
            raw_load<float>(x[i], g.x + (int64_t)m * g.ldx + k, m < g.r.rows ? g.K - k : 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (TRANS) raw_load<float>(w[i], g.w + (int64_t)(n + i) * g.ldw + k, n + i < g.N ? g.K - k : 0);
            else raw_load<float>(w[i], g.w + (int64_t)(k + i) * g.ldw + n, k + i < g.K ? g.N - n : 0);
        }
    }
    __device__ __forceinline__ void run(f32x4 (&acc)[MT][4]) const {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(TRANS ? w[t][s] : w[s][t], x[i][s], acc[i][t], 0, 0, 0);
    }
};

template <class T, int MT, bool TRANS>
__global__ __launch_bounds__(64 * kFewWaves) void project_few_kernel(ProjectArgs<T> g, int splits, float* part, unsigned int* tickets) {
    typedef FewStep<T, MT, TRANS> Step;
    __shared__ f32x4 s_part[kFewWaves][MT * 4][64];
    __shared__ int s_adapter[MT * 16];
    __shared__ bool s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 64, m0 = blockIdx.y * MT * 16, split = blockIdx.z;
    const Requests& r = g.r;

    // the rows' adapters: -2 behind or before the requests, -1 none
    if (tid < MT * 16) s_adapter[tid] = -2;
    __syncthreads();
    const int m1 = min(m0 + MT * 16, r.rows);
    for (int q = first_request(r, m0) + tid; q < r.n && r.offsets[q] < m1; q += 64 * kFewWaves) {
        const Span sp = span_of(r, q, m0, m1);
        for (int m = sp.lo; m < sp.hi; ++m) s_adapter[m - m0] = sp.s;
    }

    f32x4 acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int steps = (g.K + Step::K - 1) / Step::K, shares = splits * kFewWaves, share = split * kFewWaves + wave;
    const int s0 = (int)((int64_t)steps * share / shares), s1 = (int)((int64_t)steps * (share + 1) / shares);
    {
        constexpr int AHEAD = MT <= 2 ? 2 : 1;
        Step st[AHEAD + 1];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) if (s0 + i < s1) st[i].load(g, m0, n0 + 4 * lr, (s0 + i) * Step::K, lr, kq);
        for (int s = s0; s < s1; s += AHEAD + 1) {
#pragma unroll
            for (int i = 0; i <= AHEAD; ++i) {
                if (s + i + AHEAD < s1) st[(i + AHEAD) % (AHEAD + 1)].load(g, m0, n0 + 4 * lr, (s + i + AHEAD) * Step::K, lr, kq);
                if (s + i < s1) st[i].run(acc);
            }
        }
    }

    // adapters: this wave's directions
    __syncthreads();
    for (int j = share; j < r.rank; j += shares) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = m0 + 16 * i + lr, s = s_adapter[16 * i + lr];
            if (s < 0) continue;
            const float h = (r.scale ? r.scale[s] : 1.f) * g.h[(int64_t)m * r.rank + j];
            const T* p = g.low + ((int64_t)s * r.rank + j) * g.N + n0 + 16 * kq;
            const int left = g.N - (n0 + 16 * kq);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                typename Vec4<T>::raw rp;
                raw_load<T>(rp, p + 4 * e, left - 4 * e);
                float f[4];
                unpack<T>(rp, f);
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[i][t][e] = fmaf(h, f[t], acc[i][t][e]);
            }
        }
    }

    // row lr, columns 16 kq + 4 e + t of this lane
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_part[wave][i * 4 + e][lane] = f32x4{acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
    __syncthreads();
    const int64_t plane = (int64_t)gridDim.y * MT * 16 * gridDim.x * 64;             // partial sums of one split, whole tiles
    const int ldp = gridDim.x * 64;
    auto finish = [&](f32x4 v, int m, int n, int s) {
        if (s == -2 || m >= r.rows || n >= g.N) return;
        float b[4] = {};
        if (g.bias) {
            typename Vec4<T>::raw rb;
            raw_load<T>(rb, g.bias + n, g.N - n);
            unpack<T>(rb, b);
        }
        const float f[4] = {v[0] + b[0], v[1] + b[1], v[2] + b[2], v[3] + b[3]};
        raw_store<T>(pack<T>(f), g.y + (int64_t)m * g.ldy + n, g.N - n);
    };
    for (int e = wave; e < MT * 4; e += kFewWaves) {
        f32x4 v = s_part[0][e][lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; ++w) v += s_part[w][e][lane];
        const int mi = (e >> 2) * 16 + lr, n = n0 + 16 * kq + 4 * (e & 3);
        if (splits == 1) finish(v, m0 + mi, n, s_adapter[mi]);
        else coherent_store(part + split * plane + (int64_t)(m0 + mi) * ldp + n, v);
    }
    if (splits == 1) return;
    stores_done();
    __syncthreads();
    if (tid == 0)
        s_last = __hip_atomic_fetch_add(&tickets[blockIdx.y * gridDim.x + blockIdx.x], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned int)splits - 1;
    __syncthreads();
    if (!s_last) return;
    for (int e = wave; e < MT * 4; e += kFewWaves) {
        const int mi = (e >> 2) * 16 + lr, n = n0 + 16 * kq + 4 * (e & 3);
        if (s_adapter[mi] == -2) continue;
        const float* p = part + (int64_t)(m0 + mi) * ldp + n;
        f32x4 v = coherent_load(p);
#pragma unroll 4
        for (int s = 1; s < splits; ++s) v += coherent_load(p + s * plane);
        finish(v, m0 + mi, n, s_adapter[mi]);
    }
}

}  // namespace
}  // namespace scs
