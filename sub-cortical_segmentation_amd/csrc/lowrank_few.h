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
// One row, 4096 x 4096, bf16: 10.5 us (3.2 TB/s) behind 4.7 us of shrink; 48 rows, 2048 x 8192, f16, 24 adapters of rank 32: 18.3 us.  W's own
// time at a copy's rate is 6.5 us of either; the rest is the start, the adapters' dependent loads and the join.  Half as many workgroups along
// the contraction: 14.3 for 14.5 us and 28 for 21.5; twice as many: 17.4 and 29.
#pragma once
#include "scs_ops.h"
#include "lowrank_rules.h"
#include "lowrank_tiles.h"

namespace scs {
namespace {

// Partial sums travel past the L2s (one per XCD): written through to, and read from, the memory that all of them share (cache policy sc0 sc1),
// so that no cache has to be written back or emptied around the ticket.  A store is there once it is acknowledged (vmcnt).
constexpr int kCoherent = 1 | 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_buffer(float* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void coherent_store(__amdgpu_buffer_rsrc_t b, int at, const f32x4& v) {
    u32x4 u;
    __builtin_memcpy(&u, &v, 16);
    __builtin_amdgcn_raw_buffer_store_b128(u, b, at * 4, 0, kCoherent);
}
__device__ __forceinline__ f32x4 coherent_load(__amdgpu_buffer_rsrc_t b, int at) {
    const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(b, at * 4, 0, kCoherent);
    f32x4 v;
    __builtin_memcpy(&v, &u, 16);
    return v;
}
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// where four columns from n on can be read from any row but W's last one (from the last one as well where N % 4 == 0)
__device__ __forceinline__ int few_column(int n, int N) { return min(n, N % 4 ? N - 1 : N - 4); }

// one step of the contraction: 32 (16-bit) or 16 (f32) values, four products of sixteen columns
template <class T, int MT, bool TRANS> struct FewStep;
template <class T, int MT, bool TRANS> struct FewStep16 {
    static constexpr int K = 32;
    typedef typename Frag<T>::v8 v8;
    u32x4 x[MT];
    u32x2 w[TRANS ? 1 : 8];
    u32x4 wt[TRANS ? 4 : 1];
    // rows and columns beyond the matrices are read as their last ones (nobody keeps what comes of them); only the last step looks at every element
    __device__ __forceinline__ void load(const ProjectArgs<T>& g, int m0, int n, int k0, int lr, int kq, bool inside) {
        const int k = k0 + 8 * kq;
        if (inside) {
#pragma unroll
            for (int i = 0; i < MT; ++i) x[i] = at16(g.x + (int64_t)min(m0 + 16 * i + lr, g.r.rows - 1) * g.ldx + k);
            if constexpr (TRANS) {
#pragma unroll
                for (int t = 0; t < 4; ++t) wt[t] = at16(g.w + (int64_t)min(n + t, g.N - 1) * g.ldw + k);
            } else {
                const T* p = g.w + (int64_t)k * g.ldw + few_column(n, g.N);
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = at4(p + i * g.ldw);
            }
            return;
        }
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
    __device__ __forceinline__ void load(const ProjectArgs<float>& g, int m0, int n, int k0, int lr, int kq, bool inside) {
        const int k = k0 + 4 * kq;
        if (inside) {
#pragma unroll
            for (int i = 0; i < MT; ++i) x[i] = at4(g.x + (int64_t)min(m0 + 16 * i + lr, g.r.rows - 1) * g.ldx + k);
            const float* p = TRANS ? g.w + k : g.w + (int64_t)k * g.ldw + few_column(n, g.N);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = at4(TRANS ? p + (int64_t)min(n + i, g.N - 1) * g.ldw : p + i * g.ldw);
            return;
        }
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

// sixteen consecutive elements (zeros behind `left`)
template <class T> struct Cols16 {
    u32x4 v[sizeof(T)];
    __device__ __forceinline__ void load(const T* p, int left) {
        constexpr int PER = 16 / sizeof(T);
        if (left >= 16) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) v[i] = reinterpret_cast<const Loose<u32x4>*>(p + i * PER)->v;
            return;
        }
        T e[16] = {};
#pragma unroll
        for (int i = 0; i < 15; ++i) if (i < left) e[i] = p[i];
        __builtin_memcpy(v, e, sizeof(v));
    }
    __device__ __forceinline__ void four(int q, float (&f)[4]) const {
        T e[16];
        __builtin_memcpy(e, v, sizeof(v));
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = to_f32(e[4 * q + i]);
    }
};

// LDS of the join: [wave][row][16 columns' quarters + 1], so that neither side of it meets a bank twice
template <int MT> struct FewShared { f32x4 part[kFewWaves][MT * 16][17]; bool last; };
struct FewGrid { int tiles_n, tiles_m, splits; };

// workgroup `id` of grid.tiles_n x grid.tiles_m x grid.splits
template <class T, int MT, bool TRANS>
__device__ __forceinline__ void project_few(const ProjectArgs<T>& g, const int* __restrict__ row_adapter, const FewGrid& grid, float* part, unsigned int* tickets, int id,
                                            FewShared<MT>& sh) {
    typedef FewStep<T, MT, TRANS> Step;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4;
    const int bn = id % grid.tiles_n, bm = id / grid.tiles_n % grid.tiles_m, split = id / (grid.tiles_n * grid.tiles_m), splits = grid.splits;
    const int n0 = bn * 64, m0 = bm * MT * 16;
    const Requests& r = g.r;

    f32x4 acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int steps = (g.K + Step::K - 1) / Step::K, shares = splits * kFewWaves, share = split * kFewWaves + wave;
    const int s0 = (int)((int64_t)steps * share / shares), s1 = (int)((int64_t)steps * (share + 1) / shares);
    // (columns beyond N in W's last but one row run into its last one, which a stride of four and more covers)
    const int inside = TRANS ? g.K : g.ldw < 4 || g.N < 4 ? 0 : g.N % 4 ? g.K - 1 : g.K;
    constexpr int AHEAD = 3;
    Step st[AHEAD + 1];
    int adapter[MT];                                       // of row lr: -2 outside the requests, -1 none
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) if (s0 + i < s1) st[i].load(g, m0, n0 + 4 * lr, (s0 + i) * Step::K, lr, kq, (s0 + i + 1) * Step::K <= inside);
#pragma unroll
    for (int i = 0; i < MT; ++i) adapter[i] = m0 + 16 * i + lr < r.rows ? row_adapter[m0 + 16 * i + lr] : -2;
    // adapters: this wave's directions, one or two at a time, each row under its own adapter (the loads of all rows in flight together)
    constexpr int U = sizeof(T) == 4 || MT == 4 ? 1 : 2;               // (two of these would not fit the registers)
    for (int j0 = share; j0 < r.rank; j0 += U * shares) {
        float h[U][MT];
        Cols16<T> p[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int j = j0 + u * shares, m = min(m0 + 16 * i + lr, r.rows - 1);
                const bool on = adapter[i] >= 0 && j < r.rank;
                const int s = on ? adapter[i] : 0;
                h[u][i] = on ? (r.scale ? r.scale[s] : 1.f) * g.h[(int64_t)m * r.rank + j] : 0.f;
                p[u][i].load(g.low + ((int64_t)s * r.rank + (on ? j : 0)) * g.N + n0 + 16 * kq, on ? g.N - (n0 + 16 * kq) : 0);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float f[4];
                    p[u][i].four(e, f);
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[i][t][e] = fmaf(h[u][i], f[t], acc[i][t][e]);          // (0 x 0 where a row takes no part)
                }
    }

    for (int s = s0; s < s1; s += AHEAD + 1) {
#pragma unroll
        for (int i = 0; i <= AHEAD; ++i) {
            const int next = s + i + AHEAD;
            if (next < s1) st[(i + AHEAD) % (AHEAD + 1)].load(g, m0, n0 + 4 * lr, next * Step::K, lr, kq, (next + 1) * Step::K <= inside);
            if (s + i < s1) st[i].run(acc);
        }
    }

    // this lane holds row lr, columns 16 kq + 4 e + t; behind the join a lane holds four columns of a row and sixteen lanes 64 of them, so that
    // stores are whole lines (as the sums lie in the registers they would be 16-byte pieces: 26 us a call instead of 14 at 48 rows, 2048 x 8192, f16)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh.part[wave][i * 16 + lr][4 * kq + e] = f32x4{acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
    __syncthreads();
    const int ldp = grid.tiles_n * 64, plane = grid.tiles_m * MT * 16 * ldp;               // partial sums of one split, whole tiles
    const __amdgpu_buffer_rsrc_t pb = part_buffer(part, (int64_t)splits * plane * 4);
    auto finish = [&](f32x4 v, int m, int n) {
        float b[4] = {};
        if (g.bias) {
            typename Vec4<T>::raw rb;
            raw_load<T>(rb, g.bias + n, g.N - n);
            unpack<T>(rb, b);
        }
        const float f[4] = {v[0] + b[0], v[1] + b[1], v[2] + b[2], v[3] + b[3]};
        raw_store<T>(pack<T>(f), g.y + (int64_t)m * g.ldy + n, g.N - n);
    };
    const int c4 = tid & 15, n = n0 + 4 * c4;
    for (int row = tid >> 4; row < MT * 16; row += 4 * kFewWaves) {
        const int m = m0 + row;
        if (m >= r.rows || n >= g.N || row_adapter[m] == -2) continue;
        f32x4 v = sh.part[0][row][c4];
#pragma unroll
        for (int w = 1; w < kFewWaves; ++w) v += sh.part[w][row][c4];
        if (splits == 1) finish(v, m, n);
        else coherent_store(pb, split * plane + m * ldp + n, v);
    }
    if (splits == 1) return;
    stores_done();
    __syncthreads();
    if (tid == 0)
        sh.last = __hip_atomic_fetch_add(&tickets[bm * grid.tiles_n + bn], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned int)splits - 1;
    __syncthreads();
    if (!sh.last) return;
    for (int row = tid >> 4; row < MT * 16; row += 4 * kFewWaves) {
        const int m = m0 + row;
        if (m >= r.rows || n >= g.N || row_adapter[m] == -2) continue;
        f32x4 v = coherent_load(pb, m * ldp + n);
#pragma unroll 8
        for (int i = 1; i < splits; ++i) v += coherent_load(pb, i * plane + m * ldp + n);
        finish(v, m, n);
    }
}

template <class T, int MT, bool TRANS>
__global__ __launch_bounds__(64 * kFewWaves) void project_few_kernel(ProjectArgs<T> g, const int* __restrict__ row_adapter, FewGrid grid, float* part, unsigned int* tickets) {
    __shared__ FewShared<MT> sh;
    project_few<T, MT, TRANS>(g, row_adapter, grid, part, tickets, blockIdx.x, sh);
}

}  // namespace
}  // namespace scs
