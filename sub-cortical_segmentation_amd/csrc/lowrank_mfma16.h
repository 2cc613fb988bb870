// The shared projection on the 16-bit matrix cores (scs_lowrank.hip): Y = X W' + scale_s H P_s for bf16 and f16.
//
// D is formed transposed (A operand = weights, B operand = rows of X: v_mfma_f32_16x16x32), so that a lane holds four consecutive columns of
// one row.  A workgroup owns BM x BN of Y; both operands pass through LDS in slabs of 64 along the contraction, double buffered, copied global ->
// LDS in 16-byte pieces without a register between (ALIGNED) or through registers (rows that start at any element).
// LDS images, 16-byte pieces swizzled so that a fragment's lanes meet no bank twice:
//   K-major  [row][64]: piece c of a row lies at c ^ (row & 7).  X always; W' where it is W^T (backward: W's rows run along the contraction)
//   N-major  [64][BN]:  32-byte unit u of row k lies at u ^ f(k), f = (k & 3) | (k >> 3 & 1) << 2.  W (forward) and the adapters' P: the transposing
//            LDS read (ds_read_b64_tr_b16) turns four rows of sixteen columns into each column's four contraction values
#pragma once
#include "scs_ops.h"

namespace scs {
namespace {

__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};            // what lies behind the end of the contraction

// eight elements at any element alignment, zeros behind `left`
template <class T> __device__ __forceinline__ u32x4 load8(const T* p, int64_t left) {
    if (left >= 8) return reinterpret_cast<const Loose<u32x4>*>(p)->v;
    T e[8] = {};
    for (int i = 0; i < 7; ++i) if (i < left) e[i] = p[i];
    u32x4 r;
    __builtin_memcpy(&r, e, 16);
    return r;
}

// four contraction values of this lane's column out of the transposing read
__device__ __forceinline__ s16x4 lds_transposed(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// tile: (WM x WN) waves of (16 MT x 16 NT)
template <class T, int WM, int WN, int MT, int NT, bool TRANS, bool ALIGNED>
__global__ __launch_bounds__(64 * WM * WN) void project16_kernel(ProjectArgs<T> g) {
    typedef typename Frag<T>::v8 v8;
    constexpr int THREADS = 64 * WM * WN, BM = WM * MT * 16, BN = WN * NT * 16, BK = 64;
    constexpr int A_IT = BM * 8 / THREADS, B_IT = BN * 8 / THREADS, NP = BN / 8;       // pieces a thread moves; pieces of an N-major row
    static_assert(THREADS / NP == 16 && THREADS % 64 == 0, "the swizzle of a thread's pieces must not depend on the pass");
    __shared__ __attribute__((aligned(16))) T s_a[2][BM * BK];
    __shared__ __attribute__((aligned(16))) T s_b[2][BN * BK];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4, wm = wave / WN, wn = wave % WN;
    const Requests& r = g.r;

    // workgroups are dealt to the eight XCDs in turn: give each XCD a run of neighbouring tiles, eight row tiles high, so that its L2
    // serves W's columns and X's rows again
    int m0, n0;
    {
        const int tm = (r.rows + BM - 1) / BM, tn = (g.N + BN - 1) / BN, total = tm * tn, pid = blockIdx.x;
        const int xcd = pid & 7, each = total >> 3, rest = total & 7;
        const int t = xcd * each + min(xcd, rest) + (pid >> 3);
        const int band = t / (8 * tn), in = t - band * 8 * tn, high = min(8, tm - band * 8);
        m0 = (band * 8 + in % high) * BM;
        n0 = in / high * BN;
    }

    const int pa = (tid & 7) ^ ((tid >> 3) & 7);                        // K-major: the piece of its row that this thread moves
    const int kb = tid / NP, fb = (kb & 3) | ((kb >> 3) & 1) << 2;      // N-major: its first row, that row's swizzle ...
    const int pb = ((((tid % NP) >> 1) ^ fb) << 1) | (tid & 1);         // ... and the piece
    const T* ga[A_IT];
    const T* gb[B_IT];
#pragma unroll
    for (int i = 0; i < A_IT; ++i) ga[i] = g.x + (int64_t)min(m0 + (tid >> 3) + i * (THREADS / 8), r.rows - 1) * g.ldx + pa * 8;
#pragma unroll
    for (int i = 0; i < B_IT; ++i) {
        if constexpr (TRANS) gb[i] = g.w + (int64_t)min(n0 + (tid >> 3) + i * (THREADS / 8), g.N - 1) * g.ldw + pa * 8;
        else gb[i] = g.w + (int64_t)(kb + 16 * i) * g.ldw + (ALIGNED ? min(n0 + pb * 8, g.N - 8) : n0 + pb * 8);
    }

    u32x4 ra[ALIGNED ? 1 : A_IT], rb[ALIGNED ? 1 : B_IT];
    auto fetch = [&](int k0, int buf) {
        const T* zero = (const T*)&kZeroPiece;
#pragma unroll
        for (int i = 0; i < A_IT; ++i) {
            if constexpr (ALIGNED)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(k0 + pa * 8 < g.K ? ga[i] + k0 : zero),
                                                 (__attribute__((address_space(3))) void*)&s_a[buf][(i * THREADS + wave * 64) * 8], 16, 0, 0);
            else ra[i] = load8(ga[i] + k0, m0 + (tid >> 3) + i * (THREADS / 8) < r.rows ? g.K - (k0 + pa * 8) : 0);
        }
#pragma unroll
        for (int i = 0; i < B_IT; ++i) {
            if constexpr (TRANS) {
                if constexpr (ALIGNED)
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(k0 + pa * 8 < g.K ? gb[i] + k0 : zero),
                                                     (__attribute__((address_space(3))) void*)&s_b[buf][(i * THREADS + wave * 64) * 8], 16, 0, 0);
                else rb[i] = load8(gb[i] + k0, n0 + (tid >> 3) + i * (THREADS / 8) < g.N ? g.K - (k0 + pa * 8) : 0);
            } else {
                const int k = k0 + kb + 16 * i;
                if constexpr (ALIGNED)
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(k < g.K ? gb[i] + (int64_t)k0 * g.ldw : zero),
                                                     (__attribute__((address_space(3))) void*)&s_b[buf][(i * THREADS + wave * 64) * 8], 16, 0, 0);
                else rb[i] = load8(gb[i] + (int64_t)k0 * g.ldw, k < g.K ? g.N - (n0 + pb * 8) : 0);
            }
        }
    };
    auto settle = [&](int buf) {                                         // (ALIGNED: the copies go to LDS by themselves)
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < A_IT; ++i) *(u32x4*)&s_a[buf][(i * THREADS + tid) * 8] = ra[i];
#pragma unroll
            for (int i = 0; i < B_IT; ++i) *(u32x4*)&s_b[buf][(i * THREADS + tid) * 8] = rb[i];
        }
    };

    // fragments: K-major, lane = row lr of a 16-row tile, contraction 32 ks + 8 kq ..+7; N-major, column lr
    auto frag_k = [&](const T* s, int tile, int ks) { return *(const v8*)&s[(tile * 16 + lr) * BK + (((ks * 4 + kq) ^ (lr & 7)) * 8)]; };
    const int fr = (lr >> 2) | (kq & 1) << 2;
    auto frag_n = [&](const T* s, int tile, int ks) {
        const T* at = &s[(ks * 32 + 8 * kq + (lr >> 2)) * BN + ((tile ^ fr) << 4) + (lr & 3) * 4];
        const s16x4 lo = lds_transposed(at), hi = lds_transposed(at + 4 * BN);
        v8 v;
        __builtin_memcpy(&v, &lo, 8);
        __builtin_memcpy((char*)&v + 8, &hi, 8);
        return v;
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int slabs = (g.K + BK - 1) / BK;
    fetch(0, 0);
    settle(0);
    __syncthreads();                                                     // (waits for the copies as well)
    for (int s = 0; s < slabs; ++s) {
        const int buf = s & 1;
        if (s + 1 < slabs) fetch((s + 1) * BK, buf ^ 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            v8 a[MT], b[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = TRANS ? frag_k(s_b[buf], wn * NT + j, ks) : frag_n(s_b[buf], wn * NT + j, ks);
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = frag_k(s_a[buf], wm * MT + i, ks);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = mfma16(b[j], a[i], acc[i][j]);
        }
        if (s + 1 < slabs) settle(buf ^ 1);
        __syncthreads();
    }

    // the adapters: 32 directions a pass, scale_s H as two 16-bit pieces side by side along the contraction ([16 upper | 16 lower] twice, P's
    // rows repeated to match), each request under the mask of its rows
    const int m1 = min(m0 + BM, r.rows), mw = m0 + wm * MT * 16, mw1 = min(mw + MT * 16, r.rows);
    Walk walk(r, m0, m1);
    int q;
    Span sp;
    while (walk.next(q, sp)) {
        if (sp.s < 0) continue;
        const T* ps = g.low + (int64_t)sp.s * r.rank * g.N;
        for (int j0 = 0; j0 < r.rank; j0 += 32) {
            for (int e = tid; e < BM * 8; e += THREADS) {
                const int m = e >> 3, c = e & 7, row = m0 + m, group = j0 / 16 + (c >> 2), groups = (r.rank + 15) / 16;
                u32x4 v = u32x4{0, 0, 0, 0};
                if (row >= sp.lo && row < sp.hi && group < groups) v = *((const u32x4*)(g.pieces + ((int64_t)row * groups + group) * 32) + (c & 3));
                *(u32x4*)&s_a[0][m * BK + ((c ^ (m & 7)) * 8)] = v;
            }
            for (int e = tid; e < 32 * NP; e += THREADS) {
                const int jj = e / NP, c = e % NP, k = (jj >> 4) * 32 + (jj & 15), j = j0 + jj;
                const u32x4 v = load8(ps + (int64_t)j * g.N + n0 + c * 8, j < r.rank ? g.N - (n0 + c * 8) : 0);
                const int f0 = (k & 3) | ((k >> 3) & 1) << 2;             // (the same for k + 16)
                const int at = ((((c >> 1) ^ f0) << 1) | (c & 1)) * 8;
                *(u32x4*)&s_b[0][k * BN + at] = v;
                *(u32x4*)&s_b[0][(k + 16) * BN + at] = v;
            }
            __syncthreads();
            if (sp.lo < mw1 && sp.hi > mw) {
                const int steps = r.rank - j0 > 16 ? 2 : 1;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    v8 b[2];
                    b[0] = frag_n(s_b[0], wn * NT + j, 0);
                    if (steps > 1) b[1] = frag_n(s_b[0], wn * NT + j, 1);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        f32x4 part = mfma16(b[0], frag_k(s_a[0], wm * MT + i, 0), f32x4{0.f, 0.f, 0.f, 0.f});
                        if (steps > 1) part = mfma16(b[1], frag_k(s_a[0], wm * MT + i, 1), part);
                        const int row = mw + i * 16 + lr;
                        if (row >= sp.lo && row < sp.hi) acc[i][j] += part;
                    }
                }
            }
            __syncthreads();
        }
    }

    const int live_lo = clamp_row(r.offsets[0], r.rows), live_hi = clamp_row(r.offsets[r.n], r.rows);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int col = n0 + (wn * NT + j) * 16 + 4 * kq;
        if (col >= g.N) continue;
        float bias[4] = {};
        if (g.bias) {
            typename Vec4<T>::raw rbias;
            raw_load<T>(rbias, g.bias + col, g.N - col);
            unpack<T>(rbias, bias);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = mw + i * 16 + lr;
            if (row < live_lo || row >= live_hi) continue;
            const float v[4] = {acc[i][j][0] + bias[0], acc[i][j][1] + bias[1], acc[i][j][2] + bias[2], acc[i][j][3] + bias[3]};
            raw_store<T>(pack<T>(v), g.y + (int64_t)row * g.ldy + col, g.N - col);
        }
    }
}

}  // namespace
}  // namespace scs
