// The shared projection on the f32 matrix cores for many rows (scs_lowrank.hip): the pipeline of lowrank_tiles.h
// (slabs of LDS, copies in flight across barriers, the next slab's fragments read while this one is multiplied) with exact f32 products.
//
// What bounds it: v_mfma_f32_16x16x4_f32, 32 cycles each on the vector ALUs, which every other vector instruction takes time from: so the copies
// go to LDS without passing registers and addresses are a uniform base and a fixed offset a lane.  A workgroup of four waves owns
// 64 MT rows x 16 NT columns (16 MT rows a wave).  60 000 x 540 x 540: 303 us, 115 TFLOP/s.  This
// instruction issued back to back sustains 139 (scs_probe_f32_mfma); the library reaches 154 at 8192 x 8192 x 8192 and 87 (401 us) at this size.
// LDS images of a slab of 16 along the contraction, in 16-byte pieces:
//   K-major [row][16]: piece c of a row at c ^ (row >> 2 & 3); a lane's piece is its operand of four products.  X, and W^T in the backward pass
//   N-major [16][BN]:  column n of row k at (n + 16 (k >> 2)) mod BN, so that a fragment's four rows lie at different banks.  W, and P
#pragma once
#include "lowrank_tiles.h"

namespace scs {
namespace {

// EVEN: N is a multiple of 4
template <int MT, int NT, bool TRANS, bool EVEN>
__global__ __launch_bounds__(256, NT <= 6 ? 3 : 2) void project_tiles32_kernel(ProjectArgs<float> g) {
    constexpr int BM = 64 * MT, BN = 16 * NT, BK = 16, STAGES = 3, NP = BN / 4, LOADS = MT + 2;
    __shared__ __attribute__((aligned(16))) float s_a[STAGES][BM * BK];
    __shared__ __attribute__((aligned(16))) float s_b[STAGES][512 * 4];           // (BN <= 128; what lies behind a slab's end is never read)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4;
    const Requests& r = g.r;

    // (a run of neighbouring tiles, eight row tiles high, for each XCD: lowrank_tiles.h)
    int m0, n0;
    {
        const int tm = (r.rows + BM - 1) / BM, tn = (g.N + BN - 1) / BN, total = tm * tn, pid = blockIdx.x;
        const int xcd = pid & 7, each = total >> 3, rest = total & 7;
        const int t = xcd * each + min(xcd, rest) + (pid >> 3);
        const int band = t / (8 * tn), in = t - band * 8 * tn, high = min(8, tm - band * 8);
        m0 = (band * 8 + in % high) * BM;
        n0 = in / high * BN;
    }

    const int pa = (tid & 3) ^ ((tid >> 4) & 3);
    const float* base_a = g.x + (int64_t)m0 * g.ldx;
    const float* base_b = TRANS ? g.w + (int64_t)n0 * g.ldw : g.w + n0;
    const int64_t step_b = TRANS ? BK : BK * g.ldw;
    unsigned int oa[MT], ob[2];
    int kb[2];                                              // contraction index of the thread's piece of W'
#pragma unroll
    for (int i = 0; i < MT; ++i) oa[i] = (unsigned int)(min((tid >> 2) + i * 64, r.rows - 1 - m0) * (int)g.ldx + pa * 4) * 4u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (TRANS) {
            kb[i] = pa * 4;
            ob[i] = (unsigned int)(min((tid >> 2) + i * 64, g.N - 1 - n0) * (int)g.ldw + pa * 4) * 4u;
        } else {
            const int l = tid + i * 256, k = min(l / NP, BK - 1), at = l - l / NP * NP, piece = (at + NP - 4 * (k >> 2) % NP) % NP;
            kb[i] = k;
            ob[i] = (unsigned int)(k * (int)g.ldw + min(piece * 4, g.nw - 4 - n0)) * 4u;
        }
    }
    const unsigned int lds_a = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_a[0][0] + wave * 1024;
    const unsigned int lds_b = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_b[0][0] + wave * 1024;
    // slab s into its stage; behind the contraction's end (the last slab's rest, whole slabs after it) zeros
    auto fetch = [&](int s) {
        const float* a = base_a + s * BK;
        const float* b = base_b + s * step_b;
        const unsigned int la = lds_a + (s % STAGES) * (BM * BK * 4), lb = lds_b + (s % STAGES) * 8192;
        if ((s + 1) * BK <= g.K) {
#pragma unroll
            for (int i = 0; i < MT; ++i) copy_to_lds(a, oa[i], la + i * 4096);
            copy_to_lds(b, ob[0], lb);
            copy_to_lds(b, ob[1], lb + 4096);
        } else {
            const char* zero = (const char*)&kZeroPiece;
#pragma unroll
            for (int i = 0; i < MT; ++i) copy_to_lds(s * BK + pa * 4 < g.K ? (const char*)a + oa[i] : zero, la + i * 4096);
#pragma unroll
            for (int i = 0; i < 2; ++i) copy_to_lds(s * BK + kb[i] < g.K ? (const char*)b + ob[i] : zero, lb + i * 4096);
        }
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int ax = (wave * 16 * MT + lr) * BK + (kq ^ (lr >> 2)) * 4, bx = lr * BK + (kq ^ (lr >> 2)) * 4;
    int bn[NT];                                             // N-major: row 4 kq of column tile t
#pragma unroll
    for (int t = 0; t < NT; ++t) bn[t] = 4 * kq * BN + ((t + kq) % NT) * 16 + lr;
    auto read = [&](int s, f32x4 (&x)[MT], f32x4 (&w)[NT]) {
        const float* a = s_a[s % STAGES];
        const float* b = s_b[s % STAGES];
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = *(const f32x4*)(a + ax + i * 16 * BK);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (TRANS) w[t] = *(const f32x4*)(b + bx + t * 16 * BK);
            else
#pragma unroll
                for (int j = 0; j < 4; ++j) w[t][j] = b[bn[t] + j * BN];
        }
    };
    auto multiply = [&](const f32x4 (&x)[MT], const f32x4 (&w)[NT]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[t][j], x[i][j], acc[i][t], 0, 0, 0);
    };
    auto spread = [&] {
        constexpr int READS = MT + (TRANS ? NT : 4 * NT), ALL = 4 * MT * NT, EACH = ALL / READS;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if constexpr (EACH) __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, ALL - EACH * READS, 0);
    };
    f32x4 x0[MT], x1[MT], w0[NT], w1[NT];
    const int slabs = (g.K + BK - 1) / BK;
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fetch(s);
    copies_but<(STAGES - 1) * LOADS>();
    workgroup_barrier();
    read(0, x0, w0);
    for (int s = 0; s < slabs; s += 2) {                    // (an odd count ends with a slab of zeros)
        copies_but<(STAGES - 2) * LOADS>();
        workgroup_barrier();
        fetch(s + STAGES);
        read(s + 1, x1, w1);
        multiply(x0, w0);
        spread();
        copies_but<(STAGES - 2) * LOADS>();
        workgroup_barrier();
        fetch(s + 1 + STAGES);
        read(s + 2, x0, w0);
        multiply(x1, w1);
        spread();
    }
    copies_but<0>();
    workgroup_barrier();

    // the adapters: 16 directions a pass, each request under the mask of its rows
    const int m1 = min(m0 + BM, r.rows), mw = m0 + wave * 16 * MT;
    Walk walk(r, m0, m1);
    int q;
    Span sp;
    while (walk.next(q, sp)) {
        const float scale = walk.scale(sp);
        const float* ps = g.low + (int64_t)max(sp.s, 0) * r.rank * g.N;
#pragma unroll 1
        for (int j0 = sp.s < 0 ? r.rank : 0; j0 < r.rank; j0 += 16) {
            for (int e = tid; e < BM * BK; e += 256) {
                const int m = e >> 4, j = e & 15, row = m0 + m;
                const bool in = row >= sp.lo && row < sp.hi && j0 + j < r.rank;
                const float h = g.h[(int64_t)min(row, r.rows - 1) * r.rank + min(j0 + j, r.rank - 1)];
                s_a[0][m * BK + (((j >> 2) ^ ((m >> 2) & 3)) * 4) + (j & 3)] = in ? scale * h : 0.f;
            }
            for (int e = tid; e < BK * NP; e += 256) {
                const int k = e / NP, c = e - k * NP;
                const float* at = ps + (int64_t)min(j0 + k, r.rank - 1) * g.N;
                f32x4 v;
                if constexpr (EVEN) v = at4(at + min(n0 + c * 4, g.N - 4));
                else raw_load<float>(v, at + n0 + c * 4, g.N - (n0 + c * 4));
                const f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
                *(f32x4*)&s_b[0][k * BN + (c + 4 * (k >> 2)) % NP * 4] = j0 + k < r.rank ? v : z;
            }
            __syncthreads();
            f32x4 x[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) x[i] = *(const f32x4*)(s_a[0] + ax + i * 16 * BK);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 part[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) part[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                const int at = 4 * kq * BN + ((t + kq) % NT) * 16 + lr;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = s_b[0][at + j * BN];
#pragma unroll
                    for (int i = 0; i < MT; ++i) part[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, x[i][j], part[i], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int row = mw + i * 16 + lr;
                    const bool in = row >= sp.lo && row < sp.hi;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][t][e] += in ? part[i][e] : 0.f;
                }
            }
            __syncthreads();
        }
    }

    const int live_lo = clamp_row(r.offsets[0], r.rows), live_hi = clamp_row(r.offsets[r.n], r.rows);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = mw + i * 16 + lr;
        if (row < live_lo || row >= live_hi) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int col = n0 + t * 16 + 4 * kq;
            if (col >= g.N) continue;
            f32x4 v = acc[i][t];
            if constexpr (EVEN) {
                if (g.bias) v += at4(g.bias + col);
                reinterpret_cast<Loose<f32x4>*>(g.y + (int64_t)row * g.ldy + col)->v = v;
            } else {
                f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
                if (g.bias) raw_load<float>(b, g.bias + col, g.N - col);
                raw_store<float>(v + b, g.y + (int64_t)row * g.ldy + col, g.N - col);
            }
        }
    }
}

}  // namespace
}  // namespace scs
