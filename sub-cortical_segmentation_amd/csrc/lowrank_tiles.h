// The shared projection on the 16-bit matrix cores for many rows and 16-byte-aligned operands (scs_lowrank.hip): a pipelined form of
// lowrank_mfma16.h (same transposed product, same two LDS images).
//
// What bounds it: LDS.  A slab of 32 along the contraction costs a workgroup (BM + BN) 64 bytes of copies into LDS, and every wave reads its
// own (16 MT + 16 NT) 64 bytes back; at 256 x 256 with four waves of 128 x 128 that is 6 bytes a cycle and matrix core of the 128 the LDS has,
// against 1024 cycles of MFMA (eight waves of 128 x 64 read 1.5 times as much).  So the wave tile is as large as the accumulators allow (256
// AGPRs), one wave per SIMD, and what hides latency is the pipeline alone: four slabs of LDS, three in flight while one is read, a slab's
// fragments read into registers while the slab before is multiplied, one barrier a slab that no copy has to be drained for.
//
// The copies are issued from inline assembly because the compiler, which tracks them, waits for every one of them before the next LDS read; the
// waits are written out instead (copies return in order: vmcnt(n) leaves the n youngest in flight).
#pragma once
#include "lowrank_mfma16.h"

namespace scs {
namespace {

// 16 bytes a lane from base + offset (bytes) to LDS byte `lds` + 16 lane; no register is written, so none can be overtaken
__device__ __forceinline__ void copy_to_lds(const void* base, unsigned int offset, unsigned int lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory"); }
__device__ __forceinline__ void workgroup_barrier() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

template <class T, int WN, int MT, int NT, bool TRANS>
__global__ __launch_bounds__(128 * WN, 2) void project_tiles_kernel(ProjectArgs<T> g) {
    typedef typename Frag<T>::v8 v8;
    constexpr int THREADS = 128 * WN, BM = 32 * MT, BN = 16 * WN * NT, BK = 32, STAGES = 4, NP = BN / 8;
    constexpr int A_IT = BM * 4 / THREADS, B_IT = BN * 4 / THREADS, LOADS = A_IT + B_IT;
    __shared__ __attribute__((aligned(16))) T s_a[STAGES][BM * BK];
    __shared__ __attribute__((aligned(16))) T s_b[STAGES][BN * BK];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4, wm = wave / WN, wn = wave % WN;
    const Requests& r = g.r;

    // (the order of lowrank_mfma16.h: a run of neighbouring tiles, eight row tiles high, for each XCD)
    int m0, n0;
    {
        const int tm = (r.rows + BM - 1) / BM, tn = (g.N + BN - 1) / BN, total = tm * tn, pid = blockIdx.x;
        const int xcd = pid & 7, each = total >> 3, rest = total & 7;
        const int t = xcd * each + min(xcd, rest) + (pid >> 3);
        const int band = t / (8 * tn), in = t - band * 8 * tn, high = min(8, tm - band * 8);
        m0 = (band * 8 + in % high) * BM;
        n0 = in / high * BN;
    }

    // K-major image [row][32]: piece c of a row at c ^ (row >> 2 & 3); N-major image [32][BN]: unit u of row k at u ^ f(k), as before.
    // Addresses are a uniform base, which moves along the contraction, and a lane's 32-bit offset inside the tile (rows and columns beyond
    // the matrices read as their last ones)
    const int pa = (tid & 3) ^ ((tid >> 4) & 3);
    const T* base_a = g.x + (int64_t)m0 * g.ldx;
    const T* base_b = TRANS ? g.w + (int64_t)n0 * g.ldw : g.w + n0;
    const int64_t step_b = TRANS ? BK : BK * g.ldw;
    unsigned int oa[A_IT], ob[B_IT];
#pragma unroll
    for (int i = 0; i < A_IT; ++i) oa[i] = (unsigned int)(min((tid >> 2) + i * (THREADS / 4), r.rows - 1 - m0) * (int)g.ldx + pa * 8) * 2u;
#pragma unroll
    for (int i = 0; i < B_IT; ++i) {
        if constexpr (TRANS) ob[i] = (unsigned int)(min((tid >> 2) + i * (THREADS / 4), g.N - 1 - n0) * (int)g.ldw + pa * 8) * 2u;
        else {
            const int k = tid / NP + i * (THREADS / NP), f = (k & 3) | ((k >> 3) & 1) << 2, piece = ((((tid % NP) >> 1) ^ f) << 1) | (tid & 1);
            ob[i] = (unsigned int)(k * (int)g.ldw + min(piece * 8, g.N - 8 - n0)) * 2u;
        }
    }
    const unsigned int lds_a = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_a[0][0] + wave * 1024;
    const unsigned int lds_b = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_b[0][0] + wave * 1024;
    const int slabs = g.K / BK;                              // (K is a multiple of 2 BK)
    // slab s into its stage; those beyond the last one are copied for the count's sake alone (the last one again, which nobody reads)
    auto fetch = [&](int s) {
        const int from = min(s, slabs - 1);
        const T* a = base_a + from * BK;
        const T* b = base_b + from * step_b;
        const unsigned int la = lds_a + (s % STAGES) * (BM * BK * 2), lb = lds_b + (s % STAGES) * (BN * BK * 2);
#pragma unroll
        for (int i = 0; i < A_IT; ++i) copy_to_lds(a, oa[i], la + i * (THREADS * 16));
#pragma unroll
        for (int i = 0; i < B_IT; ++i) copy_to_lds(b, ob[i], lb + i * (THREADS * 16));
    };

    const int ka = (wm * MT * 16 + lr) * BK + ((kq ^ (lr >> 2)) * 8);                                  // (row >> 2 & 3 is lr >> 2: tiles are 16 rows)
    const int kt = (wn * NT * 16 + lr) * BK + ((kq ^ (lr >> 2)) * 8);
    const int fr = (lr >> 2) | (kq & 1) << 2, nb = (8 * kq + (lr >> 2)) * BN + (lr & 3) * 4;
    auto frag_x = [&](int st, int i) { return *(const v8*)&s_a[st][ka + i * 16 * BK]; };
    auto frag_n = [&](int st, int tile) {
        const T* at = &s_b[st][nb + ((tile ^ fr) << 4)];
        const s16x4 lo = lds_transposed(at), hi = lds_transposed(at + 4 * BN);
        v8 v;
        __builtin_memcpy(&v, &lo, 8);
        __builtin_memcpy((char*)&v + 8, &hi, 8);
        return v;
    };
    auto frag_w = [&](int st, int j) {
        if constexpr (TRANS) return *(const v8*)&s_b[st][kt + j * 16 * BK];
        else return frag_n(st, wn * NT + j);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    v8 x0[MT], w0[NT], x1[MT], w1[NT];
    auto read = [&](int s, v8 (&x)[MT], v8 (&w)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = frag_w(s % STAGES, j);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = frag_x(s % STAGES, i);
    };
    auto multiply = [&](const v8 (&x)[MT], const v8 (&w)[NT]) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mfma16(w[j], x[i], acc[i][j]);
    };
    // fragment reads of the next slab spread evenly between this slab's products
    auto spread = [&] {
        constexpr int READS = MT + (TRANS ? NT : 2 * NT), EACH = MT * NT / READS;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);          // one LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);       // EACH matrix instructions
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MT * NT - EACH * READS, 0);
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fetch(s);
    copies_but<(STAGES - 1) * LOADS>();
    workgroup_barrier();
    read(0, x0, w0);
    for (int s = 0; s < slabs; s += 2) {
        copies_but<(STAGES - 2) * LOADS>();                             // slab s + 1 is there, and every wave has its fragments of slab s
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
    copies_but<0>();                                                     // (none may land in LDS that holds something else by then)
    workgroup_barrier();

    // the adapters: 16 directions a pass, scale_s H as its upper and lower 16-bit piece side by side along the contraction, P's rows repeated
    const int m1 = min(m0 + BM, r.rows), mw = m0 + wm * MT * 16;
    auto frag_x_at = [&](int lr, int kq, int tile) { return *(const v8*)&s_a[0][(tile * 16 + lr) * BK + ((kq ^ (lr >> 2)) * 8)]; };
    auto frag_n_at = [&](int lr, int kq, int tile) {
        const T* at = &s_b[0][(8 * kq + (lr >> 2)) * BN + ((tile ^ ((lr >> 2) | (kq & 1) << 2)) << 4) + (lr & 3) * 4];
        const s16x4 lo = lds_transposed(at), hi = lds_transposed(at + 4 * BN);
        v8 v;
        __builtin_memcpy(&v, &lo, 8);
        __builtin_memcpy((char*)&v + 8, &hi, 8);
        return v;
    };
    Walk walk(r, m0, m1);
    int q;
    Span sp;
    while (walk.next(q, sp)) {
        const T* ps = g.low + (int64_t)max(sp.s, 0) * r.rank * g.N;
#pragma unroll 1
        for (int j0 = sp.s < 0 ? r.rank : 0; j0 < r.rank; j0 += 16) {
            // (opaque copies: addresses formed from them are formed here, not kept in registers beside the sums from the kernel's start on)
            int tid = threadIdx.x, lr = tid & 15, kq = (tid >> 4) & 3;
            asm volatile("" : "+v"(tid), "+v"(lr), "+v"(kq));
            for (int e = tid; e < BM * 4; e += THREADS) {
                const int m = e >> 2, c = e & 3, row = m0 + m;
                const u32x4* at = (const u32x4*)(g.pieces + ((int64_t)min(row, r.rows - 1) * ((r.rank + 15) / 16) + j0 / 16) * 32) + c;
                const u32x4 v = *at;
                const bool in = row >= sp.lo && row < sp.hi;
                *(u32x4*)&s_a[0][m * BK + ((c ^ ((m >> 2) & 3)) * 8)] = in ? v : u32x4{0, 0, 0, 0};
            }
            for (int e = tid; e < 16 * NP; e += THREADS) {
                const int k = e / NP, c = e % NP, j = j0 + k;
                const u32x4 v = at16(ps + (int64_t)min(j, r.rank - 1) * g.N + min(n0 + c * 8, g.N - 8));
                const u32x4 w = j < r.rank ? v : u32x4{0, 0, 0, 0};
                const int f = (k & 3) | ((k >> 3) & 1) << 2, at = ((((c >> 1) ^ f) << 1) | (c & 1)) * 8;       // (the same for row k + 16)
                *(u32x4*)&s_b[0][k * BN + at] = w;
                *(u32x4*)&s_b[0][(k + 16) * BN + at] = w;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const v8 w = frag_n_at(lr, kq, wn * NT + j);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const f32x4 part = mfma16(w, frag_x_at(lr, kq, wm * MT + i), f32x4{0.f, 0.f, 0.f, 0.f});
                    const int row = mw + i * 16 + lr;
                    const bool in = row >= sp.lo && row < sp.hi;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] += in ? part[e] : 0.f;
                }
                __builtin_amdgcn_sched_barrier(0);                      // (all columns' partial products at once do not fit beside the sums)
            }
            __syncthreads();
        }
    }

    const int live_lo = clamp_row(r.offsets[0], r.rows), live_hi = clamp_row(r.offsets[r.n], r.rows);
    int el = threadIdx.x & 63;
    asm volatile("" : "+v"(el));
    const int col = n0 + wn * NT * 16 + 4 * (el >> 4);                    // (N is a multiple of 8: four columns or none)
    float bias[NT][4] = {};
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < NT; ++j) unpack<T>(at4(g.bias + min(col + j * 16, g.N - 4)), bias[j]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = mw + i * 16 + (el & 15);
        if (row >= live_lo && row < live_hi) {
            T* y = g.y + (int64_t)row * g.ldy + col;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float v[4] = {acc[i][j][0] + bias[j][0], acc[i][j][1] + bias[j][1], acc[i][j][2] + bias[j][2], acc[i][j][3] + bias[j][3]};
                if (col + j * 16 < g.N) reinterpret_cast<Loose<u32x2>*>(y + j * 16)->v = pack<T>(v);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

}  // namespace
}  // namespace scs
