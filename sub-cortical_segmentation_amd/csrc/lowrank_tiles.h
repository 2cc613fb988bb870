// The shared projection on the 16-bit matrix cores for many rows (scs_lowrank.hip): Y = X W' + scale_s H P_s for bf16 and f16.
//
// D is formed transposed (A operand = weights, B operand = rows of X: v_mfma_f32_16x16x32), so that a lane holds four consecutive columns of
// one row.  A workgroup owns BM x BN of Y; both operands pass through LDS in slabs of 32 along the contraction, copied global -> LDS in 16-byte
// pieces without a register between.  LDS images, swizzled so that a fragment's lanes meet no bank twice:
//   K-major [row][32]: 16-byte piece c of a row lies at c ^ (row >> 2 & 3).  X always; W' where it is W^T (backward: W's rows run along the contraction)
//   N-major [32][BN]:  32-byte unit u of row k lies at u ^ f(k), f = (k & 3) | (k >> 3 & 1) << 2 (as many of its bits as there are units).  W (forward) and the adapters' P: the transposing
//            LDS read (ds_read_b64_tr_b16) turns four rows of sixteen columns into each column's four contraction values
//
// What bounds it: LDS and the matrix cores alike.  A slab costs a 256 x 256 tile 32 KB of copies into LDS and eight waves of 128 x 64 96 KB of
// fragment reads, 1024 cycles of the LDS's 128 bytes a cycle against 1024 of MFMA.  Four waves of 128 x 128 would read a third less, but
// their 256 sums leave the compiler too few registers: 530 us instead of 260 at 8192 x 4096 x 4096.  What hides latency is the pipeline: four slabs
// of LDS, three in flight while one is read, a slab's fragments read into registers while the slab before is multiplied, one barrier a slab
// that no copy has to be drained for (drained at every slab: 350 us).  8192 x 4096 x 4096, bf16: about 230 us, 1200 TFLOP/s.  The largest tile spills
// registers (bf16 23 to 26 a lane, f16 54 to 55), all of them behind the loop over the contraction: in the adapters' pass and at the end, once a tile.
// The adapters' pass costs a tile two barriers and a masked product of the WHOLE tile for every request in it and 16 directions: many requests of a row
// or two are its worst case (4096 x 4096, bf16, rank 16: 128 rows of 128 requests 97 us, of four requests 30; 1024 rows 394 and 53, the shrink's passes
// over the contraction, one a request of a row tile, among them).
//
// The copies are issued from inline assembly because the compiler, which tracks them, waits for every one of them before the next LDS read; the
// waits are written out instead (copies return in order: vmcnt(n) leaves the n youngest in flight).
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

// 16 bytes a lane from base + offset (bytes) to LDS byte `lds` + 16 lane; no register is written, so none can be overtaken
// (m0 belongs to the compiler, which has to be told; it warns that it may not save it across the statement, and nothing needs it saved)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(const void* base, unsigned int offset, unsigned int lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
// ... and from an address of the lane's own
__device__ __forceinline__ void copy_to_lds(const void* src, unsigned int lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory"); }
__device__ __forceinline__ void workgroup_barrier() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

template <class T, int WN, int MT, int NT> struct TilesShared {
    __attribute__((aligned(16))) T a[4][32 * MT * 32];
    __attribute__((aligned(16))) T b[4][16 * WN * NT * 32];
};

// Tile `pid` (in the order of the workgroups).  EVEN: N is a multiple of 8 (outputs, bias and P are read and written four and eight columns at a time)
template <class T, int WN, int MT, int NT, bool TRANS, bool EVEN>
__device__ __forceinline__ void project_tile(const ProjectArgs<T>& g, int pid, TilesShared<T, WN, MT, NT>& sh) {
    typedef typename Frag<T>::v8 v8;
    constexpr int THREADS = 128 * WN, BM = 32 * MT, BN = 16 * WN * NT, BK = 32, STAGES = 4, NP = BN / 8;
    constexpr int UNITS = BN / 16 < 8 ? BN / 16 - 1 : 7;               // bits of f(k) that a row has units for
    constexpr int A_IT = BM * 4 / THREADS, B_IT = BN * 4 / THREADS, LOADS = A_IT + B_IT;
    auto& s_a = sh.a;
    auto& s_b = sh.b;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, kq = lane >> 4, wm = wave / WN, wn = wave % WN;
    const Requests& r = g.r;

    // workgroups are dealt to the eight XCDs in turn: give each XCD a run of neighbouring tiles, eight row tiles high, so that its L2
    // serves W's columns and X's rows again
    int m0, n0;
    {
        const int tm = (r.rows + BM - 1) / BM, tn = (g.N + BN - 1) / BN, total = tm * tn;
        const int xcd = pid & 7, each = total >> 3, rest = total & 7;
        const int t = xcd * each + min(xcd, rest) + (pid >> 3);
        const int band = t / (8 * tn), in = t - band * 8 * tn, high = min(8, tm - band * 8);
        m0 = (band * 8 + in % high) * BM;
        n0 = in / high * BN;
    }

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
            const int k = tid / NP + i * (THREADS / NP), f = ((k & 3) | ((k >> 3) & 1) << 2) & UNITS, piece = ((((tid % NP) >> 1) ^ f) << 1) | (tid & 1);
            ob[i] = (unsigned int)(k * (int)g.ldw + min(piece * 8, g.nw - 8 - n0)) * 2u;
        }
    }
    const unsigned int lds_a = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_a[0][0] + wave * 1024;
    const unsigned int lds_b = (unsigned int)(uintptr_t)(__attribute__((address_space(3))) void*)&s_b[0][0] + wave * 1024;
    const int slabs = g.K / BK;                              // (K is a multiple of 64)
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
    const int fr = ((lr >> 2) | (kq & 1) << 2) & UNITS, nb = (8 * kq + (lr >> 2)) * BN + (lr & 3) * 4;
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

    // the adapters, 16 directions a pass.  bf16: scale_s H as its upper and lower 16-bit piece side by side along the contraction, P's rows
    // repeated.  f16: on the f32 matrix cores, because scale_s H may lie outside f16's range (or among its smallest steps) where Y does not
    const int m1 = min(m0 + BM, r.rows), mw = m0 + wm * MT * 16;
    auto frag_x_at = [&](int lr, int kq, int tile) { return *(const v8*)&s_a[0][(tile * 16 + lr) * BK + ((kq ^ (lr >> 2)) * 8)]; };
    auto frag_n_at = [&](int lr, int kq, int tile) {
        const T* at = &s_b[0][(8 * kq + (lr >> 2)) * BN + ((tile ^ (((lr >> 2) | (kq & 1) << 2) & UNITS)) << 4) + (lr & 3) * 4];
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
            auto piece_of_p = [&](int j, int c) {
                const T* at_p = ps + (int64_t)min(j, r.rank - 1) * g.N;
                const u32x4 v = EVEN ? at16(at_p + min(n0 + c * 8, g.N - 8)) : load8(at_p + n0 + c * 8, g.N - (n0 + c * 8));
                return j < r.rank ? v : u32x4{0, 0, 0, 0};
            };
            if constexpr (sizeof(T) == 2 && !kPieces<T>) {
                float* s_h = (float*)&s_a[0][0];                        // [row][16], direction j at j + row
                const float sc = walk.scale(sp);
                for (int e = tid; e < BM * 16; e += THREADS) {
                    const int m = e >> 4, j = j0 + (e & 15), row = m0 + m;
                    const bool in = row >= sp.lo && row < sp.hi && j < r.rank;
                    s_h[m * 16 + ((j + m) & 15)] = in ? sc * g.h[(int64_t)row * r.rank + j] : 0.f;
                }
                for (int e = tid; e < 16 * NP; e += THREADS) {
                    const int k = e / NP, c = e % NP;
                    *(u32x4*)&s_b[0][k * BN + ((((c >> 1) ^ (k & 3)) << 1) | (c & 1)) * 8] = piece_of_p(j0 + k, c);
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = to_f32(s_b[0][(4 * k + kq) * BN + (((wn * NT + j) ^ kq) << 4) + lr]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const int m = (wm * MT + i) * 16 + lr, row = m0 + m;
                        f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < 4; ++k) part = __builtin_amdgcn_mfma_f32_16x16x4f32(w[k], s_h[m * 16 + ((4 * k + kq + m) & 15)], part, 0, 0, 0);
                        const bool in = row >= sp.lo && row < sp.hi;
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] += in ? part[e] : 0.f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                for (int e = tid; e < BM * 4; e += THREADS) {
                    const int m = e >> 2, c = e & 3, row = m0 + m;
                    const u32x4* at = (const u32x4*)(g.pieces + ((int64_t)min(row, r.rows - 1) * ((r.rank + 15) / 16) + j0 / 16) * 32) + c;
                    const u32x4 v = *at;
                    const bool in = row >= sp.lo && row < sp.hi;
                    *(u32x4*)&s_a[0][m * BK + ((c ^ ((m >> 2) & 3)) * 8)] = in ? v : u32x4{0, 0, 0, 0};
                }
                for (int e = tid; e < 16 * NP; e += THREADS) {
                    const int k = e / NP, c = e % NP, j = j0 + k;
                    const u32x4 w = piece_of_p(j, c);
                    const int f = ((k & 3) | ((k >> 3) & 1) << 2) & UNITS, at = ((((c >> 1) ^ f) << 1) | (c & 1)) * 8;       // (the same for row k + 16)
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
            }
            __syncthreads();
        }
    }

    const int live_lo = clamp_row(r.offsets[0], r.rows), live_hi = clamp_row(r.offsets[r.n], r.rows);
    int el = threadIdx.x & 63;
    asm volatile("" : "+v"(el));
    const int col = n0 + wn * NT * 16 + 4 * (el >> 4);
    float bias[NT][4] = {};
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            typename Vec4<T>::raw b = {};
            if constexpr (EVEN) b = at4(g.bias + min(col + j * 16, g.N - 4));
            else raw_load<T>(b, g.bias + col + j * 16, g.N - (col + j * 16));
            unpack<T>(b, bias[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = mw + i * 16 + (el & 15);
        if (row >= live_lo && row < live_hi) {
            T* y = g.y + (int64_t)row * g.ldy + col;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float v[4] = {acc[i][j][0] + bias[j][0], acc[i][j][1] + bias[j][1], acc[i][j][2] + bias[j][2], acc[i][j][3] + bias[j][3]};
                if constexpr (EVEN) {
                    if (col + j * 16 < g.N) reinterpret_cast<Loose<u32x2>*>(y + j * 16)->v = pack<T>(v);
                } else raw_store<T>(pack<T>(v), y + j * 16, g.N - (col + j * 16));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <class T, int WN, int MT, int NT, bool TRANS, bool EVEN>
__global__ __launch_bounds__(128 * WN, 2) void project_tiles_kernel(ProjectArgs<T> g) {
    __shared__ TilesShared<T, WN, MT, NT> sh;
    project_tile<T, WN, MT, NT, TRANS, EVEN>(g, blockIdx.x, sh);
}

}  // namespace
}  // namespace scs
