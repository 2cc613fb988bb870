// A shared projection with a low-rank adapter per request, forward and backward (scs_lowrank_*, include/scs.h).
//
//   y_i  = x_i W + bias + scale_s (x_i A_s^T) B_s                      s = the adapter of row i's request
//   dx_i = dy_i W^T + scale_s (dy_i B_s^T) A_s
//   dA_s = scale_s sum_i (dy_i B_s^T)^T x_i          dB_s = scale_s sum_i (x_i A_s^T)^T dy_i
//
// A and B are both [rank][features], so that one set of kernels serves both directions:
//   shrink  H = X P_s^T     (X = x, P = A, or X = dy, P = B): rows to rank, f32 result
//   project Y = X W' + scale_s H P_s   (W' = W, P = B, or W' = W^T, P = A)
//   wgrad   G_s = scale_s sum H^T X    (H of dy with X = x: dA; H of x with X = dy: dB)
// A row's request is found from the offsets inside the kernels.  A 16-row tile that several requests share is multiplied with each one's
// adapter, and every product is added under the mask of its own rows: an adapter that holds infinities touches its own requests only.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "scs_ops.h"

namespace scs {
namespace {

struct Requests {
    const int32_t* offsets;
    const int32_t* adapters;
    const float* scale;
    int32_t n, n_adapters, rank;
    int32_t rows;
};

__device__ __forceinline__ int clamp_row(int o, int rows) { return o < 0 ? 0 : o > rows ? rows : o; }

struct Span { int lo, hi, s; };           // rows of a request inside [m0, m1) and its adapter (-1: none)

// The requests that own rows of [m0, m1), one after the other.  A wave holds 64 requests in its lanes - three loads at once, whatever
// comes of them - and deals them out by lane reads; where there are more, a binary search finds the first window.  Whole waves call.
struct Walk {
    const Requests& r;
    int m0, m1, base, at;
    int lo, hi, ad;                                    // of request base + lane
    __device__ __forceinline__ Walk(const Requests& req, int from, int to) : r(req), m0(from), m1(to), base(0), at(0) {
        int end = r.n;
        while (end - base > 64) {
            const int mid = (base + end) >> 1;
            if (r.offsets[mid + 1] <= m0) base = mid + 1; else end = mid;
        }
        window();
    }
    __device__ __forceinline__ void window() {
        const int q = base + (int)(threadIdx.x & 63), c = max(min(q, r.n - 1), 0);
        lo = r.offsets[c];
        hi = q < r.n ? r.offsets[c + 1] : 0x7fffffff;
        ad = r.n ? r.adapters[c] : -1;
        at = -1;
    }
    // the next request with rows inside (its number in q), false behind the last one
    __device__ __forceinline__ bool next(int& q, Span& p) {
        for (;;) {
            if (at < 0) {                              // skip what ends before m0
                const unsigned long long below = __ballot(hi <= m0);
                at = ~below == 0ull ? 64 : __builtin_ctzll(~below);
            }
            if (base + at >= r.n) return false;
            if (at >= 64) { base += 64; window(); continue; }
            q = base + at;
            const int a = __builtin_amdgcn_readlane(lo, at), b = __builtin_amdgcn_readlane(hi, at), s = __builtin_amdgcn_readlane(ad, at);
            ++at;
            if (a >= m1) return false;
            p.lo = max(m0, clamp_row(a, r.rows));
            p.hi = min(m1, clamp_row(b, r.rows));
            if (p.lo >= p.hi) continue;
            p.s = (unsigned)s < (unsigned)r.n_adapters ? s : -1;
            return true;
        }
    }
    __device__ __forceinline__ float scale(const Span& p) const { return p.s >= 0 && r.scale ? r.scale[p.s] : 1.f; }
};

// ------------------------------------------------------------------------------------------------------------------ shrink
// H[row][j] = sum_k X[row][k] P_s[j][k] (0 without an adapter).  Many rows: reading X once is the work.  A workgroup of W waves owns 16 MT
// rows, each wave a share of the contraction, joined through LDS; operands go from global memory to the matrix cores without a stop (both are
// contiguous along the contraction: a lane's 16 bytes are its operand of one 16-bit product or of four f32 ones, whose contraction
// indices are permuted alike on both sides), four steps' loads in flight.  8192 x 4096, bf16, rank 16: 27 us, half the rate of a copy (other
// numbers of waves and row tiles measured alike); 60 000 x 540, f32: 38 us.  Every request of a row tile is a pass over the whole contraction.
template <class T> __device__ __forceinline__ f32x4 product16(const u32x4& a, const u32x4& b, f32x4 c) {
    if constexpr (sizeof(T) == 4) {
        f32x4 x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
        return c;
    } else {
        typename Frag<T>::v8 x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return mfma16(x, y, c);
    }
}

// a value as the nearest bf16 one and what is left of it (2^-17 of the value is lost)
template <class T> constexpr bool kPieces = std::is_same<T, __bf16>::value;
template <class T> __device__ __forceinline__ void write_pieces(T* pieces, int64_t row, int j, int rank, float v) {
    if constexpr (kPieces<T>) {
        T* at = pieces + (row * ((rank + 15) / 16) + j / 16) * 32 + j % 16;
        const T hi = from_f32<T>(v);
        const float up = to_f32(hi);
        at[0] = hi;
        at[16] = from_f32<T>(fabsf(up) <= 3.4e38f ? v - up : 0.f);
    }
}

// The tile kernels copy 16-byte pieces: rows that start at any element, or sizes that end inside a piece, are first laid out anew with zeros
// behind their ends (up to two matrices; their bytes once read and once written), by workgroups of their own in the shrink's launch
// (1000 x 777 and 1111 x 777, f16: 3 us less than as a launch).
struct PackMatrix { const void* src; void* dst; int64_t ld; int32_t rows, cols, rows_out, cols_out; };
struct PackArgs { PackMatrix m[2]; int32_t groups; };             // groups: workgroups that do it (0: nothing to do)
template <class T> __device__ __forceinline__ void pack_pieces(const PackArgs& g, int group) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const PackMatrix& m = g.m[k];
        const int pieces = m.cols_out / PER;
        const int64_t n = (int64_t)m.rows_out * pieces;
        for (int64_t i = (int64_t)group * blockDim.x + threadIdx.x; i < n; i += (int64_t)g.groups * blockDim.x) {
            const int64_t row = i / pieces;
            const int col = (int)(i - row * pieces) * PER;
            ((u32x4*)m.dst)[i] = load16((const T*)m.src + row * m.ld + col, row < m.rows ? m.cols - col : 0);
        }
    }
}
template <class T> __global__ __launch_bounds__(256) void pack_kernel(PackArgs g) { pack_pieces<T>(g, blockIdx.x); }

template <class T, int JT, int MT, int W>
__global__ __launch_bounds__(64 * W) void shrink_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ p, int K, float* __restrict__ h, T* __restrict__ pieces, Requests r,
                                                             int* __restrict__ row_adapter, unsigned int* __restrict__ tickets, int n_tickets, PackArgs pk) {
    constexpr int STEP = 64 / sizeof(T), PER = 16 / sizeof(T), UNROLL = JT <= 2 ? 4 : 2, UNIT = UNROLL * STEP;      // contraction values
    __shared__ float s_part[W][MT * JT * 4][64];
    const int groups = gridDim.x - pk.groups;
    if ((int)blockIdx.x >= groups) {
        pack_pieces<T>(pk, blockIdx.x - groups);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, kq = lane >> 4;
    const int m0 = blockIdx.x * 16 * MT, m1 = min(m0 + 16 * MT, r.rows);
    // the contraction in units of 256 bytes of a row, dealt to the waves in turn and from another start in each workgroup: rows lie at the
    // same L2 channel where their stride is a multiple of 4 KB, and neighbouring units at neighbouring channels
    const int units = (K + UNIT - 1) / UNIT;
    auto start = [&](int v) { return (int)((v + blockIdx.x) % (unsigned)units) * UNIT; };
    Walk walk(r, m0, m1);
    const T* xr[MT];
    u32x4 first[UNROLL][MT];                            // X of this wave's first unit, on its way while the requests are looked up
    const int k_first = start(wave);
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = x + (int64_t)min(m0 + 16 * i + lr, r.rows - 1) * ldx + kq * PER;
    if (wave < units && k_first + UNIT <= K) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) first[u][i] = at16(xr[i] + k_first + u * STEP);
    }
    for (int i = blockIdx.x * 64 * W + threadIdx.x; i < n_tickets; i += groups * 64 * W) tickets[i] = 0;
    int mine = -2, q;
    Span sp;
    while (walk.next(q, sp)) {
        if (m0 + (int)threadIdx.x >= sp.lo && m0 + (int)threadIdx.x < sp.hi) mine = sp.s;
        const float scale = walk.scale(sp);
        f32x4 acc[MT][JT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < JT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (sp.s >= 0) {
            const T* pr[JT];
#pragma unroll
            for (int t = 0; t < JT; ++t) pr[t] = p + ((int64_t)sp.s * r.rank + min(t * 16 + lr, r.rank - 1)) * K + kq * PER;
            for (int v = wave; v < units; v += W) {
                const int k0 = start(v);
                if (k0 + UNIT <= K) {
                    u32x4 a[UNROLL][MT], b[UNROLL][JT];
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
                        for (int t = 0; t < JT; ++t) b[u][t] = at16(pr[t] + k0 + u * STEP);
#pragma unroll
                        for (int i = 0; i < MT; ++i) a[u][i] = v == wave ? first[u][i] : at16(xr[i] + k0 + u * STEP);
                    }
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int t = 0; t < JT; ++t) acc[i][t] = product16<T>(a[u][i], b[u][t], acc[i][t]);
                    continue;
                }
                for (int k = k0; k < K; k += STEP) {
                    const int left = K - k - kq * PER;
                    u32x4 a[MT];
#pragma unroll
                    for (int i = 0; i < MT; ++i) a[i] = load16(xr[i] + k, left);
#pragma unroll
                    for (int t = 0; t < JT; ++t) {
                        const u32x4 b = load16(pr[t] + k, left);
#pragma unroll
                        for (int i = 0; i < MT; ++i) acc[i][t] = product16<T>(a[i], b, acc[i][t]);
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < JT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_part[wave][(i * JT + t) * 4 + e][lane] = acc[i][t][e];
        __syncthreads();
        for (int e = wave; e < MT * JT * 4; e += W) {
            float v = s_part[0][e][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) v += s_part[w][e][lane];
            const int i = e / (4 * JT), t = (e >> 2) % JT, m = m0 + 16 * i + 4 * kq + (e & 3), j = t * 16 + lr;
            if (m < sp.lo || m >= sp.hi) continue;
            if (j < r.rank) h[(int64_t)m * r.rank + j] = v;
            if (pieces && t < (r.rank + 15) / 16) write_pieces<T>(pieces, m, j, r.rank, j < r.rank ? scale * v : 0.f);
        }
    }
    if (threadIdx.x < 16 * MT && m0 + (int)threadIdx.x < r.rows) row_adapter[m0 + threadIdx.x] = mine;
}

// Few rows: a workgroup owns four directions of one row, its four waves a quarter of the contraction each (every load of the quarter of a
// 4096-long row is in flight at once), joined through LDS.  It also clears the
// tickets of the projection behind it (lowrank_few.h); both shrink kernels leave every row's adapter (-2 outside the requests, -1 none).
template <class T> __device__ __forceinline__ void load8f(const T* p, int left, float (&f)[8]) {
    typename Vec4<T>::raw a, b;
    raw_load<T>(a, p, left);
    raw_load<T>(b, p + 4, left - 4);
    float lo[4], hi[4];
    unpack<T>(a, lo);
    unpack<T>(b, hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[4 + i] = hi[i]; }
}
template <class T>
__global__ __launch_bounds__(256) void shrink_dots_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ p, int K, float* __restrict__ h, T* __restrict__ pieces, Requests r,
                                                          int* __restrict__ row_adapter, unsigned int* __restrict__ tickets, int n_tickets) {
    __shared__ float s_part[4][4];
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < n_tickets; i += gridDim.x * gridDim.y * 256) tickets[i] = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x, j0 = blockIdx.y * 4;
    const T* xr = x + (int64_t)row * ldx;
    const int per = (K + 2047) / 2048 * 512, k_lo = wave * per + lane * 8, k_hi = min(K, (wave + 1) * per);
    Walk walk(r, row, row + 1);
    float first[8];                                     // the row's first piece, on its way while its request is looked up
    load8f(xr + min(k_lo, K - 1), k_lo < k_hi ? K - k_lo : 0, first);
    int q;
    Span sp;
    const bool owned = walk.next(q, sp);
    if (threadIdx.x == 0 && blockIdx.y == 0) row_adapter[row] = owned ? sp.s : -2;
    if (!owned) return;
    float sum[4] = {};
    if (sp.s >= 0) {
        const T* pr = p + ((int64_t)sp.s * r.rank + j0) * K;
#pragma unroll 2
        for (int k = k_lo; k < k_hi; k += 512) {
            float a[8], b[4][8];
            if (k == k_lo)
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = first[i];
            else load8f(xr + k, K - k, a);
#pragma unroll
            for (int j = 0; j < 4; ++j) load8f(pr + (int64_t)min(j, r.rank - 1 - j0) * K + k, K - k, b[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[j] = fmaf(a[i], b[j][i], sum[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int o = 32; o; o >>= 1) sum[j] += __shfl_xor(sum[j], o);
    }
    if (lane == 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_part[wave][j] = sum[j];
    __syncthreads();
    const int j = j0 + (int)threadIdx.x;
    const int all = (r.rank + 15) / 16 * 16, last = blockIdx.y == gridDim.y - 1 ? all - j0 : 4;       // (the last one fills its 16 pieces up with zeros)
    if ((int)threadIdx.x < last) {
        const float v = j < r.rank ? (s_part[0][threadIdx.x & 3] + s_part[1][threadIdx.x & 3]) + (s_part[2][threadIdx.x & 3] + s_part[3][threadIdx.x & 3]) : 0.f;
        if (j < r.rank) h[(int64_t)row * r.rank + j] = v;
        if (pieces) write_pieces<T>(pieces, row, j, r.rank, walk.scale(sp) * v);
    }
}

// ------------------------------------------------------------------------------------------------------------------ project
template <class T>
struct ProjectArgs {
    const T* x; int64_t ldx;
    const T* w; int64_t ldw;          // W' as stored: [K][N], or [N][K] where TRANS
    const T* bias;
    const T* low;                     // P: [n_adapters][rank][N]
    const float* h;                   // [rows][rank]
    const T* pieces;                  // bf16, many rows: scale_s h as two pieces, [rows][ceil(rank / 16)][16 upper | 16 lower]
    T* y; int64_t ldy;
    int32_t K, N;
    int32_t nw;                       // columns of W's rows that can be read (N-major W: N, or more where it was laid out anew)
    Requests r;
};

}  // namespace
}  // namespace scs
#include "lowrank_rules.h"
#include "lowrank_tiles.h"
#include "lowrank_tiles32.h"
#include "lowrank_few.h"
namespace scs {
namespace {

// ------------------------------------------------------------------------------------------------------------------ wgrad
// G_s[j][k] = scale_s sum over the rows of s of H[row][j] X[row][k], f32: reading X once is the work.  A workgroup owns 64 columns; a lane's
// vector of X (four columns of a row) is its operand of four f32 products (columns 4 c + t of product t), its waves take the rows in
// turn, sixteen at a time, and are joined through LDS in a fixed order.  dA and dB are one launch.
//   by blocks: a workgroup owns a block of rows as well and leaves one partial sum for each request in it, in slot request + block (along the
//              rows one of the two grows from each partial sum to the next: no slot is met twice); wgrad_join_kernel adds an adapter's slots up
//   direct:    a workgroup owns one adapter and walks its requests (few rows, or requests so many and short that their slots would outweigh X)
// 8192 rows of 4096 + 4096 columns, bf16, rank 16, ten requests: 46 us and 8 us of join, 2.9 TB/s of X.
template <class T> struct WgradProblem { const float* h; const T* x; int64_t ldx; float* out; float* part; int32_t F; };
template <class T> struct WgradArgs { WgradProblem<T> p[2]; int32_t block_rows; Requests r; };

template <int JT> constexpr int kWgradRows = JT <= 2 ? 16 : 8;               // rows that a wave takes at once
// rows [lo, hi) of one request into the accumulators
template <class T, int JT, int W> __device__ __forceinline__ void wgrad_rows(const WgradProblem<T>& w, const Requests& r, int col, int lo, int hi, int wave, f32x4 (&acc)[JT][4]) {
    constexpr int UNROLL = kWgradRows<JT> / 4;
    const int lane = threadIdx.x & 63, lr = lane & 15, kq = lane >> 4, left = w.F - col;
    for (int b = lo + wave * 4 * UNROLL; b < hi; b += 4 * W * UNROLL) {
        typename Vec4<T>::raw rx[UNROLL];
        float a[UNROLL][JT];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int row = b + 4 * u + kq, at = min(row, hi - 1);
            raw_load<T>(rx[u], w.x + (int64_t)at * w.ldx + col, left);
#pragma unroll
            for (int t = 0; t < JT; ++t) a[u][t] = w.h[(int64_t)at * r.rank + min(t * 16 + lr, r.rank - 1)];
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const bool in = b + 4 * u + kq < hi;                  // (a row of another request takes no part, whatever it holds)
            float f[4];
            unpack<T>(rx[u], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = in ? f[i] : 0.f;
#pragma unroll
            for (int t = 0; t < JT; ++t) {
                const float h = in && t * 16 + lr < r.rank ? a[u][t] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(h, f[i], acc[t][i], 0, 0, 0);
            }
        }
    }
}
// the waves' sums, in their order, times sc, to out [rank][F]
template <int JT, int W> __device__ __forceinline__ void wgrad_store(float (&s_part)[W - 1][JT * 16][64], const f32x4 (&acc)[JT][4], int wave, int rank, int F, int col, float sc, float* out) {
    const int lane = threadIdx.x & 63, kq = lane >> 4, left = F - col;
    __syncthreads();
    if (wave) {
#pragma unroll
        for (int t = 0; t < JT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_part[wave - 1][t * 16 + i * 4 + e][lane] = acc[t][i][e];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int t = 0; t < JT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = t * 16 + 4 * kq + e;
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = t * 16 + i * 4 + e;
                float sum = acc[t][i][e];
#pragma unroll
                for (int w = 0; w < W - 1; ++w) sum += s_part[w][at][lane];
                v[i] = sc * sum;
            }
            if (j < rank) raw_store<float>(v, out + (int64_t)j * F + col, left);
        }
}
template <int JT> __device__ __forceinline__ void wgrad_clear(f32x4 (&acc)[JT][4]) {
#pragma unroll
    for (int t = 0; t < JT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
}

template <class T, int JT>
__device__ __forceinline__ void wgrad_block(const WgradArgs<T>& g, int tile, int block, int problem, float (&s_part)[3][JT * 16][64]) {
    const WgradProblem<T>& w = g.p[problem];
    const Requests& r = g.r;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = tile * 64, col = c0 + 4 * (threadIdx.x & 15);
    if (c0 >= w.F) return;
    const int m0 = block * g.block_rows, m1 = min(m0 + g.block_rows, r.rows);
    Walk walk(r, m0, m1);
    int q;
    Span sp;
    while (walk.next(q, sp)) {
        if (sp.s < 0) continue;
        f32x4 acc[JT][4];
        wgrad_clear<JT>(acc);
        wgrad_rows<T, JT, 4>(w, r, col, sp.lo, sp.hi, wave, acc);
        wgrad_store<JT, 4>(s_part, acc, wave, r.rank, w.F, col, 1.f, w.part + (int64_t)(q + block) * r.rank * w.F);
    }
}
template <class T, int JT>
__global__ __launch_bounds__(256) void wgrad_blocks_kernel(WgradArgs<T> g) {
    __shared__ float s_part[3][JT * 16][64];
    wgrad_block<T, JT>(g, blockIdx.x, blockIdx.y, blockIdx.z, s_part);
}

// dx in small tiles and the adapters' gradients by blocks of rows in one launch, the tiles first: neither fills the card (1000 rows, 777 x 1111, f16:
// 19 us together, 18 and 14 one after the other)
template <class T, int JT, bool EVEN>
__global__ __launch_bounds__(256, 2) void tiles_and_wgrad_kernel(ProjectArgs<T> g, int n_tiles, WgradArgs<T> w, int tiles, int blocks) {
    __shared__ union Shared {
        __device__ Shared() {}
        TilesShared<T, 2, 2, 2> tile;
        float part[3][JT * 16][64];
    } sh;
    if ((int)blockIdx.x < n_tiles) {
        project_tile<T, 2, 2, 2, true, EVEN>(g, blockIdx.x, sh.tile);
        return;
    }
    const int id = blockIdx.x - n_tiles, rest = id / tiles;
    wgrad_block<T, JT>(w, id % tiles, rest % blocks, rest / blocks, sh.part);
}

template <class T, int JT, int W>
__device__ __forceinline__ void wgrad_direct(const WgradProblem<T>& w, const Requests& r, int tile, int s, float (&s_part)[W - 1][JT * 16][64]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = tile * 64, col = c0 + 4 * (lane & 15);
    if (c0 >= w.F) return;
    f32x4 acc[JT][4];
    wgrad_clear<JT>(acc);
    int turn = 0;                                             // (requests of a row or two each: the waves take them in turn)
    bool used = false;                                        // (an adapter without rows: zeros, whatever its scale holds)
    for (int q0 = 0; q0 < r.n; q0 += 64) {
        const int q = q0 + lane, c = min(q, r.n - 1);
        const int lo = clamp_row(r.offsets[c], r.rows), hi = clamp_row(r.offsets[c + 1], r.rows);
        unsigned long long todo = __ballot(q < r.n && r.adapters[c] == s && lo < hi);
        used |= todo != 0;
        for (; todo; todo &= todo - 1) {
            const int at = __builtin_ctzll(todo);
            const int a = __builtin_amdgcn_readlane(lo, at), b = __builtin_amdgcn_readlane(hi, at);
            wgrad_rows<T, JT, W>(w, r, col, a, b, (wave + W - turn) % W, acc);
            turn = (turn + (b - a + kWgradRows<JT> - 1) / kWgradRows<JT>) % W;
        }
    }
    wgrad_store<JT, W>(s_part, acc, wave, r.rank, w.F, col, used && r.scale ? r.scale[s] : 1.f, w.out + (int64_t)s * r.rank * w.F);
}

template <int JT> constexpr int direct_waves() { return JT <= 2 ? kFewWaves : 4; }             // (the join's LDS)
template <class T, int JT>
__global__ __launch_bounds__(64 * direct_waves<JT>()) void wgrad_direct_kernel(WgradArgs<T> g) {
    __shared__ float s_part[direct_waves<JT>() - 1][JT * 16][64];
    wgrad_direct<T, JT, direct_waves<JT>()>(g.p[blockIdx.z], g.r, blockIdx.x, blockIdx.y, s_part);
}

// dx of few rows and the adapters' gradients in one launch: both follow from u alone, and neither fills the card (a mini-batch of 256 rows at 540 x
// 540: 11 us together, 11 and 7 one after the other)
template <class T, int MT, int JT>
__global__ __launch_bounds__(64 * kFewWaves) void few_and_wgrad_kernel(ProjectArgs<T> g, const int* __restrict__ row_adapter, FewGrid grid, float* part, unsigned int* tickets,
                                                                       WgradArgs<T> w, int tiles) {
    __shared__ union Shared {
        __device__ Shared() {}
        FewShared<MT> few;
        float part[kFewWaves - 1][JT * 16][64];
    } sh;
    const int few = grid.tiles_n * grid.tiles_m * grid.splits;
    if ((int)blockIdx.x < few) {
        project_few<T, MT, true>(g, row_adapter, grid, part, tickets, blockIdx.x, sh.few);
        return;
    }
    const int id = blockIdx.x - few, tile = id % tiles, rest = id / tiles;
    wgrad_direct<T, JT, kFewWaves>(w.p[rest / w.r.n_adapters], w.r, tile, rest % w.r.n_adapters, sh.part);
}

// an adapter's gradient from its requests' slots, in the order of the rows
template <class T>
__global__ __launch_bounds__(256) void wgrad_join_kernel(WgradArgs<T> g) {
    const WgradProblem<T>& w = g.p[blockIdx.z];
    const Requests& r = g.r;
    const int s = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t n = (int64_t)r.rank * w.F, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if ((int64_t)blockIdx.x * 1024 >= n) return;
    const int left = (int)min(n - i, (int64_t)4);
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
    bool used = false;                                        // (as in wgrad_direct)
    for (int q0 = 0; q0 < r.n; q0 += 64) {
        const int q = q0 + lane, c = min(q, r.n - 1);
        const int lo = clamp_row(r.offsets[c], r.rows), hi = clamp_row(r.offsets[c + 1], r.rows);
        unsigned long long todo = __ballot(q < r.n && r.adapters[c] == s && lo < hi);
        used |= todo != 0;
        for (; todo; todo &= todo - 1) {
            const int at = __builtin_ctzll(todo);
            const int b_lo = __builtin_amdgcn_readlane(lo, at) / g.block_rows, b_hi = (__builtin_amdgcn_readlane(hi, at) - 1) / g.block_rows;
#pragma unroll 4
            for (int b = b_lo; b <= b_hi; ++b) {
                f32x4 v;
                raw_load<float>(v, w.part + (int64_t)(q0 + at + b) * n + i, left);
                sum += v;
            }
        }
    }
    if (left > 0) raw_store<float>(sum * (used && r.scale ? r.scale[s] : 1.f), w.out + (int64_t)s * n + i, left);
}

// ------------------------------------------------------------------------------------------------------------------ host side
size_t up(size_t b) { return (b + 255) & ~(size_t)255; }

struct Layout { size_t hid = 0, hid2 = 0, part = 0, tickets = 0, rows = 0, rows2 = 0, slots = 0, pieces = 0, pack_x = 0, pack_w = 0, bytes = 0; };
Layout layout_of(const scs_lowrank& p, bool backward, const void* x, int64_t ldx) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t o = at; at += up(b); return o; };
    l.hid = take((size_t)p.rows * p.rank * 4);
    const Few f = backward ? few_of(p, p.out_features, p.in_features) : few_of(p, p.in_features, p.out_features);
    size_t part = f.part;
    l.tickets = take((size_t)f.tickets * 4);
    l.rows = take((size_t)p.rows * 4);
    if (p.dtype == SCS_BF16 && !f.mt) l.pieces = take((size_t)p.rows * ((p.rank + 15) / 16) * 64);
    if (backward) {
        l.rows2 = take((size_t)p.rows * 4);
        l.hid2 = take((size_t)p.rows * p.rank * 4);
        if (const int b = wgrad_block_rows(p)) l.slots = take((size_t)(p.n_requests + (p.rows + b - 1) / b) * p.rank * (p.in_features + p.out_features) * 4);
    }
    l.part = take(part);
    if (!f.mt) {
        const Pack k = backward ? pack_of(p, p.out_features, p.in_features, true, x, ldx) : pack_of(p, p.in_features, p.out_features, false, x, ldx);
        l.pack_x = take(k.x_bytes);
        l.pack_w = take(k.w_bytes);
    }
    l.bytes = at;
    return l;
}

int check(const scs_lowrank* p) {
    SCS_ARG(p != nullptr, "the call's description is NULL");
    SCS_ARG(p->dtype == SCS_F32 || p->dtype == SCS_BF16 || p->dtype == SCS_F16, "dtype is SCS_F32, SCS_BF16 or SCS_F16");
    SCS_ARG(p->rank >= 1 && p->rank <= 128, "rank lies in 1..128");
    SCS_ARG(p->n_adapters >= 1 && p->n_adapters <= 65535, "n_adapters lies in 1..65535");
    SCS_ARG(p->n_requests >= 0 && p->n_requests <= (1 << 24), "n_requests lies in 0..2^24");
    SCS_ARG(p->rows >= 0 && p->rows <= (1 << 26), "rows lies in 0..2^26");             // (a launch has at most 2^32 threads along x)
    SCS_ARG(p->in_features >= 1 && p->in_features <= (1 << 20) && p->out_features >= 1 && p->out_features <= (1 << 20), "features lie in 1..2^20");
    SCS_ARG(p->ldw >= p->out_features, "ldw is below out_features");
    SCS_ARG(p->w && p->a && p->b && p->offsets && (p->adapters || p->n_requests == 0), "a table is NULL");
    const size_t e = p->dtype == SCS_F32 ? 4 : 2;
    SCS_ARG((uintptr_t)p->w % e == 0 && (uintptr_t)p->bias % e == 0 && (uintptr_t)p->a % e == 0 && (uintptr_t)p->b % e == 0, "a matrix is not aligned to its elements");
    SCS_ARG((uintptr_t)p->scale % 4 == 0 && (uintptr_t)p->offsets % 4 == 0 && (uintptr_t)p->adapters % 4 == 0, "a table is not aligned to its elements");
    return SCS_OK;
}

Requests requests_of(const scs_lowrank& p) { return Requests{p.offsets, p.adapters, p.scale, p.n_requests, p.n_adapters, p.rank, (int32_t)p.rows}; }

template <class F> void by_tiles(int rank, F&& f) {
    const int t = rank_tiles(rank);
    if (t == 1) f(std::integral_constant<int, 1>{});
    else if (t == 2) f(std::integral_constant<int, 2>{});
    else if (t == 4) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 8>{});
}

template <class T> void shrink(const scs_lowrank& p, const T* x, int64_t ldx, const T* low, int K, float* h, T* pieces, hipStream_t st, int* row_adapter, unsigned int* tickets = nullptr, int n_tickets = 0,
                               const PackArgs& pk = PackArgs{}) {
    const Requests r = requests_of(p);
    if (p.rows <= kDotRows) {
        if (pk.groups) hipLaunchKernelGGL(pack_kernel<T>, dim3(pk.groups), dim3(256), 0, st, pk);
        hipLaunchKernelGGL(shrink_dots_kernel<T>, dim3((unsigned)p.rows, (p.rank + 3) / 4), dim3(256), 0, st, x, ldx, low, K, h, pieces, r, row_adapter, tickets, n_tickets);
        return;
    }
    const ShrinkForm f = shrink_form(p, K);
    by_tiles(p.rank, [&](auto jt) {
        auto go = [&](auto mt, auto w) {
            hipLaunchKernelGGL((shrink_rows_kernel<T, jt.value, mt.value, w.value>), dim3((unsigned)((p.rows + 16 * mt.value - 1) / (16 * mt.value) + pk.groups)), dim3(64 * w.value), 0, st,
                               x, ldx, low, K, h, pieces, r, row_adapter, tickets, n_tickets, pk);
        };
        constexpr int MT = jt.value <= 2 ? 2 : 1, MOST = jt.value <= 2 ? 16 : 8;
        typedef std::integral_constant<int, 1> One;
        if (f.mt == 2) {
            if (f.waves == 8) go(std::integral_constant<int, MT>{}, std::integral_constant<int, 8>{});
            else go(std::integral_constant<int, MT>{}, std::integral_constant<int, 4>{});
        } else if (f.waves == MOST) go(One{}, std::integral_constant<int, MOST>{});
        else if (f.waves == 8) go(One{}, std::integral_constant<int, 8>{});
        else go(One{}, std::integral_constant<int, 4>{});
    });
}

template <class T, bool TRANS> void launch_few(const ProjectArgs<T>& g, const Few& f, const int* rows, float* part, unsigned int* tickets, hipStream_t st) {
    const FewGrid grid{f.tiles_n, f.tiles_m, f.splits};
    auto go = [&](auto mt) {
        hipLaunchKernelGGL((project_few_kernel<T, mt.value, TRANS>), dim3(f.tiles_n * f.tiles_m * f.splits), dim3(64 * kFewWaves), 0, st, g, rows, grid, part, tickets);
    };
    if (f.mt == 1) go(std::integral_constant<int, 1>{});
    else if (f.mt == 2) go(std::integral_constant<int, 2>{});
    else if constexpr (sizeof(T) == 2) {
        if (f.mt == 3) go(std::integral_constant<int, 3>{});
        else go(std::integral_constant<int, 4>{});
    }
}

template <class T, bool TRANS, bool EVEN> void project_tiles(const ProjectArgs<T>& g, hipStream_t st) {
    auto tiles = [&](int64_t bm, int64_t bn) { return (g.r.rows + bm - 1) / bm * ((g.N + bn - 1) / bn); };
    if constexpr (sizeof(T) == 2) {
        if (tile16(g.r.rows, g.N) == 256) hipLaunchKernelGGL((project_tiles_kernel<T, 4, 8, 4, TRANS, EVEN>), dim3((unsigned)tiles(256, 256)), dim3(512), 0, st, g);
        else if (tile16(g.r.rows, g.N) == 128) hipLaunchKernelGGL((project_tiles_kernel<T, 2, 4, 4, TRANS, EVEN>), dim3((unsigned)tiles(128, 128)), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((project_tiles_kernel<T, 2, 2, 2, TRANS, EVEN>), dim3((unsigned)tiles(64, 64)), dim3(256), 0, st, g);
    } else {
        const int nt = f32_columns(g.N), mt = f32_rows(g.r.rows, g.N);
        auto go = [&](auto n) {
            if (mt == 2) hipLaunchKernelGGL((project_tiles32_kernel<2, n.value, TRANS, EVEN>), dim3((unsigned)tiles(128, 16 * n.value)), dim3(256), 0, st, g);
            else hipLaunchKernelGGL((project_tiles32_kernel<1, n.value, TRANS, EVEN>), dim3((unsigned)tiles(64, 16 * n.value)), dim3(256), 0, st, g);
        };
        if (nt == 8) go(std::integral_constant<int, 8>{});
        else if (nt == 7) go(std::integral_constant<int, 7>{});
        else if (nt == 6) go(std::integral_constant<int, 6>{});
        else if (nt == 5) go(std::integral_constant<int, 5>{});
        else go(std::integral_constant<int, 4>{});
    }
}

// what has to be laid out anew of the tile kernels' operands (for the shrink's launch), the projection's arguments turned to where it will lie
template <class T, bool TRANS> PackArgs pack(const scs_lowrank& p, ProjectArgs<T>& g, T* pack_x, T* pack_w) {
    g.nw = g.N;
    const Pack k = pack_of(p, g.K, g.N, TRANS, g.x, g.ldx);
    PackArgs pa{};
    int n = 0;
    if (k.x) {
        pa.m[n++] = PackMatrix{g.x, pack_x, g.ldx, g.r.rows, g.K, g.r.rows, (int)k.K};
        g.x = pack_x;
        g.ldx = k.K;
    }
    if (k.w) {
        pa.m[n++] = PackMatrix{g.w, pack_w, g.ldw, TRANS ? g.N : g.K, TRANS ? g.K : g.N, (int)k.w_rows, (int)k.w_cols};
        g.w = pack_w;
        g.ldw = k.w_cols;
        g.nw = (int)k.nw;
    }
    if (n) pa.groups = (int)std::min<int64_t>((int64_t)(std::max(k.x_bytes, k.w_bytes) / 16 + 255) / 256, 8192);
    g.K = (int)k.K;
    return pa;
}

template <class T, bool TRANS> void project(const ProjectArgs<T>& g, const Few& f, const int* rows, float* part, unsigned int* tickets, hipStream_t st) {
    if (f.mt) launch_few<T, TRANS>(g, f, rows, part, tickets, st);
    else if (g.N % (sizeof(T) == 2 ? 8 : 4) == 0) project_tiles<T, TRANS, true>(g, st);
    else project_tiles<T, TRANS, false>(g, st);
}

// beside(arguments, tiles, blocks): whether the partial sums of the by-blocks form are formed in a launch of the caller's
template <class T, class Beside> void wgrad(const scs_lowrank& p, const WgradProblem<T> (&problems)[2], int n, float* slots, hipStream_t st, Beside&& beside) {
    WgradArgs<T> g{{problems[0], problems[1]}, wgrad_block_rows(p), requests_of(p)};
    const int F = std::max(problems[0].F, n > 1 ? problems[1].F : 0), tiles = (F + 63) / 64;
    if (!g.block_rows) {
        by_tiles(p.rank, [&](auto jt) {
            hipLaunchKernelGGL((wgrad_direct_kernel<T, jt.value>), dim3(tiles, p.n_adapters, n), dim3(64 * direct_waves<jt.value>()), 0, st, g);
        });
        return;
    }
    const int64_t blocks = (p.rows + g.block_rows - 1) / g.block_rows;
    g.p[0].part = slots;
    g.p[1].part = slots + (p.n_requests + blocks) * p.rank * problems[0].F;
    if (!beside(g, tiles, (int)blocks))
        by_tiles(p.rank, [&](auto jt) { hipLaunchKernelGGL((wgrad_blocks_kernel<T, jt.value>), dim3(tiles, (unsigned)blocks, n), dim3(256), 0, st, g); });
    hipLaunchKernelGGL(wgrad_join_kernel<T>, dim3((unsigned)(((int64_t)p.rank * F + 1023) / 1024), p.n_adapters, n), dim3(256), 0, st, g);
}

template <class T>
int forward(const scs_lowrank& p, const void* x, int64_t ldx, void* y, int64_t ldy, float* hidden, unsigned char* ws, hipStream_t st) {
    const Layout l = layout_of(p, false, x, ldx);
    float* h = hidden ? hidden : (float*)(ws + l.hid);
    const Few f = few_of(p, p.in_features, p.out_features);
    int* rows = (int*)(ws + l.rows);
    T* pieces = kPieces<T> && !f.mt ? (T*)(ws + l.pieces) : nullptr;
    ProjectArgs<T> g{(const T*)x, ldx, (const T*)p.w, p.ldw, (const T*)p.bias, (const T*)p.b, h, pieces, (T*)y, ldy, (int)p.in_features, (int)p.out_features, (int)p.out_features, requests_of(p)};
    const PackArgs pk = f.mt ? PackArgs{} : pack<T, false>(p, g, (T*)(ws + l.pack_x), (T*)(ws + l.pack_w));
    shrink<T>(p, (const T*)x, ldx, (const T*)p.a, (int)p.in_features, h, pieces, st, rows, (unsigned int*)(ws + l.tickets), f.tickets, pk);
    project<T, false>(g, f, rows, (float*)(ws + l.part), (unsigned int*)(ws + l.tickets), st);
    SCS_HIP(hipGetLastError());
    return SCS_OK;
}

template <class T>
int backward(const scs_lowrank& p, const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* hidden, void* dx, int64_t lddx, float* da, float* db,
             unsigned char* ws, hipStream_t st) {
    const Layout l = layout_of(p, true, dy, lddy);
    float* u = (float*)(ws + l.hid);
    float* part = (float*)(ws + l.part);
    const bool any = p.rows > 0 && p.n_requests > 0;          // (without rows dA and dB are zeros: the wgrad kernels write them)
    const Few f = few_of(p, p.out_features, p.in_features);
    int* rows = (int*)(ws + l.rows);
    int* rows2 = (int*)(ws + l.rows2);                 // (of the second shrink: the same numbers)
    T* pieces = kPieces<T> && !f.mt ? (T*)(ws + l.pieces) : nullptr;
    ProjectArgs<T> back{(const T*)dy, lddy, (const T*)p.w, p.ldw, nullptr, (const T*)p.a, u, pieces, (T*)dx, lddx, (int)p.out_features, (int)p.in_features, (int)p.in_features, requests_of(p)};
    const PackArgs pk = f.mt || !dx ? PackArgs{} : pack<T, true>(p, back, (T*)(ws + l.pack_x), (T*)(ws + l.pack_w));
    if (any && (dx || da)) shrink<T>(p, (const T*)dy, lddy, (const T*)p.b, (int)p.out_features, u, pieces, st, rows, (unsigned int*)(ws + l.tickets), f.tickets, pk);
    WgradProblem<T> w[2]{};
    int n = 0;
    if (da) w[n++] = WgradProblem<T>{u, (const T*)x, ldx, da, nullptr, (int)p.in_features};
    if (db) {
        const float* h = hidden;
        if (!h) {
            h = (float*)(ws + l.hid2);
            if (any) shrink<T>(p, (const T*)x, ldx, (const T*)p.a, (int)p.in_features, (float*)(ws + l.hid2), (T*)nullptr, st, rows2);
        }
        w[n++] = WgradProblem<T>{h, (const T*)dy, lddy, db, nullptr, (int)p.out_features};
    }
    if (dx && n && few_beside_wgrad(p, f)) {
        const int tiles = (std::max(w[0].F, n > 1 ? w[1].F : 0) + 63) / 64;
        const FewGrid grid{f.tiles_n, f.tiles_m, f.splits};
        const WgradArgs<T> wa{{w[0], w[1]}, 0, requests_of(p)};
        const dim3 all((unsigned)(f.tiles_n * f.tiles_m * f.splits + tiles * p.n_adapters * n));
        auto go = [&](auto mt, auto jt) {
            hipLaunchKernelGGL((few_and_wgrad_kernel<T, mt.value, jt.value>), all, dim3(64 * kFewWaves), 0, st, back, rows, grid, part, (unsigned int*)(ws + l.tickets), wa, tiles);
        };
        typedef std::integral_constant<int, 1> One;
        typedef std::integral_constant<int, 2> Two;
        if (f.mt == 1) { if (p.rank <= 16) go(One{}, One{}); else go(One{}, Two{}); }
        else { if (p.rank <= 16) go(Two{}, One{}); else go(Two{}, Two{}); }
    } else if (dx && n && tiles_beside_wgrad(p, f)) {
        // neither dx in small tiles nor the partial sums fill the card: one launch
        if constexpr (sizeof(T) == 2) {
            const int n_tiles = (int)((p.rows + 63) / 64 * ((p.in_features + 63) / 64));
            wgrad<T>(p, w, n, (float*)(ws + l.slots), st, [&](const WgradArgs<T>& wa, int tiles, int blocks) {
                auto go = [&](auto jt, auto even) {
                    hipLaunchKernelGGL((tiles_and_wgrad_kernel<T, jt.value, even.value>), dim3(n_tiles + tiles * blocks * n), dim3(256), 0, st, back, n_tiles, wa, tiles, blocks);
                };
                auto by_even = [&](auto jt) {
                    if (back.N % 8 == 0) go(jt, std::true_type{});
                    else go(jt, std::false_type{});
                };
                if (p.rank <= 16) by_even(std::integral_constant<int, 1>{});
                else by_even(std::integral_constant<int, 2>{});
                return true;
            });
        }
    } else {
        if (dx) project<T, true>(back, f, rows, part, (unsigned int*)(ws + l.tickets), st);
        if (n) wgrad<T>(p, w, n, (float*)(ws + l.slots), st, [](const WgradArgs<T>&, int, int) { return false; });
    }
    SCS_HIP(hipGetLastError());
    return SCS_OK;
}

}  // namespace
}  // namespace scs

using namespace scs;

extern "C" {

int scs_lowrank_workspace(scs_handle h, const scs_lowrank* p, int backward_call, const void* rows_dev, int64_t ld, size_t* bytes) {
    SCS_ARG(h && bytes, "null handle or output");
    const int rc = check(p);
    if (rc != SCS_OK) return rc;
    *bytes = layout_of(*p, backward_call != 0, rows_dev, ld).bytes;
    return SCS_OK;
}

int scs_lowrank_forward(scs_handle h, const scs_lowrank* p, const void* x_dev, int64_t ldx, void* y_dev, int64_t ldy, float* hidden_dev,
                        void* workspace_dev, size_t workspace_bytes, void* stream) {
    SCS_ARG(h != nullptr, "null handle");
    int rc = check(p);
    if (rc != SCS_OK) return rc;
    if (p->rows == 0 || p->n_requests == 0) return SCS_OK;
    const size_t e = p->dtype == SCS_F32 ? 4 : 2;
    SCS_ARG(x_dev && y_dev, "x or y is NULL");
    SCS_ARG(ldx >= p->in_features && ldy >= p->out_features, "a row stride is below the row's length");
    SCS_ARG((uintptr_t)x_dev % e == 0 && (uintptr_t)y_dev % e == 0 && (uintptr_t)hidden_dev % 4 == 0, "a matrix is not aligned to its elements");
    const size_t need = layout_of(*p, false, x_dev, ldx).bytes;
    SCS_ARG(workspace_bytes >= need && workspace_dev && (uintptr_t)workspace_dev % 16 == 0, "the workspace is too small, NULL or not aligned to 16 bytes (scs_lowrank_workspace)");
    DeviceGuard dev(handle_device(h));
    if (dev.rc != SCS_OK) return dev.rc;
    unsigned char* ws = (unsigned char*)workspace_dev;
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == SCS_F32) return forward<float>(*p, x_dev, ldx, y_dev, ldy, hidden_dev, ws, st);
    if (p->dtype == SCS_BF16) return forward<__bf16>(*p, x_dev, ldx, y_dev, ldy, hidden_dev, ws, st);
    return forward<_Float16>(*p, x_dev, ldx, y_dev, ldy, hidden_dev, ws, st);
}

int scs_lowrank_backward(scs_handle h, const scs_lowrank* p, const void* x_dev, int64_t ldx, const void* dy_dev, int64_t lddy,
                         const float* hidden_dev, void* dx_dev, int64_t lddx, float* da_dev, float* db_dev,
                         void* workspace_dev, size_t workspace_bytes, void* stream) {
    SCS_ARG(h != nullptr, "null handle");
    int rc = check(p);
    if (rc != SCS_OK) return rc;
    SCS_ARG(dx_dev || da_dev || db_dev, "no output is asked for");
    const size_t e = p->dtype == SCS_F32 ? 4 : 2;
    const bool none = p->rows == 0 || p->n_requests == 0;
    SCS_ARG(none || (dy_dev && lddy >= p->out_features), "dy is NULL or its row stride below the row's length");
    SCS_ARG(none || (!da_dev && !(db_dev && !hidden_dev)) || (x_dev && ldx >= p->in_features), "x is NULL or its row stride below the row's length");
    SCS_ARG(none || !dx_dev || lddx >= p->in_features, "the row stride of dx is below the row's length");
    SCS_ARG((uintptr_t)x_dev % e == 0 && (uintptr_t)dy_dev % e == 0 && (uintptr_t)dx_dev % e == 0 && (uintptr_t)hidden_dev % 4 == 0 &&
            (uintptr_t)da_dev % 4 == 0 && (uintptr_t)db_dev % 4 == 0, "a matrix is not aligned to its elements");
    const size_t need = layout_of(*p, true, dy_dev, lddy).bytes;
    SCS_ARG(need == 0 || (workspace_bytes >= need && workspace_dev && (uintptr_t)workspace_dev % 16 == 0),
            "the workspace is too small, NULL or not aligned to 16 bytes (scs_lowrank_workspace)");
    DeviceGuard dev(handle_device(h));
    if (dev.rc != SCS_OK) return dev.rc;
    unsigned char* ws = (unsigned char*)workspace_dev;
    hipStream_t st = (hipStream_t)stream;
    if (none) dx_dev = nullptr;
    if (p->dtype == SCS_F32) return backward<float>(*p, x_dev, ldx, dy_dev, lddy, hidden_dev, dx_dev, lddx, da_dev, db_dev, ws, st);
    if (p->dtype == SCS_BF16) return backward<__bf16>(*p, x_dev, ldx, dy_dev, lddy, hidden_dev, dx_dev, lddx, da_dev, db_dev, ws, st);
    return backward<_Float16>(*p, x_dev, ldx, dy_dev, lddy, hidden_dev, dx_dev, lddx, da_dev, db_dev, ws, st);
}

}  // extern "C"
