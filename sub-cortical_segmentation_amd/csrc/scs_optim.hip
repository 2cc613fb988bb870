// AdamW over many tensors at once (scs_adamw_*, include/scs.h): one launch for all tensors, moments in 32 bits or in 8 bits with one
// scale per block of 256 elements.  Beside lasagne.updates.adam over the parameter arena (scs_train.hip; nets.py:236-237).
//
//   g' = c g            c = grad_scale min(1, max_norm / (norm + 1e-6)), norm = |grad_scale| sqrt(sum g^2) over all tensors, in double
//   m' = b1 m + (1 - b1) g',   v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - m' / (sqrt(v') / sqrt(1 - b2^t) + eps) * lr / (1 - b1^t)
//
// Every operation above is ONE f32 rounding (no contraction, IEEE division and root), so that the codes of the 8-bit moments - decided
// at borders between two values - do not hang on how a compiler groups them.  b^t, the norm and 1 - lr wd are formed in double.
//
// Moments in 8 bits: a block holds m = q |q| s, s = max|m| / 127^2, q = -127..127, and u = sqrt(v) = q^2 s, s = max u / 255^2,
// q = 0..255; q is the code of the nearest value (the border between q and q + 1 is q^2 + q + 1/2 in units of s: exact in f32).  The
// square law gives small moments of a block a finer step than a linear one: 2 / q of the value, 0.8 % at the block's largest m, and reaches
// 6e-5 (m) and 1.5e-5 (u) of the largest.  v is held as its root because the update needs the root and squaring it doubles the range in v.
// A v that is not zero never takes the code 0: m / (0 + eps) would be a step of 1 / eps.
//
// What bounds it: HBM.  f32 parameters and moments move 28 B an element, bf16 parameters and gradients with 8-bit moments 10.1 B
// (at those bytes the division and three roots an element are the second bound: ~70 vector instructions).  96 M elements of 60 tensors: f32 520 us,
// 5.2 TB/s, a copy's rate; bf16 with 8-bit moments 280 us, 3.5 TB/s, and 64 us for the norm; the 77 trained tensors of the net, 0.88 M: 7 us and 7 us.  Work unit: a wave takes four
// blocks of 256 elements (one where there are few), a lane 4 consecutive elements of each (16-byte loads of f32, all four blocks' loads in flight before the first
// use); a workgroup = 4 waves = one chunk of 16 (4) blocks of one tensor; blocks never cross tensors.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "scs_ops.h"

namespace scs {
namespace {

constexpr int kOptBlock = 256;             // elements that share a scale
constexpr int kChunkBlocks = 16;           // blocks of one workgroup ...
constexpr int kSmallBlocks = 4;            // ... and where that would make fewer than kManyChunks of them (a net of 883 455 parameters: 290)
constexpr int kManyChunks = 2048;
constexpr int kGradsPerLaunch = 384;       // gradient pointers that travel by value in one launch's arguments (at most 4 KB of them)
constexpr int kNormGroups = 1024;          // workgroups of the norm's first stage = partial sums in double
constexpr int kTickets = 64;               // leaves of the ticket tree, one 128-byte line each
constexpr float kK127 = (float)(1.0 / 16129.0), kK255 = (float)(1.0 / 65025.0);

// one workgroup's share of one tensor: up to kChunkBlocks blocks (64 bytes, one load)
struct OptChunk {
    void* p;                 // parameter at the chunk's first element
    float* master;           // f32 value of a 16-bit parameter there, or null
    int64_t block;           // first block in the moment arenas
    int64_t first;           // first element, counted inside the tensor
    double wd;
    int32_t left;            // elements of the chunk
    int32_t tensor;
    int32_t type;            // of the parameter
    int32_t pad;
};
struct OptState {            // device words of one optimiser
    int64_t step;            // steps taken
    double norm;             // of the last clipped step
    float gscale;            // its c
    int32_t skip;            // 1: its norm was not finite: parameters, moments and step stay
    unsigned int pad[24];
    unsigned int ticket[(kTickets + 1) * 32];
};

struct GradArgs {
    const void* g[kGradsPerLaunch];
    uint8_t type[kGradsPerLaunch];
    int32_t tensor0;         // g[0] belongs to this tensor
};
struct StepArgs {
    const OptChunk* chunks;
    void* m; void* v; float* ms; float* vs;
    OptState* st;
    double lr, b1, b2;
    float eps, gscale;
    int32_t clipped;         // gscale / skip come from st
    int32_t last;            // the step's last launch: its last workgroup counts the step
};
static_assert(sizeof(GradArgs) + sizeof(StepArgs) <= 4096, "kernel arguments");

struct Coef { float b1, c1, b2, c2, size, root, eps, keep, gscale; };

#pragma clang fp contract(off)

__device__ __forceinline__ void adamw_elem(float& p, float& m, float v, float& vn, float& u, float g, const Coef& k) {
    g = g * k.gscale;
    m = m * k.b1 + g * k.c1;
    vn = v * k.b2 + (g * g) * k.c2;
    u = sqrtf(vn);                      // (correctly rounded, as the division is; the hardware root alone is off by an ulp now and then)
    p = p * k.keep - __fdiv_rn(m, u * k.root + k.eps) * k.size;
}

// nearest code of t = |x| / s: q with q^2 - q + 1/2 <= t < q^2 + q + 1/2.  floor(sqrt(t - 1/4) + 1/2) from the hardware root (off by an ulp, below 4e-5
// here), started low by 1e-4: that is q or q - 1, and one exact comparison tells.  No t exceeds the largest code's upper border.
__device__ __forceinline__ float nearest_code(float t) {
    const float q = floorf(__builtin_amdgcn_sqrtf(fabsf(t - 0.25f)) + (0.5f - 1e-4f));
    return t >= fmaf(q, q, q + 0.5f) ? q + 1.f : q;
}

// block maximum of non-negative values over a wave, as integers so that a NaN counts as the largest value; in lane 63's row reductions and two
// broadcasts (no LDS)
__device__ __forceinline__ float wave_max_abs(float a, float b, float c, float d) {
    auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
    unsigned int r = max(max(bits(a), bits(b)), max(bits(c), bits(d)));
    auto step = [&](auto ctrl, auto rows) {
        r = max(r, (unsigned int)__builtin_amdgcn_update_dpp(0, (int)r, ctrl.value, rows.value, 0xf, true));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});        // row_shr 1, 2, 4, 8: lane 15 of a row has the row's
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});        // row_bcast 15 into rows 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});        // row_bcast 31 into rows 2 and 3
    return __uint_as_float((unsigned int)__builtin_amdgcn_readlane((int)r, 63));
}
__device__ __forceinline__ float block_scale(float amax, float k) {
    const float s = amax * k;
    return s < 0x1p-126f ? 0.f : s;              // (a subnormal scale has no reciprocal: such a block holds zeros)
}

// one wave's blocks of one chunk; the moments' arenas are padded to whole blocks, the pads hold zeros and are written as such
template <class PT, class GT, int BITS, int NB>
__device__ __forceinline__ void adamw_wave(const StepArgs& a, const OptChunk& c, const GT* __restrict__ g, int wave, const Coef& k) {
    const int lane = threadIdx.x & 63, at0 = wave * NB * kOptBlock + lane * 4;
    const bool full = c.left == 4 * NB * kOptBlock;
    typename Vec4<PT>::raw rp[NB];
    typename Vec4<GT>::raw rg[NB];
    f32x4 rw[NB], rm[NB], rv[NB];
    unsigned int qm[NB], qv[NB];
    float sm[NB], sv[NB];
    PT* __restrict__ p = (PT*)c.p;
    float* __restrict__ master = c.master;
    const int64_t b0 = c.block + wave * NB;
    const int mine = full ? NB : min(NB, (c.left + kOptBlock - 1) / kOptBlock - wave * NB);          // blocks of this wave
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        if (j >= mine) continue;
        const int at = at0 + j * kOptBlock;
        const int64_t bb = b0 + j;
        if (full) {
            rg[j] = at4(g + at);
            rp[j] = at4(p + at);
            if (master) rw[j] = at4(master + at);
        } else {
            raw_load<GT>(rg[j], g + at, c.left - at);
            raw_load<PT>(rp[j], p + at, c.left - at);
            if (master) raw_load<float>(rw[j], master + at, c.left - at);
        }
        if constexpr (BITS == 32) {
            rm[j] = ((const f32x4*)a.m)[bb * 64 + lane];
            rv[j] = ((const f32x4*)a.v)[bb * 64 + lane];
        } else {
            qm[j] = ((const unsigned int*)a.m)[bb * 64 + lane];
            qv[j] = ((const unsigned int*)a.v)[bb * 64 + lane];
            sm[j] = a.ms[bb];
            sv[j] = a.vs[bb];
        }
    }
    f32x4 um[NB], uu[NB];                                  // 8 bits: the new m and root of v of every block, until their scales are known
    float top[2 * NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        top[2 * j] = top[2 * j + 1] = 0.f;
        if (j >= mine) continue;
        const int at = at0 + j * kOptBlock;
        const int64_t bb = b0 + j;
        float gf[4], pf[4], m[4], v[4], u[4];
        unpack<GT>(rg[j], gf);
        if (master) { pf[0] = rw[j].x; pf[1] = rw[j].y; pf[2] = rw[j].z; pf[3] = rw[j].w; }
        else unpack<PT>(rp[j], pf);
        if constexpr (BITS == 32) {
            m[0] = rm[j].x; m[1] = rm[j].y; m[2] = rm[j].z; m[3] = rm[j].w;
            v[0] = rv[j].x; v[1] = rv[j].y; v[2] = rv[j].z; v[3] = rv[j].w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = (float)(int8_t)(qm[j] >> (8 * i)), r = (float)((qv[j] >> (8 * i)) & 255u);
                m[i] = q * fabsf(q) * sm[j];
                u[i] = r * r * sv[j];
                v[i] = u[i] * u[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float vn;
            adamw_elem(pf[i], m[i], v[i], vn, u[i], gf[i], k);
            v[i] = vn;
        }
        if (!full) {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i >= c.left - at) { m[i] = 0.f; v[i] = 0.f; u[i] = 0.f; }
            if (master) raw_store<float>(f32x4{pf[0], pf[1], pf[2], pf[3]}, master + at, c.left - at);
            raw_store<PT>(pack<PT>(pf), p + at, c.left - at);
        } else {
            if (master) reinterpret_cast<Loose<f32x4>*>(master + at)->v = f32x4{pf[0], pf[1], pf[2], pf[3]};
            reinterpret_cast<Loose<typename Vec4<PT>::raw>*>(p + at)->v = pack<PT>(pf);
        }
        if constexpr (BITS == 32) {
            ((f32x4*)a.m)[bb * 64 + lane] = f32x4{m[0], m[1], m[2], m[3]};
            ((f32x4*)a.v)[bb * 64 + lane] = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            um[j] = f32x4{m[0], m[1], m[2], m[3]};
            uu[j] = f32x4{u[0], u[1], u[2], u[3]};
            top[2 * j] = wave_max_abs(m[0], m[1], m[2], m[3]);
            top[2 * j + 1] = wave_max_abs(u[0], u[1], u[2], u[3]);
        }
    }
    if constexpr (BITS == 8) {
        // the eight scales side by side in eight lanes: one division gives all their reciprocals
        float mine_top = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) mine_top = lane == i ? top[i] : mine_top;
        const float scale = block_scale(mine_top, lane & 1 ? kK255 : kK127);
        const float inverse = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if (j >= mine) continue;
            const int64_t bb = b0 + j;
            const float is = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inverse), 2 * j));
            const float iw = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inverse), 2 * j + 1));
            unsigned int cm = 0, cv = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = (int)copysignf(nearest_code(fabsf(um[j][i]) * is), um[j][i]);
                int r = (int)nearest_code(uu[j][i] * iw);
                r = uu[j][i] > 0.f ? max(r, 1) : r;
                cm |= ((unsigned int)q & 255u) << (8 * i);
                cv |= (unsigned int)r << (8 * i);
            }
            ((unsigned int*)a.m)[bb * 64 + lane] = cm;
            ((unsigned int*)a.v)[bb * 64 + lane] = cv;
        }
        if (lane < 2 * mine) (lane & 1 ? a.vs : a.ms)[b0 + (lane >> 1)] = scale;
    }
}

// b1^t and b2^t by squaring (a library power of two doubles takes several times as long as the rest of a small step)
__device__ __forceinline__ void powers(double b1, double b2, int64_t t, double& r1, double& r2) {
    r1 = r2 = 1.0;
    for (; t > 0; t >>= 1) {
        if (t & 1) { r1 *= b1; r2 *= b2; }
        b1 *= b1;
        b2 *= b2;
    }
}

// Whether this is the last of `n` workgroups: a ticket tree of two levels (1024 tickets of one counter take 10 us), its counters left at zero for the
// next launch.
__device__ __forceinline__ bool last_ticket(OptState* st, unsigned int id, unsigned int n) {
    const unsigned int leaf = id % kTickets, members = n / kTickets + (leaf < n % kTickets ? 1u : 0u);
    unsigned int* leaf_ticket = &st->ticket[32 * (1 + leaf)];
    if (__hip_atomic_fetch_add(leaf_ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != members - 1) return false;
    __hip_atomic_store(leaf_ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__hip_atomic_fetch_add(&st->ticket[0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != min(n, (unsigned int)kTickets) - 1) return false;
    __hip_atomic_store(&st->ticket[0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

template <int BITS, int NB>
__global__ __launch_bounds__(256) void adamw_kernel(StepArgs a, GradArgs ga) {
    __shared__ Coef s_k;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const OptChunk c = a.chunks[blockIdx.x];
    const bool skip = a.clipped && a.st->skip;
    if (tid == 0) {
        double r1, r2;
        powers(a.b1, a.b2, a.st->step + 1, r1, r2);
        s_k.b1 = (float)a.b1; s_k.c1 = (float)(1.0 - a.b1);
        s_k.b2 = (float)a.b2; s_k.c2 = (float)(1.0 - a.b2);
        s_k.size = (float)(a.lr / (1.0 - r1));
        s_k.root = (float)(1.0 / sqrt(1.0 - r2));
        s_k.eps = a.eps;
        s_k.keep = (float)(1.0 - a.lr * c.wd);
        s_k.gscale = a.clipped ? a.st->gscale : a.gscale;
    }
    __syncthreads();
    const Coef k = s_k;
    if (!skip) {
        const void* g = ga.g[c.tensor - ga.tensor0];
        const int gt = ga.type[c.tensor - ga.tensor0];
        auto by_grad = [&](auto pt) {
            using PT = decltype(pt);
            if (gt == SCS_F32) adamw_wave<PT, float, BITS, NB>(a, c, (const float*)g + c.first, wave, k);
            else if (gt == SCS_BF16) adamw_wave<PT, __bf16, BITS, NB>(a, c, (const __bf16*)g + c.first, wave, k);
            else adamw_wave<PT, _Float16, BITS, NB>(a, c, (const _Float16*)g + c.first, wave, k);
        };
        if (c.type == SCS_F32) by_grad(float{});
        else if (c.type == SCS_BF16) by_grad(__bf16{});
        else by_grad(_Float16{});
    }
    // the step is counted by the workgroup that finishes last (every workgroup has read the count by then)
    if (a.last && tid == 0 && last_ticket(a.st, blockIdx.x, gridDim.x) && !skip) a.st->step += 1;
}

// sum of squares of every gradient, in double: workgroup i takes chunks i, i + groups, ..., the last one to finish adds the partial sums
// in their order (the result does not depend on which one that is)
__device__ __forceinline__ double block_sum256(double v, double* s_red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = ((s_red[0] + s_red[1]) + s_red[2]) + s_red[3];
    __syncthreads();
    return v;
}

template <class GT, int NB> struct ChunkLoad {
    typename Vec4<GT>::raw r[NB];
    __device__ __forceinline__ void load(const GT* __restrict__ g, int n) {
        const int base = threadIdx.x * 4;
        if (n == 4 * NB * kOptBlock) {
#pragma unroll
            for (int j = 0; j < NB; ++j) r[j] = at4(g + base + j * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < NB; ++j) raw_load<GT>(r[j], g + base + j * 1024, n - (base + j * 1024));
        }
    }
    __device__ __forceinline__ double squares() const {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float f[4];
            unpack<GT>(r[j], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += (double)f[i] * (double)f[i];
        }
        return sum;
    }
};

struct NormArgs {
    const OptChunk* chunks; int32_t n_chunks;
    double* partial;          // [launches][kNormGroups]
    int32_t launch, n_partial, group0, total_groups;
    int32_t type;             // of every gradient of the launch, -1: they differ
    OptState* st; double grad_scale, max_norm; float* norm_out;
};
static_assert(sizeof(GradArgs) + sizeof(NormArgs) <= 4096, "kernel arguments");

// one type throughout: the next two chunks are on their way while one is added up
template <class GT, int NB> __device__ __forceinline__ double squares_of(const NormArgs& a, const GradArgs& ga) {
    constexpr int AHEAD = 2;
    ChunkLoad<GT, NB> l[AHEAD + 1];
    auto load = [&](ChunkLoad<GT, NB>& to, int c) {
        const OptChunk& ch = a.chunks[c];
        to.load((const GT*)ga.g[ch.tensor - ga.tensor0] + ch.first, ch.left);
    };
    const int step = gridDim.x;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) if ((int)blockIdx.x + i * step < a.n_chunks) load(l[i], blockIdx.x + i * step);
    for (int c = blockIdx.x; c < a.n_chunks; c += (AHEAD + 1) * step) {
#pragma unroll
        for (int i = 0; i <= AHEAD; ++i) {
            if (c + (i + AHEAD) * step < a.n_chunks) load(l[(i + AHEAD) % (AHEAD + 1)], c + (i + AHEAD) * step);
            if (c + i * step < a.n_chunks) sum += l[i].squares();
        }
    }
    return sum;
}
template <class GT, int NB> __device__ __forceinline__ double chunk_squares(const void* g, const OptChunk& c) {
    ChunkLoad<GT, NB> l;
    l.load((const GT*)g + c.first, c.left);
    return l.squares();
}

template <int NB>
__global__ __launch_bounds__(256) void adamw_norm_kernel(NormArgs a, GradArgs ga) {
    __shared__ double s_red[4];
    __shared__ bool s_last;
    double sum = 0.0;
    if (a.type == SCS_F32) sum = squares_of<float, NB>(a, ga);
    else if (a.type == SCS_BF16) sum = squares_of<__bf16, NB>(a, ga);
    else if (a.type == SCS_F16) sum = squares_of<_Float16, NB>(a, ga);
    else for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
        const OptChunk& ch = a.chunks[c];
        const void* g = ga.g[ch.tensor - ga.tensor0];
        const int gt = ga.type[ch.tensor - ga.tensor0];
        if (gt == SCS_F32) sum += chunk_squares<float, NB>(g, ch);
        else if (gt == SCS_BF16) sum += chunk_squares<__bf16, NB>(g, ch);
        else sum += chunk_squares<_Float16, NB>(g, ch);
    }
    sum = block_sum256(sum, s_red);
    if (threadIdx.x == 0) {
        // (device scope: the workgroup that adds them up may sit on another XCD, behind another L2)
        __hip_atomic_store(&a.partial[(int64_t)a.launch * kNormGroups + blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // (written through to what all XCDs share: no cache has to be written back)
        s_last = last_ticket(a.st, a.group0 + blockIdx.x, a.total_groups);
    }
    __syncthreads();
    if (!s_last) return;
    double all = 0.0;
    for (int i = threadIdx.x; i < a.n_partial; i += 256) all += __hip_atomic_load(&a.partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all = block_sum256(all, s_red);
    if (threadIdx.x == 0) {
        const double norm = fabs(a.grad_scale) * sqrt(all);
        const double f = a.max_norm / (norm + 1e-6);
        a.st->norm = norm;
        a.st->gscale = (float)(a.grad_scale * (f < 1.0 ? f : 1.0));
        a.st->skip = !(norm <= 1.7e308);
        if (a.norm_out) *a.norm_out = (float)norm;
    }
}

__global__ __launch_bounds__(256) void adamw_states_kernel(const unsigned int* __restrict__ m, const unsigned int* __restrict__ v,
                                                           const float* __restrict__ ms, const float* __restrict__ vs, int64_t blocks,
                                                           f32x4* __restrict__ mo, f32x4* __restrict__ vo) {
    const int64_t words = blocks * 64;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const unsigned int qm = m[i], qv = v[i];
        const float sm = ms[i >> 6], sv = vs[i >> 6];
        float a[4], b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = (float)(int8_t)(qm >> (8 * e)), r = (float)((qv >> (8 * e)) & 255u);
            const float u = r * r * sv;
            a[e] = q * fabsf(q) * sm;
            b[e] = u * u;
        }
        mo[i] = f32x4{a[0], a[1], a[2], a[3]};
        vo[i] = f32x4{b[0], b[1], b[2], b[3]};
    }
}

__global__ void adamw_set_step_kernel(OptState* st, int64_t step) { st->step = step; }
__global__ void adamw_count_kernel(OptState* st, int32_t clipped) { if (!(clipped && st->skip)) st->step += 1; }

}  // namespace
}  // namespace scs

struct scs_adamw_ctx {
    int device = 0, bits = 32, chunk_blocks = scs::kChunkBlocks;
    int n = 0;
    int64_t blocks = 0;
    void *m = nullptr, *v = nullptr;
    float *ms = nullptr, *vs = nullptr;
    std::vector<int64_t> sizes;
    std::vector<int32_t> chunk0;               // first chunk of every tensor, and the number of chunks
    unsigned char* mem = nullptr;              // OptState, partial sums, tensors, chunks
    scs::OptState* st = nullptr;
    double* partial = nullptr;
    scs::OptChunk* chunks = nullptr;
    int launches = 0;
};

using namespace scs;

extern "C" {

int scs_adamw_create(scs_handle h, const scs_adamw_tensor* tensors, int32_t n, int state_bits, void* m_dev, void* v_dev,
                     float* m_scale_dev, float* v_scale_dev, int64_t step, scs_adamw* out) {
    SCS_ARG(out != nullptr, "out is NULL");
    *out = nullptr;
    SCS_ARG(h && tensors, "null handle or tensor table");
    SCS_ARG(n >= 1 && n <= (1 << 20), "between 1 and 2^20 tensors");
    SCS_ARG(state_bits == 32 || state_bits == 8, "state_bits is 32 or 8");
    SCS_ARG(step >= 0, "the step count is negative");
    return guarded([&]() -> int {
        std::vector<OptChunk> ch;
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;
        scs_adamw_ctx* o = new scs_adamw_ctx();
        struct Drop { scs_adamw_ctx*& o; ~Drop() { if (o) { if (o->mem) (void)hipFree(o->mem); delete o; } } } drop{o};
        o->bits = state_bits; o->n = n;
        int64_t chunks = 0;
        for (int i = 0; i < n; ++i) if (tensors[i].n > 0) chunks += (tensors[i].n + kChunkBlocks * kOptBlock - 1) / (kChunkBlocks * kOptBlock);
        if (chunks < kManyChunks) o->chunk_blocks = kSmallBlocks;
        for (int i = 0; i < n; ++i) {
            const scs_adamw_tensor& t = tensors[i];
            SCS_ARG(t.n >= 0 && t.n <= ((int64_t)1 << 38), "a tensor's size is negative or above 2^38");
            SCS_ARG(t.type == SCS_F32 || t.type == SCS_BF16 || t.type == SCS_F16, "parameters are SCS_F32, SCS_BF16 or SCS_F16");
            SCS_ARG(t.n == 0 || t.param, "a parameter is NULL");
            SCS_ARG(!t.master || t.type != SCS_F32, "an f32 parameter takes no master copy");
            SCS_ARG(std::isfinite(t.weight_decay), "a weight decay is not finite");
            const size_t e = t.type == SCS_F32 ? 4 : 2;
            SCS_ARG((uintptr_t)t.param % e == 0 && (uintptr_t)t.master % 4 == 0, "a parameter is not aligned to its elements");
            if (t.n) {
                spans.emplace_back((uintptr_t)t.param, (uintptr_t)t.param + (uintptr_t)t.n * e);
                if (t.master) spans.emplace_back((uintptr_t)t.master, (uintptr_t)t.master + (uintptr_t)t.n * 4);
            }
            const int64_t blocks = (t.n + kOptBlock - 1) / kOptBlock;
            o->chunk0.push_back((int32_t)ch.size());
            for (int64_t b = 0; b < blocks; b += o->chunk_blocks) {
                const int64_t at = b * kOptBlock;
                ch.push_back(OptChunk{(char*)t.param + at * (int64_t)e, t.master ? t.master + at : nullptr, o->blocks + b, at, t.weight_decay,
                                      (int32_t)std::min<int64_t>(t.n - at, o->chunk_blocks * kOptBlock), i, t.type, 0});
            }
            SCS_ARG(ch.size() < ((size_t)1 << 30), "more elements than one optimiser takes");
            o->blocks += blocks;
            o->sizes.push_back(t.n);
        }
        o->chunk0.push_back((int32_t)ch.size());
        SCS_ARG(o->blocks == 0 || (m_dev && v_dev), "the moments are NULL");
        SCS_ARG(state_bits == 32 || o->blocks == 0 || (m_scale_dev && v_scale_dev), "8-bit moments need their scales");
        SCS_ARG((uintptr_t)m_dev % 16 == 0 && (uintptr_t)v_dev % 16 == 0 && (uintptr_t)m_scale_dev % 4 == 0 && (uintptr_t)v_scale_dev % 4 == 0,
                "the moments must be aligned to 16 bytes");
        // what a step writes shares no memory: parameters, masters, moments, scales
        auto arena = [&](const void* p, size_t b) { if (p && o->blocks) spans.emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)o->blocks * b); };
        arena(m_dev, kOptBlock * (state_bits == 32 ? 4 : 1));
        arena(v_dev, kOptBlock * (state_bits == 32 ? 4 : 1));
        if (state_bits == 8) { arena(m_scale_dev, 4); arena(v_scale_dev, 4); }
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            SCS_ARG(spans[i - 1].second <= spans[i].first, "two of the parameters, masters and moments overlap (the same tensor twice?)");
        o->m = m_dev; o->v = v_dev; o->ms = m_scale_dev; o->vs = v_scale_dev;
        o->launches = (n + kGradsPerLaunch - 1) / kGradsPerLaunch;
        o->device = handle_device(h);
        DeviceGuard dev(o->device);
        if (dev.rc != SCS_OK) return dev.rc;
        auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
        const size_t b_st = up(sizeof(OptState)), b_pa = up(sizeof(double) * kNormGroups * o->launches),
                     b_ch = up(sizeof(OptChunk) * std::max<size_t>(1, ch.size()));
        SCS_HIP(hipMalloc(&o->mem, b_st + b_pa + b_ch));
        std::vector<unsigned char> host(b_st + b_pa + b_ch, 0);
        o->st = (OptState*)o->mem;
        o->partial = (double*)(o->mem + b_st);
        o->chunks = (OptChunk*)(o->mem + b_st + b_pa);
        memcpy(host.data() + offsetof(OptState, step), &step, sizeof(step));
        if (!ch.empty()) memcpy(host.data() + b_st + b_pa, ch.data(), sizeof(OptChunk) * ch.size());
        SCS_HIP(hipMemcpy(o->mem, host.data(), host.size(), hipMemcpyHostToDevice));
        *out = o;
        o = nullptr;
        return SCS_OK;
    });
}

int scs_adamw_destroy(scs_adamw o) {
    if (!o) return SCS_OK;
    DeviceGuard dev(o->device);
    if (o->mem) (void)hipFree(o->mem);           // (waits for the device)
    delete o;
    return SCS_OK;
}

int scs_adamw_step(scs_adamw o, const void* const* grads, const int32_t* grad_types, double lr, double beta1, double beta2, double eps,
                   double grad_scale, double max_norm, float* norm_dev, void* stream) {
    SCS_ARG(o && grads && grad_types, "null optimiser, gradients or gradient types");
    SCS_ARG(std::isfinite(lr) && std::isfinite(grad_scale), "lr and grad_scale must be finite");
    SCS_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas lie in [0, 1)");
    SCS_ARG(eps > 0 && std::isfinite(eps) && (float)eps > 0.f, "eps must be positive in f32");
    SCS_ARG(max_norm >= 0, "max_norm is negative");
    SCS_ARG(!norm_dev || max_norm > 0, "the norm is formed only where max_norm is given");
    for (int i = 0; i < o->n; ++i) {
        const int32_t ty = grad_types[i];
        SCS_ARG(ty == SCS_F32 || ty == SCS_BF16 || ty == SCS_F16, "gradients are SCS_F32, SCS_BF16 or SCS_F16");
        SCS_ARG(o->sizes[i] == 0 || grads[i], "a gradient is NULL");
        SCS_ARG((uintptr_t)grads[i] % (ty == SCS_F32 ? 4 : 2) == 0, "a gradient is not aligned to its elements");
    }
    DeviceGuard dev(o->device);
    if (dev.rc != SCS_OK) return dev.rc;
    hipStream_t st = (hipStream_t)stream;
    GradArgs ga;
    auto fill = [&](int l) {
        const int lo = l * kGradsPerLaunch, hi = std::min(o->n, lo + kGradsPerLaunch);
        ga.tensor0 = lo;
        for (int i = lo; i < hi; ++i) { ga.g[i - lo] = grads[i]; ga.type[i - lo] = (uint8_t)grad_types[i]; }
        return std::make_pair(o->chunk0[lo], o->chunk0[hi]);
    };
    auto groups = [&](int l) {
        const int lo = l * kGradsPerLaunch, hi = std::min(o->n, lo + kGradsPerLaunch);
        // one at least: the last one writes the result
        return std::max(1, std::min(o->chunk_blocks == kChunkBlocks ? kNormGroups : kNormGroups / 4, (int)(o->chunk0[hi] - o->chunk0[lo])));
    };
    auto type_of = [&](int l) {
        const int lo = l * kGradsPerLaunch, hi = std::min(o->n, lo + kGradsPerLaunch);
        for (int i = lo; i < hi; ++i) if (grad_types[i] != grad_types[lo]) return -1;
        return (int)grad_types[lo];
    };
    if (max_norm > 0) {
        // every launch has a row of kNormGroups partial sums; those that a short launch leaves out were cleared at creation and stay zero
        int total = 0;
        for (int l = 0; l < o->launches; ++l) total += groups(l);
        for (int l = 0, at = 0; l < o->launches; at += groups(l), ++l) {
            const auto c = fill(l);
            NormArgs na{o->chunks + c.first, c.second - c.first, o->partial, l, kNormGroups * o->launches, at, total, type_of(l), o->st, grad_scale, max_norm, norm_dev};
            if (o->chunk_blocks == kChunkBlocks) hipLaunchKernelGGL(adamw_norm_kernel<kChunkBlocks / 4>, dim3(groups(l)), dim3(256), 0, st, na, ga);
            else hipLaunchKernelGGL(adamw_norm_kernel<kSmallBlocks / 4>, dim3(groups(l)), dim3(256), 0, st, na, ga);
        }
    }
    int last = -1;
    for (int l = 0; l < o->launches; ++l) {
        const int lo = l * kGradsPerLaunch, hi = std::min(o->n, lo + kGradsPerLaunch);
        if (o->chunk0[hi] > o->chunk0[lo]) last = l;
    }
    // (no element at all: nothing is updated, the step counts)
    if (last < 0) hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(1), 0, st, o->st, (int32_t)(max_norm > 0));
    for (int l = 0; l <= last; ++l) {
        const auto c = fill(l);
        if (c.second == c.first) continue;
        StepArgs sa{o->chunks + c.first, o->m, o->v, o->ms, o->vs, o->st, lr, beta1, beta2, (float)eps, (float)grad_scale, max_norm > 0, l == last};
        const dim3 grid(c.second - c.first);
        if (o->chunk_blocks == kChunkBlocks) {
            if (o->bits == 32) hipLaunchKernelGGL((adamw_kernel<32, kChunkBlocks / 4>), grid, dim3(256), 0, st, sa, ga);
            else hipLaunchKernelGGL((adamw_kernel<8, kChunkBlocks / 4>), grid, dim3(256), 0, st, sa, ga);
        } else {
            if (o->bits == 32) hipLaunchKernelGGL((adamw_kernel<32, kSmallBlocks / 4>), grid, dim3(256), 0, st, sa, ga);
            else hipLaunchKernelGGL((adamw_kernel<8, kSmallBlocks / 4>), grid, dim3(256), 0, st, sa, ga);
        }
    }
    SCS_HIP(hipGetLastError());
    return SCS_OK;
}

int scs_adamw_states(scs_adamw o, float* m_out_dev, float* v_out_dev, void* stream) {
    SCS_ARG(o && m_out_dev && v_out_dev, "null optimiser or outputs");
    SCS_ARG(o->bits == 8, "moments in 32 bits are read where they lie");
    SCS_ARG((uintptr_t)m_out_dev % 16 == 0 && (uintptr_t)v_out_dev % 16 == 0, "the outputs must be aligned to 16 bytes");
    if (!o->blocks) return SCS_OK;
    DeviceGuard dev(o->device);
    if (dev.rc != SCS_OK) return dev.rc;
    const int grid = (int)std::min<int64_t>((o->blocks * 64 + 255) / 256, 1 << 16);
    hipLaunchKernelGGL(adamw_states_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const unsigned int*)o->m, (const unsigned int*)o->v, o->ms, o->vs,
                       o->blocks, (f32x4*)m_out_dev, (f32x4*)v_out_dev);
    SCS_HIP(hipGetLastError());
    return SCS_OK;
}

int scs_adamw_get_step(scs_adamw o, int64_t* step, void* stream) {
    SCS_ARG(o && step, "null optimiser or output");
    DeviceGuard dev(o->device);
    if (dev.rc != SCS_OK) return dev.rc;
    SCS_HIP(hipMemcpyAsync(step, &o->st->step, sizeof(*step), hipMemcpyDeviceToHost, (hipStream_t)stream));
    SCS_HIP(hipStreamSynchronize((hipStream_t)stream));
    return SCS_OK;
}

int scs_adamw_set_step(scs_adamw o, int64_t step, void* stream) {
    SCS_ARG(o && step >= 0, "null optimiser or negative step");
    DeviceGuard dev(o->device);
    if (dev.rc != SCS_OK) return dev.rc;
    hipLaunchKernelGGL(adamw_set_step_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, o->st, step);
    SCS_HIP(hipGetLastError());
    return SCS_OK;
}

}  // extern "C"
