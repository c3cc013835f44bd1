// Layer norm over rows of C elements, forward and backward, beside the BatchNorm kernels of elementwise.hip: a row is one
// token, or one pixel of an NHWC activation (its channels are the innermost dimension in memory).
//
//   s = x (+ r, the sum rounded to the activations' type: it is an output and what backward reads)
//   mu = mean(s)   rstd = 1 / sqrt(mean((s - mu)^2) + eps)   xh = (s - mu) * rstd   y = xh * w + b
//   gw = g * w     ds = rstd * (gw - mean(gw) - xh * mean(gw * xh)) (+ gs)          dx = dr = ds
//   dw = sum over rows of g * xh      db = sum over rows of g
//
// Bound: HBM.  Forward moves 2 (4 with the residual sum) elements per element of x, backward 3 (4).  A row is read once: it
// stays in the registers of its TEAM of TS threads (NV 16-byte vectors each), the two statistics are two reductions over the
// team, the variance from (s - mu) and not from a difference of sums.  All sums are fp32.
//
// A team is a part of a wavefront up to 64 threads (DPP and permlane-swap reductions, no LDS), a workgroup of 128 .. 1024 above
// (one LDS exchange per reduction).  The smallest capacity TS * NV * (16 bytes) that holds C is taken; longer rows go to the
// kernels that walk a row in pieces and read it again from the cache.
//
// Rows need no alignment and C no divisor: a vector load or store of a global address needs only the element's alignment on
// gfx950, and the last vector of a row is moved back so that it ENDS at the row's end.  The elements it shares with its
// neighbour are left out of the sums (index below `skip`) and stored twice with the same value.
#include "common.h"

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef __bf16 bf16_t;

namespace {

template <typename T, int VE> struct Vec { typedef T type __attribute__((ext_vector_type(VE), aligned(sizeof(T)))); };
template <typename T> struct Vec<T, 1> { typedef T type; };

template <typename T, int VE>
__device__ __forceinline__ void widen(const typename Vec<T, VE>::type& raw, float (&v)[VE]) {
    if constexpr (VE == 1) v[0] = (float)raw;
    else {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = (float)raw[e];
    }
}
template <typename T, int VE>
__device__ __forceinline__ void load(const T* p, float (&v)[VE]) {
    widen<T, VE>(*reinterpret_cast<const typename Vec<T, VE>::type*>(p), v);
}
// ONCE: past the caches.  Taken where a pass moves more than they hold (256 MB): what is read for the last time (backward's
// operands) or not soon again (y, dx).  16384 x 4096 bf16 forward + backward: 148 -> 135 us, with the residual sum 225 -> 200;
// forward's operands are left in, backward reads them again.  Below that size the next operator finds y and dx in the cache.
template <bool ONCE, typename V, typename T>
__device__ __forceinline__ V raw_load(const T* p) {
    const V* q = reinterpret_cast<const V*>(p);
    if constexpr (ONCE) return __builtin_nontemporal_load(q);
    else return *q;
}
template <typename T, int VE, bool ONCE = false>
__device__ __forceinline__ void store(T* p, const float (&v)[VE]) {
    typename Vec<T, VE>::type raw;
    if constexpr (VE == 1) raw = (T)v[0];
    else {
#pragma unroll
        for (int e = 0; e < VE; ++e) raw[e] = (T)v[e];
    }
    auto* q = reinterpret_cast<typename Vec<T, VE>::type*>(p);
    if constexpr (ONCE) __builtin_nontemporal_store(raw, q);
    else *q = raw;
}

// a vector of the gain / bias, whose type is a run-time value (fp32 masters or the activations' type); null: `dflt`
template <int VE>
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t i, float dflt, float (&v)[VE]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = dflt;
    } else if (dtype == AYOLO_F32) load<float, VE>((const float*)p + i, v);
    else if (dtype == AYOLO_F16) load<half_t, VE>((const half_t*)p + i, v);
    else load<bf16_t, VE>((const bf16_t*)p + i, v);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == AYOLO_F32) ((float*)p)[i] = v;
    else if (dtype == AYOLO_F16) ((half_t*)p)[i] = (half_t)v;
    else ((bf16_t*)p)[i] = (bf16_t)v;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over aligned groups of N <= 64 lanes, left in every lane of the group
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (N >= 2) v += dpp<0xB1>(v);      // quad_perm [1,0,3,2]
    if constexpr (N >= 4) v += dpp<0x4E>(v);      // quad_perm [2,3,0,1]
    if constexpr (N >= 8) v += dpp<0x141>(v);     // row_half_mirror
    if constexpr (N >= 16) v += dpp<0x140>(v);    // row_mirror
    if constexpr (N >= 32) {                      // the two 16-lane rows of a half, then the two halves
        const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (N >= 64) {
        const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
// sums of NS values over the team.  Teams of several wavefronts exchange one value per wavefront through `ex`; `phase`
// alternates between two halves of it, so that one barrier per reduction is enough.
template <int TS, int NS>
__device__ __forceinline__ void team_sum(float (&v)[NS], float* ex, int& phase) {
#pragma unroll
    for (int k = 0; k < NS; ++k) v[k] = lanes_sum<(TS < 64 ? TS : 64)>(v[k]);
    if constexpr (TS > 64) {
        constexpr int NW = TS / 64;
        float* buf = ex + phase * (2 * NW);
        phase ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < NS; ++k) buf[(threadIdx.x >> 6) * NS + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) t += buf[w * NS + k];
            v[k] = t;
        }
    }
}

// first element of row `r` of an operand whose rows lie in groups of `inner`
__device__ __forceinline__ int64_t row_at(const ayolo_rows& t, unsigned r) {
    if (t.inner <= 0) return (int64_t)r * t.stride;
    const unsigned q = r / (unsigned)t.inner;
    return (int64_t)q * t.outer_stride + (int64_t)(r - q * (unsigned)t.inner) * t.stride;
}

struct Fwd {
    ayolo_rows x, r;
    void *y, *s;
    const void *w, *b;
    float *mean, *rstd;
    unsigned rows;
    int C, wdtype;
    float eps;
};
struct Bwd {
    ayolo_rows s, gy, gs;
    void* dx;
    const void* w;
    const float *mean, *rstd;
    float* part;              // [workgroups][2][C], or null
    unsigned rows;
    int C, wdtype;
};

// where vector v of thread l lies in a row: columns c .. c + VE - 1, those below c + skip not its own
template <int VE>
struct Place {
    int c, skip;
    __device__ __forceinline__ Place(int i, int C) {
        const int at = i * VE;
        c = at + VE <= C ? at : C - VE;
        skip = at < C ? at - c : VE;
    }
    __device__ __forceinline__ bool own(int e) const { return e >= skip; }
    __device__ __forceinline__ bool any() const { return skip < VE; }
};
// A thread's columns, the same in every row.  The smallest team is taken, so that all vectors but the last of each thread lie
// whole inside the row: only the last has elements to leave out (`mine`: 1 or 0 for each of its elements).
template <int VE, int TS, int NV>
struct Columns {
    int c[NV];
    bool stores;              // the last vector holds an element of the row
    float mine[VE];
    __device__ __forceinline__ Columns(int l, int C) {
#pragma unroll
        for (int k = 0; k < NV - 1; ++k) c[k] = (k * TS + l) * VE;
        const Place<VE> at((NV - 1) * TS + l, C);
        c[NV - 1] = at.c;
        stores = at.any();
#pragma unroll
        for (int e = 0; e < VE; ++e) mine[e] = at.own(e) ? 1.0f : 0.0f;
    }
};
// 1 / sqrt(x) by the hardware (1 ulp); it takes subnormal arguments for zero, which can be only where eps is that small
__device__ __forceinline__ float inv_sqrt(float x, float eps) { return eps >= 1e-30f ? __builtin_amdgcn_rsqf(x) : 1.0f / sqrtf(x); }

// Teams walk rows base + team, base + team + step, ...; the next row's loads are issued before the present row is reduced.
template <typename T, int VE, int TS, int NV, bool RES, bool ONCE>
__global__ __launch_bounds__(TS < 128 ? 256 : TS) void k_ln_fwd(Fwd P) {
    constexpr int NT = TS < 128 ? 256 : TS, TEAMS = NT / TS;
    typedef typename Vec<T, VE>::type V;
    __shared__ float ex[TS > 64 ? 4 * (TS / 64) : 1];
    int phase = 0;
    const int team = threadIdx.x / TS, l = threadIdx.x % TS, C = P.C;
    const Columns<VE, TS, NV> col(l, C);
    const float inv = 1.0f / (float)C;
    const unsigned step = gridDim.x * TEAMS;
    V x[NV], r[RES ? NV : 1];
    auto fetch = [&](unsigned row) {
        const T* xr = (const T*)P.x.data + row_at(P.x, row);
#pragma unroll
        for (int k = 0; k < NV; ++k) x[k] = *reinterpret_cast<const V*>(xr + col.c[k]);
        if constexpr (RES) {
            const T* rr = (const T*)P.r.data + row_at(P.r, row);
#pragma unroll
            for (int k = 0; k < NV; ++k) r[k] = *reinterpret_cast<const V*>(rr + col.c[k]);
        }
    };
    unsigned base = blockIdx.x * TEAMS;
    fetch(min(base + team, P.rows - 1));
    float w[NV][VE], b[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_param<VE>(P.w, P.wdtype, col.c[k], 1.0f, w[k]);
        load_param<VE>(P.b, P.wdtype, col.c[k], 0.0f, b[k]);
    }
    for (; base < P.rows; base += step) {
        const bool live = base + team < P.rows;            // a team past the last row repeats that row and stores nothing
        const unsigned row = live ? base + team : P.rows - 1;
        float v[NV][VE];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            widen<T, VE>(x[k], v[k]);
            if constexpr (RES) {
                float u[VE];
                widen<T, VE>(r[k], u);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[k][e] = (float)(T)(v[k][e] + u[e]);
                if (live && (k < NV - 1 || col.stores)) store<T, VE>((T*)P.s + (int64_t)row * C + col.c[k], v[k]);
            }
        }
        if (base + step < P.rows) fetch(min(base + step + team, P.rows - 1));
        float t[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) t[0] = k < NV - 1 ? t[0] + v[k][e] : __builtin_fmaf(col.mine[e], v[k][e], t[0]);
        team_sum<TS, 1>(t, ex, phase);
        const float mu = t[0] * inv;
        t[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                v[k][e] -= mu;
                t[0] = __builtin_fmaf(k < NV - 1 ? v[k][e] : v[k][e] * col.mine[e], v[k][e], t[0]);
            }
        team_sum<TS, 1>(t, ex, phase);
        const float rstd = inv_sqrt(__builtin_fmaf(t[0], inv, P.eps), P.eps);
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int e = 0; e < VE; ++e) v[k][e] = __builtin_fmaf(v[k][e] * rstd, w[k][e], b[k][e]);
                if (k < NV - 1 || col.stores) store<T, VE, ONCE>((T*)P.y + (int64_t)row * C + col.c[k], v[k]);
            }
            if (P.mean && l == 0) {
                P.mean[row] = mu;
                P.rstd[row] = rstd;
            }
        }
    }
}

// Rows longer than the widest team's registers: one workgroup per row, three passes over it (mean, variance, output; the residual
// sum is formed again in each, from the same roundings).
template <typename T, int VE, bool RES>
__global__ __launch_bounds__(1024) void k_ln_fwd_long(Fwd P) {
    __shared__ float ex[64];
    int phase = 0;
    const int C = P.C;
    const float inv = 1.0f / (float)C;
    for (unsigned row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T* xr = (const T*)P.x.data + row_at(P.x, row);
        const T* rr = RES ? (const T*)P.r.data + row_at(P.r, row) : nullptr;
        auto value = [&](const Place<VE>& at, float (&v)[VE]) {
            load<T, VE>(xr + at.c, v);
            if constexpr (RES) {
                float u[VE];
                load<T, VE>(rr + at.c, u);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[e] = (float)(T)(v[e] + u[e]);
            }
        };
        float t[1] = {0.0f};
        for (int i = threadIdx.x; i * (int64_t)VE < C; i += 1024) {
            const Place<VE> at(i, C);
            float v[VE];
            value(at, v);
            if constexpr (RES) store<T, VE>((T*)P.s + (int64_t)row * C + at.c, v);
#pragma unroll
            for (int e = 0; e < VE; ++e) t[0] += at.own(e) ? v[e] : 0.0f;
        }
        team_sum<1024, 1>(t, ex, phase);
        const float mu = t[0] * inv;
        t[0] = 0.0f;
        for (int i = threadIdx.x; i * (int64_t)VE < C; i += 1024) {
            const Place<VE> at(i, C);
            float v[VE];
            value(at, v);
#pragma unroll
            for (int e = 0; e < VE; ++e) t[0] += at.own(e) ? (v[e] - mu) * (v[e] - mu) : 0.0f;
        }
        team_sum<1024, 1>(t, ex, phase);
        const float rstd = inv_sqrt(__builtin_fmaf(t[0], inv, P.eps), P.eps);
        for (int i = threadIdx.x; i * (int64_t)VE < C; i += 1024) {
            const Place<VE> at(i, C);
            float v[VE], w[VE], b[VE];
            value(at, v);
            load_param<VE>(P.w, P.wdtype, at.c, 1.0f, w);
            load_param<VE>(P.b, P.wdtype, at.c, 0.0f, b);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[e] = __builtin_fmaf((v[e] - mu) * rstd, w[e], b[e]);
            store<T, VE>((T*)P.y + (int64_t)row * C + at.c, v);
        }
        if (P.mean && threadIdx.x == 0) {
            P.mean[row] = mu;
            P.rstd[row] = rstd;
        }
    }
}

// Backward.  A thread holds the same columns in every row its team walks, so the weight's and the bias's gradients are summed
// over those rows in its registers; at the end the teams of a wavefront are added by shuffles, its wavefronts through LDS, in a
// fixed order, and the workgroup writes one line [2][C] of partial sums.  k_ln_params adds the lines.  No atomics: the same call
// gives the same bits.
template <typename T, int VE, int TS, int NV, bool RES, bool ONCE>
__global__ __launch_bounds__(TS < 128 ? 256 : TS) void k_ln_bwd(Bwd P) {
    constexpr int NT = TS < 128 ? 256 : TS, TEAMS = NT / TS, CAP = TS * NV * VE;
    typedef typename Vec<T, VE>::type V;
    __shared__ float ex[TS > 64 ? 4 * (TS / 64) : 1];
    __shared__ float lines[TS > 64 ? 1 : 4 * 2 * CAP];
    int phase = 0;
    const int team = threadIdx.x / TS, l = threadIdx.x % TS, C = P.C;
    const Columns<VE, TS, NV> col(l, C);
    const float inv = 1.0f / (float)C;
    const unsigned step = gridDim.x * TEAMS;
    V x[NV], gy[NV], gs[RES ? NV : 1];
    float mu, rstd;
    auto fetch = [&](unsigned row) {
        const T *sr = (const T*)P.s.data + row_at(P.s, row), *gr = (const T*)P.gy.data + row_at(P.gy, row);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            x[k] = raw_load<ONCE, V>(sr + col.c[k]);
            gy[k] = raw_load<ONCE, V>(gr + col.c[k]);
        }
        if constexpr (RES) {
            const T* qr = (const T*)P.gs.data + row_at(P.gs, row);
#pragma unroll
            for (int k = 0; k < NV; ++k) gs[k] = raw_load<ONCE, V>(qr + col.c[k]);
        }
        mu = P.mean[row];
        rstd = P.rstd[row];
    };
    constexpr bool AHEAD = TS < 1024;                      // 16 wavefronts leave 128 registers each: no room for a second row
    unsigned base = blockIdx.x * TEAMS;
    if (AHEAD) fetch(min(base + team, P.rows - 1));
    float w[NV][VE], own_w[VE], dw[NV][VE], db[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_param<VE>(P.w, P.wdtype, col.c[k], 1.0f, w[k]);
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[k][e] = db[k][e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) own_w[e] = w[NV - 1][e] * col.mine[e];
    for (; base < P.rows; base += step) {
        const bool live = base + team < P.rows;
        const unsigned row = live ? base + team : P.rows - 1;
        if (!AHEAD) fetch(row);
        float v[NV][VE], g[NV][VE], q[RES ? NV : 1][VE];
        const float m = mu, s = rstd;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            widen<T, VE>(x[k], v[k]);
            widen<T, VE>(gy[k], g[k]);
            if constexpr (RES) widen<T, VE>(gs[k], q[k]);
        }
        if (AHEAD && base + step < P.rows) fetch(min(base + step + team, P.rows - 1));
        float t[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                v[k][e] = (v[k][e] - m) * s;
                const float gw = g[k][e] * (k < NV - 1 ? w[k][e] : own_w[e]);
                t[0] += gw;
                t[1] = __builtin_fmaf(gw, v[k][e], t[1]);
            }
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    dw[k][e] = __builtin_fmaf(g[k][e], v[k][e], dw[k][e]);
                    db[k][e] += g[k][e];
                }
        }
        if (P.dx) {
            team_sum<TS, 2>(t, ex, phase);
            const float c1 = t[0] * inv, c2 = t[1] * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float d = __builtin_fmaf(-v[k][e], c2, __builtin_fmaf(g[k][e], w[k][e], -c1));
                    g[k][e] = RES ? __builtin_fmaf(s, d, q[RES ? k : 0][e]) : s * d;
                }
                if (live && (k < NV - 1 || col.stores)) store<T, VE, ONCE>((T*)P.dx + (int64_t)row * C + col.c[k], g[k]);
            }
        }
    }
    if (!P.part) return;
    float* line = P.part + (int64_t)blockIdx.x * 2 * C;
    const Place<VE> last((NV - 1) * TS + l, C);
    if constexpr (TS < 64) {                               // the wavefront's teams: lanes that hold the same columns
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e)
#pragma unroll
                for (int d = TS; d < 64; d *= 2) {
                    dw[k][e] += __shfl_xor(dw[k][e], d);
                    db[k][e] += __shfl_xor(db[k][e], d);
                }
    }
    float* to = TS > 64 ? line : lines + (threadIdx.x >> 6) * 2 * C;
    if (TS >= 64 || (threadIdx.x & 63) < TS) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (k < NV - 1 || last.own(e)) {
                    to[col.c[k] + e] = dw[k][e];
                    to[C + col.c[k] + e] = db[k][e];
                }
    }
    if constexpr (TS <= 64) {
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * C; i += NT) line[i] = (lines[i] + lines[2 * C + i]) + (lines[4 * C + i] + lines[6 * C + i]);
    }
}

// The long rows' backward: dx needs two passes over the row; the parameters' gradients are summed by k_ln_bwd_long_params.
template <typename T, int VE, bool RES>
__global__ __launch_bounds__(1024) void k_ln_bwd_long(Bwd P) {
    __shared__ float ex[64];
    int phase = 0;
    const int C = P.C;
    const float inv = 1.0f / (float)C;
    for (unsigned row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T* sr = (const T*)P.s.data + row_at(P.s, row);
        const T* gr = (const T*)P.gy.data + row_at(P.gy, row);
        const T* qr = RES ? (const T*)P.gs.data + row_at(P.gs, row) : nullptr;
        const float mu = P.mean[row], rstd = P.rstd[row];
        float t[2] = {0.0f, 0.0f};
        for (int i = threadIdx.x; i * (int64_t)VE < C; i += 1024) {
            const Place<VE> at(i, C);
            float v[VE], g[VE], w[VE];
            load<T, VE>(sr + at.c, v);
            load<T, VE>(gr + at.c, g);
            load_param<VE>(P.w, P.wdtype, at.c, 1.0f, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float gw = at.own(e) ? g[e] * w[e] : 0.0f;
                t[0] += gw;
                t[1] += at.own(e) ? gw * ((v[e] - mu) * rstd) : 0.0f;
            }
        }
        team_sum<1024, 2>(t, ex, phase);
        const float c1 = t[0] * inv, c2 = t[1] * inv;
        for (int i = threadIdx.x; i * (int64_t)VE < C; i += 1024) {
            const Place<VE> at(i, C);
            float v[VE], g[VE], w[VE];
            load<T, VE>(sr + at.c, v);
            load<T, VE>(gr + at.c, g);
            load_param<VE>(P.w, P.wdtype, at.c, 1.0f, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) g[e] = rstd * (__builtin_fmaf(g[e], w[e], -c1) - (v[e] - mu) * rstd * c2);
            if constexpr (RES) {
                float q[VE];
                load<T, VE>(qr + at.c, q);
#pragma unroll
                for (int e = 0; e < VE; ++e) g[e] += q[e];
            }
            store<T, VE>((T*)P.dx + (int64_t)row * C + at.c, g);
        }
    }
}
// partial sums of the long rows: workgroup (x, y) takes 256 columns and every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void k_ln_bwd_long_params(Bwd P) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= P.C) return;
    float dw = 0.0f, db = 0.0f;
    for (unsigned row = blockIdx.y; row < P.rows; row += gridDim.y) {
        const float s = (float)((const T*)P.s.data)[row_at(P.s, row) + c], g = (float)((const T*)P.gy.data)[row_at(P.gy, row) + c];
        dw = __builtin_fmaf(g, (s - P.mean[row]) * P.rstd[row], dw);
        db += g;
    }
    float* line = P.part + (int64_t)blockIdx.y * 2 * P.C;
    line[c] = dw;
    line[P.C + c] = db;
}

// dw[c], db[c] = the sums of the `n` lines [2][C], in a fixed order: 32 columns x 32 slices of the lines per workgroup
__global__ __launch_bounds__(1024) void k_ln_params(const float* part, int n, int C, void* dw, void* db, int wdtype) {
    __shared__ float sum[32][33];
    const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + c;
    float t = 0.0f;
    if (i < 2 * (int64_t)C) {
        int k = slice;
        for (; k + 7 * 32 < n; k += 8 * 32) {              // eight loads in flight
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[(int64_t)(k + 32 * u) * 2 * C + i];
            t += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; k < n; k += 32) t += part[(int64_t)k * 2 * C + i];
    }
    sum[slice][c] = t;
    __syncthreads();
    if (slice == 0 && i < 2 * (int64_t)C) {
        t = 0.0f;
        for (int k = 0; k < 32; ++k) t += sum[k][c];
        if (i < C) { if (dw) store_param(dw, wdtype, i, t); }
        else if (db) store_param(db, wdtype, i - C, t);
    }
}

int cus() {
    static const int n = [] {                              // (once, whichever thread comes first)
        int dev = 0, v = 0;
        return hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0 ? v : 256;
    }();
    return n;
}

// the team that takes rows of `nvec` vectors: threads and vectors per thread
struct Team { int ts, nv; };
Team team_of(int64_t nvec) {
    static const Team teams[] = {{4, 1}, {8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {128, 2}, {256, 2}, {512, 2}, {1024, 2}};
    for (const Team& t : teams)
        if (nvec <= (int64_t)t.ts * t.nv) return t;
    return {0, 0};                                         // long rows
}
int ve_of(int dtype, int C) { const int ve = dtype == AYOLO_F32 ? 4 : 8; return C < ve ? 1 : ve; }
int rows_per_wg(const Team& t) { return t.ts == 0 || t.ts >= 128 ? 1 : 256 / t.ts; }

int threads_of(const Team& t) { return t.ts < 128 ? 256 : t.ts; }

// Workgroups of the backward pass (= lines of partial sums): eight wavefronts per CU.  Each writes and k_ln_params reads a line
// of 8 C bytes, and its rows are prefetched, so more wavefronts cost more than they hide: 16384 x 4096 bf16 takes 114 / 87 / 102 /
// 120 us with 4 / 8 / 16 / 32 of them, 4096 x 8192 bf16 47 / 58 / 85 us with 8 / 16 / 32, 30000 x 640 fp32 66 / 48 / 48 us with
// 4 / 8 / 16.  And six rows a line, so that the lines stay below the rows' own bytes: 3001 x 1023 fp32 takes 13 us with 512 lines
// and 16 us with 1024.
int bwd_groups(int dtype, int64_t rows, int C) {
    const Team t = team_of(cdiv64(C, ve_of(dtype, C)));
    if (t.ts == 0) return (int)(rows < 64 ? rows : 64);
    int64_t n = cdiv64(rows, rows_per_wg(t));
    const int64_t nt = threads_of(t), most = (int64_t)cus() * (nt < 512 ? 512 / nt : 1), few = rows / 6 > 64 ? rows / 6 : 64;
    if (n > most) n = most;
    return (int)(n < few ? n : few);
}

// Workgroups of the forward pass: what the CUs hold at once (2048 threads each), so that a team walks several rows with its gain
// and bias in registers; up to twice that every team has one row, which spreads better than one or two (25600 x 256 fp16: 7.6
// against 8.3 us).
int64_t fwd_groups(int64_t rows, const Team& t) {
    const int64_t need = cdiv64(rows, rows_per_wg(t)), most = (int64_t)cus() * (2048 / threads_of(t));
    return need <= 2 * most ? need : most;
}

// whether `streams` operands of rows x C elements are more than the caches hold
template <typename T> bool past_caches(unsigned rows, int C, int streams) { return (int64_t)rows * C * sizeof(T) * streams > (256ll << 20); }

template <typename T, int VE, bool RES>
void run_fwd(const Fwd& P, const Team& t, hipStream_t s) {
    if constexpr (VE > 1) if (t.ts == 0) {
        hipLaunchKernelGGL((k_ln_fwd_long<T, VE, RES>), dim3(P.rows < 65536u ? P.rows : 65536u), dim3(1024), 0, s, P);
        return;
    }
    const dim3 grid((unsigned)fwd_groups(P.rows, t));
    const bool once = VE > 1 && past_caches<T>(P.rows, P.C, RES ? 4 : 2);
#define AY_LN(TS_, NV_)                                                                                                        \
    if (t.ts == TS_ && t.nv == NV_) {                                                                                          \
        if (once) hipLaunchKernelGGL((k_ln_fwd<T, VE, TS_, NV_, RES, VE != 1>), grid, dim3(threads_of(t)), 0, s, P);            \
        else hipLaunchKernelGGL((k_ln_fwd<T, VE, TS_, NV_, RES, false>), grid, dim3(threads_of(t)), 0, s, P);                  \
    }
    AY_LN(4, 1) AY_LN(8, 1)
    if constexpr (VE > 1) { AY_LN(16, 1) AY_LN(32, 1) AY_LN(64, 1) AY_LN(64, 2) AY_LN(128, 2) AY_LN(256, 2) AY_LN(512, 2) AY_LN(1024, 2) }
#undef AY_LN
}
template <typename T, int VE, bool RES>
void run_bwd(const Bwd& P, const Team& t, int groups, hipStream_t s) {
    if constexpr (VE > 1) if (t.ts == 0) {
        if (P.dx) hipLaunchKernelGGL((k_ln_bwd_long<T, VE, RES>), dim3(P.rows < 65536u ? P.rows : 65536u), dim3(1024), 0, s, P);
        if (P.part) hipLaunchKernelGGL((k_ln_bwd_long_params<T>), dim3((unsigned)cdiv(P.C, 256), (unsigned)groups), dim3(256), 0, s, P);
        return;
    }
    const dim3 grid((unsigned)groups);
    const bool once = VE > 1 && past_caches<T>(P.rows, P.C, RES ? 4 : 3);
#define AY_LN(TS_, NV_)                                                                                                        \
    if (t.ts == TS_ && t.nv == NV_) {                                                                                          \
        if (once) hipLaunchKernelGGL((k_ln_bwd<T, VE, TS_, NV_, RES, VE != 1>), grid, dim3(threads_of(t)), 0, s, P);            \
        else hipLaunchKernelGGL((k_ln_bwd<T, VE, TS_, NV_, RES, false>), grid, dim3(threads_of(t)), 0, s, P);                  \
    }
    AY_LN(4, 1) AY_LN(8, 1)
    if constexpr (VE > 1) { AY_LN(16, 1) AY_LN(32, 1) AY_LN(64, 1) AY_LN(64, 2) AY_LN(128, 2) AY_LN(256, 2) AY_LN(512, 2) AY_LN(1024, 2) }
#undef AY_LN
}

int check(const char* what, int dtype, int wdtype, int64_t rows, int64_t C) {
    AY_CHECK_ARG(dtype == AYOLO_F16 || dtype == AYOLO_F32 || dtype == AYOLO_BF16, "%s: dtype=%d", what, dtype);
    AY_CHECK_ARG(wdtype == AYOLO_F32 || wdtype == dtype, "%s: the gain and bias are fp32 or of the activations' type (got %d for %d)", what, wdtype, dtype);
    AY_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && C > 0 && C < (1ll << 30), "%s: rows=%lld C=%lld", what, (long long)rows, (long long)C);
    return AYOLO_OK;
}

}  // namespace

extern "C" int ayolo_layer_norm_fwd(int dtype, const ayolo_rows* x, const ayolo_rows* residual, int64_t rows, int64_t C, const void* weight,
                                    const void* bias, int wdtype, float eps, void* y, void* sum, float* mean, float* rstd, ayolo_stream st) {
    if (const int rc = check("layer_norm_fwd", dtype, wdtype, rows, C)) return rc;
    AY_CHECK_ARG(rows == 0 || (x && x->data && y && (!residual || (residual->data && sum)) && !mean == !rstd), "layer_norm_fwd: null buffer");
    if (rows == 0) return AYOLO_OK;
    Fwd P{};
    P.x = *x;
    if (residual) P.r = *residual;
    P.y = y; P.s = sum; P.w = weight; P.b = bias; P.mean = mean; P.rstd = rstd;
    P.rows = (unsigned)rows; P.C = (int)C; P.wdtype = wdtype; P.eps = eps;
    const int ve = ve_of(dtype, P.C);
    const Team t = team_of(cdiv64(C, ve));
    hipStream_t s = (hipStream_t)st;
#define AY_LN(T_, VE_)                                  \
    do {                                                \
        if (residual) run_fwd<T_, VE_, true>(P, t, s);  \
        else run_fwd<T_, VE_, false>(P, t, s);          \
    } while (0)
    if (dtype == AYOLO_F32) { if (ve == 1) AY_LN(float, 1); else AY_LN(float, 4); }
    else if (dtype == AYOLO_F16) { if (ve == 1) AY_LN(half_t, 1); else AY_LN(half_t, 8); }
    else { if (ve == 1) AY_LN(bf16_t, 1); else AY_LN(bf16_t, 8); }
#undef AY_LN
    AY_CHECK_LAUNCH("k_ln_fwd");
    return AYOLO_OK;
}

extern "C" size_t ayolo_layer_norm_bwd_workspace(int dtype, int64_t rows, int64_t C) {
    if (rows <= 0 || C <= 0 || rows >= (1ll << 31) || C >= (1ll << 30)) return 0;
    return (size_t)bwd_groups(dtype, rows, (int)C) * 2 * (size_t)C * sizeof(float);
}

extern "C" int ayolo_layer_norm_bwd(int dtype, const ayolo_rows* sum, const ayolo_rows* dy, const ayolo_rows* dsum, int64_t rows, int64_t C,
                                    const void* weight, int wdtype, const float* mean, const float* rstd, void* dx, void* dweight,
                                    void* dbias, void* ws, size_t ws_bytes, ayolo_stream st) {
    if (const int rc = check("layer_norm_bwd", dtype, wdtype, rows, C)) return rc;
    AY_CHECK_ARG(rows == 0 || (sum && sum->data && dy && dy->data && mean && rstd && (!dsum || dsum->data)), "layer_norm_bwd: null buffer");
    const bool params = dweight || dbias;
    if (!params && (!dx || rows == 0)) return AYOLO_OK;
    hipStream_t s = (hipStream_t)st;
    const int groups = rows ? bwd_groups(dtype, rows, (int)C) : 0;
    if (params && rows) {
        const size_t need = ayolo_layer_norm_bwd_workspace(dtype, rows, C);
        if (!ws || ws_bytes < need) { ayolo_set_error("layer_norm_bwd: workspace %zu < %zu", ws_bytes, need); return AYOLO_ENOSPC; }
    }
    if (rows) {
        Bwd P{};
        P.s = *sum; P.gy = *dy;
        if (dsum) P.gs = *dsum;
        P.dx = dx; P.w = weight; P.mean = mean; P.rstd = rstd; P.part = params ? (float*)ws : nullptr;
        P.rows = (unsigned)rows; P.C = (int)C; P.wdtype = wdtype;
        const int ve = ve_of(dtype, P.C);
        const Team t = team_of(cdiv64(C, ve));
#define AY_LN(T_, VE_)                                         \
    do {                                                       \
        if (dsum) run_bwd<T_, VE_, true>(P, t, groups, s);     \
        else run_bwd<T_, VE_, false>(P, t, groups, s);         \
    } while (0)
        if (dtype == AYOLO_F32) { if (ve == 1) AY_LN(float, 1); else AY_LN(float, 4); }
        else if (dtype == AYOLO_F16) { if (ve == 1) AY_LN(half_t, 1); else AY_LN(half_t, 8); }
        else { if (ve == 1) AY_LN(bf16_t, 1); else AY_LN(bf16_t, 8); }
#undef AY_LN
        AY_CHECK_LAUNCH("k_ln_bwd");
    }
    if (params) {                                              // no rows: zeros
        hipLaunchKernelGGL(k_ln_params, dim3((unsigned)cdiv64(2 * C, 32)), dim3(1024), 0, s, (const float*)ws, groups, (int)C, dweight, dbias, wdtype);
        AY_CHECK_LAUNCH("k_ln_params");
    }
    return AYOLO_OK;
}
