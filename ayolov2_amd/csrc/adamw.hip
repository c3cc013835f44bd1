// The optimiser's side of a training step over MANY tensors at once, beside the SGD step of optim.hip: the 2-norm of all
// gradients, their clipping, and AdamW with its two moments in 32 or in 8 bits.
//
//   norm = sqrt(sum g^2) / grad_scale            clip: g *= min(1, max_norm / (norm + 1e-6))
//   t += 1   g' = (+-) g / grad_scale * min(1, max_norm / (norm + 1e-6))
//   m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p -= lr wd p + lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  Per fp32 parameter 4 B for the norm, 8 B for the clipping, 28 B for AdamW with 32-bit moments and 16 B with 8-bit
// ones.  The tensors come as a list on the host and travel BY VALUE in the kernel arguments (up to 4 KB per launch), so nothing is
// copied to the device, nothing has to be kept between calls, and a captured call replays as it is.  An address is kept as its low
// half and the number of its 4 GB window, of which a launch knows 16 (an allocator's segments lie far apart), so that a launch
// takes 332 gradients, 141 tensors with 32-bit and 109 with 8-bit moments: every further launch costs some 4 us of start and drain.
// A workgroup takes a chunk of one tensor; it finds its tensor by comparing the jobs' first workgroups 64 at a time.
#include "common.h"
#include <math.h>
#include <algorithm>
#include <vector>

typedef __bf16 bf16_t;
typedef unsigned v2u __attribute__((ext_vector_type(2)));

namespace {

// Elements per workgroup of 256 threads, as vectors of four that all are loaded before the first is used.  One tensor's chunks
// are many and short, so that the drain of a launch is short too: 46.5 M bf16 parameters take 169 / 179 / 192 / 206 us with 2048 /
// 4096 / 8192 / 16384 elements a workgroup, 86.7 M with 8-bit moments 399 / 408 / 442 / 476.  The norm and the clipping, with one
// vector to load per element, take 104 / 97 / 98 / 99.
constexpr int CHUNK_ADAMW = 2048, CHUNK_GRAD = 4096, CHUNK_VALUES = 4096;
constexpr unsigned PART = 1u << 30;                        // a larger tensor travels as several jobs (a multiple of every chunk)
constexpr unsigned MOST_WGS = 1u << 20;                    // of a launch, before its last job (at most 2^19 more)

template <typename T> struct V4 { typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };
// ONCE: past the caches, for what is not used again before the caches have seen everything else.  The gradients, the moments and
// unpacked values move that way, parameters on their way in; with 32-bit moments 46.5 M bf16 parameters take 177 us instead of
// 211 (183 where the parameters are stored that way too), with 8-bit ones 86.7 M fp32 parameters and their unpacked moments 399
// instead of 465 (442 where the parameters are stored the ordinary way).  Codes are better off in the caches (417 us past them),
// and so are the gradients that the norm reads when the clipping reads them next (93 us against 100 for 46.5 M).
template <bool ONCE, typename T> __device__ __forceinline__ float4v load4(const T* p) {
    const auto* q = reinterpret_cast<const typename V4<T>::type*>(p);
    const typename V4<T>::type r = ONCE ? __builtin_nontemporal_load(q) : *q;
    return float4v{(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
}
template <bool ONCE, typename T> __device__ __forceinline__ void store4(T* p, float4v v) {
    typename V4<T>::type r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (T)v[e];
    auto* q = reinterpret_cast<typename V4<T>::type*>(p);
    if constexpr (ONCE) __builtin_nontemporal_store(r, q);
    else *q = r;
}
// the first `n` of four elements; the others read as zero and are not written
template <typename T> __device__ __forceinline__ float4v load_upto(const T* p, int n) {
    if (n >= 4) return load4<false>(p);
    float4v v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) v[e] = (float)p[e];
    return v;
}
template <typename T> __device__ __forceinline__ void store_upto(T* p, float4v v, int n) {
    if (n >= 4) { store4<false>(p, v); return; }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = (T)v[e];
}

// Four elements at `i` of `n`.  A chunk that lies whole inside its tensor (FULL, a uniform condition) has no guards: a load under
// a per-lane condition is a branch with a wait behind it, and nothing else would be in flight.
template <bool FULL> struct At {
    unsigned i;
    int left;
    __device__ __forceinline__ At(unsigned at, int k, unsigned n) {
        i = at + k * 1024 + threadIdx.x * 4;
        left = FULL ? 4 : i < n ? (int)min(n - i, 4u) : 0;
        if (!FULL && i >= n) i = 0;
    }
    template <bool ONCE = false, typename T> __device__ __forceinline__ float4v load(const T* p) const { return FULL ? load4<ONCE>(p + i) : load_upto(p + i, left); }
    template <bool ONCE = false, typename T> __device__ __forceinline__ void store(T* p, float4v v) const {
        if (FULL) store4<ONCE>(p + i, v);
        else if (left > 0) store_upto(p + i, v, left);
    }
};
// A whole chunk goes at once; the others go one vector per thread at a time (they are few, and the code stays small).
template <bool FULL, int CHUNK> constexpr int U = FULL ? CHUNK / 1024 : 1;
template <int CHUNK, typename F>
__device__ __forceinline__ void each_part(unsigned at, unsigned n, F f) {
    for (unsigned i = at; i < at + CHUNK && i < n; i += 1024) f(i);
}

// A launch's tensors.  HEAD: what the kernel needs besides; N addresses per tensor.
struct Where { unsigned first, tag, tensor; };             // first workgroup; two bits of the caller's; place in the caller's list
// 4 GB windows of addresses: the high halves, by number
struct Windows {
    static constexpr int MAX = 16;
    unsigned hi[MAX];
    // (through the global address space: an address made of numbers would be taken for a generic one)
    __device__ __forceinline__ void* at(unsigned which, unsigned lo) const {
        return (void*)(__attribute__((address_space(1))) void*)((uint64_t)hi[which] << 32 | lo);
    }
    // host: the number of an address's window among the first `n`, added where it is new; -1: no room
    int number(int& n, const void* p) {
        const unsigned h = (unsigned)((uintptr_t)p >> 32);
        for (int k = 0; k < n; ++k)
            if (hi[k] == h) return k;
        if (n == MAX) return -1;
        hi[n] = h;
        return n++;
    }
};
// a job's numbers: low halves of its addresses, four bits of window for each, elements; first workgroup (21 bits), tag (2), place (9)
template <int N> struct AddressJob {
    unsigned lo[N], windows, n, meta;
    __device__ __forceinline__ unsigned window(int a) const { return windows >> 4 * a & 15u; }
    __device__ __forceinline__ unsigned place() const { return meta >> 23; }
    void set(unsigned first, unsigned tag, unsigned at, unsigned w) { meta = first | tag << 21 | at << 23; windows = w; }
};
template <> struct AddressJob<1> {                         // a single address and no place: the window takes the place's bits
    unsigned lo[1], n, meta;
    __device__ __forceinline__ unsigned window(int) const { return meta >> 23; }
    __device__ __forceinline__ unsigned place() const { return 0; }
    void set(unsigned first, unsigned tag, unsigned, unsigned w) { meta = first | tag << 21 | w << 23; }
};
template <typename HEAD, int N, int CH> struct Jobs {
    static constexpr int ADDRESSES = N, CHUNK = CH;
    typedef AddressJob<N> Job;
    static constexpr int MAX = (4096 - (int)sizeof(HEAD) - (int)sizeof(Windows) - 16) / (int)sizeof(Job);
    HEAD h;
    Windows w;
    int njobs;
    unsigned tensor0;
    Job j[MAX];
    template <typename T> __device__ __forceinline__ T* at(int k, int a) const { return (T*)w.at(j[k].window(a), j[k].lo[a]); }
    __device__ __forceinline__ Where where(int k) const {
        const unsigned m = j[k].meta;
        return Where{m & 0x1fffffu, m >> 21 & 3u, tensor0 + j[k].place()};
    }
    // the job whose workgroups hold this one (`first` ascends): every `s`-th job first, then the ones behind it
    __device__ __forceinline__ int mine() const {
        const int lane = (int)(threadIdx.x & 63), s = (njobs + 63) / 64;
        auto below = [&](int i, bool ask) { return __popcll(__ballot(ask && (j[ask ? i : 0].meta & 0x1fffffu) <= blockIdx.x)); };
        int k = (below(lane * s, lane * s < njobs) - 1) * s;
        if (s > 1) k += below(k + lane, lane < s && k + lane < njobs) - 1;
        return __builtin_amdgcn_readfirstlane(k);
    }
};

// ------------------------------------------------------------------------------------------------ norm and clipping
struct GHead {
    const float* norm;
    double* part;
    float max_norm;
};
typedef Jobs<GHead, 1, CHUNK_GRAD> GJobs;                  // tag: the gradient's type
static_assert(sizeof(GJobs) <= 4096 && GJobs::MAX == 332, "kernel arguments");

template <bool FULL, typename T>
__device__ __forceinline__ double squares(const T* g, unsigned n, unsigned at) {
    float4v x[U<FULL, CHUNK_GRAD>];
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_GRAD>; ++k) x[k] = At<FULL>(at, k, n).load(g);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_GRAD>; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += (double)x[k][e] * (double)x[k][e];
    return s;
}
__device__ __forceinline__ double wave_sum(double v) {
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}
// one partial sum per workgroup, in fp64: squares of fp32 values neither overflow nor vanish, and the order of the additions
// does not show in the rounded result.  fp64 runs at half the fp32 rate here and stays far below the memory time.
__global__ __launch_bounds__(256) void k_grad_squares(GJobs P) {
    __shared__ double w[4];
    const int j = P.mine();
    const Where J = P.where(j);
    const unsigned at = (blockIdx.x - J.first) * CHUNK_GRAD, n = P.j[j].n;
    auto of = [&](auto* g) {
        if (at + CHUNK_GRAD <= n) return squares<true>(g, n, at);
        double t = 0.0;
        each_part<CHUNK_GRAD>(at, n, [&](unsigned i) { t += squares<false>(g, n, i); });
        return t;
    };
    double s = J.tag == AYOLO_F32   ? of(P.at<const float>(j, 0))
               : J.tag == AYOLO_F16 ? of(P.at<const half_t>(j, 0))
                                    : of(P.at<const bf16_t>(j, 0));
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) P.h.part[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}
__global__ __launch_bounds__(1024) void k_grad_norm(const double* part, int64_t n, const float* grad_scale, float* out) {
    __shared__ double w[16];
    double s = 0.0;
    int64_t i = threadIdx.x;
    for (; i + 7 * 1024 < n; i += 8 * 1024) {              // eight loads in flight
        double v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = part[i + 1024 * k];
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; i < n; i += 1024) s += part[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += w[i];
        t = sqrt(t);
        *out = (float)(grad_scale ? t / (double)*grad_scale : t);
    }
}

// min(1, max_norm / (norm + 1e-6)); a NaN norm gives NaN, as the formula does
__device__ __forceinline__ float clip_factor(const float* norm, float max_norm) {
    const float c = max_norm / (*norm + 1e-6f);
    return c > 1.0f ? 1.0f : c;
}

template <bool FULL, typename T>
__device__ __forceinline__ void scale(T* g, unsigned n, unsigned at, float f) {
    float4v x[U<FULL, CHUNK_GRAD>];
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_GRAD>; ++k) x[k] = At<FULL>(at, k, n).template load<true>(g);
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_GRAD>; ++k) At<FULL>(at, k, n).template store<true>(g, x[k] * f);
}
__global__ __launch_bounds__(256) void k_grad_clip(GJobs P) {
    const int j = P.mine();
    const Where J = P.where(j);
    const unsigned at = (blockIdx.x - J.first) * CHUNK_GRAD, n = P.j[j].n;
    const float f = clip_factor(P.h.norm, P.h.max_norm);
    if (f == 1.0f) return;                                 // nothing to clip: the gradients stay as they are
    auto of = [&](auto* g) {
        if (at + CHUNK_GRAD <= n) scale<true>(g, n, at, f);
        else each_part<CHUNK_GRAD>(at, n, [&](unsigned i) { scale<false>(g, n, i, f); });
    };
    if (J.tag == AYOLO_F32) of(P.at<float>(j, 0));
    else if (J.tag == AYOLO_F16) of(P.at<half_t>(j, 0));
    else of(P.at<bf16_t>(j, 0));
}

// -------------------------------------------------------------------------------------------------- 8-bit moments
// A moment in 8 bits: one byte per element and one exponent byte E per block of 128 elements (memory order), the biased fp32
// exponent of the block's largest finite magnitude.  m: sign, 4 exponent bits, 3 mantissa bits; v: 5 exponent bits, 3 mantissa
// bits.  Read as the top bits of an fp32 number (code << 20) and scaled by 2^(E - B), B = 14 (m) or 30 (v): the block's largest
// value has exponent field B, field B + 1 takes the carry of a rounding up and the codes of infinity and NaN, field 0 holds the
// subnormals, whose spacing fp32's own subnormals give without a branch.
//
// The ranges fit each other: m keeps 2^-17 of its block's largest value, v 2^-33 (sqrt: 2^-16.5), and a v above zero never
// becomes zero, so that the smallest kept m over the smallest kept sqrt(v) stays a step of ordinary size.
//
// Rounding is stochastic, E[stored] = value (but for a v above zero and below its block's smallest code, which becomes that code):
// at b2 = 0.999 a step moves v by 0.1 % and a 3-bit mantissa by 6 % or nothing, so that rounding to nearest would hold v where it
// first was.  16 random bits (and a half of the next) per rounding come from a
// hash of (seed, t, position of the tensor, element): a call's result depends on its arguments alone.
constexpr int M_BIAS = 14, V_BIAS = 30, M_LEAST = 1, V_LEAST = 10;      // least E: keeps every value a multiple of 2^-149

__device__ __forceinline__ unsigned mix(unsigned x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;                                      // odd: the first bits of the fractions of sqrt(2) and sqrt(3)
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
constexpr unsigned STRIDE = 0x9E3779B1u;                   // 2^32 / golden ratio, odd

// One code at a time, every value: the way of a wavefront that holds an infinity or a NaN.
template <bool SIGNED>
__device__ __forceinline__ float decode(unsigned code, int e) {
    const unsigned mag = SIGNED ? code & 0x7fu : code, top = SIGNED ? 0x7fu : 0xffu;
    float x = __builtin_ldexpf(__uint_as_float(mag << 20), e - (SIGNED ? M_BIAS : V_BIAS));
    if (mag >= top - 1) x = mag == top ? __uint_as_float(0x7fc00000u) : __uint_as_float(0x7f800000u);
    return SIGNED && (code & 0x80u) ? -x : x;
}
template <bool SIGNED>
__device__ __forceinline__ unsigned encode(float x, int e, unsigned r16) {
    const unsigned top = SIGNED ? 0x7fu : 0xffu, bits = __float_as_uint(x) & 0x7fffffffu;
    const float y = __builtin_ldexpf(__uint_as_float(bits), (SIGNED ? M_BIAS : V_BIAS) - e);
    unsigned code = (__float_as_uint(y) + (r16 << 4 | 8u)) >> 20;
    if (!SIGNED && code == 0 && bits != 0) code = 1;
    if (bits >= 0x7f800000u) code = bits == 0x7f800000u ? top - 1 : top;
    return SIGNED && bits <= 0x7f800000u ? code | (__float_as_uint(x) >> 24 & 0x80u) : code;
}
// Four codes.  An e4m3 byte is m's code as the hardware's conversion reads it (exponent bias 7), but for the infinity's; v's is
// put into place as it is.
template <bool SIGNED>
__device__ __forceinline__ float4v decode4(unsigned c, int e) {
    const unsigned high = ((c & 0x7f7f7f7fu) + 0x02020202u) & 0x80808080u;      // the low seven bits of a byte above 0x7d
    if (__ballot((SIGNED ? high : high & c) != 0)) {
        return float4v{decode<SIGNED>(c & 255u, e), decode<SIGNED>(c >> 8 & 255u, e), decode<SIGNED>(c >> 16 & 255u, e), decode<SIGNED>(c >> 24, e)};
    }
    float4v x;
    if constexpr (SIGNED) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
        x = float4v{lo[0], lo[1], hi[0], hi[1]};
        e -= M_BIAS + 127 - 7;
    } else {
        x = float4v{__uint_as_float(c << 20 & 0x0ff00000u), __uint_as_float(c << 12 & 0x0ff00000u), __uint_as_float(c << 4 & 0x0ff00000u),
                    __uint_as_float(c >> 4 & 0x0ff00000u)};
        e -= V_BIAS;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __builtin_ldexpf(x[k], e);
    return x;
}
// the largest over the 32 lanes of a block, in all of them
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ unsigned block_max(unsigned v) {
    v = dpp_max<0xB1>(v);
    v = dpp_max<0x4E>(v);
    v = dpp_max<0x141>(v);
    v = dpp_max<0x140>(v);
    const v2u r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(r[0], r[1]);
}
// Four values of a block into codes; `e`: the block's exponent, r: 16 random bits each.
template <bool SIGNED>
__device__ __forceinline__ unsigned encode4(float4v x, const unsigned (&r)[4], int& e) {
    constexpr int BIAS = SIGNED ? M_BIAS : V_BIAS, LEAST = SIGNED ? M_LEAST : V_LEAST;
    unsigned b[4], top = 0, c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, b[k] = __float_as_uint(x[k]) & 0x7fffffffu);
    top = block_max(top);
    if (__ballot(top >= 0x7f800000u)) {                    // the largest finite one
        top = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = b[k] < 0x7f800000u ? max(top, b[k]) : top;
        e = max((int)(block_max(top) >> 23), LEAST);
#pragma unroll
        for (int k = 0; k < 4; ++k) c |= encode<SIGNED>(x[k], e, r[k]) << 8 * k;
        return c;
    }
    e = max((int)(top >> 23), LEAST);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        unsigned t = (__float_as_uint(__builtin_ldexpf(x[k], BIAS - e)) + (r[k] << 4 | 8u)) >> 20;
        if constexpr (SIGNED) t = (t & 0x7fu) | (t >> 4 & 0x80u);
        else t = max(t, min(b[k], 1u));
        c |= t << 8 * k;
    }
    return c;
}
__device__ __forceinline__ unsigned load_codes(const uint8_t* p, int n) {
    typedef unsigned u1 __attribute__((aligned(1)));
    if (n >= 4) return *reinterpret_cast<const u1*>(p);
    unsigned c = 0;
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) c |= (unsigned)p[e] << 8 * e;
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, unsigned c, int n) {
    typedef unsigned u1 __attribute__((aligned(1)));
    if (n >= 4) { *reinterpret_cast<u1*>(p) = c; return; }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = (uint8_t)(c >> 8 * e);
}
// ----------------------------------------------------------------------------------------------------------- AdamW
struct Coef { float step, decay, root; unsigned key; };    // lr / (1 - b1^t), lr wd, 1 / sqrt(1 - b2^t), the tensor's random key

// Tensors that share a learning rate and decay share an entry of `pair`.
struct PrepJobs {
    static constexpr int MAX = 420, PAIRS = 64;
    double ln_b1, ln_b2;
    const float *lr, *found_inf;
    Coef* out;
    unsigned seed, place0;
    int n, pairs;
    Windows w;
    struct { float lr, wd; } pair[PAIRS];
    struct { unsigned lo, which; } j[MAX];                 // the step count's address; pair (6 bits), window (4), place in the list - place0 (22)
};
static_assert(sizeof(PrepJobs) <= 4096, "kernel arguments");

// One thread per tensor: count the step and leave what depends on it to the update kernels.  1 - b^t in fp64: for b = 0.999 and
// the first steps an fp32 difference would keep few of its bits.
__global__ __launch_bounds__(512) void k_adamw_prepare(PrepJobs P) {
    const int i = threadIdx.x;
    if (i >= P.n) return;
    if (P.found_inf && *P.found_inf != 0.0f) return;
    float* step = (float*)P.w.at(P.j[i].which >> 6 & 15u, P.j[i].lo);
    const unsigned pair = P.j[i].which & 63u, place = P.place0 + (P.j[i].which >> 10);
    const float t = *step + 1.0f;
    *step = t;
    const double lr = P.lr ? (double)*P.lr : (double)P.pair[pair].lr;
    Coef c;
    c.step = (float)(lr / -expm1((double)t * P.ln_b1));
    c.decay = (float)(lr * (double)P.pair[pair].wd);
    c.root = (float)(1.0 / sqrt(-expm1((double)t * P.ln_b2)));
    c.key = mix(mix(P.seed + STRIDE * (unsigned)t) + STRIDE * (place + 1));
    P.out[place] = c;
}

struct Hyper {
    const float *grad_scale, *found_inf, *norm;
    const Coef* coef;
    float b1, c1, b2, c2, eps, max_norm;
    int maximize;
};
// p, g, m, v (and the moments' exponents); tag: which 2^30 elements of its tensor a job is
template <bool BITS8> using AJobs = Jobs<Hyper, BITS8 ? 6 : 4, CHUNK_ADAMW>;
static_assert(sizeof(AJobs<false>) <= 4096 && AJobs<false>::MAX == 141 && sizeof(AJobs<true>) <= 4096 && AJobs<true>::MAX == 109, "kernel arguments");
template <typename T, bool BITS8> struct Tensor;
template <typename T> struct Tensor<T, false> {
    T* p;
    const T* g;
    float *m, *v;
    unsigned n;
    __device__ __forceinline__ Tensor(const AJobs<false>& P, int j)
        : p(P.template at<T>(j, 0)), g(P.template at<const T>(j, 1)), m(P.template at<float>(j, 2)), v(P.template at<float>(j, 3)),
          n(P.j[j].n) {}
};
template <typename T> struct Tensor<T, true> {
    T* p;
    const T* g;
    uint8_t *m, *v, *me, *ve;
    unsigned n, origin;                                    // origin: the job's first element in its tensor
    __device__ __forceinline__ Tensor(const AJobs<true>& P, int j)
        : p(P.template at<T>(j, 0)), g(P.template at<const T>(j, 1)), m(P.template at<uint8_t>(j, 2)), v(P.template at<uint8_t>(j, 3)),
          me(P.template at<uint8_t>(j, 4)), ve(P.template at<uint8_t>(j, 5)), n(P.j[j].n), origin(P.where(j).tag * PART) {}
};

struct Scalars { float scale, factor; bool scaled; };
__device__ __forceinline__ float4v true_grad(float4v g, const Scalars& c) {
    if (c.scaled)
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = g[e] / c.scale;
    return g * c.factor;
}
// the moments, one rounding per operation (compiled without contraction): a plain sequence of the formula's products and sums
__device__ __forceinline__ void moments(float4v g, const Hyper& h, float4v& m, float4v& v) {
    m = m * h.b1 + g * h.c1;
    v = v * h.b2 + g * g * h.c2;
}
// Square root and quotient by the hardware's own functions, each 1 ulp: with the two roundings around them below 4 u of the
// step.  They take subnormal numbers for zero: a root below 2^-63, times c.root, must be nothing beside eps, i.e. at most 2^-26 of
// it.  So it is from eps = 2.3e-10 on in the first step of b2 = 0.999, 7.3e-12 in the late ones; below, the exact functions are used.
__device__ __forceinline__ float4v stepped(float4v p, float4v m, float4v v, const Coef& c, float eps) {
    if (eps >= c.root * 0x1p-37f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = __builtin_fmaf(__builtin_amdgcn_sqrtf(v[e]), c.root, eps);
            p[e] -= __builtin_fmaf(p[e], c.decay, c.step * m[e] * __builtin_amdgcn_rcpf(d));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = __builtin_fmaf(sqrtf(v[e]), c.root, eps);
            p[e] -= __builtin_fmaf(p[e], c.decay, c.step * (m[e] / d));
        }
    }
    return p;
}

template <bool FULL, typename T>
__device__ __forceinline__ void step_chunk(const Tensor<T, false>& J, const Hyper& h, const Coef& c, const Scalars& sc, unsigned at) {
    float4v x[U<FULL, CHUNK_ADAMW>], d[U<FULL, CHUNK_ADAMW>], m[U<FULL, CHUNK_ADAMW>], v[U<FULL, CHUNK_ADAMW>];
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_ADAMW>; ++k) {
        const At<FULL> a(at, k, J.n);
        d[k] = a.template load<true>(J.g);
        m[k] = a.template load<true>(J.m);
        v[k] = a.template load<true>(J.v);
        x[k] = a.template load<true>(J.p);
    }
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_ADAMW>; ++k) {
        const At<FULL> a(at, k, J.n);
        moments(true_grad(d[k], sc), h, m[k], v[k]);
        a.template store<true>(J.m, m[k]);
        a.template store<true>(J.v, v[k]);
        a.store(J.p, stepped(x[k], m[k], v[k], c, h.eps));
    }
}
// 32 lanes hold one block of 128
template <bool FULL, typename T>
__device__ __forceinline__ void step_chunk(const Tensor<T, true>& J, const Hyper& h, const Coef& c, const Scalars& sc, unsigned at) {
    float4v x[U<FULL, CHUNK_ADAMW>], d[U<FULL, CHUNK_ADAMW>];
    unsigned mc[U<FULL, CHUNK_ADAMW>], vc[U<FULL, CHUNK_ADAMW>];
    int me[U<FULL, CHUNK_ADAMW>], ve[U<FULL, CHUNK_ADAMW>];
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_ADAMW>; ++k) {
        const At<FULL> a(at, k, J.n);
        d[k] = a.template load<true>(J.g);
        mc[k] = load_codes(J.m + a.i, a.left);
        vc[k] = load_codes(J.v + a.i, a.left);
        me[k] = J.me[a.i / 128];
        ve[k] = J.ve[a.i / 128];
        x[k] = a.template load<true>(J.p);
    }
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_ADAMW>; ++k) {
        const At<FULL> a(at, k, J.n);
        float4v m = decode4<true>(mc[k], me[k]), v = decode4<false>(vc[k], ve[k]);
        moments(true_grad(d[k], sc), h, m, v);
        if constexpr (!FULL) {
#pragma unroll
            for (int e = 0; e < 4; ++e)                    // past the end: not part of the block
                if (e >= a.left) m[e] = v[e] = 0.0f;
        }
        a.template store<true>(J.p, stepped(x[k], m, v, c, h.eps));
        unsigned rm[4], rv[4];
        const unsigned first = (J.origin + a.i) * STRIDE;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned r = mix((first + e * STRIDE) ^ c.key);
            rm[e] = r >> 16;
            rv[e] = r & 0xffffu;
        }
        int em, ev;
        const unsigned cm = encode4<true>(m, rm, em), cv = encode4<false>(v, rv, ev);
        if (FULL || a.left > 0) {
            store_codes(J.m + a.i, cm, a.left);
            store_codes(J.v + a.i, cv, a.left);
            if ((threadIdx.x & 31) == 0) {
                J.me[a.i / 128] = (uint8_t)em;
                J.ve[a.i / 128] = (uint8_t)ev;
            }
        }
    }
}

template <typename T, bool BITS8>
__global__ __launch_bounds__(256) void k_adamw(AJobs<BITS8> P) {
    const Hyper& h = P.h;
    if (h.found_inf && *h.found_inf != 0.0f) return;
    const int j = P.mine();
    const Where W = P.where(j);
    const Tensor<T, BITS8> J(P, j);
    const Coef c = h.coef[W.tensor];
    Scalars sc;
    sc.scaled = h.grad_scale != nullptr;
    sc.scale = sc.scaled ? *h.grad_scale : 1.0f;
    sc.factor = (h.norm ? clip_factor(h.norm, h.max_norm) : 1.0f) * (h.maximize ? -1.0f : 1.0f);
    const unsigned at = (blockIdx.x - W.first) * CHUNK_ADAMW;
    if (at + CHUNK_ADAMW <= J.n) step_chunk<true>(J, h, c, sc, at);
    else each_part<CHUNK_ADAMW>(at, J.n, [&](unsigned i) { step_chunk<false>(J, h, c, sc, i); });
}

struct None {};
typedef Jobs<None, 3, CHUNK_VALUES> UJobs;                               // codes, exponents, values
static_assert(sizeof(UJobs) <= 4096, "kernel arguments");
template <bool SIGNED, bool FULL>
__device__ __forceinline__ void values_chunk(const uint8_t* codes, const uint8_t* exps, float* out, unsigned n, unsigned at) {
    unsigned c[U<FULL, CHUNK_VALUES>];
    int e[U<FULL, CHUNK_VALUES>];
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_VALUES>; ++k) {
        const At<FULL> a(at, k, n);
        c[k] = load_codes(codes + a.i, a.left);
        e[k] = exps[a.i / 128];
    }
#pragma unroll
    for (int k = 0; k < U<FULL, CHUNK_VALUES>; ++k) At<FULL>(at, k, n).template store<true>(out, decode4<SIGNED>(c[k], e[k]));
}
template <bool SIGNED>
__global__ __launch_bounds__(256) void k_moment_values(UJobs P) {
    const int j = P.mine();
    const unsigned at = (blockIdx.x - P.where(j).first) * CHUNK_VALUES, n = P.j[j].n;
    const uint8_t *codes = P.at<const uint8_t>(j, 0), *exps = P.at<const uint8_t>(j, 1);
    float* out = P.at<float>(j, 2);
    if (at + CHUNK_VALUES <= n) values_chunk<SIGNED, true>(codes, exps, out, n, at);
    else each_part<CHUNK_VALUES>(at, n, [&](unsigned i) { values_chunk<SIGNED, false>(codes, exps, out, n, i); });
}

// ------------------------------------------------------------------------------------------------------------- host
int es_of(int dtype) { return dtype == AYOLO_F32 ? 4 : dtype == AYOLO_U8 ? 1 : 2; }
bool is_float(int dtype) { return dtype == AYOLO_F32 || dtype == AYOLO_F16 || dtype == AYOLO_BF16; }

// every tensor of the list is a dense block of device memory of one device, of a type that `ok` takes
template <typename OK>
int check_list(const char* what, const char* name, const ayolo_tensor* t, int n, int& device, OK ok) {
    for (int i = 0; i < n; ++i) {
        if (!t[i].present) continue;
        AY_CHECK_ARG(t[i].device >= 0, "%s: %s[%d] is not on a GPU (the HIP path has no CPU fallback)", what, name, i);
        if (device < 0) device = t[i].device;
        AY_CHECK_ARG(t[i].device == device, "%s: %s[%d] is on device %d, others on %d", what, name, i, t[i].device, device);
        AY_CHECK_ARG(ok(t[i].dtype), "%s: %s[%d] has an unsupported type", what, name, i);
        AY_CHECK_ARG(t[i].layout != 0, "%s: %s[%d] is not a dense block of memory", what, name, i);
        AY_CHECK_ARG(t[i].numel == 0 || t[i].data, "%s: %s[%d] has no memory", what, name, i);
        AY_CHECK_ARG(((uintptr_t)t[i].data & (es_of(t[i].dtype) - 1)) == 0, "%s: %s[%d] is not aligned to its type", what, name, i);
    }
    return AYOLO_OK;
}
// Whether a tensor that is written shares memory with another one: sorted by address, does a range begin before a written one has
// ended, or a written one before any has?  Two that are only read may share.  A model has some thousand ranges per step.  Lists that
// are views of a few blocks ascend for long, and where the stretches in which they do lie apart there is nothing to sort; where they
// do not, ten bits at a time at most, of those in which the addresses differ, sort them in a few us of host time.
struct Range {
    uintptr_t from, end;                                   // end: its top bit says that the range is written
    bool written() const { return end >> 63; }
    uintptr_t to() const { return end & ~(uintptr_t)0 >> 1; }
};
size_t bytes_of(const ayolo_tensor& t) { return (size_t)t.numel * es_of(t.dtype); }
template <typename F>
void each_range(const ayolo_tensor* t, int n, bool written, F f, const ayolo_tensor* given = nullptr) {
    f(nullptr, 0, false);                                  // (a list of its own: a stretch that went on would span what lies between)
    for (int i = 0; i < n; ++i)
        if (t[i].present && (!given || given[i].present)) f(t[i].data, bytes_of(t[i]), written);
}
struct Stretches {
    static constexpr int MOST = 32;
    struct { uintptr_t from, to; } of[MOST];
    int n = 0;
    uintptr_t from = 0, to = 0;
    void close() {
        if (to && n < MOST) of[n].from = from, of[n].to = to;
        n += to != 0;
    }
    void add(uintptr_t a, size_t bytes) {                  // nothing (a new list): the stretch ends
        if (a < to || !to || !bytes) {
            close();
            from = a;
        }
        to = bytes ? a + bytes : 0;
    }
    bool apart() {
        close();
        if (n > MOST) return false;
        std::sort(of, of + n, [](const auto& x, const auto& y) { return x.from < y.from; });
        for (int k = 1; k < n; ++k)
            if (of[k].from < of[k - 1].to) return false;
        return true;
    }
};
void sort_ranges(std::vector<Range>& r) {
    if (r.size() < 128) {
        std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
        return;
    }
    uintptr_t differ = 0;
    for (const Range& x : r) differ |= x.from ^ r[0].from;
    if (!differ) return;
    const unsigned low = __builtin_ctzll(differ), width = 64 - __builtin_clzll(differ) - low, passes = (width + 9) / 10;
    const unsigned bits = (width + passes - 1) / passes, mask = (1u << bits) - 1;
    std::vector<Range> other(r.size());
    for (unsigned shift = low, k = 0; k < passes; ++k, shift += bits) {
        unsigned at[1025];
        std::fill(at, at + mask + 2, 0u);
        for (const Range& x : r) ++at[(x.from >> shift & mask) + 1];
        for (unsigned i = 0; i < mask; ++i) at[i + 1] += at[i];
        for (const Range& x : r) other[at[x.from >> shift & mask]++] = x;
        r.swap(other);
    }
}
// each(f): calls f(address, bytes, written) for every range of the call
template <typename EACH>
bool overlap(size_t most, EACH each) {
    Stretches s;
    each([&](const void* p, size_t bytes, bool) { s.add((uintptr_t)p, p ? bytes : 0); });
    if (s.apart()) return false;
    std::vector<Range> r;
    r.reserve(most);
    each([&](const void* p, size_t bytes, bool written) {
        if (p && bytes) r.push_back(Range{(uintptr_t)p, ((uintptr_t)p + bytes) | (uintptr_t)written << 63});
    });
    sort_ranges(r);
    uintptr_t any = 0, written = 0;                        // where the ranges before this one have ended
    for (const Range& x : r) {
        if (x.from < (x.written() ? any : written)) return true;
        any = std::max(any, x.to());
        if (x.written()) written = std::max(written, x.to());
    }
    return false;
}

// Splits a list into launches.  where(i, off, address): a job's addresses, from element `off` of tensor i on; tag(i, part): its two
// bits; go(jobs, workgroups) launches what has gathered.
template <typename JOBS, typename WHERE, typename TAG, typename GO>
int each_launch(JOBS& P, const ayolo_tensor* t, int n, WHERE where, TAG tag, GO go) {
    constexpr int N = JOBS::ADDRESSES;
    static_assert(N <= 8, "four bits of window per address");
    unsigned wgs = 0;
    int windows = 0;
    P.njobs = 0;
    auto flush = [&]() -> int {
        const int rc = P.njobs ? go(P, wgs) : AYOLO_OK;
        P.njobs = windows = 0;
        wgs = 0;
        return rc;
    };
    for (int i = 0; i < n; ++i) {
        if (!t[i].present) continue;
        for (int64_t off = 0; off < t[i].numel; off += PART) {
            char* a[N];
            where(i, off, a);
            unsigned which = 0;
            auto fits = [&]() {
                if (P.njobs == JOBS::MAX || wgs >= MOST_WGS || (P.njobs && (unsigned)i - P.tensor0 >= 512u)) return false;
                which = 0;
                for (int k = 0; k < N; ++k) {
                    const int w = P.w.number(windows, a[k]);
                    if (w < 0) return false;
                    which |= (unsigned)w << 4 * k;
                }
                return true;
            };
            if (!fits()) {
                if (const int rc = flush()) return rc;
                fits();                                    // alone it does: N windows at most
            }
            if (P.njobs == 0) P.tensor0 = (unsigned)i;
            auto& J = P.j[P.njobs++];
            for (int k = 0; k < N; ++k) J.lo[k] = (unsigned)(uintptr_t)a[k];
            J.n = (unsigned)std::min<int64_t>(PART, t[i].numel - off);
            J.set(wgs, tag(i, (unsigned)(off / PART)), (unsigned)i - P.tensor0, which);
            wgs += (J.n + JOBS::CHUNK - 1) / JOBS::CHUNK;
        }
    }
    return flush();
}

int64_t chunks_of(const ayolo_tensor* t, int n) {
    int64_t c = 0;
    for (int i = 0; i < n; ++i)
        if (t[i].present)
            for (int64_t off = 0; off < t[i].numel; off += PART) c += cdiv64(std::min<int64_t>(PART, t[i].numel - off), CHUNK_GRAD);
    return c;
}

template <typename GO>
int grad_launches(GJobs& P, const ayolo_tensor* grads, int n, GO go) {
    return each_launch(P, grads, n, [&](int i, int64_t off, char** a) { a[0] = (char*)grads[i].data + off * es_of(grads[i].dtype); },
                       [&](int i, unsigned) { return (unsigned)grads[i].dtype; }, go);
}

}  // namespace

extern "C" size_t ayolo_grad_norm_workspace(const ayolo_tensor* grads, int n) {
    return grads && n > 0 ? (size_t)std::max<int64_t>(chunks_of(grads, n), 1) * sizeof(double) : sizeof(double);
}

extern "C" int ayolo_grad_norm(const ayolo_tensor* grads, int n, const float* grad_scale, float* norm, void* ws, size_t ws_bytes, ayolo_stream st) {
    AY_CHECK_ARG(n >= 0 && (n == 0 || grads) && norm, "grad_norm: null argument");
    int dev = -1;
    if (const int rc = check_list("grad_norm", "grads", grads, n, dev, is_float)) return rc;
    const int64_t chunks = chunks_of(grads, n);
    if (!ws || ws_bytes < ayolo_grad_norm_workspace(grads, n)) { ayolo_set_error("grad_norm: workspace %zu < %zu", ws_bytes, ayolo_grad_norm_workspace(grads, n)); return AYOLO_ENOSPC; }
    hipStream_t s = (hipStream_t)st;
    GJobs P{};
    P.h.part = (double*)ws;
    const int rc = grad_launches(P, grads, n, [&](GJobs& Q, unsigned wgs) {
        hipLaunchKernelGGL(k_grad_squares, dim3(wgs), dim3(256), 0, s, Q);
        Q.h.part += wgs;
        AY_CHECK_LAUNCH("k_grad_squares");
        return AYOLO_OK;
    });
    if (rc) return rc;
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(1024), 0, s, (const double*)ws, chunks, grad_scale, norm);
    AY_CHECK_LAUNCH("k_grad_norm");
    return AYOLO_OK;
}

extern "C" int ayolo_grad_clip(const ayolo_tensor* grads, int n, const float* norm, float max_norm, ayolo_stream st) {
    AY_CHECK_ARG(n >= 0 && (n == 0 || grads) && norm && max_norm >= 0.0f, "grad_clip: null argument or max_norm=%g", (double)max_norm);
    int dev = -1;
    if (const int rc = check_list("grad_clip", "grads", grads, n, dev, is_float)) return rc;
    try {
        auto each = [&](auto f) {
            each_range(grads, n, true, f);
            f(nullptr, 0, false);
            f(norm, sizeof(float), false);
        };
        AY_CHECK_ARG(!overlap((size_t)n + 1, each), "grad_clip: two of the gradients, or one and the norm, share memory");
    } catch (...) { ayolo_set_error("grad_clip: out of host memory"); return AYOLO_ENOSPC; }
    hipStream_t s = (hipStream_t)st;
    GJobs P{};
    P.h.norm = norm;
    P.h.max_norm = max_norm;
    return grad_launches(P, grads, n, [&](GJobs& Q, unsigned wgs) {
        hipLaunchKernelGGL(k_grad_clip, dim3(wgs), dim3(256), 0, s, Q);
        AY_CHECK_LAUNCH("k_grad_clip");
        return AYOLO_OK;
    });
}

namespace {
template <bool BITS8>
int adamw_launches(const ayolo_adamw_list& L, const Hyper& h, hipStream_t s) {
    AJobs<BITS8> P{};
    P.h = h;
    int dtype = -1;                                        // of the jobs that have gathered: a launch has one
    auto go = [&](AJobs<BITS8>& Q, unsigned wgs) {
        if (dtype == AYOLO_F32) hipLaunchKernelGGL((k_adamw<float, BITS8>), dim3(wgs), dim3(256), 0, s, Q);
        else if (dtype == AYOLO_F16) hipLaunchKernelGGL((k_adamw<half_t, BITS8>), dim3(wgs), dim3(256), 0, s, Q);
        else hipLaunchKernelGGL((k_adamw<bf16_t, BITS8>), dim3(wgs), dim3(256), 0, s, Q);
        AY_CHECK_LAUNCH("k_adamw");
        return AYOLO_OK;
    };
    int from = 0;
    while (from < L.n) {                                   // runs of one type
        int to = from;
        dtype = -1;
        for (; to < L.n; ++to) {
            if (!L.g[to].present) continue;
            if (dtype >= 0 && L.p[to].dtype != dtype) break;
            dtype = L.p[to].dtype;
        }
        const int es = es_of(dtype);
        auto where = [&](int i, int64_t off, char** a) {
            i += from;
            a[0] = (char*)L.p[i].data + off * es;
            a[1] = (char*)L.g[i].data + off * es;
            a[2] = (char*)L.m[i].data + off * (BITS8 ? 1 : 4);
            a[3] = (char*)L.v[i].data + off * (BITS8 ? 1 : 4);
            if constexpr (BITS8) {
                a[4] = (char*)L.me[i].data + off / 128;
                a[5] = (char*)L.ve[i].data + off / 128;
            }
        };
        auto part = [](int, unsigned p) { return p & 3u; };
        P.h.coef = h.coef + from;
        if (const int rc = each_launch(P, L.g + from, to - from, where, part, go)) return rc;
        from = to;
    }
    return AYOLO_OK;
}
}  // namespace

extern "C" size_t ayolo_adamw_workspace(int n) { return n > 0 ? (size_t)n * sizeof(Coef) : sizeof(Coef); }

extern "C" int ayolo_adamw_step(const ayolo_adamw_list* L, const ayolo_adamw_hyper* H, void* ws, size_t ws_bytes, ayolo_stream st) {
    AY_CHECK_ARG(L && H && L->n >= 0, "adamw_step: null argument");
    const int n = L->n;
    if (n == 0) return AYOLO_OK;
    AY_CHECK_ARG(L->p && L->g && L->m && L->v && L->step && !L->me == !L->ve, "adamw_step: null list");
    const bool bits8 = L->me != nullptr;
    AY_CHECK_ARG(H->beta1 >= 0.0 && H->beta1 < 1.0 && H->beta2 >= 0.0 && H->beta2 < 1.0, "adamw_step: betas=(%g, %g)", H->beta1, H->beta2);
    AY_CHECK_ARG(H->eps >= 0.0f, "adamw_step: eps=%g", (double)H->eps);
    AY_CHECK_ARG(!H->norm || H->max_norm >= 0.0f, "adamw_step: max_norm=%g", (double)H->max_norm);
    int dev = -1;
    auto is_f32 = [](int d) { return d == AYOLO_F32; };
    auto is_state = [&](int d) { return d == (bits8 ? AYOLO_U8 : AYOLO_F32); };
    auto is_u8 = [](int d) { return d == AYOLO_U8; };
    if (const int rc = check_list("adamw_step", "params", L->p, n, dev, is_float)) return rc;
    if (const int rc = check_list("adamw_step", "grads", L->g, n, dev, is_float)) return rc;
    if (const int rc = check_list("adamw_step", "exp_avgs", L->m, n, dev, is_state)) return rc;
    if (const int rc = check_list("adamw_step", "exp_avg_sqs", L->v, n, dev, is_state)) return rc;
    if (const int rc = check_list("adamw_step", "steps", L->step, n, dev, is_f32)) return rc;
    if (bits8) {
        if (const int rc = check_list("adamw_step", "exponents of exp_avgs", L->me, n, dev, is_u8)) return rc;
        if (const int rc = check_list("adamw_step", "exponents of exp_avg_sqs", L->ve, n, dev, is_u8)) return rc;
    }
    auto number = [](float x) { return x >= 0.0f && x < INFINITY; };
    AY_CHECK_ARG(H->lr_dev || L->lr || number(H->lr), "adamw_step: lr=%g", (double)H->lr);
    AY_CHECK_ARG(L->weight_decay || number(H->weight_decay), "adamw_step: weight_decay=%g", (double)H->weight_decay);
    for (int i = 0; i < n; ++i) {
        AY_CHECK_ARG(H->lr_dev || !L->lr || number(L->lr[i]), "adamw_step: lr[%d]=%g", i, (double)L->lr[i]);
        AY_CHECK_ARG(!L->weight_decay || number(L->weight_decay[i]), "adamw_step: weight_decay[%d]=%g", i, (double)L->weight_decay[i]);
        if (!L->g[i].present) continue;
        const ayolo_tensor &p = L->p[i], &g = L->g[i], &m = L->m[i], &v = L->v[i];
        AY_CHECK_ARG(p.present && m.present && v.present && L->step[i].present, "adamw_step: tensor %d has a gradient and no parameter, state or step", i);
        AY_CHECK_ARG(g.dtype == p.dtype, "adamw_step: tensor %d: the gradient's type is not the parameter's", i);
        AY_CHECK_ARG(g.numel == p.numel && m.numel == p.numel && v.numel == p.numel, "adamw_step: tensor %d: sizes differ", i);
        AY_CHECK_ARG(g.layout == p.layout && m.layout == p.layout && v.layout == p.layout, "adamw_step: tensor %d: gradient or state in another shape or memory order than the parameter", i);
        AY_CHECK_ARG(L->step[i].numel == 1, "adamw_step: steps[%d] is not one number", i);
        if (bits8) {
            const int64_t nb = cdiv64(p.numel, 128);
            AY_CHECK_ARG(L->me[i].present && L->ve[i].present && L->me[i].numel == nb && L->ve[i].numel == nb, "adamw_step: tensor %d needs %lld exponents", i, (long long)nb);
        }
    }
    try {
        // (a gradient that IS its parameter or moment is read where it is written, by the same thread and before)
        auto is = [](const ayolo_tensor& a, const ayolo_tensor& b) { return a.data == b.data && bytes_of(a) == bytes_of(b); };
        auto each = [&](auto f) {
            for (const ayolo_tensor* t : {L->p, L->m, L->v, L->me, L->ve, L->step})
                if (t) each_range(t, n, true, f, L->g);    // (without a gradient, nothing is written)
            f(nullptr, 0, false);
            for (int i = 0; i < n; ++i)
                if (const ayolo_tensor& g = L->g[i]; g.present && !is(g, L->p[i]) && !is(g, L->m[i]) && !is(g, L->v[i])) f(g.data, bytes_of(g), false);
            for (const float* x : {H->lr_dev, H->grad_scale, H->found_inf, H->norm}) {
                f(nullptr, 0, false);
                f(x, sizeof(float), false);
            }
        };
        AY_CHECK_ARG(!overlap((size_t)n * 7 + 4, each), "adamw_step: two of the parameters, states or steps, or one and what is read, share memory");
    } catch (...) { ayolo_set_error("adamw_step: out of host memory"); return AYOLO_ENOSPC; }
    const size_t need = ayolo_adamw_workspace(n);
    if (!ws || ws_bytes < need) { ayolo_set_error("adamw_step: workspace %zu < %zu", ws_bytes, need); return AYOLO_ENOSPC; }
    hipStream_t s = (hipStream_t)st;
    PrepJobs Q{};
    Q.ln_b1 = log(H->beta1);
    Q.ln_b2 = log(H->beta2);
    Q.lr = H->lr_dev;
    Q.found_inf = H->found_inf;
    Q.out = (Coef*)ws;
    Q.seed = H->seed;
    int windows = 0;
    auto prepare = [&]() -> int {
        if (Q.n == 0) return AYOLO_OK;
        hipLaunchKernelGGL(k_adamw_prepare, dim3(1), dim3(512), 0, s, Q);
        AY_CHECK_LAUNCH("k_adamw_prepare");
        Q.n = Q.pairs = windows = 0;
        return AYOLO_OK;
    };
    for (int i = 0; i < n; ++i) {
        if (!L->g[i].present) continue;
        const float lr = L->lr ? L->lr[i] : H->lr, wd = L->weight_decay ? L->weight_decay[i] : H->weight_decay;
        int pair = 0, w = 0;
        auto fits = [&]() {
            if (Q.n == PrepJobs::MAX || (Q.n && (unsigned)i - Q.place0 >= 1u << 22)) return false;
            for (pair = 0; pair < Q.pairs && !(Q.pair[pair].lr == lr && Q.pair[pair].wd == wd);) ++pair;
            return pair < PrepJobs::PAIRS && (w = Q.w.number(windows, L->step[i].data)) >= 0;
        };
        if (!fits()) {
            if (const int rc = prepare()) return rc;
            fits();
        }
        if (Q.n == 0) Q.place0 = (unsigned)i;
        if (pair == Q.pairs) {
            Q.pair[pair].lr = lr;
            Q.pair[pair].wd = wd;
            ++Q.pairs;
        }
        Q.j[Q.n].lo = (unsigned)(uintptr_t)L->step[i].data;
        Q.j[Q.n].which = (unsigned)pair | (unsigned)w << 6 | ((unsigned)i - Q.place0) << 10;
        ++Q.n;
    }
    if (const int rc = prepare()) return rc;
    Hyper h{};
    h.grad_scale = H->grad_scale;
    h.found_inf = H->found_inf;
    h.norm = H->norm;
    h.coef = (const Coef*)ws;
    h.b1 = (float)H->beta1;
    h.c1 = (float)(1.0 - H->beta1);
    h.b2 = (float)H->beta2;
    h.c2 = (float)(1.0 - H->beta2);
    h.eps = H->eps;
    h.max_norm = H->max_norm;
    h.maximize = H->maximize;
    return bits8 ? adamw_launches<true>(*L, h, s) : adamw_launches<false>(*L, h, s);
}

extern "C" int ayolo_moment_values(const ayolo_tensor* codes, const ayolo_tensor* exps, const ayolo_tensor* out, int n, int is_signed, ayolo_stream st) {
    AY_CHECK_ARG(n >= 0 && (n == 0 || (codes && exps && out)), "moment_values: null list");
    int dev = -1;
    auto is_u8 = [](int d) { return d == AYOLO_U8; };
    if (const int rc = check_list("moment_values", "codes", codes, n, dev, is_u8)) return rc;
    if (const int rc = check_list("moment_values", "exponents", exps, n, dev, is_u8)) return rc;
    if (const int rc = check_list("moment_values", "out", out, n, dev, [](int d) { return d == AYOLO_F32; })) return rc;
    for (int i = 0; i < n; ++i) {
        AY_CHECK_ARG(codes[i].present && exps[i].present && out[i].present, "moment_values: tensor %d is missing", i);
        AY_CHECK_ARG(out[i].numel == codes[i].numel && out[i].layout == codes[i].layout && exps[i].numel == cdiv64(codes[i].numel, 128), "moment_values: tensor %d: sizes or memory orders differ", i);
    }
    try {
        auto each = [&](auto f) {
            each_range(codes, n, false, f);
            each_range(exps, n, false, f);
            each_range(out, n, true, f);
        };
        AY_CHECK_ARG(!overlap((size_t)n * 3, each), "moment_values: two outputs, or one and the moments, share memory");
    } catch (...) { ayolo_set_error("moment_values: out of host memory"); return AYOLO_ENOSPC; }
    hipStream_t s = (hipStream_t)st;
    UJobs P{};
    return each_launch(P, codes, n,
        [&](int i, int64_t off, char** a) {
            a[0] = (char*)codes[i].data + off;
            a[1] = (char*)exps[i].data + off / 128;
            a[2] = (char*)out[i].data + off * 4;
        },
        [](int, unsigned) { return 0u; },
        [&](UJobs& Q, unsigned wgs) {
            if (is_signed) hipLaunchKernelGGL(k_moment_values<true>, dim3(wgs), dim3(256), 0, s, Q);
            else hipLaunchKernelGGL(k_moment_values<false>, dim3(wgs), dim3(256), 0, s, Q);
            AY_CHECK_LAUNCH("k_moment_values");
            return AYOLO_OK;
        });
}
