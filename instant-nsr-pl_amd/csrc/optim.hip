// AdamW over many tensors of any size in few launches, moments in 32 bits or in 8, with the norm of all gradients and the
// decision to clip or to leave the step out on the device (torch.optim.AdamW as the reference configures it:
// systems/utils.py:314-325, configs/nerf-blender.yaml:74-79; GradScaler of `precision: 16`: configs/nerf-blender.yaml:103).
//
// Per element, g' = g * (unscale and clip factor):
//   m' = b1 m + (1 - b1) g',   v' = b2 v + (1 - b2) g'^2,
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// An element whose g' is not finite keeps p, m and v, as with every other AdamW kernel of the library; 8-bit moments of it are
// encoded again with their block, whose scale may be another now.
//
// 8-bit moments: blocks of 256 consecutive elements share one fp32 scale per moment; m and r = sqrt(v) are e4m3 codes,
// scale = (largest magnitude of the block) / 448.  The root is held and not v because e4m3 spans 2^17.8: of r that is 2^35.6
// of v.  Codes are rounded stochastically: one step changes v by a share (1 - b2) of the distance to g'^2, far under half a
// lattice step (2^-4), so rounding to nearest would never move it; with random bits the expectation moves as it should.  r > 0
// keeps at least the smallest code (2^-9 of 448), so m is never divided by eps alone because r fell under the lattice.
#include "elem.h"

#include <type_traits>

namespace {

constexpr int OPT_THREADS = 256;
constexpr int OPT_BLOCK = 256;          // elements under one scale: one wave, 4 elements a lane
// Elements per workgroup of the update: one pass of 4 a lane.  Twice and four times as many in one workgroup were slower at
// every size (12.6 M fp32 parameters, 32 bits: 68.8 / 70.8 / 76.1 us; 8 bits: 42.2 / 43.9 / 54.1 us): more workgroups hide
// more latency than more loads in flight in each.
constexpr int OPT_CHUNK = OPT_THREADS * 4;
// Of the gradient norm: 4 (fp32) or 2 (16 bits) vectors a lane in flight, one or few chunks a workgroup, a partial sum for each
// workgroup (27.9 M fp32 gradients: 28 us; chunks of 8192 in at most 1024 workgroups 33 us, 2048 in 8192 as fast but twice the
// sums to add).
constexpr int NORM_CHUNK = 4096;
constexpr uint32_t NORM_MAX_GRID = 4096;  // partial sums per launch
constexpr float E4M3_TOP = 448.f, E4M3_INV_TOP = 1.f / 448.f;
constexpr float LEAST_TOP = 7.888609052210118e-31f;    // 2^-100: keeps 448 / top and top / 448 normal numbers
constexpr float ROOT_MOST = 1.8446743e19f;             // sqrt of the largest float: a root stays finite in 8 bits
constexpr float TO_LATTICE = 7.52316384526264e-37f;    // 2^-120: e4m3's exponent bias (7) in fp32's place (127)

// Descriptors travel as kernel arguments, of which 4 KB are sure: 64 tensors with what the plain 32-bit update needs, 36 with
// everything, 128 for the norm.  size: elements in the low 40 bits, flags above.
struct PlainTensor {
    void *p;
    const void *g;
    void *m, *v;
    uint64_t size;
    float lr, decay;  // lr: lr / (1 - b1^t) where the step count is the host's
};
struct FullTensor : PlainTensor {
    float *sm, *sr;
    _Float16 *image;
    const float *lr_dev;
    uint64_t index0;
    float wd;
};
struct NormTensor { const void *g; uint64_t size; };
constexpr int SIZE_BITS = 40;
enum : uint32_t { DT_MASK = 3, STATE8 = 4 };  // flags: the type's code, and these

template <class D, int MOST>
struct Launch {
    D t[MOST];
    uint32_t first[MOST];  // first chunk of each tensor
    uint32_t n_tensors, n_chunks;
};
using PlainLaunch = Launch<PlainTensor, 64>;
using FullLaunch = Launch<FullTensor, 36>;
using NormLaunch = Launch<NormTensor, 128>;
static_assert(sizeof(PlainLaunch) <= 3840 && sizeof(FullLaunch) <= 3840 && sizeof(NormLaunch) <= 3840,
              "kernel arguments stay under 4 KB");

// the tensor that owns a chunk: lanes compare the tensors' first chunks, those in front of it are counted
template <class D, int MOST>
__device__ __forceinline__ uint32_t tensor_of(const Launch<D, MOST> &a, uint32_t chunk)
{
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < MOST; k += 64) {
        const uint32_t i = k + (threadIdx.x & 63);
        n += __popcll(__ballot(i < a.n_tensors && a.first[i < MOST ? i : 0] <= chunk));
    }
    return (uint32_t)__builtin_amdgcn_readfirstlane(n - 1);
}

struct OptScalars { float scale, step, root, decay, b1, c1, b2, c2, eps; };  // c = 1 - b, root = 1 / sqrt(1 - b2^t)

__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) <= 3.4028234e38f; }

// one element; r = sqrt(v') comes back for the 8-bit state
__device__ __forceinline__ void adamw_elem(float &p, float &m, float &v, float g, const OptScalars &s, float &r)
{
    g *= s.scale;
    const float m1 = s.b1 * m + s.c1 * g, v1 = s.b2 * v + s.c2 * (g * g);
    const bool take = is_finite(g);
    m = take ? m1 : m;
    v = take ? v1 : v;
    r = sqrtf(v);
    // (the reciprocal instruction is good to 1 ulp, of an update that is a small part of p; the division cost the 8-bit form 4 %)
    const float p1 = p * s.decay - s.step * (m * __builtin_amdgcn_rcpf(r * s.root + s.eps));
    p = take ? p1 : p;
}

// ---- random bits and e4m3 ------------------------------------------------------------------------------------------------
// (steps and constants: the 32-bit finaliser published with MurmurHash3, in the public domain)
__device__ __forceinline__ uint32_t mix32(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x85ebca6bu;
    x ^= x >> 13;
    x *= 0xc2b2ae35u;
    return x ^ (x >> 16);
}

// y >= 0, at most 448 (1 + 2^-23): y 2^-120 carries the e4m3 code (3 mantissa bits, subnormals included) in front of 20 more
// bits of its own; the random bits, a half unit under their last one, decide about the carry
__device__ __forceinline__ uint32_t e4m3_stochastic(float y, uint32_t bits16)
{
    const uint32_t c = (__float_as_uint(y * TO_LATTICE) + (bits16 << 4 | 8u)) >> 20;
    return c < 0x7eu ? c : 0x7eu;
}

__device__ __forceinline__ float wave_max_nonnegative(float v)  // (bits of non-negative floats are ordered like the floats)
{
    uint32_t x = __float_as_uint(v);
    auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    x = up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
    x = up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));   // quad_perm 2 3 0 1
    x = up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));  // row_half_mirror
    x = up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));  // row_mirror
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = up(r[0], r[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __uint_as_float(up(q[0], q[1]));
}

__device__ __forceinline__ float e4m3_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }
__device__ __forceinline__ void e4m3_values(uint32_t codes, float (&v)[4])
{
    v[0] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 0);
    v[1] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 1);
    v[2] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 2);
    v[3] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 3);
}

// the four elements that a lane holds of one block of 256: new codes, and the block's scales where `first`
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&r)[4], const uint32_t (&h)[4], uint32_t &cm,
                                             uint32_t &cr, float &sm, float &sr)
{
    float tm = LEAST_TOP, tr = LEAST_TOP;
#pragma unroll
    for (int k = 0; k < 4; ++k) { tm = fmaxf(tm, fabsf(m[k])); tr = fmaxf(tr, r[k]); }
    tm = wave_max_nonnegative(tm);
    tr = wave_max_nonnegative(tr);
    const float im = E4M3_TOP / tm, ir = E4M3_TOP / tr;
    sm = tm * E4M3_INV_TOP;
    sr = tr * E4M3_INV_TOP;
    cm = cr = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t sign = (__float_as_uint(m[k]) >> 24) & 0x80u;
        uint32_t c = e4m3_stochastic(fabsf(m[k]) * im, h[k] >> 16);
        cm |= (m[k] != 0.f ? c | sign : 0u) << (8 * k);
        c = e4m3_stochastic(r[k] * ir, h[k] & 0xffffu);
        cr |= (r[k] > 0.f ? (c ? c : 1u) : 0u) << (8 * k);
    }
}

// ---- the chunk of one workgroup ------------------------------------------------------------------------------------------
template <class V, class T> __device__ __forceinline__ V get(const T *p)  // (global memory takes vectors at any element)
{
    V v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class V, class T> __device__ __forceinline__ void put(T *p, const V &v)
{
    __builtin_memcpy(p, &v, sizeof(v));
}

__device__ __forceinline__ uint32_t random_bits(uint64_t e, uint32_t key0)
{
    return mix32((uint32_t)e ^ (key0 + (uint32_t)(e >> 32) * 0x9e3779b9u));
}

// a whole chunk inside the tensor: a lane holds 4 consecutive elements, a wave one block of 256
template <int DT, bool S8, class D>
__device__ __forceinline__ void chunk_whole(const D &t, uint64_t base, const OptScalars &s, uint32_t key0)
{
    using T = typename Elem<DT>::T;
    const uint64_t i = base + 4 * threadIdx.x;
    Vec<T, 4> pv = get<Vec<T, 4>>((const T *)t.p + i);
    const Vec<T, 4> gv = get<Vec<T, 4>>((const T *)t.g + i);
    if constexpr (S8) {
        const uint64_t blk = i / OPT_BLOCK;
        const uint32_t mc = get<uint32_t>((const uint8_t *)t.m + i), rc = get<uint32_t>((const uint8_t *)t.v + i);
        const float sm = t.sm[blk], sr = t.sr[blk];
        float mf[4], rf[4], nm, nr;
        uint32_t h[4], cm, cr;
        e4m3_values(mc, mf);
        e4m3_values(rc, rf);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float pf = (float)pv.e[k], vf = rf[k] * sr;
            mf[k] *= sm;
            vf *= vf;
            adamw_elem(pf, mf[k], vf, (float)gv.e[k], s, rf[k]);
            rf[k] = fminf(rf[k], ROOT_MOST);
            pv.e[k] = (T)pf;
            h[k] = random_bits(t.index0 + i + k, key0);
        }
        encode_block(mf, rf, h, cm, cr, nm, nr);
        put((uint8_t *)t.m + i, cm);
        put((uint8_t *)t.v + i, cr);
        if ((threadIdx.x & 63) == 0) { t.sm[blk] = nm; t.sr[blk] = nr; }
    } else {
        Vec<float, 4> m = get<Vec<float, 4>>((const float *)t.m + i), v = get<Vec<float, 4>>((const float *)t.v + i);
        float r;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float pf = (float)pv.e[k];
            adamw_elem(pf, m.e[k], v.e[k], (float)gv.e[k], s, r);
            pv.e[k] = (T)pf;
        }
        put((float *)t.m + i, m);
        put((float *)t.v + i, v);
    }
    put((T *)t.p + i, pv);
    if constexpr (std::is_same<D, FullTensor>::value)
        if (t.image) {
            Vec<_Float16, 4> hv;
#pragma unroll
            for (int k = 0; k < 4; ++k) hv.e[k] = (_Float16)(float)pv.e[k];
            put(t.image + i, hv);
        }
}

// the tensor's last chunk: a wave has its block of 256 all the same, its lanes hold elements 64 apart
template <int DT, bool S8, class D>
__device__ __forceinline__ void chunk_last(const D &t, uint64_t base, uint64_t n, const OptScalars &s, uint32_t key0)
{
    using T = typename Elem<DT>::T;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t b0 = base + (threadIdx.x >> 6) * OPT_BLOCK, blk = b0 / OPT_BLOCK;
    if (b0 >= n) return;  // (the whole wave)
    float mf[4], rf[4], sm = 0.f, sr = 0.f;
    uint32_t h[4];
    if constexpr (S8) { sm = t.sm[blk]; sr = t.sr[blk]; }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint64_t i = b0 + k * 64 + lane;
        mf[k] = rf[k] = 0.f;
        h[k] = 0;
        if (i >= n) continue;
        float pf = (float)((const T *)t.p)[i], vf;
        if constexpr (S8) {
            mf[k] = e4m3_value(((const uint8_t *)t.m)[i]) * sm;
            vf = e4m3_value(((const uint8_t *)t.v)[i]) * sr;
            vf *= vf;
            h[k] = random_bits(t.index0 + i, key0);
        } else {
            mf[k] = ((const float *)t.m)[i];
            vf = ((const float *)t.v)[i];
        }
        adamw_elem(pf, mf[k], vf, (float)((const T *)t.g)[i], s, rf[k]);
        rf[k] = fminf(rf[k], ROOT_MOST);
        const T pt = (T)pf;
        ((T *)t.p)[i] = pt;
        if constexpr (std::is_same<D, FullTensor>::value)
            if (t.image) t.image[i] = (_Float16)(float)pt;
        if constexpr (!S8) {
            ((float *)t.m)[i] = mf[k];
            ((float *)t.v)[i] = vf;
        }
    }
    if constexpr (S8) {
        uint32_t cm, cr;
        float nm, nr;
        encode_block(mf, rf, h, cm, cr, nm, nr);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint64_t i = b0 + k * 64 + lane;
            if (i < n) {
                ((uint8_t *)t.m)[i] = (uint8_t)(cm >> (8 * k));
                ((uint8_t *)t.v)[i] = (uint8_t)(cr >> (8 * k));
            }
        }
        if (lane == 0) { t.sm[blk] = nm; t.sr[blk] = nr; }
    }
}

template <int DT, bool S8, class D>
__device__ __forceinline__ void run_chunk(const D &t, uint64_t base, uint64_t n, const OptScalars &s, uint32_t key0)
{
    base + OPT_CHUNK <= n ? chunk_whole<DT, S8>(t, base, s, key0) : chunk_last<DT, S8>(t, base, n, s, key0);
}

// The update.  Bound by HBM: 28 bytes an fp32 element with 32-bit moments (12.6 M elements: 67 us, 5.2 TB/s), 16.06 bytes with
// 8-bit ones (2^27 elements: 367 us, 5.9 TB/s), 22 bytes a bf16 element (3.5 M: 15 us, 5.1 TB/s).  The 8-bit form keeps the vector
// units 80 % busy as well: about 100 instructions an element, of which the two roundings, the hash and the exact root (its codes
// are to be the same on every machine) are most.  One chunk a workgroup; the tensor is found by one comparison a lane.
// hyper of nsr_adamw_begin: {gradient factor, 1 / (1 - b1^t), 1 / sqrt(1 - b2^t), leave out?, t, norm}
template <class D, int MOST>
__global__ void __launch_bounds__(OPT_THREADS)
k_adamw_tensors(const Launch<D, MOST> a, OptScalars s, uint32_t seed, uint32_t step, const float *__restrict__ hyper)
{
    constexpr bool FULL = std::is_same<D, FullTensor>::value;
    if (hyper) {
        if (__float_as_int(hyper[3])) return;
        s.scale *= hyper[0];
        s.root = hyper[2];
        step = (uint32_t)__float_as_int(hyper[4]);
    }
    // from the last chunk to the first: the gradients that the norm (or the backward pass) touched last are nearest in the
    // caches (1 to 2 % for 8-bit moments)
    const uint32_t chunk = gridDim.x - 1 - blockIdx.x;
    const uint32_t which = tensor_of(a, chunk);
    const D &t = a.t[which];
    const uint32_t flags = (uint32_t)(t.size >> SIZE_BITS);
    const uint64_t n = t.size & ((1ull << SIZE_BITS) - 1), base = (uint64_t)(chunk - a.first[which]) * OPT_CHUNK;
    float lr = t.lr;
    s.decay = t.decay;
    uint32_t key0 = 0;
    if constexpr (FULL) {
        if (t.lr_dev) {
            lr = *t.lr_dev;
            s.decay = 1.f - lr * t.wd;
        }
        key0 = mix32(mix32(step) ^ seed);
    }
    s.step = hyper ? lr * hyper[1] : lr;
    const uint32_t dt = flags & DT_MASK;
    if constexpr (FULL)
        if (flags & STATE8) {
            if (dt == DT_F32) run_chunk<DT_F32, true>(t, base, n, s, key0);
            else if (dt == DT_F16) run_chunk<DT_F16, true>(t, base, n, s, key0);
            else run_chunk<DT_BF16, true>(t, base, n, s, key0);
            return;
        }
    if (dt == DT_F32) run_chunk<DT_F32, false>(t, base, n, s, key0);
    else if (dt == DT_F16) run_chunk<DT_F16, false>(t, base, n, s, key0);
    else run_chunk<DT_BF16, false>(t, base, n, s, key0);
}

// ---- norm of all gradients -----------------------------------------------------------------------------------------------
// Squares and sums in 64 bits: no overflow for any finite gradient, and the same value for every order that matters in fp32.
// Bound by HBM reads: 27.9 M fp32 gradients in 28 us (3.9 TB/s) behind an update whose results still drain from the caches; a
// bare read of as much clean memory takes 23 us.
template <int DT>
__device__ __forceinline__ double chunk_squares(const void *grad, uint64_t n, uint64_t base)
{
    using T = typename Elem<DT>::T;
    constexpr int N = 16 / sizeof(T), PASSES = NORM_CHUNK / (OPT_THREADS * N);
    const T *g = (const T *)grad + base;
    double acc[2] = {0.0, 0.0};  // (two chains of additions)
    const uint32_t left = n - base < NORM_CHUNK ? (uint32_t)(n - base) : NORM_CHUNK;
    Vec<T, N> v[PASSES];
#pragma unroll
    for (int it = 0; it < PASSES; ++it) {
        const uint32_t i = (it * OPT_THREADS + threadIdx.x % OPT_THREADS) * N;
        if (i + N <= left) {
            v[it] = get<Vec<T, N>>(g + i);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) v[it].e[k] = i + k < left ? g[i + k] : (T)0.f;
        }
    }
#pragma unroll
    for (int it = 0; it < PASSES; ++it)
#pragma unroll
        for (int k = 0; k < N; ++k) { const double d = (double)(float)v[it].e[k]; acc[k & 1] = fma(d, d, acc[k & 1]); }
    return acc[0] + acc[1];
}

__device__ __forceinline__ double wave_sum64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// sums of squares of every `stride`th chunk from `chunk` on, by 256 threads
__device__ __forceinline__ double squares_of_chunks(const NormLaunch &a, uint32_t chunk, uint32_t stride)
{
    double acc = 0.0;
    for (; chunk < a.n_chunks; chunk += stride) {
        const uint32_t which = tensor_of(a, chunk);
        const NormTensor &t = a.t[which];
        const uint64_t n = t.size & ((1ull << SIZE_BITS) - 1), base = (uint64_t)(chunk - a.first[which]) * NORM_CHUNK;
        const uint32_t dt = (uint32_t)(t.size >> SIZE_BITS) & DT_MASK;
        if (dt == DT_F32) acc += chunk_squares<DT_F32>(t.g, n, base);
        else if (dt == DT_F16) acc += chunk_squares<DT_F16>(t.g, n, base);
        else acc += chunk_squares<DT_BF16>(t.g, n, base);
    }
    return acc;
}

__global__ void __launch_bounds__(OPT_THREADS)
k_grad_squares(const NormLaunch a, double *__restrict__ partials)
{
    const double acc = wave_sum64(squares_of_chunks(a, blockIdx.x, gridDim.x));
    __shared__ double part[OPT_THREADS / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partials[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// one workgroup: each thread's share of the sum of squares in a fixed order, then the step's scalars.  Two threads have worked
// out b^t = exp(t ln b) in 64 bits meanwhile (its error, t |ln b| 2^-53 of it, is far under fp32's; pow took twice as long as
// the whole kernel does now).
constexpr int BEGIN_THREADS = 1024;
struct Begin {
    int32_t *step;
    float *hyper;
    double ln_b1, ln_b2, max_norm;
    const float *grad_scale, *found_inf;
};
__device__ __forceinline__ void begin_step(const Begin &b, double acc, bool clip)
{
    __shared__ double part[BEGIN_THREADS / 64], power[2];
    const int32_t taken = *b.step;
    if (threadIdx.x == 64 || threadIdx.x == 128)
        power[threadIdx.x / 128] = exp((taken + 1.0) * (threadIdx.x == 64 ? b.ln_b1 : b.ln_b2));
    acc = wave_sum64(acc);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x != 0) return;
    const double unscale = b.grad_scale ? 1.0 / (double)*b.grad_scale : 1.0;
    double factor = unscale;
    bool skip = b.found_inf && *b.found_inf != 0.f;
    if (clip) {
        double sum = part[0];
        for (int k = 1; k < BEGIN_THREADS / 64; ++k) sum += part[k];
        const double norm = sqrt(sum) * unscale;
        const double ratio = b.max_norm / (norm + 1e-6);  // torch.nn.utils.clip_grad_norm_
        factor *= ratio < 1.0 ? ratio : 1.0;
        skip = skip || !(norm <= 1.7976931348623157e308);
        b.hyper[5] = (float)norm;
    }
    if (!skip) *b.step = taken + 1;
    b.hyper[0] = (float)factor;
    b.hyper[1] = (float)(1.0 / (1.0 - power[0]));
    b.hyper[2] = (float)(1.0 / sqrt(1.0 - power[1]));
    b.hyper[3] = __int_as_float(skip ? 1 : 0);
    b.hyper[4] = __int_as_float(taken + 1);  // (read only where the step is taken)
}

__global__ void __launch_bounds__(BEGIN_THREADS)
k_adamw_begin(const Begin b, const double *__restrict__ partials, uint32_t n_partials)
{
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < n_partials; i += BEGIN_THREADS) acc += partials[i];
    begin_step(b, acc, partials != nullptr);
}

// few gradients: the workgroup sums their squares itself, four chunks at a time
__global__ void __launch_bounds__(BEGIN_THREADS)
k_adamw_begin_few(const Begin b, const NormLaunch a)
{
    constexpr uint32_t AT_ONCE = BEGIN_THREADS / OPT_THREADS;
    begin_step(b, squares_of_chunks(a, (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / OPT_THREADS), AT_ONCE), true);
}
static_assert(sizeof(NormLaunch) + sizeof(Begin) <= 3840, "kernel arguments stay under 4 KB");
// (up to 131072 elements; a clipped step of that size: 18.2 us a call, 20.6 us with the sums in a launch of their own)
constexpr uint32_t FEW_CHUNKS = 32;

// ---- host ----------------------------------------------------------------------------------------------------------------
// 2^23 chunks of 256 threads are 2^31 threads: a grid stays under the launch limit of 2^32 with the next tensor's chunks too.
// A tensor of more chunks is several pieces.
constexpr uint32_t LAUNCH_CHUNKS = 1u << 23;

int check_grads(const char *what, const NsrAdamwTensor *tensors, uint32_t n_tensors)
{
    NSR_REQUIRE(n_tensors == 0 || tensors, "%s: NULL descriptors", what);
    for (uint32_t i = 0; i < n_tensors; ++i) {
        const NsrAdamwTensor &x = tensors[i];
        NSR_REQUIRE(x.n < (1ull << 35), "%s: tensor %u has 2^35 elements or more", what, i);
        NSR_REQUIRE(x.dtype <= DT_BF16, "%s: tensor %u: dtype %u (0 fp32, 1 fp16, 2 bf16)", what, i, x.dtype);
        NSR_REQUIRE(x.n == 0 || x.grad, "%s: tensor %u has a NULL gradient", what, i);
        NSR_REQUIRE(((uintptr_t)x.grad & (dtype_size(x.dtype) - 1)) == 0, "%s: tensor %u: misaligned gradient", what, i);
    }
    return NSR_OK;
}

int check_states(const char *what, const NsrAdamwTensor *tensors, uint32_t n_tensors, bool lr_on_device)
{
    for (uint32_t i = 0; i < n_tensors; ++i) {
        const NsrAdamwTensor &x = tensors[i];
        if (x.n == 0) continue;
        NSR_REQUIRE(x.params && x.exp_avg && x.exp_avg_sq, "%s: tensor %u has a NULL pointer", what, i);
        NSR_REQUIRE(x.state_bits == 32 || x.state_bits == 8, "%s: tensor %u: moments in %u bits (32 or 8)", what, i, x.state_bits);
        NSR_REQUIRE(x.state_bits == 32 || (x.scales_m && x.scales_r), "%s: tensor %u: 8-bit moments need scales", what, i);
        NSR_REQUIRE(!x.lr_dev || lr_on_device, "%s: tensor %u: lr_dev needs the device-side step count (hyper)", what, i);
        NSR_REQUIRE(x.index0 % OPT_BLOCK == 0, "%s: tensor %u: index0 must be a multiple of %d", what, i, OPT_BLOCK);
        const uintptr_t fp32 = (uintptr_t)x.scales_m | (uintptr_t)x.scales_r | (uintptr_t)x.lr_dev |
                               (x.state_bits == 32 ? (uintptr_t)x.exp_avg | (uintptr_t)x.exp_avg_sq : 0);
        NSR_REQUIRE((fp32 & 3) == 0 && ((uintptr_t)x.params & (dtype_size(x.dtype) - 1)) == 0 && ((uintptr_t)x.image & 1) == 0,
                    "%s: tensor %u: misaligned pointer", what, i);
    }
    return NSR_OK;
}

// fills launches of at most MOST tensors (or pieces of tensors: fill(descriptor, tensor, first element, elements)) and hands
// each to `go`
template <class D, int MOST, class Fill, class Go>
int each_launch(const NsrAdamwTensor *tensors, uint32_t n_tensors, uint32_t chunk, Fill fill, Go go)
{
    Launch<D, MOST> a;
    a.n_tensors = a.n_chunks = 0;
    for (uint32_t i = 0; i < n_tensors; ++i) {
        const uint64_t n = tensors[i].n, most = (uint64_t)LAUNCH_CHUNKS * chunk;
        for (uint64_t at = 0; at < n; at += most) {
            const uint64_t part = n - at < most ? n - at : most;
            fill(a.t[a.n_tensors], tensors[i], at, part);
            a.first[a.n_tensors++] = a.n_chunks;
            a.n_chunks += nsr_div_up(part, chunk);
            if (a.n_tensors == MOST || a.n_chunks >= LAUNCH_CHUNKS - 1) {
                const int rc = go(a);
                if (rc != NSR_OK) return rc;
                a.n_tensors = a.n_chunks = 0;
            }
        }
    }
    return a.n_tensors ? go(a) : NSR_OK;
}

void fill_norm(NormTensor &t, const NsrAdamwTensor &x, uint64_t at, uint64_t n)
{
    t.g = (const char *)x.grad + at * dtype_size(x.dtype);
    t.size = n | (uint64_t)x.dtype << SIZE_BITS;
}

}  // namespace

extern "C" int nsr_adamw_tensors(const NsrAdamwTensor *tensors, uint32_t n_tensors, double beta1, double beta2, double eps,
                                 int32_t step, const float *hyper, double grad_unscale, uint32_t seed, void *stream)
{
    NSR_REQUIRE(hyper || step >= 1, "nsr_adamw_tensors: step counts from 1");
    NSR_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "nsr_adamw_tensors: betas in [0, 1)");
    NSR_REQUIRE(eps >= 0.0, "nsr_adamw_tensors: eps >= 0");
    int rc = check_grads("nsr_adamw_tensors", tensors, n_tensors);
    if (rc == NSR_OK) rc = check_states("nsr_adamw_tensors", tensors, n_tensors, hyper != nullptr);
    if (rc != NSR_OK) return rc;
    const double c1 = hyper ? 1.0 : 1.0 - pow(beta1, (double)step), c2 = hyper ? 1.0 : 1.0 - pow(beta2, (double)step);
    OptScalars s;
    s.scale = (float)grad_unscale; s.step = 0.f; s.root = (float)(1.0 / sqrt(c2)); s.decay = 1.f;
    s.b1 = (float)beta1; s.c1 = (float)(1.0 - beta1); s.b2 = (float)beta2; s.c2 = (float)(1.0 - beta2); s.eps = (float)eps;
    bool plain = true;
    for (uint32_t i = 0; i < n_tensors; ++i)
        plain = plain && (tensors[i].n == 0 || (tensors[i].state_bits == 32 && !tensors[i].image && !tensors[i].lr_dev));
    auto fill = [&](PlainTensor &t, const NsrAdamwTensor &x, uint64_t at, uint64_t n) {
        const uint64_t e = at * dtype_size(x.dtype), st = at * x.state_bits / 8;
        t.p = (char *)x.params + e; t.g = (const char *)x.grad + e; t.m = (char *)x.exp_avg + st; t.v = (char *)x.exp_avg_sq + st;
        t.size = n | (uint64_t)(x.dtype | (x.state_bits == 8 ? STATE8 : 0)) << SIZE_BITS;
        t.lr = (float)(x.lr / c1); t.decay = (float)(1.0 - x.lr * x.weight_decay);
    };
    auto fill_all = [&](FullTensor &t, const NsrAdamwTensor &x, uint64_t at, uint64_t n) {
        fill(t, x, at, n);
        t.sm = x.scales_m ? x.scales_m + at / OPT_BLOCK : nullptr; t.sr = x.scales_r ? x.scales_r + at / OPT_BLOCK : nullptr;
        t.image = x.image ? (_Float16 *)x.image + at : nullptr; t.lr_dev = x.lr_dev;
        t.index0 = x.index0 + at; t.wd = (float)x.weight_decay;
    };
    auto go = [&](const auto &a, auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.n_chunks), dim3(OPT_THREADS), 0, (hipStream_t)stream, a, s, seed, (uint32_t)step, hyper);
        NSR_CHECK_LAUNCH("nsr_adamw_tensors");
        return NSR_OK;
    };
    if (plain)
        return each_launch<PlainTensor, 64>(tensors, n_tensors, OPT_CHUNK, fill,
                                            [&](const PlainLaunch &a) { return go(a, k_adamw_tensors<PlainTensor, 64>); });
    return each_launch<FullTensor, 36>(tensors, n_tensors, OPT_CHUNK, fill_all,
                                       [&](const FullLaunch &a) { return go(a, k_adamw_tensors<FullTensor, 36>); });
}

extern "C" uint32_t nsr_grad_squares_capacity(const NsrAdamwTensor *tensors, uint32_t n_tensors)
{
    // a launch ends after 128 tensors (or pieces) or LAUNCH_CHUNKS - 1 chunks, whichever comes first
    uint64_t chunks = 0;
    for (uint32_t i = 0; tensors && i < n_tensors; ++i) chunks += nsr_div_up(tensors[i].n, NORM_CHUNK);
    return (uint32_t)((nsr_div_up(n_tensors, 128) + 2 * (chunks / (LAUNCH_CHUNKS - 1)) + 1) * NORM_MAX_GRID);
}

extern "C" int nsr_grad_squares(const NsrAdamwTensor *tensors, uint32_t n_tensors, double *partials, uint32_t capacity,
                                uint32_t *n_partials, void *stream)
{
    NSR_REQUIRE(partials && n_partials, "nsr_grad_squares: NULL pointer");
    NSR_REQUIRE(((uintptr_t)partials & 7) == 0, "nsr_grad_squares: partials must be 8-byte aligned");
    *n_partials = 0;
    const int rc = check_grads("nsr_grad_squares", tensors, n_tensors);
    if (rc != NSR_OK) return rc;
    return each_launch<NormTensor, 128>(tensors, n_tensors, NORM_CHUNK, fill_norm, [&](const NormLaunch &a) {
        const uint32_t grid = a.n_chunks < NORM_MAX_GRID ? a.n_chunks : NORM_MAX_GRID;
        NSR_REQUIRE(capacity - *n_partials >= grid, "nsr_grad_squares: room for %u partial sums is too little", capacity);
        hipLaunchKernelGGL(k_grad_squares, dim3(grid), dim3(OPT_THREADS), 0, (hipStream_t)stream, a, partials + *n_partials);
        NSR_CHECK_LAUNCH("nsr_grad_squares");
        *n_partials += grid;
        return NSR_OK;
    });
}

extern "C" int nsr_adamw_begin(int32_t *step, float *hyper, double beta1, double beta2, const double *partials,
                               uint32_t n_partials, double max_norm, const float *grad_scale, const float *found_inf,
                               void *stream)
{
    NSR_REQUIRE(step && hyper, "nsr_adamw_begin: NULL pointer");
    NSR_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "nsr_adamw_begin: betas in [0, 1)");
    NSR_REQUIRE(!partials || max_norm > 0.0, "nsr_adamw_begin: max_norm > 0");
    const Begin b{step, hyper, log(beta1), log(beta2), max_norm, grad_scale, found_inf};
    hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(BEGIN_THREADS), 0, (hipStream_t)stream, b, partials, partials ? n_partials : 0);
    NSR_CHECK_LAUNCH("nsr_adamw_begin");
    return NSR_OK;
}

extern "C" int nsr_adamw_begin_clipped(const NsrAdamwTensor *tensors, uint32_t n_tensors, double *partials, uint32_t capacity,
                                       int32_t *step, float *hyper, double beta1, double beta2, double max_norm,
                                       const float *grad_scale, const float *found_inf, void *stream)
{
    NSR_REQUIRE(step && hyper && partials, "nsr_adamw_begin_clipped: NULL pointer");
    NSR_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "nsr_adamw_begin_clipped: betas in [0, 1)");
    NSR_REQUIRE(max_norm > 0.0, "nsr_adamw_begin_clipped: max_norm > 0");
    int rc = check_grads("nsr_adamw_begin_clipped", tensors, n_tensors);
    if (rc != NSR_OK) return rc;
    uint64_t chunks = 0, live = 0;
    for (uint32_t i = 0; i < n_tensors; ++i) { chunks += nsr_div_up(tensors[i].n, NORM_CHUNK); live += tensors[i].n != 0; }
    if (chunks == 0 || chunks > FEW_CHUNKS || live > 128) {
        uint32_t n = 0;
        rc = nsr_grad_squares(tensors, n_tensors, partials, capacity, &n, stream);
        return rc != NSR_OK ? rc : nsr_adamw_begin(step, hyper, beta1, beta2, partials, n, max_norm, grad_scale, found_inf, stream);
    }
    const Begin b{step, hyper, log(beta1), log(beta2), max_norm, grad_scale, found_inf};
    return each_launch<NormTensor, 128>(tensors, n_tensors, NORM_CHUNK, fill_norm, [&](const NormLaunch &a) {
        hipLaunchKernelGGL(k_adamw_begin_few, dim3(1), dim3(BEGIN_THREADS), 0, (hipStream_t)stream, b, a);
        NSR_CHECK_LAUNCH("nsr_adamw_begin_clipped");
        return NSR_OK;
    });
}
