// AdamW over many tensors of any size in few launches, moments in 32 bits or in 8, with the norm of all gradients and the
// decision to clip or to leave the step out on the device (torch.optim.AdamW as the reference configures it:
// systems/utils.py:314-325, configs/nerf-blender.yaml:74-79; GradScaler of `precision: 16`: configs/nerf-blender.yaml:103).
//
// Per element, g' = g * (unscale and clip factor):
//   m' = b1 m + (1 - b1) g',   v' = b2 v + (1 - b2) g'^2,
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// An element whose g' is not finite keeps p, m and v, as with every other AdamW kernel of the library.
//
// 8-bit moments: blocks of 256 consecutive elements share one fp32 scale per moment; m and r = sqrt(v) are e4m3 codes,
// scale = (largest magnitude of the block) / 448.  The root is held and not v because e4m3 spans 2^17.8: of r that is 2^35.6
// of v.  Codes are rounded stochastically: one step changes v by a share (1 - b2) of the distance to g'^2, far under half a
// lattice step (2^-4), so rounding to nearest would never move it; with random bits the expectation moves as it should.  r > 0
// keeps at least the smallest code (2^-9 of 448), so m is never divided by eps alone because r fell under the lattice.
#include "elem.h"

namespace {

constexpr int OPT_THREADS = 256;
constexpr int OPT_BLOCK = 256;          // elements under one scale: one wave, 4 elements a lane
constexpr int OPT_CHUNK = 4096;         // elements per workgroup: 4 passes of 256 threads x 4 elements
constexpr int OPT_TENSORS = 36;         // tensors per launch: their descriptors travel as kernel arguments (4 KB)
constexpr int NORM_MAX_GRID = 1024;     // partial sums per launch of the gradient norm
constexpr float E4M3_TOP = 448.f, E4M3_INV_TOP = 1.f / 448.f;
constexpr float LEAST_TOP = 7.888609052210118e-31f;    // 2^-100: keeps 448 / top and top / 448 normal numbers
constexpr float TO_LATTICE = 7.52316384526264e-37f;    // 2^-120: e4m3's exponent bias (7) in fp32's place (127)

struct OptTensor {
    void *p;
    const void *g;
    void *m, *v;
    float *sm, *sr;
    __half *image;
    const float *lr_dev;
    uint64_t n, index0;
    float lr, decay, wd;  // lr: lr / (1 - b1^t) where the step count is the host's
    uint32_t flags;
};
enum : uint32_t { DT_MASK = 3, STATE8 = 4, ALIGNED = 8 };  // flags: the type's code, and these

struct OptLaunch {
    OptTensor t[OPT_TENSORS];
    uint32_t first[OPT_TENSORS];  // first chunk of each tensor
    uint32_t n_tensors, n_chunks;
};
static_assert(sizeof(OptLaunch) <= 3840, "kernel arguments stay under 4 KB");

// the tensor that owns a chunk: one lane per tensor compares, the tensors in front of the chunk are counted
__device__ __forceinline__ uint32_t tensor_of(const OptLaunch &a, uint32_t chunk)
{
    const uint32_t lane = threadIdx.x & 63;
    const bool before = lane < a.n_tensors && a.first[lane < a.n_tensors ? lane : 0] <= chunk;
    return (uint32_t)__builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
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
    const float p1 = p * s.decay - s.step * (m / (r * s.root + s.eps));
    p = take ? p1 : p;
}

// ---- random bits and e4m3 ------------------------------------------------------------------------------------------------
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
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
        x = y > x ? y : x;
    }
    return __uint_as_float(x);
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

constexpr float ROOT_MOST = 1.8446743e19f;  // sqrt of the largest float: a root stays finite in 8 bits

// ---- the chunk of one workgroup ------------------------------------------------------------------------------------------
// vector form: whole chunk inside the tensor, all pointers aligned; lane holds 4 consecutive elements
template <int DT>
__device__ __forceinline__ void chunk_vector(const OptTensor &t, uint64_t base, const OptScalars &s, uint32_t key0)
{
    using T = typename Elem<DT>::T;
    using V = Vec<T, 4>;
    V *p = reinterpret_cast<V *>((T *)t.p + base);
    const V *g = reinterpret_cast<const V *>((const T *)t.g + base);
#pragma unroll
    for (int it = 0; it < OPT_CHUNK / (OPT_THREADS * 4); ++it) {
        const uint32_t q = it * OPT_THREADS + threadIdx.x;
        V pv = p[q];
        const V gv = g[q];
        float pf[4], mf[4], vf[4], rf[4];
        if (!(t.flags & STATE8)) {
            float4 *mp = reinterpret_cast<float4 *>((float *)t.m + base) + q, *vp = reinterpret_cast<float4 *>((float *)t.v + base) + q;
            *reinterpret_cast<float4 *>(mf) = *mp;
            *reinterpret_cast<float4 *>(vf) = *vp;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                pf[k] = (float)pv.e[k];
                adamw_elem(pf[k], mf[k], vf[k], (float)gv.e[k], s, rf[k]);
                pv.e[k] = (T)pf[k];
            }
            *mp = *reinterpret_cast<float4 *>(mf);
            *vp = *reinterpret_cast<float4 *>(vf);
        } else {
            const uint64_t blk = base / OPT_BLOCK + q / 64;
            uint32_t *mp = (uint32_t *)t.m + base / 4 + q, *vp = (uint32_t *)t.v + base / 4 + q;
            const uint32_t mc = *mp, rc = *vp;
            const float sm = t.sm[blk], sr = t.sr[blk];
            const uint64_t e = t.index0 + base + 4 * (uint64_t)q;
            const uint32_t key = key0 + (uint32_t)(e >> 32) * 0x9e3779b9u;
            uint32_t h[4];
            e4m3_values(mc, mf);
            e4m3_values(rc, rf);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                pf[k] = (float)pv.e[k];
                mf[k] *= sm;
                rf[k] *= sr;
                vf[k] = rf[k] * rf[k];
                adamw_elem(pf[k], mf[k], vf[k], (float)gv.e[k], s, rf[k]);
                rf[k] = fminf(rf[k], ROOT_MOST);
                pv.e[k] = (T)pf[k];
                h[k] = mix32(((uint32_t)e + k) ^ key);
            }
            uint32_t cm, cr;
            float nm, nr;
            encode_block(mf, rf, h, cm, cr, nm, nr);
            *mp = cm;
            *vp = cr;
            if ((threadIdx.x & 63) == 0) { t.sm[blk] = nm; t.sr[blk] = nr; }
        }
        p[q] = pv;
        if (t.image) {
            Vec<_Float16, 4> hv;
#pragma unroll
            for (int k = 0; k < 4; ++k) hv.e[k] = (_Float16)(float)pv.e[k];
            reinterpret_cast<Vec<_Float16, 4> *>((_Float16 *)t.image + base)[q] = hv;
        }
    }
}

// element form: the tensor's last chunk, or pointers that no vector load takes; lanes hold elements 64 apart
template <int DT>
__device__ __forceinline__ void chunk_element(const OptTensor &t, uint64_t base, const OptScalars &s, uint32_t key0)
{
    using T = typename Elem<DT>::T;
    T *p = (T *)t.p;
    const T *g = (const T *)t.g;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int it = 0; it < OPT_CHUNK / (OPT_THREADS * 4); ++it) {
        const uint64_t b0 = base + (it * 4 + wave) * (uint64_t)OPT_BLOCK;
        if (b0 >= t.n) return;  // (the whole wave leaves)
        float mf[4], rf[4];
        uint32_t h[4];
        const uint64_t blk = b0 / OPT_BLOCK;
        const float sm = t.flags & STATE8 ? t.sm[blk] : 0.f, sr = t.flags & STATE8 ? t.sr[blk] : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint64_t i = b0 + k * 64 + lane;
            mf[k] = rf[k] = 0.f;
            h[k] = 0;
            if (i >= t.n) continue;
            float pf = (float)p[i], vf;
            if (t.flags & STATE8) {
                mf[k] = e4m3_value(((const uint8_t *)t.m)[i]) * sm;
                const float r0 = e4m3_value(((const uint8_t *)t.v)[i]) * sr;
                vf = r0 * r0;
                const uint64_t e = t.index0 + i;
                h[k] = mix32((uint32_t)e ^ (key0 + (uint32_t)(e >> 32) * 0x9e3779b9u));
            } else {
                mf[k] = ((const float *)t.m)[i];
                vf = ((const float *)t.v)[i];
            }
            adamw_elem(pf, mf[k], vf, (float)g[i], s, rf[k]);
            rf[k] = fminf(rf[k], ROOT_MOST);
            const T pt = (T)pf;
            p[i] = pt;
            if (t.image) ((_Float16 *)t.image)[i] = (_Float16)(float)pt;
            if (!(t.flags & STATE8)) {
                ((float *)t.m)[i] = mf[k];
                ((float *)t.v)[i] = vf;
            }
        }
        if (t.flags & STATE8) {
            uint32_t cm, cr;
            float nm, nr;
            encode_block(mf, rf, h, cm, cr, nm, nr);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t i = b0 + k * 64 + lane;
                if (i < t.n) {
                    ((uint8_t *)t.m)[i] = (uint8_t)(cm >> (8 * k));
                    ((uint8_t *)t.v)[i] = (uint8_t)(cr >> (8 * k));
                }
            }
            if (lane == 0) { t.sm[blk] = nm; t.sr[blk] = nr; }
        }
    }
}

// hyper of nsr_adamw_begin: {gradient factor, 1 / (1 - b1^t), 1 / sqrt(1 - b2^t), leave out?, t, norm}
__global__ void __launch_bounds__(OPT_THREADS)
k_adamw_tensors(const OptLaunch a, OptScalars s, uint32_t seed, uint32_t step, const float *__restrict__ hyper)
{
    if (hyper) {
        if (__float_as_int(hyper[3])) return;
        s.scale *= hyper[0];
        s.root = hyper[2];
        step = (uint32_t)__float_as_int(hyper[4]);
    }
    const uint32_t which = tensor_of(a, blockIdx.x);
    const OptTensor &t = a.t[which];
    float lr = t.lr;
    s.decay = t.decay;
    if (t.lr_dev) {
        lr = *t.lr_dev;
        s.decay = 1.f - lr * t.wd;
    }
    s.step = hyper ? lr * hyper[1] : lr;
    const uint32_t key0 = mix32(mix32(step) ^ seed);
    const uint64_t base = (uint64_t)(blockIdx.x - a.first[which]) * OPT_CHUNK;
    const bool vec = (t.flags & ALIGNED) && base + OPT_CHUNK <= t.n;
    switch (t.flags & DT_MASK) {
    case DT_F32: vec ? chunk_vector<DT_F32>(t, base, s, key0) : chunk_element<DT_F32>(t, base, s, key0); break;
    case DT_F16: vec ? chunk_vector<DT_F16>(t, base, s, key0) : chunk_element<DT_F16>(t, base, s, key0); break;
    default: vec ? chunk_vector<DT_BF16>(t, base, s, key0) : chunk_element<DT_BF16>(t, base, s, key0); break;
    }
}

// ---- norm of all gradients -----------------------------------------------------------------------------------------------
// squares and sums in 64 bits: no overflow for any finite gradient, and the same value for every order that matters in fp32
template <int DT>
__device__ __forceinline__ double chunk_squares(const OptTensor &t, uint64_t base)
{
    using T = typename Elem<DT>::T;
    const T *g = (const T *)t.g + base;
    const uint64_t left = t.n - base;
    double acc = 0.0;
    if ((t.flags & ALIGNED) && left >= OPT_CHUNK) {
        Vec<T, 4> v[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) v[it] = reinterpret_cast<const Vec<T, 4> *>(g)[it * OPT_THREADS + threadIdx.x];
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int k = 0; k < 4; ++k) { const double d = (double)v[it].e[k]; acc += d * d; }
    } else {
        const uint32_t n = left < OPT_CHUNK ? (uint32_t)left : OPT_CHUNK;
        for (uint32_t i = threadIdx.x; i < n; i += OPT_THREADS) { const double d = (double)g[i]; acc += d * d; }
    }
    return acc;
}

__global__ void __launch_bounds__(OPT_THREADS)
k_grad_squares(const OptLaunch a, double *__restrict__ partials)
{
    double acc = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < a.n_chunks; chunk += gridDim.x) {
        const uint32_t which = tensor_of(a, chunk);
        const OptTensor &t = a.t[which];
        const uint64_t base = (uint64_t)(chunk - a.first[which]) * OPT_CHUNK;
        switch (t.flags & DT_MASK) {
        case DT_F32: acc += chunk_squares<DT_F32>(t, base); break;
        case DT_F16: acc += chunk_squares<DT_F16>(t, base); break;
        default: acc += chunk_squares<DT_BF16>(t, base); break;
        }
    }
    __shared__ double part[OPT_THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partials[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// one workgroup: the partial sums in a fixed order, then the step's scalars
__global__ void __launch_bounds__(OPT_THREADS)
k_adamw_begin(int32_t *__restrict__ step, float *__restrict__ hyper, double b1, double b2, const double *__restrict__ partials,
              uint32_t n_partials, double max_norm, const float *__restrict__ grad_scale, const float *__restrict__ found_inf)
{
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < n_partials; i += OPT_THREADS) acc += partials[i];
    __shared__ double part[OPT_THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x != 0) return;
    const double unscale = grad_scale ? 1.0 / (double)*grad_scale : 1.0;
    double factor = unscale;
    bool skip = found_inf && *found_inf != 0.f;
    if (partials) {
        const double norm = sqrt((part[0] + part[1]) + (part[2] + part[3])) * unscale;
        const double ratio = max_norm / (norm + 1e-6);  // torch.nn.utils.clip_grad_norm_
        factor *= ratio < 1.0 ? ratio : 1.0;
        skip = skip || !(norm <= 1.7976931348623157e308);
        hyper[5] = (float)norm;
    }
    const int32_t t = skip ? *step : *step + 1;
    if (!skip) *step = t;
    hyper[0] = (float)factor;
    hyper[1] = (float)(1.0 / (1.0 - pow(b1, (double)t)));
    hyper[2] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    hyper[3] = __int_as_float(skip ? 1 : 0);
    hyper[4] = __int_as_float(t);
}

// ---- host ----------------------------------------------------------------------------------------------------------------
bool all_aligned(const OptTensor &t)
{
    const uintptr_t own = (uintptr_t)t.p | (uintptr_t)t.g, state = (uintptr_t)t.m | (uintptr_t)t.v;
    const uintptr_t need = (t.flags & DT_MASK) == DT_F32 ? 15 : 7, need_state = t.flags & STATE8 ? 3 : 15;
    return (own & need) == 0 && (state & need_state) == 0 && ((uintptr_t)t.image & 7) == 0;
}

// fills launches of at most OPT_TENSORS tensors and hands each to `go`; grads_only: the norm, which reads nothing else
template <class Go>
int each_launch(const char *what, const NsrAdamwTensor *tensors, uint32_t n_tensors, bool grads_only, bool lr_on_device, double b1_correction, Go go)
{
    NSR_REQUIRE(n_tensors == 0 || tensors, "%s: NULL descriptors", what);
    for (uint32_t i = 0; i < n_tensors; ++i) {  // refuse before anything is launched
        const NsrAdamwTensor &x = tensors[i];
        NSR_REQUIRE(x.n < (1ull << 35), "%s: tensor %u has 2^35 elements or more", what, i);
        NSR_REQUIRE(x.dtype <= 2, "%s: tensor %u: dtype %u (0 fp32, 1 fp16, 2 bf16)", what, i, x.dtype);
        NSR_REQUIRE(x.n == 0 || x.grad, "%s: tensor %u has a NULL gradient", what, i);
        NSR_REQUIRE(((uintptr_t)x.grad & (x.dtype == 0 ? 3 : 1)) == 0, "%s: tensor %u: misaligned gradient", what, i);
        if (grads_only || x.n == 0) continue;
        NSR_REQUIRE(x.params && x.exp_avg && x.exp_avg_sq, "%s: tensor %u has a NULL pointer", what, i);
        NSR_REQUIRE(x.state_bits == 32 || x.state_bits == 8, "%s: tensor %u: moments in %u bits (32 or 8)", what, i, x.state_bits);
        NSR_REQUIRE(x.state_bits == 32 || (x.scales_m && x.scales_r), "%s: tensor %u: 8-bit moments need scales", what, i);
        NSR_REQUIRE(!x.lr_dev || lr_on_device, "%s: tensor %u: lr_dev needs the device-side step count (hyper)", what, i);
        NSR_REQUIRE(x.index0 % OPT_BLOCK == 0, "%s: tensor %u: index0 must be a multiple of %d", what, i, OPT_BLOCK);
        const uintptr_t fp32 = (uintptr_t)x.scales_m | (uintptr_t)x.scales_r | (uintptr_t)x.lr_dev |
                               (x.state_bits == 32 ? (uintptr_t)x.exp_avg | (uintptr_t)x.exp_avg_sq : 0);
        NSR_REQUIRE((fp32 & 3) == 0 && ((uintptr_t)x.params & (x.dtype == 0 ? 3 : 1)) == 0 && ((uintptr_t)x.image & 1) == 0,
                    "%s: tensor %u: misaligned pointer", what, i);
    }
    OptLaunch a;
    a.n_tensors = a.n_chunks = 0;
    for (uint32_t i = 0; i < n_tensors; ++i) {
        const NsrAdamwTensor &x = tensors[i];
        if (x.n) {
            OptTensor &t = a.t[a.n_tensors];
            t.p = x.params; t.g = x.grad; t.m = x.exp_avg; t.v = x.exp_avg_sq;
            t.sm = x.scales_m; t.sr = x.scales_r; t.image = (__half *)x.image; t.lr_dev = x.lr_dev;
            t.n = x.n; t.index0 = x.index0;
            t.lr = (float)(x.lr / b1_correction); t.decay = (float)(1.0 - x.lr * x.weight_decay); t.wd = (float)x.weight_decay;
            t.flags = x.dtype | (x.state_bits == 8 ? STATE8 : 0);
            if (grads_only) t.flags |= ((uintptr_t)x.grad & (x.dtype == 0 ? 15 : 7)) == 0 ? ALIGNED : 0;
            else t.flags |= all_aligned(t) ? ALIGNED : 0;
            a.first[a.n_tensors++] = a.n_chunks;
            a.n_chunks += nsr_div_up(x.n, OPT_CHUNK);
        }
        // 2^23 chunks are 2^31 threads: the grid stays under the launch limit (2^32 threads) with the next tensor's 2^23 more
        if (a.n_tensors && (a.n_tensors == OPT_TENSORS || a.n_chunks >= (1u << 23) - 1 || i + 1 == n_tensors)) {
            const int rc = go(a);
            if (rc != NSR_OK) return rc;
            a.n_tensors = a.n_chunks = 0;
        }
    }
    return NSR_OK;
}

}  // namespace

extern "C" int nsr_adamw_tensors(const NsrAdamwTensor *tensors, uint32_t n_tensors, double beta1, double beta2, double eps,
                                 int32_t step, const float *hyper, double grad_unscale, uint32_t seed, void *stream)
{
    NSR_REQUIRE(hyper || step >= 1, "nsr_adamw_tensors: step counts from 1");
    NSR_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "nsr_adamw_tensors: betas in [0, 1)");
    NSR_REQUIRE(eps >= 0.0, "nsr_adamw_tensors: eps >= 0");
    double c1 = 1.0, c2 = 1.0;
    if (!hyper) { c1 = 1.0 - pow(beta1, (double)step); c2 = 1.0 - pow(beta2, (double)step); }
    OptScalars s;
    s.scale = (float)grad_unscale; s.step = 0.f; s.root = (float)(1.0 / sqrt(c2)); s.decay = 1.f;
    s.b1 = (float)beta1; s.c1 = (float)(1.0 - beta1); s.b2 = (float)beta2; s.c2 = (float)(1.0 - beta2); s.eps = (float)eps;
    return each_launch("nsr_adamw_tensors", tensors, n_tensors, false, hyper != nullptr, c1, [&](const OptLaunch &a) {
        hipLaunchKernelGGL(k_adamw_tensors, dim3(a.n_chunks), dim3(OPT_THREADS), 0, (hipStream_t)stream, a, s, seed,
                           (uint32_t)step, hyper);
        NSR_CHECK_LAUNCH("nsr_adamw_tensors");
        return NSR_OK;
    });
}

extern "C" uint32_t nsr_grad_squares_capacity(const NsrAdamwTensor *tensors, uint32_t n_tensors)
{
    // a launch ends after OPT_TENSORS tensors or 2^23 - 1 chunks, whichever comes first
    uint64_t chunks = 0;
    for (uint32_t i = 0; tensors && i < n_tensors; ++i) chunks += nsr_div_up(tensors[i].n, OPT_CHUNK);
    const uint64_t launches = nsr_div_up(n_tensors, OPT_TENSORS) + chunks / ((1u << 23) - 1) + 1;
    return (uint32_t)(launches * NORM_MAX_GRID);
}

extern "C" int nsr_grad_squares(const NsrAdamwTensor *tensors, uint32_t n_tensors, double *partials, uint32_t capacity,
                                uint32_t *n_partials, void *stream)
{
    NSR_REQUIRE(partials && n_partials, "nsr_grad_squares: NULL pointer");
    NSR_REQUIRE(((uintptr_t)partials & 7) == 0, "nsr_grad_squares: partials must be 8-byte aligned");
    *n_partials = 0;
    return each_launch("nsr_grad_squares", tensors, n_tensors, true, true, 1.0, [&](const OptLaunch &a) {
        const uint32_t grid = a.n_chunks < (uint32_t)NORM_MAX_GRID ? a.n_chunks : NORM_MAX_GRID;
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
    hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(OPT_THREADS), 0, (hipStream_t)stream, step, hyper, beta1, beta2, partials,
                       partials ? n_partials : 0, max_norm, grad_scale, found_inf);
    NSR_CHECK_LAUNCH("nsr_adamw_begin");
    return NSR_OK;
}
