// AdamW step over many tensors in one launch:
//   t += 1,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps),
// the states float32 or 8-bit codes in blocks of 256 elements with one float32
// scale each:  m = s sgn(c) (c / 127)^2, c in -127 .. 127;  v = s (c / 255)^4, c
// in 0 .. 255.  The powers give small values their own codes (m from 6e-5 of s
// on, sqrt(v) from 1.5e-5 sqrt(s) on); a v above 0 keeps a code above 0, so no
// first moment that is kept meets a second moment rounded to 0.  s is the power
// of two at or above the block's largest: a scale rounded to float32 instead
// would hang on the last bit of the 64-bit sums (0.9 s + 0.1 g is a tie of two
// float32 one time in ten), and the codes on it; it costs the codes a factor
// of sqrt(2) (m) or 2^(1/4) (v) of their range at most.
//
// Bound by HBM: 28 bytes an element with float32 states, 16 with 8-bit ones
// (float32 parameters and gradients).  86.6 M elements with float32 states 476
// us, 5.1 TB/s; 304 M with 8-bit states 1,190 us, 4.1 TB/s, where the codes' decisions
// cost about a fifth beside the memory's time.
#include "rpfq_device.h"

namespace rpfq {

// Elements of a workgroup: 4096, or 1024 where those would not fill the chip
// (769,000 elements 7.1 -> 5.1 us).
constexpr int kAdamChunk = 4096, kAdamSmallChunk = 1024;

struct AdamLaunch {
    AdamTensor t[kAdamTensors];
    int start[kAdamTensors + 1];  // first chunk of each tensor
    int count, chunk;
    const float* coef;
    double b1, b2;
    float eps;
};

// b^t for a whole t >= 0 in 64 bits, by squares.
__device__ __forceinline__ double adam_pow(double b, double t) {
    double r = 1.0;
    for (uint32_t n = (uint32_t)t; n; n >>= 1, b *= b)
        if (n & 1) r *= b;
    return r;
}

// coef: 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 / grad_scale, 1 (0: the
// step is left out).  The powers in 64 bits, as torch takes them on the host;
// here so that a captured step counts on when it is replayed.
__global__ void adam_coef_kernel(float* step, AdamHyper h, const float* lr_dev, const float* grad_scale, const float* found_inf,
                                 float* coef) {
    const bool skip = found_inf && *found_inf != 0.0f;
    const double t = (double)*step + (skip ? 0.0 : 1.0), lr = lr_dev ? (double)*lr_dev : h.lr;
    if (!skip) *step = (float)t;
    coef[0] = (float)(1.0 - lr * h.weight_decay);
    coef[1] = (float)(lr / (1.0 - adam_pow(h.beta1, t)));
    coef[2] = (float)(1.0 / sqrt(1.0 - adam_pow(h.beta2, t)));
    coef[3] = grad_scale ? (float)(1.0 / (double)*grad_scale) : 1.0f;
    coef[4] = skip ? 0.0f : 1.0f;
}

template <int DT>
__device__ __forceinline__ float adam_load(const void* p, int64_t i) {
    if (DT == RPFQ_F32) return reinterpret_cast<const float*>(p)[i];
    if (DT == RPFQ_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// 4 elements from i on, those below n (vec: all four, 16- or 8-byte aligned).
template <int DT>
__device__ __forceinline__ f32x4 adam_load4(const void* p, int64_t i, int64_t n, bool vec) {
    f32x4 v = {0, 0, 0, 0};
    if (vec) {
        if constexpr (DT == RPFQ_F32) {
            v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
            const uint32_t w[2] = {u.x, u.y};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint16_t b = (uint16_t)(w[t >> 1] >> (16 * (t & 1)));
                v[t] = DT == RPFQ_F16 ? (float)__builtin_bit_cast(_Float16, b) : bf16_to_f32(b);
            }
        }
        return v;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (i + t < n) v[t] = adam_load<DT>(p, i + t);
    return v;
}

template <int DT>
__device__ __forceinline__ void adam_store4(void* p, int64_t i, int64_t n, bool vec, f32x4 v) {
    if (vec) {
        if constexpr (DT == RPFQ_F32) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i) = v;
        } else {
            uint2 o;
            o.x = DT == RPFQ_F16 ? cvt_pk(v[0], v[1]) : pack_bf2(v[0], v[1]);
            o.y = DT == RPFQ_F16 ? cvt_pk(v[2], v[3]) : pack_bf2(v[2], v[3]);
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = o;
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (i + t < n) store1<DT>(p, i + t, v[t]);
}

// The update; v_sqrt and v_rcp are within one unit of the last place.
__device__ __forceinline__ float adam_param(float p, float m, float v, const float* coef, float eps) {
    const float d = __builtin_fmaf(__builtin_amdgcn_sqrtf(v), coef[2], eps);
    // a denominator that v_rcp takes for 0 (eps = 0 and v = 0 among them) is divided by
    const float q = d >= 0x1p-126f ? coef[1] * m * __builtin_amdgcn_rcpf(d) : coef[1] * m / d;
    return __builtin_fmaf(p, coef[0], -q);
}

// 8-bit states.  The codes are those of the definition in 64 bits, found in
// float32 wherever that decides: a block with a value that float32's error
// (2^-20 of the sums' terms) leaves between two codes or two scales, about one
// in thirty, is done over in 64 bits.
constexpr float kAdamTol = 0x1p-20f;
constexpr double kM2 = 1.0 / (127.0 * 127.0), kV4 = 1.0 / (255.0 * 255.0 * 255.0 * 255.0);

__device__ __forceinline__ uint32_t wave_max(uint32_t mx) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    return mx;
}

// The scale of a block from the bits of its largest: the power of two at or
// above it, 2^-126 at least, 0 for zeros, NaN where a value is inf or NaN or the
// power is past float32.
__device__ __forceinline__ float adam_scale(uint32_t mx) {
    if (mx == 0) return 0.0f;
    const uint32_t up = (mx + 0x7fffffu) & 0x7f800000u;
    return up >= 0x7f800000u || mx >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(up), 0x1p-126f);
}

// The code of a >= 0 under c -> s (c / MAX)^P (P = 2 or 4), nearest, from u = a
// / s <= 1: v_sqrt finds it to within one, and (2 c +- 1)^P, whole numbers, are
// the middles next to it.  unsure: a is within err of one of them.
template <int P, class T>
__device__ __forceinline__ float adam_code(float u, T exact_u, float err, bool& unsure) {
    constexpr float MAX = P == 2 ? 127.0f : 255.0f;
    const float root = __builtin_amdgcn_sqrtf(u);
    float c = fminf(__builtin_rintf(MAX * (P == 2 ? root : __builtin_amdgcn_sqrtf(root))), MAX);
    constexpr T UNIT = P == 2 ? (T)(4.0 / kM2) : (T)(16.0 / kV4);
    const T a = exact_u * UNIT;
    const T hi = (T)(2.0f * c + 1.0f), lo = (T)(2.0f * c - 1.0f);
    const T h2 = hi * hi, l2 = lo * lo, h = P == 2 ? h2 : h2 * h2, l = P == 2 ? l2 : l2 * l2;
    unsure |= fabsf((float)(a - h)) <= err * (float)UNIT || fabsf((float)(a - l)) <= err * (float)UNIT;
    if (a > h) c += 1.0f;
    else if (c > 0.0f && a < l) c -= 1.0f;
    return fminf(c, MAX);
}
__device__ __forceinline__ double adam_m(int c, float scale) { return (double)(c * abs(c)) * ((double)scale * kM2); }
__device__ __forceinline__ double adam_v(int c, float scale) {
    const double q = (double)(c * c);
    return q * q * ((double)scale * kV4);
}

// 4 elements of a block of 64 lanes: old codes and scales in, new ones out, and
// the moments as float32.
struct AdamSmall {
    uint32_t cm, cv;
    float sm, sv;
};
__device__ __forceinline__ float inv_power(float s) { return s > 0.0f ? 1.0f / s : 0.0f; }  // exact, s a power of two

__device__ __forceinline__ void adam_small_exact(AdamSmall& q, f32x4 g, double b1, double b2, f32x4& m, f32x4& v) {
    double md[4], vd[4];
    uint32_t um = 0, uv = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double gd = (double)g[e];
        md[e] = b1 * adam_m((int8_t)(q.cm >> (8 * e)), q.sm) + (1.0 - b1) * gd;
        vd[e] = b2 * adam_v((int)((q.cv >> (8 * e)) & 0xffu), q.sv) + (1.0 - b2) * gd * gd;
        m[e] = (float)md[e];
        v[e] = (float)vd[e];
        // to float32 upwards, so that the power of two is that of the 64-bit value
        um = max(um, (__float_as_uint(m[e]) & 0x7fffffffu) + ((double)fabsf(m[e]) < fabs(md[e]) ? 1u : 0u));
        uv = max(uv, __float_as_uint(v[e]) + ((double)v[e] < vd[e] ? 1u : 0u));
    }
    q.sm = adam_scale(wave_max(um));
    q.sv = adam_scale(wave_max(uv));
    const float im = inv_power(q.sm), iv = inv_power(q.sv);
    uint32_t cm = 0, cv = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bool unsure = false;
        const double a = fabs(md[e]) * (double)im, b = vd[e] * (double)iv;
        const int c = im > 0.0f ? (int)adam_code<2>((float)a, a, 0.0f, unsure) : 0;
        const int u = iv > 0.0f ? (int)adam_code<4>((float)b, b, 0.0f, unsure) : 0;
        cm |= (uint32_t)((md[e] < 0.0 ? -c : c) & 0xff) << (8 * e);
        cv |= (uint32_t)(u == 0 && vd[e] > 0.0 && iv > 0.0f ? 1 : u) << (8 * e);
    }
    q.cm = cm;
    q.cv = cv;
}

__device__ __forceinline__ void adam_small(AdamSmall& q, f32x4 g, double b1, double b2, f32x4& m, f32x4& v) {
    const float f1 = (float)b1, f2 = (float)b2, d1 = (float)(1.0 - b1), d2 = (float)(1.0 - b2);
    const float km = q.sm * (float)kM2, kv = q.sv * (float)kV4;
    // blocks of zeros without a gradient stay that
    if (!__any((q.cm | q.cv) != 0 || g[0] != 0.0f || g[1] != 0.0f || g[2] != 0.0f || g[3] != 0.0f)) {
        q.sm = q.sv = 0.0f;
        m = v = (f32x4){0, 0, 0, 0};
        return;
    }
    float em[4];  // what m's error is relative to
    uint32_t um = 0, uv = 0, ue = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float c = (float)(int8_t)(q.cm >> (8 * e)), u = (float)((q.cv >> (8 * e)) & 0xffu);
        const float was = f1 * (c * fabsf(c) * km), add = d1 * g[e], u2 = u * u;
        m[e] = was + add;
        v[e] = __builtin_fmaf(f2, u2 * u2 * kv, d2 * (g[e] * g[e]));
        em[e] = fabsf(was) + fabsf(add);
        ue = max(ue, __float_as_uint(em[e]));
        um = max(um, __float_as_uint(m[e]) & 0x7fffffffu);
        uv = max(uv, __float_as_uint(v[e]));
    }
    um = wave_max(um);
    uv = wave_max(uv);
    ue = wave_max(ue);
    const float sm = adam_scale(um), sv = adam_scale(uv), im = inv_power(sm), iv = inv_power(sv);
    // what float32 does not decide: special values and zeros, numbers near the
    // ends of its range, a largest within err of a power of two
    auto apart = [](uint32_t u, float s, float err) {
        const float x = __uint_as_float(u);
        return !(x > 0x1p-60f && x < 0x1p60f) || x + err >= s || x - err <= 0.5f * s;
    };
    bool unsure = apart(um, sm, __uint_as_float(ue) * kAdamTol) || apart(uv, sv, __uint_as_float(uv) * kAdamTol);
    uint32_t cm = 0, cv = 0;
    if (!unsure) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = fabsf(m[e]) * im, b = v[e] * iv;
            const int c = (int)adam_code<2>(a, a, em[e] * im * kAdamTol, unsure);
            const int u = (int)adam_code<4>(b, b, b * kAdamTol, unsure);
            cm |= (uint32_t)((m[e] < 0.0f ? -c : c) & 0xff) << (8 * e);
            cv |= (uint32_t)(u == 0 && v[e] > 0.0f ? 1 : u) << (8 * e);
            // a v above 0 that has left float32's range
            unsure |= v[e] < 0x1p-120f && (g[e] != 0.0f || ((q.cv >> (8 * e)) & 0xffu) != 0);
        }
    }
    if (__any(unsure)) {
        adam_small_exact(q, g, b1, b2, m, v);
        return;
    }
    q = {cm, cv, sm, sv};
}

template <int PDT, int GDT, bool SMALL>
__global__ void __launch_bounds__(256) adam_kernel(AdamLaunch a) {
    const float* cf = a.coef;
    if (cf[4] == 0.0f) return;
    const float coef[3] = {cf[0], cf[1], cf[2]};
    const float inv = cf[3];
    int lo = 0, hi = a.count;  // the chunk's tensor
    const int chunk = blockIdx.x;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.start[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    const AdamTensor t = a.t[lo];
    const int64_t n = t.numel < 0 ? -t.numel : t.numel;  // negative: some pointer is not aligned for whole vectors
    const int64_t first = (int64_t)(chunk - a.start[lo]) * a.chunk;
    const int64_t last = first + a.chunk < n ? first + a.chunk : n;
    const bool aligned = t.numel > 0;
    const float b1 = (float)a.b1, b2 = (float)a.b2, d1 = (float)(1.0 - a.b1), d2 = (float)(1.0 - a.b2);
    for (int64_t i = first + 4 * threadIdx.x; i < (SMALL ? first + a.chunk : last); i += 1024) {
        const bool vec = aligned && i + 4 <= n;
        f32x4 p = adam_load4<PDT>(t.param, i, n, vec), g = adam_load4<GDT>(t.grad, i, n, vec) * inv;
        f32x4 m, v;
        if constexpr (!SMALL) {
            float* mp = reinterpret_cast<float*>(t.exp_avg);
            float* vp = reinterpret_cast<float*>(t.exp_avg_sq);
            m = adam_load4<RPFQ_F32>(mp, i, n, vec);
            v = adam_load4<RPFQ_F32>(vp, i, n, vec);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = m[e] * b1 + g[e] * d1;
                v[e] = v[e] * b2 + g[e] * g[e] * d2;
            }
            adam_store4<RPFQ_F32>(mp, i, n, vec, m);
            adam_store4<RPFQ_F32>(vp, i, n, vec, v);
        } else {
            // a wave's 64 x 4 elements are one block; blocks past the tensor
            // have no scale, and whole waves leave together
            if ((i & ~(int64_t)255) >= n) return;
            int8_t* mp = reinterpret_cast<int8_t*>(t.exp_avg);
            uint8_t* vp = reinterpret_cast<uint8_t*>(t.exp_avg_sq);
            const float sm = t.exp_avg_scale[i >> 8], sv = t.exp_avg_sq_scale[i >> 8];
            uint32_t cm = 0, cv = 0;
            if (vec) {
                cm = *reinterpret_cast<const uint32_t*>(mp + i);
                cv = *reinterpret_cast<const uint32_t*>(vp + i);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < n) cm |= (uint32_t)(uint8_t)mp[i + e] << (8 * e), cv |= (uint32_t)vp[i + e] << (8 * e);
            }
            AdamSmall q = {cm, cv, sm, sv};
            adam_small(q, g, a.b1, a.b2, m, v);
            cm = q.cm, cv = q.cv;
            if (vec) {
                *reinterpret_cast<uint32_t*>(mp + i) = cm;
                *reinterpret_cast<uint32_t*>(vp + i) = cv;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < n) mp[i + e] = (int8_t)(cm >> (8 * e)), vp[i + e] = (uint8_t)(cv >> (8 * e));
            }
            if ((threadIdx.x & 63) == 0) {
                t.exp_avg_scale[i >> 8] = q.sm;
                t.exp_avg_sq_scale[i >> 8] = q.sv;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = adam_param(p[e], m[e], v[e], coef, a.eps);
        adam_store4<PDT>(t.param, i, n, vec, p);
    }
}

// The values of 8-bit states, float32: 5 bytes an element and moment (2 x 304 M
// 500 us, 6.1 TB/s).
struct AdamValues {
    const void* c[kAdamTensors];
    const float* s[kAdamTensors];
    float* out[kAdamTensors];
    int64_t n[kAdamTensors];  // negative: codes of v
    int start[kAdamTensors + 1];
    int count;
};
__global__ void __launch_bounds__(256) adam_values_kernel(AdamValues a) {
    int lo = 0, hi = a.count;
    const int chunk = blockIdx.x;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.start[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    const bool second = a.n[lo] < 0;
    const int64_t n = second ? -a.n[lo] : a.n[lo], first = (int64_t)(chunk - a.start[lo]) * kAdamChunk;
    const uint8_t* c = reinterpret_cast<const uint8_t*>(a.c[lo]);
    const float* s = a.s[lo];
    float* out = a.out[lo];
    const bool aligned = ((reinterpret_cast<uintptr_t>(c) & 3) | (reinterpret_cast<uintptr_t>(out) & 15)) == 0;
    for (int64_t i = first + 4 * threadIdx.x; i < first + kAdamChunk && i < n; i += 1024) {
        const float scale = s[i >> 8];
        const bool vec = aligned && i + 4 <= n;
        uint32_t w = 0;
        if (vec) {
            w = *reinterpret_cast<const uint32_t*>(c + i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) w |= (uint32_t)c[i + e] << (8 * e);
        }
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t b = (w >> (8 * e)) & 0xffu;
            v[e] = (float)(second ? adam_v((int)b, scale) : adam_m((int8_t)b, scale));
        }
        adam_store4<RPFQ_F32>(out, i, n, vec, v);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
template <int PDT, int GDT>
static void adam_go(const AdamLaunch& a, bool small, int chunks, hipStream_t s) {
    if (small) hipLaunchKernelGGL((adam_kernel<PDT, GDT, true>), dim3(chunks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((adam_kernel<PDT, GDT, false>), dim3(chunks), dim3(256), 0, s, a);
}

hipError_t launch_adamw(const AdamTensor* t, int64_t count, int pdt, int bits, const AdamHyper& h, float* step,
                        const float* lr_dev, const float* grad_scale, const float* found_inf, float* coef, hipStream_t s) {
    hipLaunchKernelGGL(adam_coef_kernel, dim3(1), dim3(1), 0, s, step, h, lr_dev, grad_scale, found_inf, coef);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    AdamLaunch a = {};
    a.coef = coef;
    a.b1 = h.beta1;
    a.b2 = h.beta2;
    a.eps = (float)h.eps;
    int64_t all = 0;
    for (int64_t i = 0; i < count; ++i) all += t[i].numel;
    a.chunk = all < 8LL * device_cus() * kAdamChunk ? kAdamSmallChunk : kAdamChunk;
    auto flush = [&]() {
        if (!a.count) return hipSuccess;
        const int chunks = a.start[a.count];
        const bool small = bits == 8;
        if (pdt == RPFQ_F32) adam_go<RPFQ_F32, RPFQ_F32>(a, small, chunks, s);
        else if (pdt == RPFQ_F16) adam_go<RPFQ_F16, RPFQ_F16>(a, small, chunks, s);
        else adam_go<RPFQ_BF16, RPFQ_BF16>(a, small, chunks, s);
        a.count = 0;
        return hipGetLastError();
    };
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].numel == 0) continue;
        const int64_t n = t[i].numel, chunks = (n + a.chunk - 1) / a.chunk;
        if (a.count == kAdamTensors || (a.count && a.start[a.count] + chunks > (1 << 30)))
            if ((e = flush()) != hipSuccess) return e;
        AdamTensor& d = a.t[a.count];
        d = t[i];
        const uintptr_t wide = reinterpret_cast<uintptr_t>(d.param) | reinterpret_cast<uintptr_t>(d.grad) |
                               (bits == 32 ? reinterpret_cast<uintptr_t>(d.exp_avg) | reinterpret_cast<uintptr_t>(d.exp_avg_sq) : 0);
        const uintptr_t codes = bits == 8 ? reinterpret_cast<uintptr_t>(d.exp_avg) | reinterpret_cast<uintptr_t>(d.exp_avg_sq) : 0;
        if ((wide & 15) || (codes & 3)) d.numel = -n;
        a.start[a.count + 1] = (a.count ? a.start[a.count] : 0) + (int)chunks;
        ++a.count;
    }
    return flush();
}

hipError_t launch_adamw_values(const void* const* codes, const float* const* scales, const int64_t* numel,
                               const int* second, float* const* out, int64_t count, hipStream_t s) {
    AdamValues a = {};
    auto flush = [&]() {
        if (!a.count) return hipSuccess;
        hipLaunchKernelGGL(adam_values_kernel, dim3(a.start[a.count]), dim3(256), 0, s, a);
        a.count = 0;
        return hipGetLastError();
    };
    hipError_t e;
    for (int64_t i = 0; i < count; ++i) {
        if (numel[i] == 0) continue;
        const int64_t chunks = (numel[i] + kAdamChunk - 1) / kAdamChunk;
        if (a.count == kAdamTensors || (a.count && a.start[a.count] + chunks > (1 << 30)))
            if ((e = flush()) != hipSuccess) return e;
        a.c[a.count] = codes[i];
        a.s[a.count] = scales[i];
        a.out[a.count] = out[i];
        a.n[a.count] = second[i] ? -numel[i] : numel[i];
        a.start[a.count + 1] = (a.count ? a.start[a.count] : 0) + (int)chunks;
        ++a.count;
    }
    return flush();
}

}  // namespace rpfq
