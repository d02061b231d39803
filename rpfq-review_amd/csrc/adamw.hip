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
// (float32 parameters and gradients).
#include "rpfq_device.h"

namespace rpfq {

constexpr int kAdamChunk = 4096;  // elements of a workgroup

struct AdamLaunch {
    AdamTensor t[kAdamTensors];
    int start[kAdamTensors + 1];  // first chunk of each tensor
    int count;
    const float* coef;
    double b1, b2;
    float eps;
};

// coef: 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 / grad_scale, 1 (0: the
// step is left out).  The powers in 64 bits, as torch takes them on the host;
// here so that a captured step counts on when it is replayed.
__global__ void adam_coef_kernel(float* step, AdamHyper h, const float* lr_dev, const float* grad_scale, const float* found_inf,
                                 float* coef) {
    const bool skip = found_inf && *found_inf != 0.0f;
    const double t = (double)*step + (skip ? 0.0 : 1.0), lr = lr_dev ? (double)*lr_dev : h.lr;
    if (!skip) *step = (float)t;
    coef[0] = (float)(1.0 - lr * h.weight_decay);
    coef[1] = (float)(lr / (1.0 - pow(h.beta1, t)));
    coef[2] = (float)(1.0 / sqrt(1.0 - pow(h.beta2, t)));
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

__device__ __forceinline__ float adam_param(float p, float m, float v, const float* coef, float eps) {
    return p * coef[0] - coef[1] * m / (sqrtf(v) * coef[2] + eps);
}

// The code of a >= 0 under c -> top_value (c / MAX)^P (P = 2 or 4), nearest.
// float32 finds it to within one; the two middles next to it are compared in 64
// bits, so the codes are those of the definition.
template <int P>
__device__ __forceinline__ int adam_code(double a, float scale) {
    constexpr int MAX = P == 2 ? 127 : 255;
    if (!(scale > 0.0f)) return 0;
    const float u = fminf((float)a / scale, 1.0f);
    float c = __builtin_rintf((float)MAX * (P == 2 ? sqrtf(u) : sqrtf(sqrtf(u))));
    const double k = (double)scale * (P == 2 ? 1.0 / (127.0 * 127.0) : 1.0 / (255.0 * 255.0 * 255.0 * 255.0));
    const double hi = (double)c + 0.5, lo = (double)c - 0.5;
    const double h2 = hi * hi, l2 = lo * lo;
    if (a > (P == 2 ? h2 : h2 * h2) * k) c += 1.0f;
    else if (c > 0.0f && a < (P == 2 ? l2 : l2 * l2) * k) c -= 1.0f;
    return (int)fminf(c, (float)MAX);
}
__device__ __forceinline__ double adam_m(int c, float scale) {
    return (double)(c * abs(c)) * ((double)scale * (1.0 / (127.0 * 127.0)));
}
__device__ __forceinline__ double adam_v(int c, float scale) {
    const double q = (double)(c * c);
    return q * q * ((double)scale * (1.0 / (255.0 * 255.0 * 255.0 * 255.0)));
}

// The scale of a block (one wave, 4 values a lane): the power of two at or above
// the largest, 2^-126 at least, 0 for zeros, NaN where a value is inf or NaN or
// the power is past float32.  Each value is taken to float32 upwards first.
__device__ __forceinline__ float adam_scale(const double (&a)[4]) {
    uint32_t mx = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const double d = fabs(a[t]);
        const float f = (float)d;
        mx = max(mx, __float_as_uint(f) + ((double)f < d ? 1u : 0u));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    if (mx == 0) return 0.0f;
    const uint32_t up = ((mx + 0x7fffffu) & 0x7f800000u);
    return up >= 0x7f800000u || mx >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(up), 0x1p-126f);
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
    const int64_t first = (int64_t)(chunk - a.start[lo]) * kAdamChunk;
    const int64_t last = first + kAdamChunk < n ? first + kAdamChunk : n;
    const bool aligned = t.numel > 0;
    const float b1 = (float)a.b1, b2 = (float)a.b2, d1 = (float)(1.0 - a.b1), d2 = (float)(1.0 - a.b2);
    for (int64_t i = first + 4 * threadIdx.x; i < (SMALL ? first + kAdamChunk : last); i += 1024) {
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
            double md[4], vd[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double gd = (double)g[e];
                md[e] = a.b1 * adam_m((int8_t)(cm >> (8 * e)), sm) + (1.0 - a.b1) * gd;
                vd[e] = a.b2 * adam_v((int)((cv >> (8 * e)) & 0xffu), sv) + (1.0 - a.b2) * gd * gd;
                m[e] = (float)md[e];
                v[e] = (float)vd[e];
            }
            const float tm = adam_scale(md), tv = adam_scale(vd);
            cm = cv = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = adam_code<2>(fabs(md[e]), tm), u = adam_code<4>(vd[e], tv);
                cm |= (uint32_t)((md[e] < 0.0 ? -c : c) & 0xff) << (8 * e);
                cv |= (uint32_t)(u == 0 && vd[e] > 0.0 && tv > 0.0f ? 1 : u) << (8 * e);
            }
            if (vec) {
                *reinterpret_cast<uint32_t*>(mp + i) = cm;
                *reinterpret_cast<uint32_t*>(vp + i) = cv;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < n) mp[i + e] = (int8_t)(cm >> (8 * e)), vp[i + e] = (uint8_t)(cv >> (8 * e));
            }
            if ((threadIdx.x & 63) == 0) {
                t.exp_avg_scale[i >> 8] = tm;
                t.exp_avg_sq_scale[i >> 8] = tv;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = adam_param(p[e], m[e], v[e], coef, a.eps);
        adam_store4<PDT>(t.param, i, n, vec, p);
    }
}

// The values of 8-bit states, float32.
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
        const int64_t n = t[i].numel, chunks = (n + kAdamChunk - 1) / kAdamChunk;
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
