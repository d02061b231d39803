// Rotary positions of several axes: pair j of a head's values turns by the angle
// position[token][axis of j] freqs[j],
//   (u, v) -> (u cos - v sin, v cos + u sin),
// in the queries and keys of one call; the gradient turns back.
#include "rpfq_device.h"

namespace rpfq {

struct RotaryArgs {
    rpfq_rotary_desc d;
    const char* in[2];
    char* out[2];
    const void* pos;
    const double* freqs;
    int pairs, tokens, units, total;  // pairs of a head; tokens of a workgroup, units of a head, of all its tokens
};

template <int DT>
constexpr int rotary_vec() { return DT == RPFQ_F32 ? 4 : 8; }

// V consecutive values as float32: 16 bytes, or one value.
template <int DT, int V>
__device__ __forceinline__ void rotary_load(const char* p, int64_t at, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = load_y1<DT>(p, at);
    } else if constexpr (DT == RPFQ_F32) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p + 4 * at);
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = a[t];
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p + 2 * at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (DT == RPFQ_F16) {
                const half2v h = __builtin_bit_cast(half2v, w[t]);
                v[2 * t] = (float)h[0], v[2 * t + 1] = (float)h[1];
            } else {
                v[2 * t] = bf16_to_f32(w[t] & 0xffffu), v[2 * t + 1] = bf16_to_f32(w[t] >> 16);
            }
        }
    }
}
template <int DT, int V>
__device__ __forceinline__ void rotary_store(char* p, int64_t at, const float (&v)[V]) {
    if constexpr (V == 1) {
        store1<DT>(p, at, v[0]);
    } else if constexpr (DT == RPFQ_F32) {
        *reinterpret_cast<f32x4*>(p + 4 * at) = (f32x4){v[0], v[1], v[2], v[3]};
    } else {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = DT == RPFQ_F16 ? cvt_pk(v[2 * t], v[2 * t + 1]) : pack_bf2(v[2 * t], v[2 * t + 1]);
        *reinterpret_cast<uint4*>(p + 2 * at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A workgroup takes `tokens` tokens: their cosines and sines go to LDS once, for
// all heads of both tensors.  The angle is formed in 64 bits and reduced to a
// part of a turn before it becomes float32, so a position of 2^31 is as exact as
// 1.  Then a thread takes V pairs at a time (V = 1: any strides and sizes).
template <int DT, int V>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
    extern __shared__ float2 turn[];  // [tokens][pairs]
    const rpfq_rotary_desc& d = a.d;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens, all = d.B * d.N;
    for (int i = threadIdx.x; i < a.tokens * a.pairs; i += 256) {
        const int tok = i / a.pairs, j = i - tok * a.pairs;
        const int64_t t = t0 + tok;
        if (t >= all) break;
        int axis = 0, end = d.sections[0];
        while (j >= end && axis < 3) end += d.sections[++axis];
        const int64_t b = t / d.N, at = b * d.pos_stride[0] + (t - b * d.N) * d.pos_stride[1] + axis;
        const double pos = d.pos_dtype == RPFQ_POS_I64   ? (double)reinterpret_cast<const int64_t*>(a.pos)[at]
                           : d.pos_dtype == RPFQ_POS_I32 ? (double)reinterpret_cast<const int32_t*>(a.pos)[at]
                                                         : (double)reinterpret_cast<const float*>(a.pos)[at];
        const double turns = pos * a.freqs[j] * 0.15915494309189533577;  // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c, d.inverse ? -s : s);
    }
    __syncthreads();
    const int heads = (int)(d.heads[0] + d.heads[1]);
    for (int i = threadIdx.x; i < a.total; i += 256) {
        const int row = i / a.units, u = i - row * a.units, tok = row / heads;
        int h = row - tok * heads;
        const int64_t t = t0 + tok;
        if (t >= all) break;
        const int which = h >= d.heads[0];
        if (which) h -= (int)d.heads[0];
        const int64_t b = t / d.N, n = t - b * d.N;
        const char* in = a.in[which];
        char* out = a.out[which];
        const int64_t from = b * d.in_stride[which][0] + n * d.in_stride[which][1] + h * d.in_stride[which][2];
        const int64_t to = b * d.out_stride[which][0] + n * d.out_stride[which][1] + h * d.out_stride[which][2];
        float x[V], y[V];
        if (u * V >= a.pairs) {  // values behind the pairs: as they are
            const int at = 2 * a.pairs + u * V - a.pairs;
            rotary_load<DT, V>(in, from + at, x);
            rotary_store<DT, V>(out, to + at, x);
            continue;
        }
        const float2* cs = turn + tok * a.pairs + u * V;
        const int first = d.interleaved ? 2 * u * V : u * V, second = d.interleaved ? first + V : a.pairs + u * V;
        rotary_load<DT, V>(in, from + first, x);
        rotary_load<DT, V>(in, from + second, y);
        float p[V], q[V];
        if (V > 1 && d.interleaved) {
#pragma unroll
            for (int t = 0; t < V / 2; ++t) {
                const float2 e = cs[t], f = cs[V / 2 + t];
                p[2 * t] = x[2 * t] * e.x - x[2 * t + 1] * e.y, p[2 * t + 1] = x[2 * t + 1] * e.x + x[2 * t] * e.y;
                q[2 * t] = y[2 * t] * f.x - y[2 * t + 1] * f.y, q[2 * t + 1] = y[2 * t + 1] * f.x + y[2 * t] * f.y;
            }
        } else {
#pragma unroll
            for (int t = 0; t < V; ++t) {
                const float2 e = cs[t];
                p[t] = x[t] * e.x - y[t] * e.y, q[t] = y[t] * e.x + x[t] * e.y;
            }
        }
        rotary_store<DT, V>(out, to + first, p);
        rotary_store<DT, V>(out, to + second, q);
    }
}

template <int DT>
static hipError_t rotary_go(RotaryArgs& a, bool vec, hipStream_t s) {
    const int v = vec ? rotary_vec<DT>() : 1;
    const int64_t all = a.d.B * a.d.N;
    a.units = a.pairs / v + (int)(a.d.D - 2 * a.pairs) / v;
    // tokens of a workgroup: an angle a thread, but fewer where the chip would not
    // be filled (2 workgroups a CU)
    const int64_t fill = all / (2 * device_cus()), most = 256 / a.pairs;
    a.tokens = (int)(most < fill ? most : fill);
    if (a.tokens < 1) a.tokens = 1;
    a.total = a.tokens * (int)(a.d.heads[0] + a.d.heads[1]) * a.units;
    const dim3 grid((unsigned)((all + a.tokens - 1) / a.tokens));
    const size_t lds = (size_t)a.tokens * a.pairs * sizeof(float2);
    if (vec) hipLaunchKernelGGL((rotary_kernel<DT, rotary_vec<DT>()>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((rotary_kernel<DT, 1>), grid, dim3(256), lds, s, a);
    return hipGetLastError();
}

hipError_t launch_rotary(const rpfq_rotary_desc& d, const void* q, const void* k, void* q_out, void* k_out, const void* pos,
                         const double* freqs, hipStream_t s) {
    RotaryArgs a = {};
    a.d = d;
    a.in[0] = reinterpret_cast<const char*>(q), a.in[1] = reinterpret_cast<const char*>(k);
    a.out[0] = reinterpret_cast<char*>(q_out), a.out[1] = reinterpret_cast<char*>(k_out);
    a.pos = pos;
    a.freqs = freqs;
    for (int i = 0; i < d.axes; ++i) a.pairs += d.sections[i];
    for (int i = d.axes; i < 4; ++i) a.d.sections[i] = 0;
    const int v = d.dtype == RPFQ_F32 ? 4 : 8;
    int64_t odd = a.pairs | d.D;  // whether any offset is no multiple of v
    uintptr_t at = 0;
    for (int i = 0; i < (d.heads[1] ? 2 : 1); ++i) {
        for (int j = 0; j < 3; ++j) odd |= d.in_stride[i][j] | d.out_stride[i][j];
        at |= reinterpret_cast<uintptr_t>(a.in[i]) | reinterpret_cast<uintptr_t>(a.out[i]);
    }
    const bool vec = odd % v == 0 && at % 16 == 0;
    switch (d.dtype) {
        case RPFQ_F32: return rotary_go<RPFQ_F32>(a, vec, s);
        case RPFQ_F16: return rotary_go<RPFQ_F16>(a, vec, s);
        default: return rotary_go<RPFQ_BF16>(a, vec, s);
    }
}

}  // namespace rpfq
