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
    int pairs, tokens;  // pairs of a head, tokens of a workgroup
    int turned, units;  // units of V values, or of V pairs, that turn; of a head (the rest are copied)
    int total;          // units of all its tokens
    int rest;           // values of a unit that is copied: V, or 1
    int64_t first;      // the launch's first token
};

// V consecutive values as float32, from any element on: gfx950 loads 16 unaligned
// bytes with one instruction.
template <int DT, int V>
__device__ __forceinline__ void rotary_load(const char* p, int64_t at, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = load_y1<DT>(p, at);
    } else if constexpr (DT == RPFQ_F32) {
        __builtin_memcpy(v, p + 4 * at, 4 * V);
    } else {
        uint32_t w[V / 2];
        __builtin_memcpy(w, p + 2 * at, 2 * V);
#pragma unroll
        for (int t = 0; t < V / 2; ++t) {
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
        __builtin_memcpy(p + 4 * at, v, 4 * V);
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int t = 0; t < V / 2; ++t) w[t] = DT == RPFQ_F16 ? cvt_pk(v[2 * t], v[2 * t + 1]) : pack_bf2(v[2 * t], v[2 * t + 1]);
        __builtin_memcpy(p + 2 * at, w, 2 * V);
    }
}

// A workgroup takes `tokens` tokens: their cosines and sines go to LDS once, for
// all heads of both tensors.  The angle is formed in 64 bits and reduced to a
// part of a turn before it becomes float32, so a position of 2^31 is as exact as
// 1.  Then a thread takes V pairs at a time, or V values of neighbours.
// Bound by HBM: 32,768 tokens x 20 heads x 128 bf16 60 us (336 MB, 5.5 TB/s).
template <int DT, int V>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
    extern __shared__ float2 turn[];  // [tokens][pairs]
    const rpfq_rotary_desc& d = a.d;
    const int64_t t0 = a.first + (int64_t)blockIdx.x * a.tokens, all = d.B * d.N;
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
        if (u >= a.turned) {  // values behind the pairs: as they are
            const int at = 2 * a.pairs + (u - a.turned) * a.rest;
            if (a.rest == V) {
                rotary_load<DT, V>(in, from + at, x);
                rotary_store<DT, V>(out, to + at, x);
            } else {
                float one[1];
                rotary_load<DT, 1>(in, from + at, one);
                rotary_store<DT, 1>(out, to + at, one);
            }
            continue;
        }
        if (V > 1 && d.interleaved) {
            const float2* cs = turn + tok * a.pairs + u * (V / 2);
            rotary_load<DT, V>(in, from + u * V, x);
#pragma unroll
            for (int t = 0; t < V / 2; ++t) {
                const float2 e = cs[t];
                y[2 * t] = x[2 * t] * e.x - x[2 * t + 1] * e.y, y[2 * t + 1] = x[2 * t + 1] * e.x + x[2 * t] * e.y;
            }
            rotary_store<DT, V>(out, to + u * V, y);
            continue;
        }
        const float2* cs = turn + tok * a.pairs + u * V;
        const int first = u * V, second = a.pairs + u * V;
        rotary_load<DT, V>(in, from + first, x);
        rotary_load<DT, V>(in, from + second, y);
        float p[V], q[V];
#pragma unroll
        for (int t = 0; t < V; ++t) {
            const float2 e = cs[t];
            p[t] = x[t] * e.x - y[t] * e.y, q[t] = y[t] * e.x + x[t] * e.y;
        }
        rotary_store<DT, V>(out, to + first, p);
        rotary_store<DT, V>(out, to + second, q);
    }
}

// V of a call: 16 bytes, or fewer where the pairs are no multiple (26 pairs of
// neighbours in float32, 1,568 x 2 tokens of 32 heads: 43 us a value at a time, so 21).
template <int DT, int V>
static hipError_t rotary_go(RotaryArgs& a, hipStream_t s) {
    if constexpr (V > 1) {
        if ((a.d.interleaved ? 2 * a.pairs : a.pairs) % V) return rotary_go<DT, V / 2>(a, s);
    }
    const int64_t all = a.d.B * a.d.N;
    const int behind = (int)a.d.D - 2 * a.pairs;
    a.rest = behind % V ? 1 : V;
    a.turned = V > 1 && a.d.interleaved ? 2 * a.pairs / V : a.pairs / V;
    a.units = a.turned + behind / a.rest;
    // tokens of a workgroup: an angle a thread, but fewer where the chip would not
    // be filled (2 workgroups a CU)
    const int64_t fill = all / (2 * device_cus()), most = 256 / a.pairs;
    a.tokens = (int)(most < fill ? most : fill);
    if (a.tokens < 1) a.tokens = 1;
    a.total = a.tokens * (int)(a.d.heads[0] + a.d.heads[1]) * a.units;
    // a grid has fewer than 2^32 threads: 2^23 workgroups of 256 a launch
    const int64_t most_blocks = 1 << 23;
    for (a.first = 0; a.first < all; a.first += most_blocks * a.tokens) {
        const int64_t blocks = (all - a.first + a.tokens - 1) / a.tokens;
        const dim3 grid((unsigned)(blocks < most_blocks ? blocks : most_blocks));
        hipLaunchKernelGGL((rotary_kernel<DT, V>), grid, dim3(256), (size_t)a.tokens * a.pairs * sizeof(float2), s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
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
    switch (d.dtype) {
        case RPFQ_F32: return rotary_go<RPFQ_F32, 4>(a, s);
        case RPFQ_F16: return rotary_go<RPFQ_F16, 8>(a, s);
        default: return rotary_go<RPFQ_BF16, 8>(a, s);
    }
}

}  // namespace rpfq
