// Root-mean-square norm of rows with the residual's addition in front of it,
//   h = x + residual (rounded to x's type),  r = 1 / sqrt(mean h^2 + eps),
//   y = h r w,
// its output in x's type or as 8-bit codes with a scale per row, and its
// gradient.
#include "rpfq_device.h"

namespace rpfq {

// 8 elements of a row from column c on (zeros past C), as they lie.  Rows may
// begin at any element: gfx950 loads 16 unaligned bytes with one instruction.
template <int DT>
struct Norm8 {
    uint32_t w[DT == RPFQ_F32 ? 8 : 4];
    __device__ __forceinline__ void load(const void* p, int64_t row, int c, int C) {
        constexpr int ES = DT == RPFQ_F32 ? 4 : 2;
        const char* src = reinterpret_cast<const char*>(p) + (row + c) * ES;
        if (c + 8 <= C) {
            __builtin_memcpy(w, src, 8 * ES);
            return;
        }
#pragma unroll
        for (int t = 0; t < (int)(sizeof(w) / 4); ++t) w[t] = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t)
            if (c + t < C) {
                if (DT == RPFQ_F32) w[t % (sizeof(w) / 4)] = reinterpret_cast<const uint32_t*>(src)[t];
                else w[t / 2 % (sizeof(w) / 4)] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[t] << (16 * (t & 1));
            }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            if (DT == RPFQ_F32) v[t] = __uint_as_float(w[t % (sizeof(w) / 4)]);
            else if (DT == RPFQ_F16) v[t] = (float)__builtin_bit_cast(half2v, w[t / 2 % (sizeof(w) / 4)])[t & 1];
            else v[t] = bf16_to_f32(t & 1 ? w[t / 2 % (sizeof(w) / 4)] >> 16 : w[t / 2 % (sizeof(w) / 4)] & 0xffffu);
        }
    }
};
template <int DT>
__device__ __forceinline__ void norm_load8(const void* p, int64_t row, int c, int C, float (&v)[8]) {
    Norm8<DT> r;
    r.load(p, row, c, C);
    r.values(v);
}
template <int DT>
__device__ __forceinline__ uint32_t norm_pack2(float a, float b) {
    return DT == RPFQ_F16 ? cvt_pk(a, b) : pack_bf2(a, b);
}
template <int DT>
__device__ __forceinline__ void norm_store8(void* p, int64_t row, int c, int C, const float (&v)[8]) {
    if (c + 8 <= C) {
        if constexpr (DT == RPFQ_F32) {
            __builtin_memcpy(reinterpret_cast<float*>(p) + row + c, v, 32);
        } else {
            const uint32_t w[4] = {norm_pack2<DT>(v[0], v[1]), norm_pack2<DT>(v[2], v[3]), norm_pack2<DT>(v[4], v[5]),
                                   norm_pack2<DT>(v[6], v[7])};
            __builtin_memcpy(reinterpret_cast<uint16_t*>(p) + row + c, w, 16);
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
        if (c + t < C) store1<DT>(p, row + c + t, v[t]);
}
__device__ __forceinline__ void norm_weight8(const void* w, int wdt, int c, int C, float (&v)[8]) {
    if (!w) {
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = 1.0f;
    } else if (wdt == RPFQ_F32) {
        norm_load8<RPFQ_F32>(w, 0, c, C, v);
    } else if (wdt == RPFQ_F16) {
        norm_load8<RPFQ_F16>(w, 0, c, C, v);
    } else {
        norm_load8<RPFQ_BF16>(w, 0, c, C, v);
    }
}
// v as x's type holds it
template <int DT>
__device__ __forceinline__ float norm_round(float v) {
    if (DT == RPFQ_F16) return (float)(_Float16)v;
    if (DT == RPFQ_BF16) return bf16_to_f32(f32_to_bf16(v));
    return v;
}

// op over the 64 lanes, in all of them: within 16 lanes by DPP, across them by
// lane swaps.  No LDS: six shuffles wait for it six times, the row's three
// reductions took a third of the 8-bit norm.
template <int CTRL>
__device__ __forceinline__ uint32_t norm_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <class V, class Op>
__device__ __forceinline__ V wave_all(V v, Op op) {
    static_assert(sizeof(V) == 4, "one register");
    v = op(v, __builtin_bit_cast(V, norm_dpp<0xb1>(__builtin_bit_cast(uint32_t, v))));   // lane ^ 1
    v = op(v, __builtin_bit_cast(V, norm_dpp<0x4e>(__builtin_bit_cast(uint32_t, v))));   // lane ^ 2
    v = op(v, __builtin_bit_cast(V, norm_dpp<0x141>(__builtin_bit_cast(uint32_t, v))));  // 7 - lane of 8
    v = op(v, __builtin_bit_cast(V, norm_dpp<0x140>(__builtin_bit_cast(uint32_t, v))));  // 15 - lane of 16
    const uint32_t a = __builtin_bit_cast(uint32_t, v);
    const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = op(__builtin_bit_cast(V, (uint32_t)x[0]), __builtin_bit_cast(V, (uint32_t)x[1]));
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return op(__builtin_bit_cast(V, (uint32_t)y[0]), __builtin_bit_cast(V, (uint32_t)y[1]));
}
template <class Op>
__device__ __forceinline__ double wave_all(double v, Op op) {  // rare
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    return v;
}
// Sum or maximum over the T threads of a row: a wave, or the workgroup of four
// through `sm` (a barrier on both sides; every thread of it calls).
template <int T, class V, class Op>
__device__ __forceinline__ V row_reduce(V v, V* sm, Op op) {
    v = wave_all(v, op);
    if constexpr (T > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
        __syncthreads();
        v = op(op(sm[0], sm[1]), op(sm[2], sm[3]));
    }
    return v;
}
struct Plus {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Most {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};

struct NormArgs {
    const void *x, *res, *w;
    int wdt, C;
    int64_t M;
    float eps;
    void *y, *h;
    float* rstd;
    int8_t* codes;
    float* scale;
};

// 1 / sqrt(mean h^2 + eps).  The squares' sum is float32; where it leaves the
// range that float32 keeps (elements past 2^60 or below 2^-50) it is summed
// again in 64 bits.
template <int T, int NC>
__device__ __forceinline__ float norm_rstd(const float (&h)[NC][8], int C, float eps, double* sm) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int t = 0; t < 8; ++t) s = fmaf(h[i][t], h[i][t], s);
    s = row_reduce<T>(s, reinterpret_cast<float*>(sm), Plus());
    if (s >= 0x1p-100f && s <= 0x1p120f) return 1.0f / sqrtf(s / (float)C + eps);
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int t = 0; t < 8; ++t) d = fma((double)h[i][t], (double)h[i][t], d);
    d = row_reduce<T>(d, sm, Plus());
    return (float)(1.0 / sqrt(d / C + (double)eps));
}

// Codes of a row, rint(127 p / max|p|) of p = h w: 1 / rms cancels, so they are
// decided by the stored h and w alone, ties to even.  float32's own quotient is
// within 2e-5; where it is within 1e-4 of the middle of two codes, 254 |p| is
// compared with (2 c + 1) max|p| exactly: 64 bits hold the products (48 of their
// 53 bits), not always their multiples, so the difference is formed by fma, with
// what (2 c + 1) max|p| was rounded by.  The largest product is taken among those
// that float32 rounds to within 2^-22 of the largest.
template <int T, int NC>
__device__ __forceinline__ void norm_codes(const NormArgs& a, const float (&h)[NC][8], const float (&w)[NC][8], float rstd, int64_t m, int col, double* sm) {
    // a power of two near 1 / rms, exact on h: products stay in float32's range
    int e = 1 - __builtin_amdgcn_frexp_expf(rstd);
    e = e < -126 ? -126 : e > 126 ? 126 : e;
    const float lift = __builtin_amdgcn_ldexpf(1.0f, -e), back = __builtin_amdgcn_ldexpf(rstd, e);
    uint32_t mx = 0;
    float p[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            p[i][t] = h[i][t] * lift * w[i][t];  // 0 past C, as h is
            mx = max(mx, __float_as_uint(p[i][t]) & 0x7fffffffu);
        }
    }
    mx = row_reduce<T>(mx, reinterpret_cast<uint32_t*>(sm), Most());
    const bool fin = mx < 0x7f800000u, ok = fin && mx >= 0x00800000u;
    const float top = __uint_as_float(mx), r = ok ? 127.0f / top : 0.0f;
    auto exact = [&](int i, int t) { return (double)(fabsf(h[i][t]) * lift) * (double)fabsf(w[i][t]); };
    double topd = 0.0;
    if (ok) {
        const float near = top * (1.0f - 0x1p-22f);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float most = 0.0f;  // one branch for 8: of a row one lane or two take it
#pragma unroll
            for (int t = 0; t < 8; ++t) most = fmaxf(most, fabsf(p[i][t]));
            if (most < near) continue;
            asm volatile("");  // the 64-bit products are not formed ahead of the branch
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (fabsf(p[i][t]) >= near) topd = fmax(topd, exact(i, t));
        }
    }
    // of a wave's row mostly one lane has candidates
    const uint64_t who = __ballot(topd > 0.0);
    if (T == 64 && (who & (who - 1)) == 0) {
        const int lane = who ? __builtin_ctzll(who) : 0;
        const uint64_t bits = __builtin_bit_cast(uint64_t, topd);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), lane);
        topd = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    } else {
        topd = row_reduce<T>(topd, sm, Most());
    }
    if ((threadIdx.x & (T - 1)) == 0) a.scale[m] = fin ? (float)(topd / 127.0 * (double)back) : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c0 = col + 8 * T * i;
        if (c0 >= a.C) continue;
        // float32 holds whole numbers around 1.5 2^23: the sum rounds to one, its
        // low byte is the code
        constexpr float WHOLE = 0x1.8p23f;
        uint32_t out[2];
        float code[8], off = 0.0f;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            code[t] = fmaf(p[i][t], r, WHOLE);
            off = fmaxf(off, fabsf(fmaf(p[i][t], r, -(code[t] - WHOLE))));
        }
        if (off > 0.5f - 1e-4f) {  // in the middle of two codes: of 8 values one in 600
            asm volatile("");
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float q = fabsf(p[i][t]) * r;
                float c = __builtin_rintf(q);
                if (fabsf(fabsf(q - c) - 0.5f) < 1e-4f) {
                    c = floorf(q);
                    const double odd = 2.0 * (double)c + 1.0, mid = odd * topd;
                    const double past = fma(254.0, exact(i, t), -mid), rest = fma(odd, topd, -mid);
                    if (past > rest || (past == rest && ((int)c & 1))) c += 1.0f;
                }
                code[t] = copysignf(c, p[i][t]) + WHOLE;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(code[4 * e + 1]), __float_as_uint(code[4 * e]), 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(code[4 * e + 3]), __float_as_uint(code[4 * e + 2]), 0x04000c0cu);
            out[e] = fin ? lo | hi : 0u;
        }
        int8_t* dst = a.codes + m * a.C + c0;
        if (c0 + 8 <= a.C) {
            __builtin_memcpy(dst, out, 8);
        } else {
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (c0 + t < a.C) dst[t] = (int8_t)(out[t >> 2] >> (8 * (t & 3)));
        }
    }
}

// A row in the registers of T threads (a wave, or a workgroup of four), 8 NC
// values each: read once, written once.  A workgroup stays for many rows, with
// the weights in registers.  Bound by HBM: 50,432 rows of 768 bf16 to codes 60 us
// (271 MB, 4.5 TB/s; a workgroup a row group 72, with the next row loaded ahead,
// at half the waves, 79), 16,384 of 4,096 to bf16 88 us (537 MB, 6.1 TB/s).
template <int DT, int T, int NC, bool CODES>
__global__ void __launch_bounds__(256) rms_norm_kernel(NormArgs a) {
    __shared__ double sm[4];
    const int col = 8 * (threadIdx.x & (T - 1));
    constexpr int ROWS = 256 / T;
    float w[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) norm_weight8(a.w, a.wdt, col + 8 * T * i, a.C, w[i]);
    for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / T; m < a.M; m += (int64_t)gridDim.x * ROWS) {
        const int64_t row = m * a.C;
        Norm8<DT> x[NC], r[NC];
        float h[NC][8];
#pragma unroll
        for (int i = 0; i < NC; ++i) x[i].load(a.x, row, col + 8 * T * i, a.C);
        if (a.res)
#pragma unroll
            for (int i = 0; i < NC; ++i) r[i].load(a.res, row, col + 8 * T * i, a.C);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            x[i].values(h[i]);
            if (!a.res) continue;
            float v[8];
            r[i].values(v);
#pragma unroll
            for (int t = 0; t < 8; ++t) h[i][t] = norm_round<DT>(h[i][t] + v[t]);
            if (col + 8 * T * i < a.C) norm_store8<DT>(a.h, row, col + 8 * T * i, a.C, h[i]);
        }
        const float rstd = norm_rstd<T, NC>(h, a.C, a.eps, sm);
        if constexpr (CODES) {
            norm_codes<T, NC>(a, h, w, rstd, m, col, sm);
        } else {
            if (a.rstd && (threadIdx.x & (T - 1)) == 0) a.rstd[m] = rstd;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int c = col + 8 * T * i;
                if (c >= a.C) continue;
                float y[8];
#pragma unroll
                for (int t = 0; t < 8; ++t) y[t] = w[i][t] * (h[i][t] * rstd);
                norm_store8<DT>(a.y, row, c, a.C, y);
            }
        }
    }
}

// With n = h r and g = gy w:  gx = r (g - n mean(g n)) + gh,  gw = sum_rows gy n.
struct NormGradArgs {
    const void *gy, *gh, *h, *w;
    int wdt, C;
    int64_t M;
    const float* rstd;
    void* gx;
    float* part;  // [gridDim.x][C] sums of gy n, or NULL
};

template <int DT, int T, int NC>
__global__ void __launch_bounds__(256) rms_norm_grad_kernel(NormGradArgs a) {
    __shared__ float sm[4];
    const int col = 8 * (threadIdx.x & (T - 1));
    constexpr int ROWS = 256 / T;
    float gw[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int t = 0; t < 8; ++t) gw[i][t] = 0.0f;
    float w[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) norm_weight8(a.w, a.wdt, col + 8 * T * i, a.C, w[i]);
    for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / T; m < a.M; m += (int64_t)gridDim.x * ROWS) {
        const int64_t row = m * a.C;
        Norm8<DT> hr[NC], gr[NC], sum[NC];
        float n[NC][8], g[NC][8];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            hr[i].load(a.h, row, col + 8 * T * i, a.C);
            gr[i].load(a.gy, row, col + 8 * T * i, a.C);
        }
        if (a.gh)
#pragma unroll
            for (int i = 0; i < NC; ++i) sum[i].load(a.gh, row, col + 8 * T * i, a.C);
        const float r = a.rstd[m];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            hr[i].values(n[i]);
            gr[i].values(g[i]);
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                n[i][t] *= r;
                gw[i][t] = fmaf(g[i][t], n[i][t], gw[i][t]);
                g[i][t] *= w[i][t];
                s = fmaf(g[i][t], n[i][t], s);
            }
        }
        const float mean = row_reduce<T>(s, sm, Plus()) / (float)a.C;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = col + 8 * T * i;
            if (c >= a.C) continue;
            float gh[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (a.gh) sum[i].values(gh);
#pragma unroll
            for (int t = 0; t < 8; ++t) gh[t] = fmaf(r, g[i][t] - n[i][t] * mean, gh[t]);
            norm_store8<DT>(a.gx, row, c, a.C, gh);
        }
    }
    if (!a.part) return;
    if constexpr (T == 64) {  // the four waves' sums, in their order
        __shared__ float acc[512 * NC];
        const int wave = threadIdx.x >> 6;
        for (int w = 0; w < 4; ++w) {
            __syncthreads();
            if (wave == w)
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        float* at = acc + col + 512 * i + t;
                        *at = w ? *at + gw[i][t] : gw[i][t];
                    }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += 256) a.part[(int64_t)blockIdx.x * a.C + c] = acc[c];
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (col + 8 * T * i + t < a.C) a.part[(int64_t)blockIdx.x * a.C + col + 8 * T * i + t] = gw[i][t];
    }
}

// gw = the column sums of [parts][C]: 64 columns a workgroup, its 16 waves every
// 16th part, added up in their order.
template <int WDT>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const float* part, int parts, int C, void* gw) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < C)
#pragma unroll 8
        for (int p = wave; p < parts; p += 16) s += part[(int64_t)p * C + c];
    sm[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < C) {
#pragma unroll
        for (int w = 1; w < 16; ++w) s += sm[w][lane];
        store1<WDT>(gw, c, s);
    }
}

// Threads of a row and values of each: a wave for up to 2,048 values, a
// workgroup for up to kNormMaxC.
template <int DT, class Go>
static hipError_t norm_form(int64_t C, Go go) {
    if (C <= 512) return go.template run<DT, 64, 1>();
    if (C <= 1024) return go.template run<DT, 64, 2>();
    if (C <= 2048) return go.template run<DT, 64, 4>();
    if (C <= 4096) return go.template run<DT, 256, 2>();
    if (C <= 8192) return go.template run<DT, 256, 4>();
    return go.template run<DT, 256, 8>();
}
template <class Go>
static hipError_t norm_dispatch(int dt, int64_t C, Go go) {
    switch (dt) {
        case RPFQ_F32: return norm_form<RPFQ_F32>(C, go);
        case RPFQ_F16: return norm_form<RPFQ_F16>(C, go);
        default: return norm_form<RPFQ_BF16>(C, go);
    }
}

struct NormGo {
    const NormArgs& a;
    hipStream_t s;
    template <int DT, int T, int NC>
    hipError_t run() {
        const int64_t blocks = (a.M + 256 / T - 1) / (256 / T);
        const int64_t most = 8 * device_cus();
        const dim3 grid((unsigned)(blocks < most ? blocks : most));
        if (a.codes) hipLaunchKernelGGL((rms_norm_kernel<DT, T, NC, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rms_norm_kernel<DT, T, NC, false>), grid, dim3(256), 0, s, a);
        return hipGetLastError();
    }
};
hipError_t launch_rms_norm(const NormCall& c, void* y, void* h, float* rstd, int8_t* codes, float* scale, hipStream_t s) {
    const NormArgs a = {c.x, c.residual, c.weight, c.weight_dtype, (int)c.C, c.M, c.eps, y, h, rstd, codes, scale};
    return norm_dispatch(c.dtype, c.C, NormGo{a, s});
}

// Workgroups of the gradient: each leaves a row of partial sums.  Four a CU: with
// two, too few loads are on their way (16,384 x 4,096 bf16, 537 MB: 165 us, with
// four 115, 4.7 TB/s).
int norm_grad_parts(int64_t M, int64_t C) {
    const int64_t rows = C <= 2048 ? 4 : 1, blocks = (M + rows - 1) / rows, most = 4 * device_cus();
    return (int)(blocks < most ? blocks : most);
}
struct NormGradGo {
    const NormGradArgs& a;
    int parts;
    hipStream_t s;
    template <int DT, int T, int NC>
    hipError_t run() {
        hipLaunchKernelGGL((rms_norm_grad_kernel<DT, T, NC>), dim3(parts), dim3(256), 0, s, a);
        return hipGetLastError();
    }
};
hipError_t launch_rms_norm_grad(const NormCall& c, const void* gy, const void* gh, const float* rstd, void* gx, void* gw,
                                void* work, hipStream_t s) {
    const int parts = norm_grad_parts(c.M, c.C);
    float* part = gw ? reinterpret_cast<float*>(work) : nullptr;
    const NormGradArgs a = {gy, gh, c.x, c.weight, c.weight_dtype, (int)c.C, c.M, rstd, gx, part};
    const hipError_t e = norm_dispatch(c.dtype, c.C, NormGradGo{a, parts, s});
    if (e != hipSuccess || !gw) return e;
    const dim3 grid((unsigned)((c.C + 63) / 64));
    switch (c.weight_dtype) {
        case RPFQ_F32: hipLaunchKernelGGL((norm_columns_kernel<RPFQ_F32>), grid, dim3(1024), 0, s, part, parts, (int)c.C, gw); break;
        case RPFQ_F16: hipLaunchKernelGGL((norm_columns_kernel<RPFQ_F16>), grid, dim3(1024), 0, s, part, parts, (int)c.C, gw); break;
        default: hipLaunchKernelGGL((norm_columns_kernel<RPFQ_BF16>), grid, dim3(1024), 0, s, part, parts, (int)c.C, gw);
    }
    return hipGetLastError();
}

}  // namespace rpfq
