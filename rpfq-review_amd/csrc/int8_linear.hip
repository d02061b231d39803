// 8-bit integer layer: y[m, n] = (sum_k cx[m, k] cw[n, k]) sx[m] sw[n] + b[n],
// cx = rint(127 x / max|x_m|) with sx = max|x_m| / 127 for each token, cw and sw
// the same of each output channel of the weight, sums exact in int32.
#include "tile_gemm.h"

namespace rpfq {

// ---------------------------------------------------------------------------
// codes and scales of rows
// ---------------------------------------------------------------------------
// rint(127 x / top), ties to even, exactly: float32's own product is within
// 2e-5 of the quotient, so where it is within 1e-4 of the middle of two codes
// the quotient is compared with that middle in 64 bits, 254 |x| against
// (2 c + 1) top, both exact there.  16-bit rows meet such ties in earnest (x =
// top / 2 is 63.5).
__device__ __forceinline__ int int8_code(float x, float top, float r) {
    const float t = fabsf(x) * r;
    float c = __builtin_rintf(t);
    if (fabsf(fabsf(t - c) - 0.5f) < 1e-4f) {
        c = floorf(t);
        const double a = 254.0 * (double)fabsf(x), mid = (2.0 * (double)c + 1.0) * (double)top;
        if (a > mid || (a == mid && ((int)c & 1))) c += 1.0f;
    }
    return (int)copysignf(c, x);
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
    if (DT == RPFQ_F32) return reinterpret_cast<const float*>(p)[i];
    if (DT == RPFQ_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == RPFQ_F32) {
        const f32x4* q = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i);
        const f32x4 a = q[0], b = q[1];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = a[t], v[4 + t] = b[t];
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
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

// The same at any alignment of the elements.
template <int DT>
__device__ __forceinline__ void load8_any(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == RPFQ_F32) {
        __builtin_memcpy(v, reinterpret_cast<const float*>(p) + i, 32);
    } else {
        uint4 u;
        __builtin_memcpy(&u, reinterpret_cast<const uint16_t*>(p) + i, 16);
        load8<DT>(&u, 0, v);
    }
}

// What a row's largest magnitude (its bits: NaN above inf above numbers)
// makes of it: the scale to store, and (top, r) for int8_code, both times a
// power of two where 127 / top would overflow.  inf or NaN: scale NaN.
struct Int8Row {
    float scale, top, r, lift;
    __device__ __forceinline__ explicit Int8Row(uint32_t bits) {
        const float mx = __uint_as_float(bits);
        const bool fin = bits < 0x7f800000u, ok = fin && mx > 0.0f;
        scale = fin ? mx / 127.0f : __uint_as_float(0x7fc00000u);
        lift = ok && mx < 0x1p-60f ? 0x1p80f : 1.0f;
        top = ok ? mx * lift : 1.0f;
        r = ok ? 127.0f / top : 0.0f;
    }
    __device__ __forceinline__ int code(float x) const { return r > 0.0f ? int8_code(x * lift, top, r) : 0; }
};

// Waves of a row each, the row in registers: K <= 512 NC, 16-byte aligned rows.
// Codes past K (up to ldq) are zero.  HBM bound: x once, a byte a value out
// (50,432 x 1,024 fp16: 37 us, 4.2 TB/s; 1,576 x 768 bf16: 4 to 5 us, a launch and a
// read's latency).
template <int DT, int NC>
__global__ void __launch_bounds__(256) int8_rows_kernel(const void* x, int64_t M, int K, int8_t* q, int64_t ldq,
                                                       float* scale) {
    const int lane = threadIdx.x & 63;
    for (int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); m < M; m += (int64_t)gridDim.x * 4) {
        float v[NC][8];
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = 8 * (lane + 64 * i);
            if (c < K) {
                load8<DT>(x, m * K + c, v[i]);
            } else {
#pragma unroll
                for (int t = 0; t < 8; ++t) v[i][t] = 0.0f;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) mx = max(mx, __float_as_uint(v[i][t]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
        const Int8Row row(mx);
        if (lane == 0) scale[m] = row.scale;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = 8 * (lane + 64 * i);
            if (c >= ldq) continue;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int t = 0; t < 8; ++t) w[t >> 2] |= (uint32_t)(row.code(v[i][t]) & 0xff) << (8 * (t & 3));
            *reinterpret_cast<uint2*>(q + m * ldq + c) = make_uint2(w[0], w[1]);
        }
    }
}

// codes [rows, K] of any K and alignment -> rows of ldq bytes, zeros past K: a
// wave a row, 16 bytes a lane.
struct Int8Pad {
    const int8_t* src;
    int64_t ld, K;
    int8_t* dst;
    int64_t ldq, rows;
    unsigned blocks;
};
__device__ __forceinline__ void int8_pad(const Int8Pad& a, unsigned block) {
    const int lane = threadIdx.x & 63;
    for (int64_t n = (int64_t)block * 4 + (threadIdx.x >> 6); n < a.rows; n += (int64_t)a.blocks * 4)
        for (int64_t k = 16 * lane; k < a.ldq; k += 1024) {
            const int8_t* src = a.src + n * a.ld + k;
            int8_t e[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            if (k + 16 <= a.K) {
                __builtin_memcpy(e, src, 16);
            } else {
#pragma unroll
                for (int t = 0; t < 16; ++t)
                    if (k + t < a.K) e[t] = src[t];
            }
            __builtin_memcpy(a.dst + n * a.ldq + k, e, 16);
        }
}
__global__ void __launch_bounds__(256) int8_pad_kernel(Int8Pad a) { int8_pad(a, blockIdx.x); }

// Any K and alignment: one workgroup a row, read twice (the second time from
// L2).  The workgroups past `blocks` copy a weight whose rows do not lie as the
// product reads them, in the same launch (777 and 333 rows of 515: 3.9 us, 6.6
// in two).
template <int DT>
__global__ void __launch_bounds__(256) int8_rows_any_kernel(const void* x, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                                                           float* scale, unsigned blocks, Int8Pad pad) {
    __shared__ uint32_t sm[4];
    if (blockIdx.x >= blocks) {
        int8_pad(pad, blockIdx.x - blocks);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t m = blockIdx.x; m < M; m += blocks) {
        uint32_t mx = 0;
        for (int64_t k = threadIdx.x; k < K; k += 256) mx = max(mx, __float_as_uint(load1<DT>(x, m * K + k)) & 0x7fffffffu);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
        if (lane == 0) sm[wave] = mx;
        __syncthreads();
        const Int8Row row(max(max(sm[0], sm[1]), max(sm[2], sm[3])));
        if (threadIdx.x == 0) scale[m] = row.scale;
        for (int64_t k = threadIdx.x; k < ldq; k += 256)
            q[m * ldq + k] = (int8_t)(k < K ? row.code(load1<DT>(x, m * K + k)) : 0);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
struct Int8Args {
    TileOperand x, w;
    const float *sx, *sw, *bias;
    void* y;
    int64_t M, N, K;  // K bytes of a code row
    int tiles_m, tiles_n, group, vec;
};

// Bound by the matrix cores' step (tile_gemm.h) and, for a wide output of a small
// K, by its stores: 50,432 x 1,024 -> 4,096 fp16, 260 to 310 us, 1.4 to 1.6 POP/s and
// 413 MB of y, which alone are 90 us at a copy's rate and hide behind nothing
// in their own workgroup.  Workgroups that walk several tiles and load the next
// one's first step during the stores measured the same (249 us against 253).
// 1,576 x 768 -> 2,304 bf16 9.5 us.
template <class G>
constexpr int kInt8Lds = G::LDS + 768 * 4;

template <int MB, int WM, int S, int KB, int YDT>
__global__ void __launch_bounds__(256 * WM, 2) int8_gemm_kernel(Int8Args a) {
    extern __shared__ __align__(16) char smem[];
    using G = TileGemm<MB, WM, S, KB, false, false, MmaI8>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int mt, nt;
    group_tile(xcd_tile(blockIdx.x, a.tiles_m * a.tiles_n), a.tiles_m, a.tiles_n, a.group, mt, nt);
    const int64_t m0 = (int64_t)mt * G::ROWS + 32 * MB * (wave >> 2), n0 = (int64_t)nt * 256, nw = n0 + 64 * (wave & 3);
    intx16 acc[2][MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[0][i] = acc[1][i] = intx16{0};
    const int steps = (int)G::steps(a.K);
    // scales and biases of the tile's columns and scales of its rows
    float* col = reinterpret_cast<float*>(smem + G::LDS);
    G::run(a.x, a.w, (int64_t)mt * G::ROWS, n0, a.K, a.K, steps, 1, 0, steps, smem, wave, lane, acc, [&] {
        for (int c = threadIdx.x; c < 256; c += G::THREADS) {
            const int64_t n = n0 + c;
            col[c] = n < a.N ? a.sw[n] : 0.0f;
            col[256 + c] = n < a.N && a.bias ? a.bias[n] : 0.0f;
            const int64_t m = (int64_t)mt * G::ROWS + c;
            if (c < G::ROWS) col[512 + c] = m < a.M ? a.sx[m] : 0.0f;
        }
    });
    const float* sxs = col + 512 + 32 * MB * (wave >> 2) + (lane & 31);
    char* epi = smem + wave * kTileEpi;
    if constexpr (YDT == RPFQ_F32) {
        const int64_t n = nw + 4 * (lane & 15);
        const float* mine = col + 64 * (wave & 3) + 4 * (lane & 15);
        const f32x4 sw = *reinterpret_cast<const f32x4*>(mine), b = *reinterpret_cast<const f32x4*>(mine + 256);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const float sx = sxs[32 * i];
            tile_rows(epi, acc[0][i], acc[1][i], lane, [&](int v, int) { return (float)v * sx; },
                      [&](int row, int, f32x4 v) {
                          const int64_t m = m0 + 32 * i + row;
                          if (m < a.M) tile_store4<YDT>(a.y, m * a.N, n, a.N, a.vec, v * sw + b);
                      });
        }
    } else {
        const float* mine = col + 64 * (wave & 3) + 4 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const float sx = sxs[32 * i];
            tile_rows_half(
                epi, acc[0][i], acc[1][i], lane,
                [&](int v0, int v1, int v2, int v3, int j, int q) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(mine + 32 * j + 8 * q);
                    const f32x4 b = *reinterpret_cast<const f32x4*>(mine + 256 + 32 * j + 8 * q);
                    const f32x4 v = (f32x4){(float)v0 * sx, (float)v1 * sx, (float)v2 * sx, (float)v3 * sx} * w + b;
                    return make_uint2(tile_pack2<YDT>(v[0], v[1]), tile_pack2<YDT>(v[2], v[3]));
                },
                [&](int row, int c, uint4 v) {
                    const int64_t m = m0 + 32 * i + row;
                    if (m < a.M) tile_store8(a.y, m * a.N, nw + c, a.N, a.vec, v);
                });
        }
    }
}

// Few rows (M <= 16, serving's single tokens): one launch, x quantized by every
// workgroup (its codes in LDS, M K <= kInt8FewCodes), the weights streamed once.
// Workgroup = 16 channels; its four waves take a quarter of K each in steps of
// 64 (v_mfma_i32_16x16x64_i8, the rows past M zero), whose loads are all
// independent, and add up their int32 sums in LDS.  Bound by the latency of
// two reads, x and the weights, and by HBM for large weights.  1 x 768 -> 1000
// fp16 5.1 us; quantizer and tile kernel 3 + 7.
constexpr int64_t kInt8FewCodes = 32768;
struct Int8Few {
    const void* x;
    const int8_t* w;
    const float *sw, *bias;
    void* y;
    int64_t ldw, N;
    int M, K;
};
constexpr int int8_few_pitch(int64_t K) { return (int)((K + 63) / 64 * 64 + 16); }

template <int XDT, int YDT>
__global__ void __launch_bounds__(256) int8_few_kernel(Int8Few a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ float sx[16];
    __shared__ int part[4][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int steps = (a.K + 63) / 64, pitch = int8_few_pitch(a.K);
    // weights of this wave's first steps, on their way while x is quantized
    const int s0 = steps * wave / 4, s1 = steps * (wave + 1) / 4;
    const int64_t row = n0 + r < a.N ? n0 + r : a.N - 1;
    const int8_t* wp = a.w + row * a.ldw + 16 * g;
    auto load = [&](int s) {  // a lane's 16 bytes begin in the row (which holds K in whole 16 bytes) or past it
        intx4 v = {0, 0, 0, 0};
        if (s < s1 && 64 * s + 16 * g < a.K) v = *reinterpret_cast<const intx4*>(wp + 64 * s);
        return v;
    };
    constexpr int AHEAD = 8;
    intx4 w[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) w[i] = load(s0 + i);
    int8_t* codes = reinterpret_cast<int8_t*>(smem);  // [16][pitch]
    for (int m = wave; m < a.M; m += 4) {
        uint32_t mx = 0;
        auto piece = [&](int k, float (&v)[8]) {  // 8 values of the row, zeros past its end
            const int64_t at = (int64_t)m * a.K + k;
            if (k + 8 <= a.K) {
                load8_any<XDT>(a.x, at, v);
            } else {
#pragma unroll
                for (int t = 0; t < 8; ++t) v[t] = k + t < a.K ? load1<XDT>(a.x, at + t) : 0.0f;
            }
        };
        for (int k = 8 * lane; k < a.K; k += 512) {
            float v[8];
            piece(k, v);
#pragma unroll
            for (int t = 0; t < 8; ++t) mx = max(mx, __float_as_uint(v[t]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
        const Int8Row q(mx);
        if (lane == 0) sx[m] = q.scale;
        for (int k = 8 * lane; k < 64 * steps; k += 512) {
            uint32_t c[2] = {0, 0};
            if (k < a.K) {
                float v[8];
                piece(k, v);
#pragma unroll
                for (int t = 0; t < 8; ++t) c[t >> 2] |= (uint32_t)(q.code(v[t]) & 0xff) << (8 * (t & 3));
            }
            *reinterpret_cast<uint2*>(codes + m * pitch + k) = make_uint2(c[0], c[1]);
        }
    }
    __syncthreads();
    intx4 acc = {0, 0, 0, 0};
    const bool used = r < a.M;
    for (int s = s0; s < s1; s += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (s + i >= s1) break;
            intx4 x = {0, 0, 0, 0};
            if (used) x = *reinterpret_cast<const intx4*>(codes + r * pitch + 64 * (s + i) + 16 * g);
            const intx4 v = w[i];
            w[i] = load(s + i + AHEAD);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(v, x, acc, 0, 0, 0);
        }
    }
    // acc[t]: channel 4 g + t, row r
#pragma unroll
    for (int t = 0; t < 4; ++t) part[wave][4 * g + t][r] = acc[t];
    __syncthreads();
    const int c = threadIdx.x & 15, m = threadIdx.x >> 4;
    const int64_t n = n0 + c;
    if (m < a.M && n < a.N) {
        const int sum = part[0][c][m] + part[1][c][m] + part[2][c][m] + part[3][c][m];
        const float v = (float)sum * sx[m] * a.sw[n];
        store1<YDT>(a.y, (int64_t)m * a.N + n, a.bias ? v + a.bias[n] : v);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static bool int8_few(int xdt, int64_t M, int64_t K) {
    return xdt >= 0 && M <= 16 && M * K <= kInt8FewCodes;
}

template <int XDT, int YDT>
static hipError_t few_go(const Int8Few& a, hipStream_t s) {
    // at most kInt8FewCodes + 16 x 79 bytes
    hipLaunchKernelGGL((int8_few_kernel<XDT, YDT>), dim3((unsigned)((a.N + 15) / 16)), dim3(256), a.M * int8_few_pitch(a.K), s, a);
    return hipGetLastError();
}
template <int XDT>
static hipError_t few_y(const Int8Few& a, int ydt, hipStream_t s) {
    switch (ydt) {
        case RPFQ_F32: return few_go<XDT, RPFQ_F32>(a, s);
        case RPFQ_F16: return few_go<XDT, RPFQ_F16>(a, s);
        default: return few_go<XDT, RPFQ_BF16>(a, s);
    }
}

static Int8Pad pad_of(const int8_t* src, int64_t ld, int64_t K, int64_t rows, int8_t* dst, int64_t ldq) {
    const int64_t blocks = (rows + 3) / 4;
    return {src, ld, K, dst, ldq, rows, (unsigned)(blocks < 16384 ? blocks : 16384)};
}
static hipError_t pad_codes(const Int8Pad& a, hipStream_t s) {
    hipLaunchKernelGGL(int8_pad_kernel, dim3(a.blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

// pad: a weight to be copied beside it, or blocks = 0
template <int DT>
static hipError_t quantize_dt(const void* x, int64_t M, int64_t K, int8_t* q, int64_t ldq, float* scale, const Int8Pad& pad,
                              hipStream_t s) {
    const bool vec = K % 8 == 0 && ldq % 8 == 0 && ldq <= 4096 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % 8 == 0;
    if (!vec) {
        const unsigned blocks = (unsigned)(M < 65536 ? M : 65536);
        hipLaunchKernelGGL((int8_rows_any_kernel<DT>), dim3(blocks + pad.blocks), dim3(256), 0, s, x, M, K, q, ldq, scale, blocks,
                           pad);
        return hipGetLastError();
    }
    if (pad.blocks) {
        const hipError_t e = pad_codes(pad, s);
        if (e != hipSuccess) return e;
    }
    // at most 2^22 workgroups: a launch's threads are counted in 32 bits
    const dim3 rows((unsigned)(M < (1LL << 24) ? (M + 3) / 4 : 1LL << 22));
#define RPFQ_ROWS(NC) hipLaunchKernelGGL((int8_rows_kernel<DT, NC>), rows, dim3(256), 0, s, x, M, (int)K, q, ldq, scale)
    if (ldq <= 512) RPFQ_ROWS(1);
    else if (ldq <= 1024) RPFQ_ROWS(2);
    else if (ldq <= 2048) RPFQ_ROWS(4);
    else RPFQ_ROWS(8);
#undef RPFQ_ROWS
    return hipGetLastError();
}

static hipError_t quantize(const void* x, int dt, int64_t M, int64_t K, int8_t* q, int64_t ldq, float* scale,
                           const Int8Pad& pad, hipStream_t s) {
    switch (dt) {
        case RPFQ_F32: return quantize_dt<RPFQ_F32>(x, M, K, q, ldq, scale, pad, s);
        case RPFQ_F16: return quantize_dt<RPFQ_F16>(x, M, K, q, ldq, scale, pad, s);
        default: return quantize_dt<RPFQ_BF16>(x, M, K, q, ldq, scale, pad, s);
    }
}
hipError_t launch_quantize_int8(const void* x, int dt, int64_t M, int64_t K, int8_t* q, int64_t ldq, float* scale,
                                hipStream_t s) {
    return quantize(x, dt, M, K, q, ldq, scale, Int8Pad{}, s);
}

template <int YDT>
struct Int8Go {
    Int8Args& a;
    hipStream_t s;
    template <int MB, int WM, int S, int KB>
    hipError_t run() {
        using G = TileGemm<MB, WM, S, KB, false, false, MmaI8>;
        static std::atomic<uint64_t> attr_done{0};
        const auto kernel = &int8_gemm_kernel<MB, WM, S, KB, YDT>;
        const hipError_t e = set_lds_attr_once(reinterpret_cast<const void*>(kernel), kInt8Lds<G>, attr_done);
        if (e != hipSuccess) return e;
        a.tiles_m = (int)((a.M + G::ROWS - 1) / G::ROWS);
        a.tiles_n = (int)((a.N + 255) / 256);
        a.group = tile_group(a.tiles_n, 256 * a.K);
        hipLaunchKernelGGL((int8_gemm_kernel<MB, WM, S, KB, YDT>), dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(G::THREADS),
                           kInt8Lds<G>, s, a);
        return hipGetLastError();
    }
};

template <int YDT>
static hipError_t gemm_y(Int8Args& a, hipStream_t s) {
    return tile_dispatch(tile_form(a.M, a.N), Int8Go<YDT>{a, s});
}

// x codes in `work` unless given, or few; w copied there if its rows are not whole 16-byte pieces
Int8Plan int8_plan(const void* x, int xdt, int64_t M, int64_t N, int64_t K, const int8_t* w, int64_t ldw) {
    Int8Plan p = {};
    p.ld = (K + 15) & ~(int64_t)15;
    p.few = int8_few(xdt, M, K);
    p.pad_w = int8_pads(w, ldw, K);
    p.copy_x = !p.few && (xdt >= 0 || int8_pads(reinterpret_cast<const int8_t*>(x), K, K));
    auto take = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += (n + 255) & ~(size_t)255;
        return at;
    };
    if (p.copy_x) {
        p.x_at = take((size_t)M * p.ld);
        p.sx_at = take((size_t)M * 4);
    }
    if (p.pad_w) p.w_at = take((size_t)N * p.ld);
    return p;
}

hipError_t launch_linear_int8(const void* x, int xdt, const float* sx, const int8_t* w, int64_t ldw, const float* sw,
                              const float* bias, int64_t M, int64_t N, int64_t K, void* y, int ydt, void* work,
                              hipStream_t s) {
    const Int8Plan p = int8_plan(x, xdt, M, N, K, w, ldw);
    char* wk = reinterpret_cast<char*>(work);
    hipError_t e;
    Int8Pad pad = {};
    if (p.pad_w) {
        int8_t* q = reinterpret_cast<int8_t*>(wk + p.w_at);
        pad = pad_of(w, ldw, K, N, q, p.ld);
        w = q;
        ldw = p.ld;
        const bool beside = p.copy_x && xdt >= 0;  // with the quantizer's launch
        if (!beside && (e = pad_codes(pad, s)) != hipSuccess) return e;
    }
    if (p.few) {
        const Int8Few f = {x, w, sw, bias, y, ldw, N, (int)M, (int)K};
        switch (xdt) {
            case RPFQ_F32: return few_y<RPFQ_F32>(f, ydt, s);
            case RPFQ_F16: return few_y<RPFQ_F16>(f, ydt, s);
            default: return few_y<RPFQ_BF16>(f, ydt, s);
        }
    }
    Int8Args a = {};
    a.x = {reinterpret_cast<const char*>(x), K, 0, M};
    a.w = {reinterpret_cast<const char*>(w), ldw, 0, N};
    a.sx = sx;
    if (p.copy_x) {
        int8_t* q = reinterpret_cast<int8_t*>(wk + p.x_at);
        float* qs = reinterpret_cast<float*>(wk + p.sx_at);
        // codes that come unaligned are copied as an unaligned weight is
        e = xdt >= 0 ? quantize(x, xdt, M, K, q, p.ld, qs, pad, s)
                     : pad_codes(pad_of(reinterpret_cast<const int8_t*>(x), K, K, M, q, p.ld), s);
        if (e != hipSuccess) return e;
        a.x = {reinterpret_cast<const char*>(q), p.ld, 0, M};
        if (xdt >= 0) a.sx = qs;
    }
    a.sw = sw;
    a.bias = bias;
    a.y = y;
    a.M = M;
    a.N = N;
    a.K = p.ld;
    const int es = ydt == RPFQ_F32 ? 4 : 2;
    a.vec = N % (16 / es) == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
    // a 16-bit output larger than the 256-MB cache behind the L2 goes past both,
    // which leaves them to the operands (50,432 x 4,096: 289 -> 277 us); a smaller
    // one is what the next layer reads
    if (a.vec && es == 2 && M * N * es > 256LL << 20) a.vec = 2;
    switch (ydt) {
        case RPFQ_F32: return gemm_y<RPFQ_F32>(a, s);
        case RPFQ_F16: return gemm_y<RPFQ_F16>(a, s);
        default: return gemm_y<RPFQ_BF16>(a, s);
    }
}

}  // namespace rpfq
