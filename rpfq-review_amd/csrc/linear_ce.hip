// Softmax cross entropy of a linear classifier over many classes and its
// gradient, without keeping the logits:
//   z = x w^T + b,  loss_m = lse(z_m) - (1 - e) z_{m,t} - (e / V) sum_v z_{m,v},
//   dz_m = g_m (softmax(z_m) - (1 - e) 1_t - e / V),
//   dx = dz w,  dw = dz^T x,  db = sum_m dz_m.
// Forward: the logits' tiles leave the matrix cores as a maximum and a sum of
// exp(z - maximum) per row and tile (float32), joined by a pass over the tiles.
// Kept of a row are its maximum, the sum's reciprocal and the target's logit,
// not lse: that one's last bit is 2^-20 of a probability near 1, which is most
// of dz where p - 1 is small.
// Backward: the logits are formed again, a piece of the classes at a time; dz
// of a piece goes to a workspace and meets w and x from there.
//
// dz as the matrix cores take it: beside 16-bit operands as two terms of their
// type, what the first leaves (at most 2^-8 of the value in bf16, 2^-11 in fp16)
// being rounded once more: 2^-16 and 2^-22 of the value are lost, and in fp16,
// where dz is taken times 2^15 so that probabilities down to 2^-29 stay normal,
// 2^-40 at least.  One term alone left gradients of 64 rows (1,000 classes, bf16)
// 2.3e-3 off, where the rounding of the result is 1.7e-3; two leave 1.7e-3 and
// cost the gradients' products twice (2,048 x 20,000 x 1,024 fp16 loss and
// gradients 413 -> 614 us, 8,192 x 65,536 x 768 bf16 3,310 -> 5,260).  The sums
// over classes and rows stay in float32 until the gradients are rounded to their
// own type.  float32 operands lose nothing: many rows go as three bf16 terms
// (tile_pair), few as they are (kCeDirectRows).  fp16 rows with upstream gradients
// of their own have dz in two bf16 terms, with 2^-16 of it for the product of the
// second terms that is left out (CePlan::wide).
#include <cmath>

#include "tile_gemm.h"

namespace rpfq {

// exp(z - a) as exp2(z log2e - a log2e), one fused operation a value, where a
// is the rounded product wherever it is used again, so its rounding cancels.
// log2e in float32 stands for 1.3e-8 too little of every logit, less than their
// own rounding.  Past 2^100 (masks of a type's lowest value) a log2e could
// overflow: there the difference comes first.
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kCeFar = 0x1p100f;
__device__ __forceinline__ float ce_exp2(float z, float a2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -a2)); }
// z - top of a logit against a row's maximum, in the units of exp2
__device__ __forceinline__ float ce_gap_z(float z, float top) {
    return fabsf(top) <= kCeFar ? __builtin_fmaf(z, kLog2e, -(top * kLog2e)) : (z - top) * kLog2e;
}
// (a - b) log2e as the two agree on it
__device__ __forceinline__ float ce_gap(float a, float b) {
    return fabsf(a) <= kCeFar && fabsf(b) <= kCeFar ? a * kLog2e - b * kLog2e : (a - b) * kLog2e;
}

// What the gradients are multiplied by in the end.
struct CeFactor {
    const float* grad;  // of the loss, [1]
    const float* coef;  // the mean's factor, or NULL
    float undo;         // of dz's scale
    __device__ __forceinline__ float operator()() const { return grad[0] * (coef ? coef[0] : 1.0f) * undo; }
};

struct CeArgs {
    TileOperand x, w;          // [M, D], [V, D], K layout
    const void* bias;          // [V] of bias_dt, or NULL
    int bias_dt;
    const int64_t* target;
    int64_t M, V;              // rows, classes (w.count: those of a piece)
    int64_t v0;                // first class of the piece
    int64_t kb;                // bytes of k
    int pairs;                 // of the planes of x and w
    int tiles_m, tiles_n, group;
    float smooth;
    // forward
    float2* part;              // [tiles_n][M] (maximum, sum of exp(z - maximum))
    float* zsum;               // [tiles_n][M] sums of z, or NULL
    float* zt;                 // [M] the target's logit
    // backward
    const float* stat;         // [3][M] maximum, 1 / sum, the target's logit
    const float* rho;          // [M] weights of the rows in dz, or NULL: 1
    int64_t ignore;
    float dz_scale;
    char* xz;                  // x without its ignored rows, to be written here; or NULL
    char* dz;                  // [terms][M][ldz bytes]
    int64_t ldz, dz_plane;
    int64_t n8;                // columns of dz that are written: the piece's, in whole 16 bytes
    float* colsum;             // [row waves][n8] or NULL
};

__device__ __forceinline__ float ce_load(const void* p, int dt, int64_t i) {
    if (dt == RPFQ_F32) return reinterpret_cast<const float*>(p)[i];
    if (dt == RPFQ_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// Adds the bias to a wave's block of logits and makes those past the last
// class -inf: columns 32 j + 8 q + 4 g + t of the wave's 64, bias in LDS.
template <int MB>
__device__ __forceinline__ void ce_bias(floatx16 (&acc)[2][MB], const float* bias, int lane) {
    const int g = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(bias + 32 * j + 8 * q + 4 * g);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[j][i][4 * q + t] += b[t];
        }
}

// What the epilogues keep in LDS past the stages: the biases of a tile's
// columns, -inf past the last class, and of dz's rows what they need.
struct CeRow {
    float top;  // the maximum
    float f;    // p's factor; 0: a row that counts nowhere, NaN: one whose target is no class
    float off;  // what is taken off every class
    float dzt;  // dz of the target
};
template <int ROWS>
struct CeLds {
    float bias[256];
    CeRow row[ROWS];
    int t[ROWS];  // the target's column in the tile, or -1
};

__device__ __forceinline__ bool ce_biased(const CeArgs& a, int64_t n0) { return a.bias || n0 + 256 > a.w.count; }
__device__ __forceinline__ void ce_stage_bias(const CeArgs& a, int64_t n0, float* sm) {
    if (!ce_biased(a, n0) || threadIdx.x >= 256) return;
    const int64_t n = n0 + threadIdx.x;
    float b = n < a.w.count ? 0.0f : -__builtin_inff();
    if (a.bias && n < a.w.count) b = ce_load(a.bias, a.bias_dt, a.v0 + n);
    sm[threadIdx.x] = b;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// Bound by the products; the exponentials (16 clocks a wave and value, and as
// much again for maximum and sum) are 3 us of a 256 x 256 tile's 27 at D = 768.
// 8,192 x 65,536 x 768 bf16 845 us, 975 TFLOP/s (a library product that writes its
// logits: 1,031, without the softmax); 500 x 131,072 x 1,024 129 us; 2,048 x 20,000
// x 1,024 fp16 101 us.  128-row tiles, two workgroups a CU, whose exponentials
// overlap the other's products: 930 us.
template <int MB, int WM, int S, int KB, class Mma>
__global__ void __launch_bounds__(256 * WM, 2) ce_stats_kernel(CeArgs a) {
    extern __shared__ __align__(16) char smem[];
    using G = TileGemm<MB, WM, S, KB, false, false, Mma>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    int mt, nt;
    group_tile(xcd_tile(blockIdx.x, a.tiles_m * a.tiles_n), a.tiles_m, a.tiles_n, a.group, mt, nt);
    const int64_t m0 = (int64_t)mt * G::ROWS, n0 = (int64_t)nt * 256, nw = n0 + 64 * (wave & 3);
    floatx16 acc[2][MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[0][i] = acc[1][i] = floatx16{0};
    const int per = (int)G::steps(a.kb), steps = a.pairs * per;
    float* sb = reinterpret_cast<float*>(smem + G::LDS);
    G::run(a.x, a.w, m0, n0, a.kb, a.kb, per, a.pairs, 0, steps, smem, wave, lane, acc, [&] { ce_stage_bias(a, n0, sb); });
    float* sp = reinterpret_cast<float*>(smem);  // [4 column waves][rows][max, sum, sum of z]
    if (ce_biased(a, n0)) ce_bias<MB>(acc, sb + 64 * (wave & 3), lane);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int row = 32 * (MB * (wave >> 2) + i) + r;
        float mx = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, acc[j][i][v]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        float sum = 0.0f, zs = 0.0f;
        if (!__any(fabsf(mx) > kCeFar)) {
            const float base = mx * kLog2e;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) sum += ce_exp2(acc[j][i][v], base);
        } else {
            const float base = mx == -__builtin_inff() ? 0.0f : mx;
            const bool far = fabsf(base) > kCeFar;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    sum += far ? __builtin_amdgcn_exp2f((acc[j][i][v] - base) * kLog2e) : ce_exp2(acc[j][i][v], base * kLog2e);
        }
        if (a.zsum) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) zs += nw + 32 * j + acc_row(v, g) < a.w.count ? acc[j][i][v] : 0.0f;
            zs += __shfl_xor(zs, 32, 64);
        }
        sum += __shfl_xor(sum, 32, 64);
        const int64_t m = m0 + row;
        if (m < a.M) {
            const int64_t t = a.target[m] - nw;
            if (t >= 0 && t < 64 && nw + t < a.V) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (t == 32 * j + acc_row(v, g)) a.zt[m] = acc[j][i][v];
            }
        }
        if (g == 0) {
            float* d = sp + ((wave & 3) * G::ROWS + row) * 3;
            d[0] = mx;
            d[1] = sum;
            d[2] = zs;
        }
    }
    __syncthreads();
    const int row = threadIdx.x;
    if (row < G::ROWS && m0 + row < a.M) {
        float mx = -__builtin_inff(), sum = 0.0f, zs = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sp[(w * G::ROWS + row) * 3]);
        // fmax passes over NaN: the sums keep it
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* d = sp + (w * G::ROWS + row) * 3;
            sum += d[0] == -__builtin_inff() ? d[1] : d[1] * __builtin_amdgcn_exp2f(ce_gap(d[0], mx));
            zs += d[2];
        }
        a.part[(int64_t)nt * a.M + m0 + row] = make_float2(mx, sum);
        if (a.zsum) a.zsum[(int64_t)nt * a.M + m0 + row] = zs;
    }
}

struct CeJoin {
    const float2* part;
    const float* zsum;
    const float* zt;
    const int64_t* target;
    int64_t M, V, ignore;
    int tiles;
    float smooth;
    int reduction;
    float* stat;  // [3][M]: maximum, 1 / sum of exp(z - maximum), the target's logit
    float* rows;  // [M] loss of each row, 0 where ignored
    float* loss;  // the sum or the mean of them
    float* coef;
};
constexpr int64_t kCeFewRows = 128;

// Sum (reduction 2) or mean (1) of the rows' losses in a fixed order, and the
// factor that the gradient takes from it: coef = 1 or 1 / count (0 where no row
// counts: its rows then have no gradient, their mean is NaN).
__device__ __forceinline__ void ce_reduce(const CeJoin& a, double s, int n) {
    __shared__ double sm[1024];
    __shared__ int cm[1024];
    const int t = threadIdx.x;
    sm[t] = s;
    cm[t] = n;
    __syncthreads();
    for (int h = 512; h > 0; h >>= 1) {
        if (t < h) {
            sm[t] += sm[t + h];
            cm[t] += cm[t + h];
        }
        __syncthreads();
    }
    if (t == 0) {
        const double c = (double)cm[0];
        a.loss[0] = (float)(a.reduction == 1 ? sm[0] / c : sm[0]);
        a.coef[0] = a.reduction == 1 ? (cm[0] ? (float)(1.0 / c) : 0.0f) : 1.0f;
    }
}

__global__ void __launch_bounds__(1024) ce_reduce_kernel(CeJoin a) {
    double s = 0.0;
    int n = 0;
    for (int64_t m = threadIdx.x; m < a.M; m += 1024) {
        s += (double)a.rows[m];
        n += a.target[m] != a.ignore;
    }
    ce_reduce(a, s, n);
}

// lse and loss of a row from its tiles: 16 threads a row, in a fixed order
// (8,192 rows of 256 tiles 10 us; 500 of 512, in 8 workgroups, 13, and 18 with a
// tile's read at a time).
// ALL: one workgroup takes all rows and reduces them.
template <bool ALL>
__global__ void __launch_bounds__(1024) ce_join_kernel(CeJoin a) {
    const int c = threadIdx.x & 63, q = threadIdx.x >> 6;  // row, one of 16 parts of the tiles
    __shared__ float sm[3][64][17];
    constexpr int AHEAD = 8;  // tiles on their way at once
    double total = 0.0;
    int count = 0;
    for (int64_t m0 = ALL ? 0 : (int64_t)blockIdx.x * 64; m0 < (ALL ? a.M : (int64_t)blockIdx.x * 64 + 64); m0 += 64) {
        const int64_t m = m0 + c;
        float mx = -__builtin_inff(), sum = 0.0f, zs = 0.0f;
        if (m < a.M)
            for (int t = q; t < a.tiles; t += 16 * AHEAD) {
                float2 p[AHEAD];
                float z[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int64_t at = (int64_t)(t + 16 * k) * a.M + m;
                    const bool there = t + 16 * k < a.tiles;
                    p[k] = there ? a.part[at] : make_float2(0.0f, 0.0f);
                    z[k] = there && a.zsum ? a.zsum[at] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (t + 16 * k >= a.tiles) break;
                    const float n = fmaxf(mx, p[k].x), base = n == -__builtin_inff() ? 0.0f : n, y = p[k].y;
                    // a tile of -inf has sum 0, one with NaN has sum NaN whatever its maximum
                    const float add = y == 0.0f || y != y ? y : y * __builtin_amdgcn_exp2f(ce_gap(p[k].x, base));
                    sum = (sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f(ce_gap(mx, base))) + add;
                    mx = n;
                    zs += z[k];
                }
            }
        sm[0][c][q] = mx;
        sm[1][c][q] = sum;
        sm[2][c][q] = zs;
        __syncthreads();
        if (q == 0 && m < a.M) {
            float top = -__builtin_inff();
            for (int i = 0; i < 16; ++i) top = fmaxf(top, sm[0][c][i]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            sum = zs = 0.0f;
            for (int i = 0; i < 16; ++i) {
                const float s = sm[1][c][i];
                sum += s == 0.0f || s != s ? s : s * __builtin_amdgcn_exp2f(ce_gap(sm[0][c][i], base));
                zs += sm[2][c][i];
            }
            // lse in 64 bits, from the exponent that the sum is relative to
            const double lse = fabsf(base) <= kCeFar ? ((double)(base * kLog2e) + log2((double)sum)) / (double)kLog2e
                                                     : (double)base + log((double)sum);
            const int64_t t = a.target[m];
            const bool labelled = t >= 0 && t < a.V;
            const float zt = labelled ? a.zt[m] : 0.0f;
            float loss = 0.0f;
            if (t != a.ignore) {
                loss = __uint_as_float(0x7fc00000u);
                if (labelled) {
                    double d = (1.0 - (double)a.smooth) * (lse - (double)zt);
                    if (a.zsum) d += (double)a.smooth * (lse - (double)zs / (double)a.V);
                    loss = (float)d;
                }
                ++count;
            }
            a.stat[m] = base;
            a.stat[a.M + m] = 1.0f / sum;
            a.stat[2 * a.M + m] = zt;
            if (!ALL) a.rows[m] = loss;
            total += (double)loss;
        }
        __syncthreads();
    }
    if (ALL) ce_reduce(a, total, count);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// reduction none: rho[m] = grad[m] over the largest finite one of the rows that
// count, so that their dz stays within [-1, 1], and that largest, factor[0].  A
// row with inf or NaN keeps it to itself and to grad_w.
__global__ void __launch_bounds__(1024) ce_rho_kernel(const float* grad, const int64_t* target, int64_t M, int64_t ignore,
                                                      float* rho, float* factor) {
    __shared__ float sm[1024];
    const int t = threadIdx.x;
    float top = 0.0f;
    for (int64_t m = t; m < M; m += 1024) {
        const float g = fabsf(grad[m]);
        if (target[m] != ignore && g <= 3.40282347e38f) top = fmaxf(top, g);
    }
    sm[t] = top;
    __syncthreads();
    for (int h = 512; h > 0; h >>= 1) {
        if (t < h) sm[t] = fmaxf(sm[t], sm[t + h]);
        __syncthreads();
    }
    top = sm[0] > 0.0f ? sm[0] : 1.0f;
    for (int64_t m = t; m < M; m += 1024) rho[m] = grad[m] / top;
    if (t == 0) factor[0] = top;
}

// A float32 as three bf16 terms, each the top 8 bits of what is left: exact for
// every finite value.
__device__ __forceinline__ void split3(float v, uint16_t& h, uint16_t& m, uint16_t& l) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) {
        h = 0x7fc0, m = l = 0;
        return;
    }
    h = (uint16_t)(u >> 16);
    const float r1 = (u & 0x7fffffffu) == 0x7f800000u ? 0.0f : v - __uint_as_float(u & 0xffff0000u);
    m = (uint16_t)(__float_as_uint(r1) >> 16);
    const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
    l = (uint16_t)(__float_as_uint(r2) >> 16);
}

// A value as two 16-bit terms, both nearest.  What an inf leaves is 0 and not
// inf - inf.
template <int DT>
__device__ __forceinline__ void ce_terms2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = tile_pack2<DT>(a, b);
    const float ha = DT == RPFQ_F16 ? (float)__builtin_bit_cast(half2v, hi)[0] : bf16_to_f32(hi & 0xffffu);
    const float hb = DT == RPFQ_F16 ? (float)__builtin_bit_cast(half2v, hi)[1] : bf16_to_f32(hi >> 16);
    const float la = a - ha, lb = b - hb;
    lo = tile_pack2<DT>(la == la ? la : 0.0f, lb == lb ? lb : 0.0f);
}

// x [M, D] and w [V, D] as operands: rows of ld elements, float32 as three planes
// of bf16 terms.  target: rows of x that it ignores are zeros, whatever they
// hold (0 x NaN would reach every class of dw); NULL: all rows as they are.
struct CeCopy {
    const void* src[2];
    uint16_t* dst[2];
    int64_t rows[2];
    int64_t D, ld;
    const int64_t* target;
    int64_t ignore;
    int lanes;
};
// MODE 0: 16-bit rows, 1: planes, 2: float32 rows, 3: fp16 as two bf16 planes
// (nearest, and what that leaves: 3 bits, exact).  `lanes` (a power of two) take
// a row, 8 elements each; whole pieces are read at once, at any alignment of
// their elements.
template <int MODE>
__global__ void __launch_bounds__(256) ce_copy_kernel(CeCopy a) {
    const int lane = threadIdx.x & (a.lanes - 1), per = (int)(a.ld / 8);
    const int64_t rows = a.rows[0] + a.rows[1], step = (int64_t)gridDim.x * (256 / a.lanes);
    for (int64_t at = (int64_t)blockIdx.x * (256 / a.lanes) + threadIdx.x / a.lanes; at < rows; at += step) {
        const int k = at >= a.rows[0];
        const int64_t m = k ? at - a.rows[0] : at;
        const bool on = k || !a.target || a.target[m] != a.ignore;
        for (int i = lane; i < per; i += a.lanes) {
            const int64_t d = 8 * i;
            uint16_t* out = a.dst[k] + (m * a.ld + d) * (MODE == 2 ? 2 : 1);
            if constexpr (MODE == 0 || MODE == 3) {
                const uint16_t* x = reinterpret_cast<const uint16_t*>(a.src[k]) + m * a.D + d;
                uint16_t e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (on && d + 8 <= a.D) {
                    __builtin_memcpy(e, x, 16);
                } else if (on) {
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (d + t < a.D) e[t] = x[t];
                }
                if constexpr (MODE == 3) {
                    uint4 h, l;
                    auto two = [&](int i, uint32_t& hi, uint32_t& lo) {
                        ce_terms2<RPFQ_BF16>((float)__builtin_bit_cast(_Float16, e[i]), (float)__builtin_bit_cast(_Float16, e[i + 1]),
                                             hi, lo);
                    };
                    two(0, h.x, l.x);
                    two(2, h.y, l.y);
                    two(4, h.z, l.z);
                    two(6, h.w, l.w);
                    __builtin_memcpy(e, &h, 16);
                    __builtin_memcpy(out + a.rows[k] * a.ld, &l, 16);
                }
                __builtin_memcpy(out, e, 16);
            } else {
                const float* x = reinterpret_cast<const float*>(a.src[k]) + m * a.D + d;
                float e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (on && d + 8 <= a.D) {
                    __builtin_memcpy(e, x, 32);
                } else if (on) {
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (d + t < a.D) e[t] = x[t];
                }
                if constexpr (MODE == 2) {
                    __builtin_memcpy(out, e, 32);
                } else {
                    const int64_t plane = a.rows[k] * a.ld;
                    uint16_t h[8], mid[8], l[8];
#pragma unroll
                    for (int t = 0; t < 8; ++t) split3(e[t], h[t], mid[t], l[t]);
                    __builtin_memcpy(out, h, 16);
                    __builtin_memcpy(out + plane, mid, 16);
                    __builtin_memcpy(out + 2 * plane, l, 16);
                }
            }
        }
    }
}

// Sums of 32 values over the 32 lanes of a half wave: lane r ends with the sum
// of value r.  Each round halves the values: a lane keeps one half and hands
// the other to its partner.
template <int M>
__device__ __forceinline__ void ce_lane_round(float (&v)[32], int lane) {
    const bool up = lane & M;
#pragma unroll
    for (int k = 0; k < M; ++k) {
        const float give = up ? v[k] : v[k + M], keep = up ? v[k + M] : v[k];
        v[k] = keep + __shfl_xor(give, M, 64);
    }
}
__device__ __forceinline__ float ce_lane_sums(float (&v)[32], int lane) {
    ce_lane_round<16>(v, lane);
    ce_lane_round<8>(v, lane);
    ce_lane_round<4>(v, lane);
    ce_lane_round<2>(v, lane);
    ce_lane_round<1>(v, lane);
    return v[0];
}

// dz of one piece of the classes.  DT: the type of dz's terms (float32: itself
// beside float32 operands, three bf16 terms beside theirs).
// The logits' product again and dz's terms written: 8,192 x 65,536 x 768 bf16 1,320
// us in two pieces, 625 TFLOP/s and 1.6 TB/s of dz; 2,048 x 20,000 x 1,024 fp16 146
// us.  With one term 950 and 114.  Stores past the caches were slower where a
// piece of dz stays in them.
template <int MB, int WM, int S, int KB, class Mma, int DT>
__global__ void __launch_bounds__(256 * WM, 2) ce_dz_kernel(CeArgs a) {
    extern __shared__ __align__(16) char smem[];
    using G = TileGemm<MB, WM, S, KB, false, false, Mma>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    int mt, nt;
    group_tile(xcd_tile(blockIdx.x, a.tiles_m * a.tiles_n), a.tiles_m, a.tiles_n, a.group, mt, nt);
    const int64_t m0 = (int64_t)mt * G::ROWS, mw = m0 + 32 * MB * (wave >> 2);
    const int64_t n0 = (int64_t)nt * 256, nw = n0 + 64 * (wave & 3);
    floatx16 acc[2][MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[0][i] = acc[1][i] = floatx16{0};
    const int per = (int)G::steps(a.kb), steps = a.pairs * per;
    CeLds<G::ROWS>& sh = *reinterpret_cast<CeLds<G::ROWS>*>(smem + G::LDS);
    const float even = a.smooth / (float)a.V;
    G::run(a.x, a.w, m0, n0, a.kb, a.kb, per, a.pairs, 0, steps, smem, wave, lane, acc, [&] {
        ce_stage_bias(a, n0, sh.bias);
        if (threadIdx.x < G::ROWS) {
            const int64_t m = m0 + threadIdx.x;
            CeRow row = {0.0f, 0.0f, 0.0f, 0.0f};
            int t = -1;
            if (m < a.M) {
                const int64_t label = a.target[m], at = label - a.v0 - n0;
                const float inv = a.stat[a.M + m], zt = a.stat[2 * a.M + m], own = a.rho ? a.rho[m] : 1.0f;
                row.top = a.stat[m];
                const float rho = label == a.ignore             ? 0.0f
                                  : label < 0 || label >= a.V ? __uint_as_float(0x7fc00000u)
                                                                : own * a.dz_scale;
                if (rho != 0.0f) {
                    row.f = inv * rho;
                    row.off = even * rho;
                    if (at >= 0 && at < 256) t = (int)at;
                    // p - 1 before the factors: what is left of a p near 1 keeps its bits
                    row.dzt = (__builtin_amdgcn_exp2f(ce_gap_z(zt, row.top)) * inv - even - (1.0f - a.smooth)) * rho;
                }
            }
            sh.row[threadIdx.x] = row;
            sh.t[threadIdx.x] = t;
        }
        if (a.xz) {  // the row tile's share of x, a part of it for each column tile
            const uint32_t per16 = (uint32_t)(a.kb / 16), rows = (uint32_t)(a.M - m0 < G::ROWS ? a.M - m0 : G::ROWS);
            const uint32_t all = rows * per16, share = (all + a.tiles_n - 1) / a.tiles_n;
            const uint32_t end = (nt + 1) * share < all ? (nt + 1) * share : all;
            for (uint32_t i = nt * share + threadIdx.x; i < end; i += G::THREADS) {
                const int64_t m = m0 + i / per16, at = m * a.kb + (i % per16) * 16;
                const uint4 v = *reinterpret_cast<const uint4*>(a.x.p + at);
                *reinterpret_cast<uint4*>(a.xz + at) = a.target[m] != a.ignore ? v : make_uint4(0, 0, 0, 0);
            }
        }
    });
    char* epi = smem + wave * kTileEpi;
    if (ce_biased(a, n0)) ce_bias<MB>(acc, sh.bias + 64 * (wave & 3), lane);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const CeRow row = sh.row[32 * (MB * (wave >> 2) + i) + r];
        const float top = row.top, f = row.f, off = row.off, dzt = row.dzt;
        // the target's column among the wave's
        int t = sh.t[32 * (MB * (wave >> 2) + i) + r] - 64 * (wave & 3);
        t = t >= 0 && t < 64 ? t : -1;
        const bool plain = !__any(fabsf(top) > kCeFar);
        const float base = top * kLog2e;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float z = acc[j][i][v];
                const float e = plain ? ce_exp2(z, base) : __builtin_amdgcn_exp2f(ce_gap_z(z, top));
                acc[j][i][v] = __builtin_fmaf(e, f, -off);
            }
        if (__any(f == 0.0f)) {  // whatever such a row holds
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[j][i][v] = f == 0.0f ? 0.0f : acc[j][i][v];
        }
        if (a.w.count - n0 < 256) {  // columns past the last class, for the operands' padding
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (nw + 32 * j + acc_row(v, g) >= a.w.count) acc[j][i][v] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (t == 32 * j + acc_row(v, g)) acc[j][i][v] = dzt;
        if constexpr (DT == RPFQ_F32) {
            const int64_t n = nw + 4 * (lane & 15);
            tile_rows(epi, acc[0][i], acc[1][i], lane, [](float v, int) { return v; },
                      [&](int row, int, f32x4 v) {
                          const int64_t m = mw + 32 * i + row;
                          if (m >= a.M || n >= a.n8) return;
                          if constexpr (Mma::ES == 4) {
                              *reinterpret_cast<f32x4*>(a.dz + m * a.ldz + 4 * n) = v;
                              return;
                          }
                          char* d = a.dz + m * a.ldz + 2 * n;
                          uint16_t h[4], k[4], l[4];
#pragma unroll
                          for (int e = 0; e < 4; ++e) split3(v[e], h[e], k[e], l[e]);
                          __builtin_memcpy(d, h, 8);
                          __builtin_memcpy(d + a.dz_plane, k, 8);
                          __builtin_memcpy(d + 2 * a.dz_plane, l, 8);
                      });
        } else {
            tile_rows8(epi, acc[0][i], acc[1][i], lane, [&](int row, int c, f32x4 v, f32x4 u) {
                const int64_t m = mw + 32 * i + row, n = nw + c;
                if (m >= a.M || n >= a.n8) return;
                uint4 h, l;
                ce_terms2<DT>(v[0], v[1], h.x, l.x);
                ce_terms2<DT>(v[2], v[3], h.y, l.y);
                ce_terms2<DT>(u[0], u[1], h.z, l.z);
                ce_terms2<DT>(u[2], u[3], h.w, l.w);
                char* d = a.dz + m * a.ldz + 2 * n;
                *reinterpret_cast<uint4*>(d) = h;
                *reinterpret_cast<uint4*>(d + a.dz_plane) = l;
            });
        }
    }
    if (a.colsum) {  // the wave's columns over its rows
        float cs[32];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                cs[16 * j + v] = acc[j][0][v];
#pragma unroll
                for (int i = 1; i < MB; ++i) cs[16 * j + v] += acc[j][i][v];
            }
        const float sum = ce_lane_sums(cs, lane);
        const int64_t n = nw + 32 * (r >> 4) + acc_row(r & 15, g);
        if (n < a.n8) a.colsum[((int64_t)mt * WM + (wave >> 2)) * a.n8 + n] = sum;
    }
}

struct CeGrad {
    TileOperand r, c;
    int64_t rk, ck;
    int64_t M, N;     // rows, columns of the gradient
    int pairs, splits;
    int tiles_m, tiles_n;
    float* part;      // [splits][M][ldp], or NULL: the gradient itself, rounded
    int64_t ldp;
    int add;          // part holds the pieces before
    CeFactor factor;
    void* out;        // [M, N]
    int vec;
};

// One product of the gradient: dx (dz in K layout, w in T) or dw (dz and x in T).
template <int MB, int WM, int S, int KB, bool RT, class Mma, int DT>
__device__ __forceinline__ void ce_grad_unit(const CeGrad& a, int bid, char* smem) {
    using G = TileGemm<MB, WM, S, KB, RT, true, Mma>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = a.tiles_m * a.tiles_n;
    const int unit = xcd_tile(bid, tiles * a.splits), sp = unit / tiles;
    int mt, nt;
    group_tile(unit - sp * tiles, a.tiles_m, a.tiles_n, a.tiles_n, mt, nt);
    const int64_t m0 = (int64_t)mt * G::ROWS, mw = m0 + 32 * MB * (wave >> 2), n0 = (int64_t)nt * 256;
    const int per = (int)G::steps(a.rk), steps = a.pairs * per;
    const int s0 = (int)((int64_t)steps * sp / a.splits), s1 = (int)((int64_t)steps * (sp + 1) / a.splits);
    floatx16 acc[2][MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[0][i] = acc[1][i] = floatx16{0};
    G::run(a.r, a.c, m0, n0, a.rk, a.ck, per, a.pairs, s0, s1, smem, wave, lane, acc, [] {});
    const int64_t n = n0 + 64 * (wave & 3) + 4 * (lane & 15);
    const float f = a.part ? 1.0f : a.factor();
    float* part = a.part ? a.part + (int64_t)sp * a.M * a.ldp : nullptr;
#pragma unroll
    for (int i = 0; i < MB; ++i)
        tile_rows(smem + wave * kTileEpi, acc[0][i], acc[1][i], lane, [&](float v, int) { return v; },
                  [&](int row, int, f32x4 v) {
                      const int64_t m = mw + 32 * i + row;
                      if (m >= a.M) return;
                      if (part) {
                          if (n >= a.ldp) return;
                          f32x4* d = reinterpret_cast<f32x4*>(part + m * a.ldp + n);
                          *d = a.add ? *d + v : v;
                      } else {
                          tile_store4<DT>(a.out, m * a.N, n, a.N, a.vec, v * f);
                      }
                  });
}

// Both products of a piece's dz in one launch: dx (dz in K layout, w in T) and dw
// (dz and x in T), the longer units first and the others into their last round
// (2,048 x 20,000 x 1,024 fp16, one term: 1.2 and 1.0 rounds of the chip; 227 us in
// two launches, 200 in one; 380 with two terms).  8,192 x 65,536 x 768 bf16, two
// terms, 2,980 us in two pieces, 1,107 TFLOP/s (library products of the same
// shapes, one term: 1,700 us).
struct CeGrads {
    CeGrad g[2];   // dx, dw; splits = 0: not wanted
    int units[2];
    int first;     // whose units come first
};
template <int MB, int WM, int S, int KB, class Mma, int DT>
__global__ void __launch_bounds__(256 * WM, 2) ce_grads_kernel(CeGrads a) {
    extern __shared__ __align__(16) char smem[];
    const int bid = blockIdx.x, lead = a.units[a.first];
    const int k = bid < lead ? a.first : 1 - a.first, at = bid < lead ? bid : bid - lead;
    if (k == 0) ce_grad_unit<MB, WM, S, KB, false, Mma, DT>(a.g[0], at, smem);
    else ce_grad_unit<MB, WM, S, KB, true, Mma, DT>(a.g[1], at, smem);
}

// out = factor * sum of the partials, in their order: of dw, db and dx, those
// that a piece leaves, in one launch.  HBM bound: 8 x 8,192 x 768 float32 15.5 us
// with the factor and rounding.
struct CeSum {
    const float* part;
    void* out;
    int64_t stride, rows, N, ldp;  // of a partial; rows, columns and row length of the sum
    int parts, dt, vec, blocks;
};
struct CeSums {
    CeSum s[3];
    CeFactor factor;
};
__global__ void __launch_bounds__(256) ce_sums_kernel(CeSums a) {
    int k = 0, bid = blockIdx.x;
    while (bid >= a.s[k].blocks) bid -= a.s[k++].blocks;
    const CeSum j = a.s[k];
    const float f = a.factor();
    const int64_t per = j.ldp / 4, total = j.rows * per;
    for (int64_t i = (int64_t)bid * 256 + threadIdx.x; i < total; i += (int64_t)j.blocks * 256) {
        const int64_t m = i / per, n = (i - m * per) * 4;
        const f32x4* p = reinterpret_cast<const f32x4*>(j.part + m * j.ldp + n);
        f32x4 v = p[0];
        int s = 1;
        for (; s + 8 <= j.parts; s += 8) {  // eight loads on their way, added in order
            f32x4 w[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) w[t] = p[(s + t) * (j.stride / 4)];
#pragma unroll
            for (int t = 0; t < 8; ++t) v += w[t];
        }
        for (; s < j.parts; ++s) v += p[s * (j.stride / 4)];
        v *= f;
        if (j.dt == RPFQ_F32) tile_store4<RPFQ_F32>(j.out, m * j.N, n, j.N, j.vec, v);
        else if (j.dt == RPFQ_F16) tile_store4<RPFQ_F16>(j.out, m * j.N, n, j.N, j.vec, v);
        else tile_store4<RPFQ_BF16>(j.out, m * j.N, n, j.N, j.vec, v);
    }
}

// ---------------------------------------------------------------------------
// plan and launches
// ---------------------------------------------------------------------------
// The form of the two gradients' launch, dx of M x D over V classes and dw of V
// x D over M rows, and the splits of their k (in steps of 64 bytes) that take
// the least time: the longest unit or the chip's share of all and half a unit,
// in steps of a 256-row tile (0.9 us), and the partials' way through memory
// (about 5 TB/s, and a launch).
static CeSplit ce_split(int64_t M, int64_t V, int64_t D, int pairs, int es) {
    // float32 as it is: twice the steps, each eight times as long
    const int64_t cost16 = es == 4 ? 16 : pairs, least = es == 4 ? 16 : 4;
    const int64_t cus = device_cus(), tn = (D + 255) / 256, kx = cost16 * ((V + 31) / 32), kw = cost16 * ((M + 31) / 32);
    static constexpr int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32, 48, 64};
    CeSplit best = {kTile128, 1, 1};
    double cost = 1e300;
    struct {
        TileForm form;
        int rows, slots;
        double step, start;
    } const forms[] = {{kTile64, 64, 1, 0.38, 4.0}, {kTile128Deep, 128, 1, 0.48, 4.0}, {kTile128, 128, 2, 1.15, 6.0}, {kTile256, 256, 1, 1.0, 5.0}};
    for (const auto& f : forms) {
        const int64_t slots = f.slots * cus;
        for (const int sx : kSplits) {
            if (sx > 1 && least * sx > kx) break;
            for (const int sw : kSplits) {
                if (sw > 1 && least * sw > kw) break;
                const double nx = (double)((kx + sx - 1) / sx) * f.step + f.start, nw = (double)((kw + sw - 1) / sw) * f.step + f.start;
                const double ux = (double)((M + f.rows - 1) / f.rows * tn * sx), uw = (double)((V + f.rows - 1) / f.rows * tn * sw);
                const double longest = nx > nw ? nx : nw, rounds = (ux * nx + uw * nw) / (double)slots;
                // the deep forms are for one round: more of them wait on the LDS fill
                if (ux + uw > (double)slots && (f.form == kTile64 || f.form == kTile128Deep)) continue;
                double c = ux + uw <= (double)slots ? longest : rounds + 0.5 * (nx < nw ? nx : nw);
                if (c < longest) c = longest;
                if (sx > 1) c += 7.0 + (double)sx * M * D * 8.0 / 4.5e6;
                if (sw > 1) c += 7.0 + (double)sw * V * D * 8.0 / 4.5e6;
                if (c < cost) {
                    cost = c;
                    best = {f.form, sx, sw};
                }
            }
        }
    }
    return best;
}

// Classes of a piece: dz within kCePiece bytes, whole tiles, pieces alike.  Pieces
// of 128 MiB to 2 GiB lie within 7 to 9% of each other (8,192 x 65,536 x 768 bf16
// 5,750 to 5,340 us, 4,096 x 131,072 x 1,024 6,520 to 7,100, float32 21,050 to 18,480).
constexpr int64_t kCePiece = 1LL << 30;
// Bytes of a row of dz with n classes: 16-byte pieces, and not a multiple of 4
// KB, where a tile's rows would all lie on the same channels.
static int64_t ce_ldz(int64_t n, int es) {
    const int64_t ld = es * ((n + 7) & ~(int64_t)7);
    return ld % 4096 == 0 ? ld + 256 : ld;
}

// float32 products of few rows: as they are, on the float32 matrix
// instructions.  Three planes of both operands cost 20 bytes an element of w and
// pass, whatever M is, but from about 256 rows on their products are 1.2 to 1.6
// times as fast (loss and gradients, us, planes -> direct: 50,000 classes x 1,024,
// 16 rows 649 -> 270, 128 773 -> 545, 256 1,017 -> 997, 512 1,626 -> 1,936;
// 10,008 x 768, 64 rows 185 -> 163, 256 both 221, 1,024 492 -> 677).
constexpr int64_t kCeDirectRows = 256;

// products of dz's terms with those of the other operand
static int ce_pairs(const CePlan& p) { return p.terms == 3 ? kPairs32 : p.wide ? kPairsHalf : p.terms; }

CePlan ce_plan(int dt, int64_t M, int64_t V, int64_t D, int reduction, bool smooth, bool backward) {
    CePlan p = {};
    // fp16 rows with upstream gradients of their own: dz, whose rows may lie far
    // apart, in bf16 terms, and x and w in as many for its products.  Under one
    // fp16 scale a row 2^-25 of the largest kept three bits.  2,048 x 20,000 x 1,024
    // loss and gradients 645 -> 809 us, 256 x 10,000 x 768 75 -> 90; through the
    // six products of float32 operands 1,632 and 192.
    p.wide = dt == RPFQ_F16 && reduction == RPFQ_REDUCE_NONE && backward;
    const bool direct = dt == RPFQ_F32 && M <= kCeDirectRows;
    const int planes = p.planes = dt == RPFQ_F32 && !direct ? 3 : 1;
    const int es = p.es = direct ? 4 : 2;
    const int terms = p.terms = direct ? 1 : planes == 3 ? 3 : 2;
    p.ldk = planes == 3 ? (D + 31) & ~(int64_t)31 : (D + 7) & ~(int64_t)7;
    p.pad = planes == 3 || D % 8 != 0;
    auto take = [&](int64_t n) {
        const size_t at = p.bytes;
        p.bytes += ((size_t)n + 255) & ~(size_t)255;
        return at;
    };
    if (p.pad) {
        p.x_at = take(es * planes * M * p.ldk);
        p.w_at = take(es * planes * V * p.ldk);
    }
    p.tiles_v = (V + 255) / 256;
    if (!backward) {
        p.part_at = take(8 * p.tiles_v * M);
        p.zsum_at = take(smooth ? 4 * p.tiles_v * M : 0);
        p.zt_at = take(4 * M);
        p.rows_at = take(reduction ? 4 * M : 0);
        return p;
    }
    if (p.wide) {  // two planes of x (without its ignored rows) and w
        p.x2_at = take(4 * M * p.ldk);
        p.w2_at = take(4 * V * p.ldk);
    } else if (!p.pad) {
        p.x_at = take(es * M * p.ldk);  // x without its ignored rows
    }
    p.rho_at = take(4 * M);
    p.factor_at = take(4);
    const int64_t fit = std::max<int64_t>(1, kCePiece / (es * terms * M * 256));
    p.pieces = (p.tiles_v + fit - 1) / fit;
    p.piece = (p.tiles_v + p.pieces - 1) / p.pieces * 256;  // classes
    if (p.piece > V) p.piece = (V + 7) & ~(int64_t)7;
    p.dz_at = take(terms * M * (es * p.piece + 256));
    p.col_at = take(4 * ((M + 31) / 32 + 8) * p.piece);
    // float32 partials, rows of whole 16 bytes
    p.ldp = (D + 3) & ~(int64_t)3;
    p.grad = ce_split(M, p.piece, D, ce_pairs(p), es);
    p.dx_at = take(p.grad.dx > 1 || p.pieces > 1 ? 4 * p.grad.dx * M * p.ldp : 0);
    p.dw_at = take(p.grad.dw > 1 ? 4 * p.grad.dw * p.piece * p.ldp : 0);
    return p;
}

static unsigned blocks_of(int64_t n) { return (unsigned)(n < 1 ? 1 : n > 16384 ? 16384 : n); }

template <int MODE>
static hipError_t ce_copy(const CePlan& p, const CeCall& c, const int64_t* target, const char* x, const char* w, hipStream_t s) {
    int lanes = 1;
    while (lanes < 64 && 8 * lanes < p.ldk) lanes *= 2;
    const CeCopy k = {{c.x, c.w},
                      {reinterpret_cast<uint16_t*>(const_cast<char*>(x)), reinterpret_cast<uint16_t*>(const_cast<char*>(w))},
                      {c.M, c.V},
                      c.D,
                      p.ldk,
                      target,
                      c.ignore,
                      lanes};
    hipLaunchKernelGGL(ce_copy_kernel<MODE>, dim3(blocks_of(((c.M + c.V) * lanes + 255) / 256)), dim3(256), 0, s, k);
    return hipGetLastError();
}

// The operands of the logits: as they are, or padded / split copies in `work`.
// target: rows of x that it ignores are zero there (backward).
static hipError_t ce_operands(const CePlan& p, const CeCall& c, const int64_t* target, char* wk, CeArgs& a, hipStream_t s) {
    a.kb = p.es * p.ldk;
    a.pairs = p.planes == 3 ? kPairs32 : 1;
    a.x = {reinterpret_cast<const char*>(c.x), a.kb, 0, c.M};
    a.w = {reinterpret_cast<const char*>(c.w), a.kb, 0, c.V};
    a.bias = c.bias;
    a.bias_dt = c.bias_dtype;
    a.target = c.target;
    a.M = c.M;
    a.V = c.V;
    a.smooth = c.smooth;
    a.ignore = c.ignore;
    if (!p.pad) return hipSuccess;
    a.x.p = wk + p.x_at;
    a.w.p = wk + p.w_at;
    a.x.plane = 2 * c.M * p.ldk;  // planes are 16-bit
    a.w.plane = 2 * c.V * p.ldk;
    return p.planes == 3 ? ce_copy<1>(p, c, target, a.x.p, a.w.p, s)
           : p.es == 4   ? ce_copy<2>(p, c, target, a.x.p, a.w.p, s)
                         : ce_copy<0>(p, c, target, a.x.p, a.w.p, s);
}

template <class K>
static hipError_t ce_lds(K kernel, int bytes, std::atomic<uint64_t>& done) {
    return set_lds_attr_once(reinterpret_cast<const void*>(kernel), bytes, done);
}

template <class Mma>
struct StatsGo {
    CeArgs& a;
    hipStream_t s;
    template <int MB, int WM, int S, int KB>
    hipError_t run() {
        using G = TileGemm<MB, WM, S, KB, false, false, Mma>;
        static std::atomic<uint64_t> done{0};
        const hipError_t e = ce_lds(&ce_stats_kernel<MB, WM, S, KB, Mma>, G::LDS + 1024, done);
        if (e != hipSuccess) return e;
        a.tiles_m = (int)((a.M + G::ROWS - 1) / G::ROWS);
        a.tiles_n = (int)((a.w.count + 255) / 256);
        a.group = tile_group(a.tiles_n, 256 * a.kb);
        hipLaunchKernelGGL((ce_stats_kernel<MB, WM, S, KB, Mma>), dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(G::THREADS),
                           G::LDS + 1024, s, a);
        return hipGetLastError();
    }
};

template <class Mma, int DT>
struct DzGo {
    CeArgs& a;
    int& col_rows;  // rows of column sums that the launch leaves
    hipStream_t s;
    template <int MB, int WM, int S, int KB>
    hipError_t run() {
        using G = TileGemm<MB, WM, S, KB, false, false, Mma>;
        constexpr int lds = G::LDS + (int)sizeof(CeLds<G::ROWS>);
        static std::atomic<uint64_t> done{0};
        const hipError_t e = ce_lds(&ce_dz_kernel<MB, WM, S, KB, Mma, DT>, lds, done);
        if (e != hipSuccess) return e;
        a.tiles_m = (int)((a.M + G::ROWS - 1) / G::ROWS);
        a.tiles_n = (int)((a.w.count + 255) / 256);
        a.group = tile_group(a.tiles_n, 256 * a.kb);
        col_rows = a.tiles_m * WM;
        hipLaunchKernelGGL((ce_dz_kernel<MB, WM, S, KB, Mma, DT>), dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(G::THREADS),
                           lds, s, a);
        return hipGetLastError();
    }
};

template <class Mma, int DT>
struct GradGo {
    CeGrads& a;
    hipStream_t s;
    template <int MB, int WM, int S, int KB>
    hipError_t run() {
        using X = TileGemm<MB, WM, S, KB, false, true, Mma>;
        using W = TileGemm<MB, WM, S, KB, true, true, Mma>;
        static_assert(X::LDS == W::LDS, "one launch");
        static std::atomic<uint64_t> done{0};
        const hipError_t e = ce_lds(&ce_grads_kernel<MB, WM, S, KB, Mma, DT>, X::LDS, done);
        if (e != hipSuccess) return e;
        double length[2];
        for (int k = 0; k < 2; ++k) {
            CeGrad& g = a.g[k];
            g.tiles_m = (int)((g.M + X::ROWS - 1) / X::ROWS);
            g.tiles_n = (int)((g.N + 255) / 256);
            a.units[k] = g.tiles_m * g.tiles_n * g.splits;
            length[k] = g.splits ? (double)(k ? W::steps(g.rk) : X::steps(g.rk)) / g.splits : 0.0;
        }
        a.first = length[1] > length[0];
        hipLaunchKernelGGL((ce_grads_kernel<MB, WM, S, KB, Mma, DT>), dim3((unsigned)(a.units[0] + a.units[1])),
                           dim3(X::THREADS), X::LDS, s, a);
        return hipGetLastError();
    }
};
static hipError_t ce_grads(int dt, const CePlan& p, CeGrads& g, hipStream_t s) {
    const TileForm form = p.grad.form;
    return p.terms == 1      ? tile_dispatch64(form, GradGo<MmaF32, RPFQ_F32>{g, s})
           : p.terms == 3    ? tile_dispatch64(form, GradGo<MmaBf16, RPFQ_F32>{g, s})
           : p.wide          ? tile_dispatch64(form, GradGo<MmaBf16, RPFQ_F16>{g, s})
           : dt == RPFQ_F16  ? tile_dispatch64(form, GradGo<MmaF16, RPFQ_F16>{g, s})
                             : tile_dispatch64(form, GradGo<MmaBf16, RPFQ_BF16>{g, s});
}

static CeSum ce_sum(int dt, const float* part, int parts, int64_t stride, int64_t rows, int64_t N, int64_t ldp, void* out) {
    const int es = dt == RPFQ_F32 ? 4 : 2;
    return {part, out, stride, rows, N, ldp, parts, dt, N % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * es) == 0,
            (int)blocks_of((rows * (ldp / 4) + 255) / 256)};
}

hipError_t launch_linear_ce(const CeCall& c, float* loss, float* stat, float* coef, void* work, hipStream_t s) {
    const CePlan p = ce_plan(c.dtype, c.M, c.V, c.D, c.reduction, c.smooth > 0.0f, false);
    char* wk = reinterpret_cast<char*>(work);
    CeArgs a = {};
    hipError_t e = ce_operands(p, c, nullptr, wk, a, s);
    if (e != hipSuccess) return e;
    a.part = reinterpret_cast<float2*>(wk + p.part_at);
    a.zsum = c.smooth > 0.0f ? reinterpret_cast<float*>(wk + p.zsum_at) : nullptr;
    a.zt = reinterpret_cast<float*>(wk + p.zt_at);
    const TileForm form = tile_form(c.M, c.V);
    e = p.es == 4              ? tile_dispatch(form, StatsGo<MmaF32>{a, s})
        : c.dtype == RPFQ_F16 ? tile_dispatch(form, StatsGo<MmaF16>{a, s})
                              : tile_dispatch(form, StatsGo<MmaBf16>{a, s});
    if (e != hipSuccess) return e;
    float* rows = c.reduction ? reinterpret_cast<float*>(wk + p.rows_at) : loss;
    const CeJoin j = {a.part, a.zsum, a.zt, c.target, c.M, c.V, c.ignore, (int)p.tiles_v, c.smooth, c.reduction, stat, rows, loss,
                      coef};
    // few rows: the sum over them by the same workgroup (one launch less, 4 us)
    if (c.reduction && c.M <= kCeFewRows) {
        hipLaunchKernelGGL(ce_join_kernel<true>, dim3(1), dim3(1024), 0, s, j);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(ce_join_kernel<false>, dim3((unsigned)((c.M + 63) / 64)), dim3(1024), 0, s, j);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (c.reduction) {
        hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, s, j);
        e = hipGetLastError();
    }
    return e;
}

hipError_t launch_linear_ce_grad(const CeCall& c, const float* stat, const float* coef, const float* grad, void* gx, void* gw,
                                 void* gb, void* work, hipStream_t s) {
    const CePlan p = ce_plan(c.dtype, c.M, c.V, c.D, c.reduction, c.smooth > 0.0f, true);
    char* wk = reinterpret_cast<char*>(work);
    const int es = c.dtype == RPFQ_F32 ? 4 : 2;
    CeArgs a = {};
    hipError_t e = ce_operands(p, c, c.target, wk, a, s);
    if (e != hipSuccess) return e;
    const float scale = c.dtype == RPFQ_F16 && !p.wide ? 32768.0f : 1.0f;
    CeFactor factor = {grad, c.reduction == 1 ? coef : nullptr, 1.0f / scale};
    if (c.reduction == 0) {
        float* rho = reinterpret_cast<float*>(wk + p.rho_at);
        float* top = reinterpret_cast<float*>(wk + p.factor_at);
        hipLaunchKernelGGL(ce_rho_kernel, dim3(1), dim3(1024), 0, s, grad, c.target, c.M, c.ignore, rho, top);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        a.rho = rho;
        factor.grad = top;
    }
    TileOperand xz = a.x, w2 = a.w;  // of the gradients' products; x's ignored rows as zeros
    if (p.wide) {
        xz.p = wk + p.x2_at;
        w2.p = wk + p.w2_at;
        xz.plane = 2 * c.M * p.ldk;
        w2.plane = 2 * c.V * p.ldk;
        if ((e = ce_copy<3>(p, c, c.target, xz.p, w2.p, s)) != hipSuccess) return e;
    } else if (gw && !p.pad) {
        xz.p = wk + p.x_at;
        a.xz = wk + p.x_at;
    }
    a.stat = stat;
    a.dz_scale = scale;
    a.dz = wk + p.dz_at;
    a.colsum = gb ? reinterpret_cast<float*>(wk + p.col_at) : nullptr;
    const TileOperand w = a.w;
    float* dxp = p.grad.dx > 1 || p.pieces > 1 ? reinterpret_cast<float*>(wk + p.dx_at) : nullptr;
    for (int64_t v0 = 0; v0 < c.V; v0 += p.piece) {
        const int64_t n = std::min(p.piece, c.V - v0);
        a.v0 = v0;
        a.w.p = w.p + v0 * w.ld;
        a.w.count = n;
        a.ldz = ce_ldz(n, p.es);
        a.n8 = (n + 7) & ~(int64_t)7;
        a.dz_plane = c.M * a.ldz;
        const TileForm form = tile_form(c.M, n);
        int col_rows = 0;
        e = p.terms == 1          ? tile_dispatch(form, DzGo<MmaF32, RPFQ_F32>{a, col_rows, s})
            : p.terms == 3        ? tile_dispatch(form, DzGo<MmaBf16, RPFQ_F32>{a, col_rows, s})
            : p.wide              ? tile_dispatch(form, DzGo<MmaF16, RPFQ_BF16>{a, col_rows, s})
            : c.dtype == RPFQ_F16 ? tile_dispatch(form, DzGo<MmaF16, RPFQ_F16>{a, col_rows, s})
                                  : tile_dispatch(form, DzGo<MmaBf16, RPFQ_BF16>{a, col_rows, s});
        if (e != hipSuccess) return e;
        a.xz = nullptr;  // written with the first piece
        const TileOperand dzk = {a.dz, a.ldz, a.dz_plane, c.M}, dzt = {a.dz, a.ldz, a.dz_plane, n};
        CeGrads both = {};
        CeGrad &dx = both.g[0], &dw = both.g[1];
        dx.pairs = dw.pairs = ce_pairs(p);
        dx.N = dw.N = c.D;
        dx.ldp = dw.ldp = p.ldp;
        dx.factor = dw.factor = factor;
        dx.r = dzk;
        dx.c = {w2.p + v0 * w2.ld, w2.ld, w2.plane, p.ldk};
        dx.rk = p.es * a.n8;
        dx.ck = n;
        dx.M = c.M;
        dx.splits = gx ? p.grad.dx : 0;
        dx.part = dxp;
        dx.add = v0 > 0;
        dx.out = gx;
        dx.vec = c.D % 4 == 0 && reinterpret_cast<uintptr_t>(gx) % (4 * es) == 0;
        dw.r = dzt;
        dw.c = {xz.p, xz.ld, xz.plane, p.ldk};
        dw.rk = dw.ck = c.M;
        dw.M = n;
        dw.splits = gw ? p.grad.dw : 0;
        dw.part = p.grad.dw > 1 ? reinterpret_cast<float*>(wk + p.dw_at) : nullptr;
        dw.out = gw ? reinterpret_cast<char*>(gw) + v0 * c.D * es : nullptr;
        dw.vec = c.D % 4 == 0 && reinterpret_cast<uintptr_t>(dw.out) % (4 * es) == 0;
        if ((gx || gw) && (e = ce_grads(c.dtype, p, both, s)) != hipSuccess) return e;
        CeSums sums = {{}, factor};
        int jobs = 0, blocks = 0;
        auto add = [&](const CeSum& j) {
            sums.s[jobs++] = j;
            blocks += j.blocks;
        };
        if (gw && dw.part) add(ce_sum(c.dtype, dw.part, dw.splits, n * p.ldp, n, c.D, p.ldp, dw.out));
        if (gx && dxp && v0 + n == c.V) add(ce_sum(c.dtype, dxp, p.grad.dx, c.M * p.ldp, c.M, c.D, p.ldp, gx));
        if (gb)  // the column sums of the row tiles, as one row each
            add(ce_sum(c.bias_dtype, a.colsum, col_rows, a.n8, 1, n, a.n8,
                       reinterpret_cast<char*>(gb) + v0 * (c.bias_dtype == RPFQ_F32 ? 4 : 2)));
        if (jobs) {
            hipLaunchKernelGGL(ce_sums_kernel, dim3((unsigned)blocks), dim3(256), 0, s, sums);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace rpfq
