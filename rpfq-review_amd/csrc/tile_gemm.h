// Tile product of two row-major operands on the matrix cores, shared by the
// int8 layer and the classifier's loss: C[rows, cols] = sum_k R[.., k] C[.., k],
// either operand lying with k contiguous ("K": rows of k) or with its own index
// contiguous ("T": one row per k).  16-bit floats or int8, 32-bit sums.
#pragma once

#include "rpfq_device.h"

namespace rpfq {

typedef int intx16 __attribute__((ext_vector_type(16)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s4_t;
typedef __attribute__((address_space(3))) const intx4* lds_i4_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The 32 x 32 products: 32 bytes of k a row (16 halves, 32 int8).
struct MmaF16 {
    using acc_t = floatx16;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
};
struct MmaBf16 {
    using acc_t = floatx16;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct MmaI8 {
    using acc_t = intx16;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
    }
};

// One operand of a product.  K layout: `count` rows of `k_bytes` at p + row ld.
// T layout: k rows at p + k ld of `count` 2-byte elements.  p, ld, k_bytes (K)
// and 2 count (T) are multiples of 16 bytes.  Planes (float32 as three bf16
// terms) lie `plane` bytes apart.
struct TileOperand {
    const char* p;
    int64_t ld;
    int64_t plane;
    int64_t count;
};

// float32 products as bf16 ones: v = h + m + l exactly (8 bits each), and of
// the nine products the six above 2^-24, smallest first.  The terms keep
// float32's exponents, so no scales are needed; 6 x the cost of one.
constexpr int kPairs32 = 6;
__device__ __forceinline__ void tile_pair(int pair, int& r, int& c) {
    // (l,h) (h,l) (m,m) (m,h) (h,m) (h,h); planes h = 0, m = 1, l = 2
    r = (0x001102 >> (4 * pair)) & 3;
    c = (0x010120 >> (4 * pair)) & 3;
}

// LDS DMA through a buffer resource: lanes with an offset past its end write
// zeros.  Asm for the reason given at dma_dwordx4; the same waits apply.  The
// wait states cover a resource whose words a VALU instruction has just written.
__device__ __forceinline__ void dma_buffer(intx4 rsrc, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc)
                 : "memory", "m0");
}
__device__ __forceinline__ intx4 tile_rsrc(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return (intx4){__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)),
                   0x7fffffff, 0x00027000};
}
constexpr uint32_t kTileOut = 0x80000000u;  // an offset past every resource's end

// W elements of one operand (a tile's rows or columns), 64 bytes of k a step.
// K layout in LDS: W rows of 64 B, chunk c of 16 B at c ^ ((row >> 2) & 3), so 16
// rows of one chunk (a read of half a wave) fall on all 64 banks once.  T
// layout: 32 k rows of 2 W bytes, chunk c at c ^ ((k & 3) << 2) (64 columns: c ^
// (k & 2) << 1): the 4 rows x 64 B of a transposed read on distinct banks.
template <int W, bool T>
struct TileSide {
    static constexpr int BYTES = W * 64;
    static constexpr int LOADS = W / 64;        // DMA loads per wave and step, 1 KB each
    static constexpr int CH = W / 8;            // T: chunks of a k row
    uint32_t v[LOADS];
    uint32_t kpos[LOADS];  // K: byte of k within a step; T: k row within a step
    const char* base;
    int64_t ld, plane;

    static __device__ __forceinline__ int swz(int k) { return CH >= 16 ? (k & 3) << 2 : (k & 2) << 1; }

    __device__ __forceinline__ void init(const TileOperand& o, int64_t first, int wave, int lane) {
        ld = o.ld;
        plane = o.plane;
        base = o.p + (T ? first * 2 : first * o.ld);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int piece = wave * LOADS + j;
            if (T) {
                const int k = piece * (64 / CH) + lane / CH, c = (lane % CH) ^ swz(k);
                kpos[j] = (uint32_t)k;
                v[j] = first + 8 * c < o.count ? (uint32_t)(k * o.ld + c * 16) : kTileOut;
            } else {
                const int row = piece * 16 + (lane >> 2), c = (lane & 3) ^ ((lane >> 4) & 3);
                kpos[j] = (uint32_t)(c * 16);
                v[j] = first + row < o.count ? (uint32_t)(row * o.ld + c * 16) : kTileOut;
            }
        }
    }
    // step `ks` of plane pl (k: bytes of a row (K) or rows (T)) to LDS at `lds`
    __device__ __forceinline__ void issue(int ks, int pl, int64_t k, uint32_t lds, int wave) {
        const intx4 rs = tile_rsrc(base + pl * plane + (T ? (int64_t)ks * 32 * ld : (int64_t)ks * 64));
        const int64_t left64 = T ? k - (int64_t)ks * 32 : k - (int64_t)ks * 64;
        const uint32_t left = (uint32_t)(left64 > 64 ? 64 : left64);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) dma_buffer(rs, kpos[j] < left ? v[j] : kTileOut, lds + (wave * LOADS + j) * 1024);
    }
    // where lane l reads block 0 of substep 0; frag() adds the rest
    static __device__ __forceinline__ uint32_t at(int lane) {
        const int r = lane & 31, g = lane >> 5;
        if (!T) return (uint32_t)(r * 64 + ((g ^ ((r >> 2) & 3)) * 16));
        const int i16 = lane & 15, hf = (lane >> 4) & 1, k = 8 * g + (i16 >> 2);
        return (uint32_t)(k * 2 * W + ((2 * hf + ((i16 & 3) >> 1)) * 16) + (i16 & 1) * 8);
    }
    // 16 bytes of k of the lane's element of block b (32 elements), substep s
    static __device__ __forceinline__ uint4 frag(uint32_t stage, uint32_t at, int b, int s, int lane) {
        if (!T) {
            // chunk 2 s + g: the swizzle is an xor, so substep 1 flips bit 1
            return __builtin_bit_cast(uint4, *((lds_i4_t)(stage + (at ^ (uint32_t)(s * 32)) + b * 2048)));
        } else {
            const int k = (lane & 15) >> 2;  // modulo 4: what the swizzle looks at
            const uint32_t a = stage + ((at + b * 64) ^ (uint32_t)(swz(k) * 16)) + s * 32 * W;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)a);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(a + 8 * W));
            return __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// Workgroup of 4 waves: 32 MB rows x 256 columns, wave w the columns 64 w ..
// 64 w + 63 of every row, acc[j][i] the 32 x 32 block of columns 32 j and rows
// 32 i: lane (r, g) holds row r and columns acc_row(v, g).  Both operands go
// global -> LDS by DMA, three stages of 64 bytes of k, two steps ahead; two
// workgroups share a CU, so one's epilogue runs beside the other's products.
template <int MB, bool RT, bool CT, class Mma>
struct TileGemm {
    static constexpr int RW = MB == 1 ? 64 : 32 * MB;  // rows of R loaded (64 at least: one DMA load a wave)
    using R = TileSide<RW, RT>;
    using C = TileSide<256, CT>;
    using acc_t = typename Mma::acc_t;
    static constexpr int STAGE = R::BYTES + C::BYTES;
    static constexpr int LDS = 3 * STAGE;
    static constexpr int LOADS = R::LOADS + C::LOADS;

    // Adds steps s0 .. s1 - 1 of the product; a step is 64 bytes of k of one
    // pair of planes, `per` steps a pair.  rk, ck: k of the operands as issue() takes it.
    static __device__ __forceinline__ void run(const TileOperand& ro, const TileOperand& co, int64_t m0, int64_t n0,
                                               int64_t rk, int64_t ck, int per, bool planes, int s0, int s1, char* smem,
                                               int wave, int lane, acc_t (&acc)[2][MB]) {
        R rs;
        C cs;
        rs.init(ro, m0, wave, lane);
        cs.init(co, n0, wave, lane);
        const uint32_t lds = lds_addr(smem);
        int pair = s0 / per, ks = s0 - pair * per;
        auto issue = [&](int st) {
            int rp = 0, cp = 0;
            if (planes) tile_pair(pair, rp, cp);
            rs.issue(ks, rp, rk, lds + st * STAGE, wave);
            cs.issue(ks, cp, ck, lds + st * STAGE + R::BYTES, wave);
            if (++ks == per) {
                ks = 0;
                ++pair;
            }
        };
        const uint32_t ra = R::at(lane), ca = C::at(lane);
        if (s0 < s1) issue(0);
        if (s0 + 1 < s1) issue(1);
        auto step = [&](int s, int st) {
            if (s + 1 < s1)
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s + 2 < s1) issue((st + 2) % 3);  // read a step ago, by every wave
            const uint32_t rst = lds + st * STAGE, cst = rst + R::BYTES;
            uint4 c0[2], c1[2], r0[MB], r1[MB];
#pragma unroll
            for (int j = 0; j < 2; ++j) c0[j] = C::frag(cst, ca, 2 * wave + j, 0, lane);
#pragma unroll
            for (int i = 0; i < MB; ++i) r0[i] = R::frag(rst, ra, i, 0, lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) c1[j] = C::frag(cst, ca, 2 * wave + j, 1, lane);
#pragma unroll
            for (int i = 0; i < MB; ++i) r1[i] = R::frag(rst, ra, i, 1, lane);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[j][i] = Mma::mma(c0[j], r0[i], acc[j][i]);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[j][i] = Mma::mma(c1[j], r1[i], acc[j][i]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        };
        int s = s0;
        for (; s + 3 <= s1; s += 3) {
            step(s, 0);
            step(s + 1, 1);
            step(s + 2, 2);
        }
        if (s < s1) step(s, 0);
        if (s + 1 < s1) step(s + 1, 1);
        __builtin_amdgcn_s_barrier();  // the stages are free for the epilogue
        asm volatile("" ::: "memory");
    }
};

// One wave's 32 x 64 block through 8 KB of LDS of its own: put(v) takes the
// accumulators' values, then out(row, column, 4 values) is called for whole
// 256-byte pieces of rows (16 lanes a row, 4 columns each).
template <class Acc, class F, class Out>
__device__ __forceinline__ void tile_rows(char* epi, const Acc& a0, const Acc& a1, int lane, F value, Out out) {
    const int r = lane & 31, g = lane >> 5, c = lane & 15, row4 = lane >> 4;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 v;
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = value((j ? a1 : a0)[4 * q + t], 32 * j + 8 * q + 4 * g + t);
            *reinterpret_cast<f32x4*>(epi + r * 256 + (((8 * j + 2 * q + g) ^ (r & 15)) * 16)) = v;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int row = 4 * j + row4;
        out(row, 4 * c, *reinterpret_cast<const f32x4*>(epi + row * 256 + ((c ^ (row & 15)) * 16)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}
constexpr int kTileEpi = 8192;  // a wave's LDS in tile_rows

// 4 values to columns n .. n + 3 of a row of N (those below N): one store
// where `vec` says that rows are 4-element aligned.
template <int YDT>
__device__ __forceinline__ void tile_store4(void* y, int64_t row_off, int64_t n, int64_t N, bool vec, f32x4 v) {
    if (vec) {
        if (n >= N) return;
        if constexpr (YDT == RPFQ_F32) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(y) + row_off + n) = v;
        } else {
            uint2 o;
            o.x = YDT == RPFQ_F16 ? cvt_pk(v[0], v[1]) : pack_bf2(v[0], v[1]);
            o.y = YDT == RPFQ_F16 ? cvt_pk(v[2], v[3]) : pack_bf2(v[2], v[3]);
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(y) + row_off + n) = o;
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (n + t < N) store1<YDT>(y, row_off + n + t, v[t]);
}

}  // namespace rpfq
