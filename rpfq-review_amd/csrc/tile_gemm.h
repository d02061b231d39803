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

// The 32 x 32 products: 32 bytes of k a row (16 halves, 32 int8, 8 floats), ES
// bytes an element.
struct MmaF16 {
    using acc_t = floatx16;
    static constexpr int ES = 2;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
};
struct MmaBf16 {
    using acc_t = floatx16;
    static constexpr int ES = 2;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct MmaI8 {
    using acc_t = intx16;
    static constexpr int ES = 1;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
    }
};

// float32 as it is, 1/16 of the 16-bit rate: lane (r, g) holds k = 4 (2 s + g) + t
// in both operands, one of them a step.
struct MmaF32 {
    using acc_t = floatx16;
    static constexpr int ES = 4;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[t], y[t], c, 0, 0, 0);
        return c;
    }
};

// One operand of a product.  K layout: `count` rows of `k_bytes` at p + row ld.
// T layout: k rows at p + k ld of `count` elements.  p, ld, k_bytes (K) and the
// bytes of count (T) are multiples of 16.  Planes (float32 as three bf16
// terms, or as two of 16 bits) lie `plane` bytes apart.
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
// fp16 products as bf16 ones, where the other operand's exponents pass fp16's: a
// fp16 is two bf16 terms exactly, the other side two terms of its own; (l,h)
// (h,l) (h,h), without the one below 2^-16.
constexpr int kPairsHalf = 3;
__device__ __forceinline__ void tile_pair(int pairs, int pair, int& r, int& c) {
    // (l,h) (h,l) (m,m) (m,h) (h,m) (h,h); planes h = 0, m = 1, l = 2
    r = ((pairs == kPairs32 ? 0x001102 : 0x001) >> (4 * pair)) & 3;
    c = ((pairs == kPairs32 ? 0x010120 : 0x010) >> (4 * pair)) & 3;
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

// W elements of one operand (a tile's rows or columns), KB bytes of k a step.
// K layout in LDS: W rows of KB bytes, chunk c of 16 at c ^ ((row >> 2) & 3) (KB =
// 64) or c ^ ((row >> 1) & 7) (128): 16 rows of one chunk, what half a wave's
// read takes, fall on all 64 banks once (5.7 clocks a 1-KB read, 16 to 32
// unswizzled).  T layout: KB / 2 k rows of 2 W bytes, chunk c at c ^ ((k & 3) <<
// 2) (64 columns: c ^ (k & 2) << 1): the 4 rows x 64 B of a transposed read on
// distinct banks.  T layout of float32: KB / 4 rows of 4 W bytes, read a value at
// a time; chunk c at c ^ 8 where k & 4, so the two halves of a wave, four rows
// apart, fall on different banks.
template <int W, bool T, int WAVES, int KB, int ES>
struct TileSide {
    static constexpr int BYTES = W * KB;
    static constexpr int LOADS = W * KB / 1024 / WAVES;  // DMA loads per wave and step, 1 KB each
    static constexpr int CH = W * ES / 16;               // T: chunks of a k row
    static constexpr int PER = T ? KB / ES : KB;         // k of a step: rows (T) or bytes of a row
    static constexpr int KC = KB / 16;                   // K: chunks of a row
    uint32_t v[LOADS];
    uint32_t kpos[LOADS];  // K: byte of k within a step; T: k row within a step
    const char* base;
    int64_t ld, plane;

    static __device__ __forceinline__ int swz(int k) { return ES == 4 ? (k & 4) << 1 : CH >= 16 ? (k & 3) << 2 : (k & 2) << 1; }
    static __device__ __forceinline__ int kswz(int row) { return KC == 4 ? (row >> 2) & 3 : (row >> 1) & 7; }

    __device__ __forceinline__ void init(const TileOperand& o, int64_t first, int wave, int lane) {
        ld = o.ld;
        plane = o.plane;
        base = o.p + (T ? first * ES : first * o.ld);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int piece = wave * LOADS + j;
            if (T) {
                const int k = piece * (64 / CH) + lane / CH, c = (lane % CH) ^ swz(k);
                kpos[j] = (uint32_t)k;
                v[j] = first + (16 / ES) * c < o.count ? (uint32_t)(k * o.ld + c * 16) : kTileOut;
            } else {
                const int row = piece * (64 / KC) + lane / KC, c = (lane % KC) ^ kswz(row);
                kpos[j] = (uint32_t)(c * 16);
                v[j] = first + row < o.count ? (uint32_t)(row * o.ld + c * 16) : kTileOut;
            }
        }
    }
    // step `ks` of plane pl (k: bytes of a row (K) or rows (T)) to LDS at `lds`
    __device__ __forceinline__ void issue(int ks, int pl, int64_t k, uint32_t lds, int wave) {
        const intx4 rs = tile_rsrc(base + pl * plane + (T ? (int64_t)ks * PER * ld : (int64_t)ks * PER));
        const int64_t left64 = k - (int64_t)ks * PER;
        const uint32_t left = (uint32_t)(left64 > PER ? PER : left64);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) dma_buffer(rs, kpos[j] < left ? v[j] : kTileOut, lds + (wave * LOADS + j) * 1024);
    }
    // where lane l reads block 0 of substep s of a stage at 0
    static __device__ __forceinline__ uint32_t at(int lane, int s) {
        const int r = lane & 31, g = lane >> 5;
        if (!T) return (uint32_t)(r * KB + (((2 * s + g) ^ kswz(r)) * 16));
        if (ES == 4) return (uint32_t)(4 * g * 4 * W + r * 4);
        const int i16 = lane & 15, hf = (lane >> 4) & 1, k = 8 * g + (i16 >> 2);
        return (uint32_t)(k * 2 * W + ((2 * hf + ((i16 & 3) >> 1)) * 16) + (i16 & 1) * 8);
    }
    // 16 bytes of k of the lane's element of block b (32 elements), substep s
    static __device__ __forceinline__ uint4 frag(uint32_t stage, const uint32_t (&at)[KB / 32], int b, int s, int lane) {
        if (!T) {
            uint32_t a = stage + at[s];
            // one register and 16-bit offsets from it: for addresses past 64 KB
            // the compiler took 8-byte reads instead (1,050 -> 1,290 TFLOP/s)
            asm("" : "+v"(a));
            return __builtin_bit_cast(uint4, *((lds_i4_t)a + b * 2 * KB));
        } else if constexpr (ES == 4) {
            const uint32_t a = stage + ((at[0] + b * 128) ^ (uint32_t)(lane >> 5 << 7)) + s * 32 * W;
            uint32_t v[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = *((lds_u32_t)(a + t * 4 * W));
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            const int k = (lane & 15) >> 2;  // modulo 4: what the swizzle looks at
            const uint32_t a = stage + ((at[0] + b * 64) ^ (uint32_t)(swz(k) * 16)) + s * 32 * W;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)a);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(a + 8 * W));
            return __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// Workgroup of 4 WM waves: 32 MB WM rows x 256 columns, wave w the columns 64
// (w % 4) .. + 63 of rows 32 MB (w / 4) .. + 32 MB - 1, acc[j][i] the 32 x 32
// block of its columns 32 j and rows 32 i: lane (r, g) holds row r and columns
// acc_row(v, g).  Both operands go global -> LDS by DMA, in S stages of KB bytes
// of k, S - 1 steps ahead (S = 2: two).  The forms that are used (bf16, normal
// operands, K layouts, the products alone; 8192 x 65536 x 768 / 8192^3):
//   256 x 256, KB 128, S 2, one workgroup a CU: 1,213 / 1,290 TFLOP/s, and
//     1,090 / 1,180 where a step begins with its first reads.  Half the LDS
//     fill per product of a 128-row tile, which is bound by it (48 of 64 bytes
//     a clock from the vector cache at full matrix rate).  Four waves of 128 x
//     128 instead of eight of 128 x 64 read less LDS, but a wave alone on its
//     SIMD waits more: 1,146 / 1,227;
//   128 x 256, KB 64, S 3, two a CU: 1,058 / 1,021 (steps overlapped 1,054 /
//     1,010);
//   64 x 256 and 128 x 256 of eight waves, KB 128, S 3, one a CU: launches of
//     fewer tiles than CUs (333 x 10,007 x 2,496: 27 and 34 us; four waves with
//     S 6 of 64 bytes 40 and 43).
template <int MB, int WM, int S, int KB, bool RT, bool CT, class Mma>
struct TileGemm {
    static constexpr int WAVES = 4 * WM, THREADS = 64 * WAVES, ROWS = 32 * MB * WM;
    static constexpr int RW = ROWS < 64 ? 64 : ROWS;  // rows of R loaded: one DMA load a wave at least
    using R = TileSide<RW, RT, WAVES, KB, Mma::ES>;
    using C = TileSide<256, CT, WAVES, KB, Mma::ES>;
    using acc_t = typename Mma::acc_t;
    static constexpr int SUB = KB / 32;
    static constexpr int STAGE = R::BYTES + C::BYTES;
    static constexpr int LDS = S * STAGE;
    static constexpr int LOADS = R::LOADS + C::LOADS;
    // steps of R's k (bytes of a row in K layout, rows in T)
    static constexpr int64_t steps(int64_t k) { return (k + R::PER - 1) / R::PER; }

    // Adds steps s0 .. s1 - 1 of the product; a step is KB bytes of k of one
    // pair of planes, `per` steps a pair.  pairs: those of tile_pair, or R's
    // planes, 1 or 2, beside one of C, the second first.  rk, ck: k of the
    // operands as issue() takes it.  meanwhile(): what the epilogue wants in LDS
    // past the stages, loaded while the first steps are on their way (s0 < s1).
    template <class F>
    static __device__ __forceinline__ void run(const TileOperand& ro, const TileOperand& co, int64_t m0, int64_t n0,
                                               int64_t rk, int64_t ck, int per, int pairs, int s0, int s1, char* smem,
                                               int wave, int lane, acc_t (&acc)[2][MB], F meanwhile) {
        R rs;
        C cs;
        rs.init(ro, m0, wave, lane);
        cs.init(co, n0, wave, lane);
        const uint32_t lds = lds_addr(smem);
        const int wc = wave & 3, wr = wave >> 2;
        int pair = s0 / per, ks = s0 - pair * per;
        auto issue = [&](int st) {
            int rp = pairs - 1 - pair, cp = 0;
            if (pairs >= kPairsHalf) tile_pair(pairs, pair, rp, cp);
            rs.issue(ks, rp, rk, lds + st * STAGE, wave);
            cs.issue(ks, cp, ck, lds + st * STAGE + R::BYTES, wave);
            if (++ks == per) {
                ks = 0;
                ++pair;
            }
        };
        uint32_t ra[SUB], ca[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) ra[u] = R::at(lane, u), ca[u] = C::at(lane, u);
        uint4 cf[2][2], rf[2][MB];  // of a substep and the next
        auto read = [&](int st, int u, int p) {
            const uint32_t rst = lds + st * STAGE, cst = rst + R::BYTES;
#pragma unroll
            for (int j = 0; j < 2; ++j) cf[p][j] = C::frag(cst, ca, 2 * wc + j, u, lane);
#pragma unroll
            for (int i = 0; i < MB; ++i) rf[p][i] = R::frag(rst, ra, MB * wr + i, u, lane);
        };
        auto products = [&](int p) {
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[j][i] = Mma::mma(cf[p][j], rf[p][i], acc[j][i]);
            __builtin_amdgcn_sched_barrier(0);
        };
        // waits for the DMA of all but the last `behind` steps, and for every wave's
        auto landed = [&](auto behind) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(behind)::value * LOADS) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        using std::integral_constant;
        if constexpr (S == 2) {
            // The steps overlap: while a step's last products run, the next one's
            // first operands are read and the stage is filled again.
            if (s0 == s1) return;
            issue(0);
            if (s0 + 1 < s1) issue(1);
            meanwhile();
            if (s0 + 1 < s1) landed(integral_constant<int, 1>());
            else landed(integral_constant<int, 0>());
            read(0, 0, 0);
            auto step = [&](int s, int st) {
#pragma unroll
                for (int u = 0; u + 1 < SUB; ++u) {
                    read(st, u + 1, (u + 1) & 1);
                    products(u & 1);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                landed(integral_constant<int, 0>());
                if (s + 1 < s1) read(st ^ 1, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (s + 2 < s1) issue(st);
                products((SUB - 1) & 1);
            };
            int s = s0;
            for (; s + 2 <= s1; s += 2) {
                step(s, 0);
                step(s + 1, 1);
            }
            if (s < s1) step(s, 0);
        } else {
#pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (s0 + i < s1) issue(i);
            meanwhile();
            auto step = [&](int s, int st) {
                // the steps behind s may still be on their way
                if (s + S - 2 < s1) landed(integral_constant<int, S - 2>());
                else landed(integral_constant<int, 0>());
                if (s + S - 1 < s1) issue((st + S - 1) % S);  // read a step ago, by every wave
                read(st, 0, 0);
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    if (u + 1 < SUB) read(st, u + 1, (u + 1) & 1);
                    products(u & 1);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            };
            int s = s0;
            for (; s + S <= s1; s += S)
#pragma unroll
                for (int i = 0; i < S; ++i) step(s + i, i);
#pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (s + i < s1) step(s + i, i);
            __builtin_amdgcn_s_barrier();  // the stages are free for the epilogue
            asm volatile("" ::: "memory");
        }
    }
};

// The form of a launch of M x N outputs: one round of the chip on the smallest
// tiles that fill it (64 rows, 32 for few rows; a step there waits on its DMA
// and not on the products), else the cheaper of 128- and 256-row tiles, whose
// rounds cost 1.15 to 1 (bf16 products).
inline TileForm tile_form(int64_t M, int64_t N) {
    const int64_t cus = device_cus(), tn = (N + 255) / 256;
    if (M <= 32) return kTile32;
    if ((M + 63) / 64 * tn <= cus) return kTile64;
    const int64_t t128 = (M + 127) / 128 * tn, t256 = (M + 255) / 256 * tn;
    if (t128 <= cus) return kTile128Deep;
    return 20 * ((t256 + cus - 1) / cus) <= 23 * ((t128 + 2 * cus - 1) / (2 * cus)) ? kTile256 : kTile128;
}
// go.run<MB, WM, S, KB>() of a form of 64 rows or more, or of any
template <class Go>
inline hipError_t tile_dispatch64(TileForm f, Go go) {
    switch (f) {
        case kTile64: return go.template run<1, 2, 3, 128>();
        case kTile128Deep: return go.template run<2, 2, 3, 128>();
        case kTile128: return go.template run<4, 1, 3, 64>();
        default: return go.template run<4, 2, 2, 128>();
    }
}
template <class Go>
inline hipError_t tile_dispatch(TileForm f, Go go) {
    return f == kTile32 ? go.template run<1, 1, 3, 128>() : tile_dispatch64(f, go);
}

// One wave's 32 x 64 block through 8 KB of LDS of its own: value(v, column)
// makes the accumulators' values, then out(row, column, 4 values) is called for
// whole 256-byte pieces of rows (16 lanes a row, 4 columns each).
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

// The same with 8 columns a lane: out(row, column, 4 values, the 4 behind them).
template <class Acc, class Out>
__device__ __forceinline__ void tile_rows8(char* epi, const Acc& a0, const Acc& a1, int lane, Out out) {
    const int r = lane & 31, g = lane >> 5, c = lane & 7, row8 = lane >> 3;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const Acc& a = j ? a1 : a0;
            const f32x4 v = {a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
            *reinterpret_cast<f32x4*>(epi + r * 256 + (((8 * j + 2 * q + g) ^ (r & 15)) * 16)) = v;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = 8 * j + row8;
        const char* from = epi + row * 256;
        out(row, 8 * c, *reinterpret_cast<const f32x4*>(from + (((2 * c) ^ (row & 15)) * 16)),
            *reinterpret_cast<const f32x4*>(from + (((2 * c + 1) ^ (row & 15)) * 16)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// The same for 16-bit outputs, half the LDS: value4(4 values, column) packs four
// columns to 8 bytes, out(row, column, 8 values) stores 128-byte pieces.
__device__ __forceinline__ int tile_half_at(int r, int c) { return r * 128 + (((c >> 3) ^ ((r >> 1) & 7)) * 16) + (c & 7) * 2; }
template <class Acc, class F, class Out>
__device__ __forceinline__ void tile_rows_half(char* epi, const Acc& a0, const Acc& a1, int lane, F value4, Out out) {
    const int r = lane & 31, g = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = 32 * j + 8 * q + 4 * g;
            const Acc& a = j ? a1 : a0;
            *reinterpret_cast<uint2*>(epi + tile_half_at(r, c)) = value4(a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3], j, q);
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = 8 * j + (lane >> 3), c = 8 * (lane & 7);
        out(row, c, *reinterpret_cast<const uint4*>(epi + tile_half_at(row, c)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}
constexpr int kTileEpi = 8192;  // a wave's LDS in tile_rows

template <int YDT>
__device__ __forceinline__ uint32_t tile_pack2(float a, float b) {
    return YDT == RPFQ_F16 ? cvt_pk(a, b) : pack_bf2(a, b);
}

// 4 values to columns n .. n + 3 of a row of N (those below N): one store
// where `vec` says that rows are 4-element aligned.
template <int YDT>
__device__ __forceinline__ void tile_store4(void* y, int64_t row_off, int64_t n, int64_t N, bool vec, f32x4 v) {
    if (vec) {
        if (n >= N) return;
        if constexpr (YDT == RPFQ_F32) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(y) + row_off + n) = v;
        } else {
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(y) + row_off + n) =
                make_uint2(tile_pack2<YDT>(v[0], v[1]), tile_pack2<YDT>(v[2], v[3]));
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (n + t < N) store1<YDT>(y, row_off + n + t, v[t]);
}

// 8 16-bit values to columns n .. n + 7 of a row of N (those below N): one store
// where `vec` says that rows are 16-byte aligned, past the caches where it is 2.
__device__ __forceinline__ void tile_store8(void* y, int64_t row_off, int64_t n, int64_t N, int vec, uint4 v) {
    uint16_t* d = reinterpret_cast<uint16_t*>(y) + row_off + n;
    if (vec) {
        if (n >= N) return;
        if (vec == 2) __builtin_nontemporal_store(__builtin_bit_cast(intx4, v), reinterpret_cast<intx4*>(d));
        else *reinterpret_cast<uint4*>(d) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int t = 0; t < 8; ++t)
        if (n + t < N) d[t] = (uint16_t)(w[t >> 1] >> (16 * (t & 1)));
}

}  // namespace rpfq
