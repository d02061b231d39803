// Attention with a sliding window and first tokens that stay visible (sinks),
// over whole sequences with its gradient, and for the last tokens over a cache.
// Query i sees key j of its sequence where
//   causal:  j <= i and (i - j < window or j < sinks),
//   else:    |i - j| < window or j < sinks or i < sinks;
//   O = P V,  P = softmax(scale Q K^T) over what is seen, 0 for a row without any.
// Gradient, with P formed again from two numbers a row, a score and log2 of the
// sum relative to it: P = exp2((S - top) scale2 - lg), scale2 = scale log2(e).
// Their sum in one number would be rounded at the scores' size, and P with it.
//   dV = P^T dO,  dS = P (dO V^T - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q.
#include "tile_gemm.h"

#include <type_traits>
#include <utility>

namespace rpfq {

// A tile's rows in LDS: DP values of 16 bits (the head's size, rounded up to
// 32; zeros behind it), chunks of 16 bytes.  Chunk c lies at c ^ swz(row): both
// reads below fall on all banks, 16 rows of one chunk (a 32 x 32 product's rows)
// and 4 rows x 64 bytes (the transposed read).
template <int DP>
struct Rows {
    static constexpr int RB = DP <= 32 ? 64 : DP <= 64 ? 128 : 256;  // bytes of a row
    static constexpr int CH = RB / 16;
    static constexpr int PER = 1024 / RB;  // rows of one DMA load
    static __device__ __forceinline__ int swz(int row) {
        return CH == 16 ? (row & 3) << 2 | ((row >> 2) & 3) : CH == 8 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row >> 2) & 3;
    }
};

// The loads of a tile of R rows by WAVES waves: rows of `ld` bytes, `left` of them
// from the tile's first on; rows behind those and chunks past D as zeros.  The
// scalar sums of an address are kept from tile to tile.
template <int DP, int R, int WAVES>
struct RowLoads {
    static constexpr int TOTAL = R / Rows<DP>::PER, LOADS = (TOTAL + WAVES - 1) / WAVES;
    static_assert(LOADS == 1 || WAVES * Rows<DP>::PER % 16 == 0, "a wave's loads lie alike");
    uint32_t off;  // of load 0; load p is WAVES p PER rows on
    uint64_t at;
    int ld, left, bytes;
    __device__ __forceinline__ void init(int64_t row_bytes, int D, int wave, int lane) {
        ld = (int)row_bytes;
        bytes = 2 * D;
        const int row = wave * Rows<DP>::PER + lane / Rows<DP>::CH, c = (lane & (Rows<DP>::CH - 1)) ^ Rows<DP>::swz(row);
        off = 8 * c < D ? (uint32_t)(row * ld + 16 * c) : kTileOut;
    }
    // to rows first .. of a tensor whose rows 0 .. n - 1 count
    __device__ __forceinline__ void seek(const char* base, int first, int n) {
        at = reinterpret_cast<uint64_t>(base) + (uint64_t)first * (uint32_t)ld;
        left = n - first;
    }
    // the tile's resource
    intx4 rsrc;
    __device__ __forceinline__ void resource() {
        const int rows = left < R ? left : R;
        rsrc = (intx4){__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)((at >> 32) & 0xffff)),
                       __builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * ld + bytes : 0), 0x00027000};
        asm volatile("" : "+v"(off));  // the loads' own sums stay in the loop: a register, not one each
    }
    // and on to the tile behind it
    __device__ __forceinline__ void next() {
        resource();
        at += (uint32_t)(R * ld);
        left -= R;
    }
    __device__ __forceinline__ void load(int p, uint32_t lds, int wave) const {
        if (TOTAL % WAVES && wave + p * WAVES >= TOTAL) return;
        const uint32_t to = lds + (wave + p * WAVES) * 1024;
        const uint32_t from = off + (uint32_t)(p * WAVES * Rows<DP>::PER * ld);
        if (p == 0) dma_buffer(rsrc, from, to);  // waits for the resource's words, for all of them
        else asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(from), "s"(rsrc) : "memory", "m0");
    }
    __device__ __forceinline__ void issue(uint32_t lds, int wave) const {
#pragma unroll
        for (int p = 0; p < LOADS; ++p) load(p, lds, wave);
    }
};

// Fragments of a tile's 32-row block: rows as they lie (the product's rows, 16
// values of a row a step), and transposed (the row index is contracted, 16 rows
// a step: lane half g holds rows 4 g .. + 3 and 8 + 4 g .. + 3, the order in
// which a 32 x 32 result holds its rows).
// A chunk's number stands in an address as bits, so that the swizzled address of
// another chunk, or of 8 rows on, is one XOR away: `at` is a multiple of 256.
template <int DP>
struct Frags {
    using T = Rows<DP>;
    uint32_t row, col;
    __device__ __forceinline__ void init(uint32_t at, int lane) {
        const int r = lane & 31, g = lane >> 5, i16 = lane & 15, hf = (lane >> 4) & 1, tr = 4 * g + (i16 >> 2);
        row = at + r * T::RB + ((g ^ T::swz(r)) * 16);
        col = at + tr * T::RB + (((2 * hf + ((i16 & 3) >> 1)) ^ T::swz(tr)) * 16) + (i16 & 1) * 8;
    }
    // to the other stage
    __device__ __forceinline__ void move(uint32_t by) { row += by, col += by; }
    __device__ __forceinline__ uint4 rows(uint32_t at, int s) const {
        return __builtin_bit_cast(uint4, *reinterpret_cast<__attribute__((address_space(3))) const u32x4*>((row ^ (uint32_t)s << 5) + at));
    }
    __device__ __forceinline__ uint4 cols(uint32_t at, int j) const {
        const uint32_t c = col ^ (uint32_t)j << 6;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(c + at));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)((c ^ 32u) + (at + 8 * T::RB)));
        return __builtin_bit_cast(uint4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// A step's fragments in the order of their products, PD of them ahead: left to
// itself the compiler reads each one right before its product and waits.
template <int N, int PD, class Read, class Use, int... E>
__device__ __forceinline__ void win_each(uint4 (&ring)[PD], Read read, Use use, std::integer_sequence<int, E...>) {
    ((use(E, ring[E % PD]), E + PD < N ? (void)(ring[E % PD] = read(E + PD)) : (void)0, __builtin_amdgcn_sched_barrier(0)), ...);
}
template <int N, int PD, class Read, class Use>
__device__ __forceinline__ void win_stream(Read read, Use use) {
    uint4 ring[PD];
#pragma unroll
    for (int e = 0; e < PD; ++e) ring[e] = read(e);
    __builtin_amdgcn_sched_barrier(0);
    win_each<N, PD>(ring, read, use, std::make_integer_sequence<int, N>());
}
#define WIN_INLINE __attribute__((always_inline))

template <bool BF>
__device__ __forceinline__ floatx16 win_mma(uint4 a, uint4 b, floatx16 c) {
    if constexpr (BF) return MmaBf16::mma(a, b, c);
    return MmaF16::mma(a, b, c);
}
template <bool BF>
__device__ __forceinline__ uint32_t win_pack(float lo, float hi) {
    if constexpr (BF) return pack_bf2(lo, hi);
    return cvt_pk(lo, hi);
}
// 8 values of a 32 x 32 result as the other operand's 16 rows
template <bool BF>
__device__ __forceinline__ uint4 win_pack8(const floatx16& s, int u) {
    return make_uint4(win_pack<BF>(s[8 * u], s[8 * u + 1]), win_pack<BF>(s[8 * u + 2], s[8 * u + 3]),
                      win_pack<BF>(s[8 * u + 4], s[8 * u + 5]), win_pack<BF>(s[8 * u + 6], s[8 * u + 7]));
}
// What win_pack, and win_pack8, rounded off, as 16-bit values in the same order.
template <bool BF>
__device__ __forceinline__ uint32_t win_rest(float lo, float hi, uint32_t p) {
    const half2v h = __builtin_bit_cast(half2v, p);
    return win_pack<BF>(lo - (BF ? bf16_to_f32(p & 0xffffu) : (float)h[0]), hi - (BF ? bf16_to_f32(p >> 16) : (float)h[1]));
}
template <bool BF>
__device__ __forceinline__ uint4 win_rest8(const floatx16& s, int u, uint4 p) {
    return make_uint4(win_rest<BF>(s[8 * u], s[8 * u + 1], p.x), win_rest<BF>(s[8 * u + 2], s[8 * u + 3], p.y),
                      win_rest<BF>(s[8 * u + 4], s[8 * u + 5], p.z), win_rest<BF>(s[8 * u + 6], s[8 * u + 7], p.w));
}
// c + lo + hi of a 16-bit pair
template <bool BF>
__device__ __forceinline__ float win_sum2(uint32_t v, float c) {
    if constexpr (BF) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, v), __builtin_bit_cast(bf2, 0x3f803f80u), c, false);
    } else {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, v), __builtin_bit_cast(half2v, 0x3c003c00u), c, false);
    }
}
// c + a . b of 8 pairs of 16 bits, in float32
template <bool BF>
__device__ __forceinline__ float win_dot8(uint4 a, uint4 b, float c) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (BF) {
            c = fmaf(bf16_to_f32(x[t] & 0xffffu), bf16_to_f32(y[t] & 0xffffu), c);
            c = fmaf(bf16_to_f32(x[t] >> 16), bf16_to_f32(y[t] >> 16), c);
        } else {
            const half2v h = __builtin_bit_cast(half2v, x[t]), k = __builtin_bit_cast(half2v, y[t]);
            c = fmaf((float)h[0], (float)k[0], c);
            c = fmaf((float)h[1], (float)k[1], c);
        }
    }
    return c;
}

// Probabilities are formed times 2^-win_shift.  fp16: 2^7, where they pass 1 by
// 2^kWinLag at most, normal down to 2^-21 of the row's largest and off by less
// than 2^-32 of it below.  bf16 has float32's range and so have its values:
// 2^-28, so that a million of them stay within float32.
template <bool BF>
constexpr float win_shift() { return BF ? 28.0f : -7.0f; }

// A tile with sinks has far more to go over than the others: every key (sinks as
// queries, where not causal), every query (sinks as keys).  What lies past the
// tile's own window is divided into `parts` workgroups of their own; each leaves
// float32 sums of the sinks' rows (slot 0: the tile's), which a join adds up in
// their order.  parts = 0: the tile goes over all of it itself, and first.
struct WinFar {
    int tiles, rows, parts;  // tiles with sinks, the sinks, parts of a tile
};
struct WinArgs {
    const char *q, *k, *v, *o, *go;     // o: out of the forward, in of the gradient
    char *out, *gq, *gk, *gv, *rests;   // rests: out of the forward, in of the gradient, contiguous
    int64_t qs[3], ks[3], vs[3], os[3], gos[3];  // bytes between batches, tokens, heads
    const int32_t* lengths;
    float *top, *stat, *delta;          // [B, H, NP]; stat: lg
    int B, N, H, KV, D, NP;
    int window, sinks, causal;
    int hw, qw, tiles;                  // heads and 32-query blocks of a workgroup; query tiles
    float scale, scale2;                // scale2 = scale log2(e)
    WinFar far, kfar;                   // of the sinks as queries, as keys
    float *part, *kpart;
    // cached
    int M, rows, blocks, splits;        // keys of the cache; queries of a key head; their 32-row blocks; parts of a row
};

__device__ __forceinline__ int win_length(const WinArgs& a, int b, int most) {
    if (!a.lengths) return most;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > most ? most : n;
}
// Keeps a rare branch one: without it the compiler computes both sides, the masks
// of every tile among them.
__device__ __forceinline__ void win_rare() { asm volatile(""); }
// What a lane's query (key) sees of the keys (queries) in a block's result: those
// from lo on, `len` more, and those up to `early` (the sinks).
struct WinMask {
    int lo, early;
    uint32_t len;
    __device__ __forceinline__ void within(int from, int to) {
        from = from < 0 ? 0 : from;
        lo = to < from ? 0x40000000 : from;
        len = to < from ? 0u : (uint32_t)(to - from);
    }
    // of query i, among keys 0 .. n - 1
    static __device__ __forceinline__ WinMask keys(const WinArgs& a, int i, int n) {
        WinMask m;
        int to = a.causal ? i : i + a.window - 1;
        to = to < n - 1 ? to : n - 1;
        m.early = a.sinks - 1 < to || !a.causal ? a.sinks - 1 : to;
        m.early = m.early < n - 1 ? m.early : n - 1;
        if (!a.causal && i < a.sinks) m.within(0, n - 1);
        else m.within(i - a.window + 1, to);
        return m;
    }
    // of key j, among the queries; those behind the end weigh nothing of themselves
    static __device__ __forceinline__ WinMask queries(const WinArgs& a, int j) {
        WinMask m;
        m.early = a.causal ? -1 : a.sinks - 1;
        m.within(a.causal || j < a.sinks ? (a.causal ? j : 0) : j - a.window + 1, j < a.sinks ? 0x3fffffff : j + a.window - 1);
        return m;
    }
    // hide(v) for the results of rows base .. base + 31 that are not seen; `first`:
    // the sinks are among them
    template <class Hide>
    __device__ __forceinline__ void operator()(int base, int g, bool first, Hide hide) const {
        const int from = lo - base - 4 * g, last = early - base - 4 * g;
        if (first) {
            win_rare();
#pragma unroll
            for (int v = 0; v < 16; ++v) hide(v, ((uint32_t)(acc_row(v, 0) - from) <= len) | (acc_row(v, 0) <= last));
        } else {
            win_rare();
#pragma unroll
            for (int v = 0; v < 16; ++v) hide(v, (uint32_t)(acc_row(v, 0) - from) <= len);
        }
    }
};

// What a wave's own queries (keys) see of a run x0 .. x1 of keys (queries): 0
// nothing, 1 some, 2 all.  Runs within [lo, hi] are seen in part, within [all_lo,
// all_hi] whole, and those that begin in front of `early` may be.
struct WinSpan {
    int lo, hi, all_lo, all_hi, early;
    // of queries q0 .. q1 (none: q1 < q0) of n
    static __device__ __forceinline__ WinSpan keys(const WinArgs& a, int q0, int q1, int n) {
        WinSpan s = {q0 - a.window + 1, a.causal ? q1 : q1 + a.window - 1, q1 - a.window + 1, a.causal ? q0 : q0 + a.window - 1, a.sinks};
        if (!a.causal && q0 < a.sinks) s.lo = -0x7fffffff, s.hi = 0x7fffffff;
        if (!a.causal && q1 < a.sinks) s.all_lo = 0, s.all_hi = n;
        s.all_hi = s.all_hi < n - 1 ? s.all_hi : n - 1;
        if (q1 < q0) s.lo = 0x7fffffff, s.all_hi = -1, s.early = 0;
        return s;
    }
    // of keys k0 .. k1; queries behind the end weigh nothing of themselves
    static __device__ __forceinline__ WinSpan queries(const WinArgs& a, int k0, int k1) {
        WinSpan s = {a.causal ? k0 : k0 - a.window + 1, k1 + a.window - 1, a.causal ? k1 : k1 - a.window + 1, k0 + a.window - 1, a.causal ? 0 : a.sinks};
        if (k0 < a.sinks) s.hi = 0x7fffffff, s.lo = a.causal ? s.lo : -0x7fffffff;
        if (k1 < a.sinks) s.all_hi = 0x7fffffff, s.all_lo = a.causal ? s.all_lo : -0x7fffffff;
        if (k1 < k0) s.lo = 0x7fffffff, s.all_hi = -1, s.early = 0;
        return s;
    }
    __device__ __forceinline__ int operator()(int x0, int x1) const {
        if (x0 >= all_lo && x1 <= all_hi) return 2;
        return (x0 <= hi && x1 >= lo) || x0 < early;
    }
};

// The tiles of T keys that queries q0 .. q1 (< n) see: `first` tiles of the
// sinks, then [t0, t1).
struct WinTiles {
    int first, t0, count;
    __device__ __forceinline__ int at(int s) const { return s < first ? s : t0 + s - first; }
    // whether step s is not the tile behind step s - 1's
    __device__ __forceinline__ bool leap(int s) const { return s == first && first > 0 && t0 > first; }
};
template <int T>
__device__ __forceinline__ WinTiles win_tiles(const WinArgs& a, int q0, int q1, int n) {
    int lo = q0 - a.window + 1, hi = a.causal ? q1 + 1 : q1 + a.window;
    if (!a.causal && q0 < a.sinks) lo = 0, hi = n;
    lo = lo < 0 ? 0 : lo;
    hi = hi > n ? n : hi;
    WinTiles t;
    t.first = ((a.sinks < lo ? a.sinks : lo) + T - 1) / T;
    t.t0 = lo / T > t.first ? lo / T : t.first;
    const int t1 = (hi + T - 1) / T;
    t.count = q1 < q0 ? 0 : t.first + (t1 > t.t0 ? t1 - t.t0 : 0);
    return t;
}

// 32 rows of DP results [d][row] as 16-bit values: after trading halves across
// the 32 lanes each lane has 8 consecutive ones.  RESTS: what that rounds off too.
template <int DP, bool BF, bool RESTS = false>
__device__ __forceinline__ void win_store(const floatx16 (&o)[DP / 32], float f, bool zero, bool inside, char* dst, int D, int g, char* rests = nullptr) {
#pragma unroll
    for (int j = 0; j < DP / 32; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            uint32_t x[2], y[2], xr[2], yr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = o[j][8 * p + 2 * e] * f, b = o[j][8 * p + 2 * e + 1] * f;
                const float c = o[j][8 * p + 4 + 2 * e] * f, h = o[j][8 * p + 5 + 2 * e] * f;
                x[e] = win_pack<BF>(a, b);
                y[e] = win_pack<BF>(c, h);
                if (RESTS) xr[e] = zero ? 0 : win_rest<BF>(a, b, x[e]), yr[e] = zero ? 0 : win_rest<BF>(c, h, y[e]);
                if (zero) x[e] = y[e] = 0;
            }
            const auto s0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
            const int d = 32 * j + 16 * p + 8 * g;
            if (inside && d < D) *reinterpret_cast<uint4*>(dst + 2 * d) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
            if constexpr (RESTS) {
                const auto r0 = __builtin_amdgcn_permlane32_swap(xr[0], yr[0], false, false);
                const auto r1 = __builtin_amdgcn_permlane32_swap(xr[1], yr[1], false, false);
                if (inside && d < D) *reinterpret_cast<uint4*>(rests + 2 * d) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
            }
        }
}

// A 16-bit row's values 16 s + 8 g .. + 7, zeros past D or where it is not inside:
// there `base`, a row that is, is read in its place, so that the loads go out
// together (behind branches the compiler waits for each).
template <int DP>
__device__ __forceinline__ void win_row(uint4 (&f)[DP / 16], const char* base, int64_t off, bool inside, int D, int g) {
    const char* src = base + (inside ? off : 0);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const bool in = 16 * s + 8 * g < D;
        f[s] = *reinterpret_cast<const uint4*>(src + (in ? 32 * s + 16 * g : 0));
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const bool in = (16 * s + 8 * g < D) & inside;
        f[s] = make_uint4(in ? f[s].x : 0, in ? f[s].y : 0, in ? f[s].z : 0, in ? f[s].w : 0);
    }
}

// The compiler's wait for a load stands here, and not at its first use: in a loop
// that would be a wait for the DMA of the next tile too, which it does not count.
template <int N>
__device__ __forceinline__ void win_arrived(uint4 (&f)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s].x), "+v"(f[s].y), "+v"(f[s].z), "+v"(f[s].w));
}
__device__ __forceinline__ void win_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// c + a b where some of a are not finite: these count where they are seen (the bits
// of `seen`, b's 8 values), a factor that was rounded to 0 among them.
template <bool BF>
__device__ __forceinline__ floatx16 win_mma_some(uint4 a, uint4 b, uint32_t seen, floatx16 c) {
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u, ONE = BF ? 0x3f80u : 0x3c00u;
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
    uint32_t fin[4], odd[4], some[4], any = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t lo = (x[t] & E) == E ? 0xffffu : 0u, hi = (x[t] & E << 16) == E << 16 ? 0xffff0000u : 0u;
        fin[t] = x[t] & ~(lo | hi);
        odd[t] = (lo | hi) & (ONE | ONE << 16);
        some[t] = (seen >> 2 * t & 1 ? ONE : 0u) | (seen >> (2 * t + 1) & 1 ? ONE << 16 : 0u);
        any |= lo | hi;
    }
    if (!__any(any != 0)) return win_mma<BF>(a, b, c);
    const floatx16 n = win_mma<BF>(make_uint4(odd[0], odd[1], odd[2], odd[3]), make_uint4(some[0], some[1], some[2], some[3]), floatx16{0});
    const floatx16 all = win_mma<BF>(a, b, floatx16{0});
    c = win_mma<BF>(make_uint4(fin[0], fin[1], fin[2], fin[3]), b, c);
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] += n[v] != 0.0f ? all[v] : 0.0f;
    return c;
}

// The larger, the sum, of what lanes l and l + 32 hold.
__device__ __forceinline__ float half_max(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// The running softmax of a lane's query over blocks of 32 keys (two lanes hold one
// query's scores, half each): `top` the score that is subtracted, `sub` = top
// scale2 + shift as it is rounded; l the sum, times 2^-win_rel relative to top.  top
// follows the largest score only where that passes it by 2^kWinLag, so that the
// sums are hardly ever scaled anew.
struct WinState {
    float top, sub, l;
};
constexpr float kWinLag = 8.0f;
// The exponent that the block's scores take off; anew(f): what was summed before
// is scaled.  NaN among them passes by: it ends in the sum.  FAR: scores past
// 2^20, where the rounding of `sub` would carry probabilities out of fp16's range,
// have the largest subtracted first.
template <bool BF, bool FAR, class Anew>
__device__ __forceinline__ float win_top(floatx16& s, WinState& st, float scale2, Anew anew) {
    float mx = s[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) mx = fmaxf(mx, s[v]);
    mx = half_max(mx);
    if (__any((mx - st.top) * scale2 > kWinLag)) {  // -inf - -inf: nothing seen yet, nothing to scale
        const float top = fmaxf(st.top, mx);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float sub = fmaf(base, scale2, win_shift<BF>());
        const float f = __builtin_amdgcn_exp2f(FAR ? (st.top - base) * scale2 : st.sub - sub);
        st.top = top;
        st.sub = top == -__builtin_inff() ? -__builtin_inff() : sub;
        st.l *= f;
        anew(f);
    }
    const bool none = st.top == -__builtin_inff();  // nothing seen yet: exp2(-inf) is 0
    if (FAR) {
        const float base = none ? 0.0f : st.top;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] -= base;
        return win_shift<BF>();
    }
    return none ? 0.0f : st.sub;
}
// log2 of what a block's sums stand under, from exp2((S - top) scale2) on: the shift,
// with the rounding of `sub` where that was subtracted.
template <bool BF, bool FAR>
__device__ __forceinline__ float win_rel(const WinState& st, float scale2) {
    return FAR || st.top == -__builtin_inff() ? win_shift<BF>() : fmaf(-st.top, scale2, st.sub);
}
// P of scores LO .. HI - 1
__device__ __forceinline__ void win_exp(floatx16& s, int lo, int hi, float scale2, float sub) {
#pragma unroll
    for (int v = 0; v < 16; ++v)
        if (v >= lo && v < hi) s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], scale2, -sub));
}
__device__ __forceinline__ void win_exp_from(floatx16& s, int lo, int hi, float top, float scale2, float lg) {
#pragma unroll
    for (int v = 0; v < 16; ++v)
        if (v >= lo && v < hi) s[v] = __builtin_amdgcn_exp2f(fmaf(s[v] - top, scale2, -lg));
}
// Where the 16 exponentials of a block stand among N products, the first `from` without.
constexpr int win_piece(int x, int from, int n) { return x < from ? 0 : x >= n ? 16 : 16 * (x - from) / (n - from); }

// Unit of a launch over `groups` x `tiles`: (group, tile, part), the parts of the
// far ranges first, or the long tiles.
struct WinUnit {
    int group, tile, part;  // part 0: the tile itself
};
__device__ __forceinline__ WinUnit win_unit(const WinFar& f, int groups, int tiles) {
    const int u = blockIdx.x, first = groups * f.tiles * (f.parts ? f.parts : 1), skip = f.parts ? 0 : f.tiles;
    if (u < first) {
        const int p = f.parts ? u % f.parts : 0, v = xcd_tile(f.parts ? u / f.parts : u, groups * f.tiles);
        return {v / f.tiles, v % f.tiles, f.parts ? 1 + p : 0};
    }
    const int v = xcd_tile(u - first, groups * (tiles - skip));
    return {v / (tiles - skip), skip + v % (tiles - skip), 0};
}
static inline int64_t win_units(const WinFar& f, int64_t groups, int tiles) { return groups * (tiles + f.tiles * f.parts); }
// The tiles that a unit goes over, of all [0, end) and up to `near` by the tile itself.
__device__ __forceinline__ WinTiles win_share(const WinFar& f, const WinUnit& u, WinTiles t, int near, int end) {
    if (!f.parts || u.tile >= f.tiles) return t;
    near = near < end ? near : end;
    if (!u.part) {
        if (t.t0 + t.count - t.first > near) t.count = near > t.t0 ? t.first + near - t.t0 : t.first;
    } else {
        const int n = end - near;
        t.first = 0;
        t.t0 = near + (int)((int64_t)n * (u.part - 1) / f.parts);
        t.count = near + (int)((int64_t)n * u.part / f.parts) - t.t0;
    }
    return t;
}

// Where a workgroup of four waves stands: wave w has head hw h0 + w % hw and the
// 32-query block w / hw of its tile.  Heads that share keys sit together, so a
// tile is narrow and its window little wider than one query's.
struct WinPlace {
    int b, h, kv, q0, q1, mine, n;  // tile's first and last query (< n), first of this wave
    WinUnit unit;
};
__device__ __forceinline__ WinPlace win_place(const WinArgs& a, int wave) {
    WinPlace p;
    const int groups = a.H / a.hw;
    p.unit = win_unit(a.far, a.B * groups, a.tiles);
    p.b = p.unit.group / groups;
    const int h0 = (p.unit.group - p.b * groups) * a.hw;
    p.h = h0 + wave % a.hw;
    p.kv = h0 / (a.H / a.KV);
    const int tile = a.causal ? a.tiles - 1 - p.unit.tile : p.unit.tile;  // the longest first
    p.q0 = tile * 32 * a.qw;
    p.mine = p.q0 + 32 * (wave / a.hw);
    p.n = win_length(a, p.b, a.N);
    p.q1 = (p.q0 + 32 * a.qw < p.n ? p.q0 + 32 * a.qw : p.n) - 1;
    return p;
}
// Its key tiles of T.
template <int T>
__device__ __forceinline__ WinTiles win_keys(const WinArgs& a, const WinPlace& p) {
    return win_share(a.far, p.unit, win_tiles<T>(a, p.q0, p.q1, p.n), (p.q0 + 32 * a.qw + a.window + T - 1) / T, p.q1 < p.q0 ? 0 : (p.n + T - 1) / T);
}

// A row's two numbers for the gradient's probabilities, which fp16 has times 2^15;
// a row without any has probabilities of 0.
template <bool BF>
__device__ __forceinline__ void win_stat(float* top, float* stat, int64_t at, bool any, float score, float lg) {
    top[at] = any ? score : 0.0f;
    stat[at] = any ? lg - (BF ? 0.0f : 15.0f) : __builtin_inff();
}

// 32 rows of DP results as a slot of their float32 sums: `o` times f, and three
// numbers behind them: the score and the sum that they are relative to, and what
// win_rel differs from the shift by.  Rows behind a sequence's end leave zeros,
// whatever the products of their zeros with its values were.
template <int DP>
__device__ __forceinline__ void win_part(float* dst, const floatx16 (&o)[DP / 32], float f, bool inside, float top, float l, float rel, int g) {
#pragma unroll
    for (int j = 0; j < DP / 32; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
            const f32x4 x = (f32x4){o[j][v] * f, o[j][v + 1] * f, o[j][v + 2] * f, o[j][v + 3] * f};
            *reinterpret_cast<f32x4*>(dst + 32 * j + acc_row(v, g)) = inside ? x : (f32x4){0, 0, 0, 0};
        }
    if (g == 0) dst[DP] = top, dst[DP + 1] = l, dst[DP + 2] = rel;
}

// Forward.  S^T = K Q^T: a lane holds one query's scores, so the softmax is
// in-lane but for one exchange, and the probabilities, rounded to 16 bits, are
// already the operand of O^T = V^T P^T.  K and V tiles of 64 keys go to LDS by
// DMA, the next one while this one is used.  Bound by the products for heads of
// 128 (8,192 tokens, 16 heads on 4, window 1,024, bf16: 88 us, 0.87 PFLOP/s of what
// the tiles compute), by few and short walks over the keys for heads of 64 (96
// heads, 1,025 tokens, 127 to both sides: 29 us).  P goes into P V rounded to 16
// bits, which costs the output up to 0.4 of its own rounding.  TWO, where a gradient
// is wanted: with the rest as a second term (115 and 36 us), since rowsum(dO O) is
// subtracted from values as large, and what O is off by is much of what is left.
// The careful pass keeps one term.
template <int DP, bool BF, bool TWO>
__global__ void __launch_bounds__(256, DP > 64 ? 2 : DP > 32 ? 3 : 4) window_forward_kernel(WinArgs a) {
    extern __shared__ __align__(256) char smem[];
    constexpr int T = 64, TILE = T * Rows<DP>::RB;  // K, then V; twice
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const WinPlace p = win_place(a, wave);
    const int i = p.mine + r, last = (p.mine + 31 < p.n - 1 ? p.mine + 31 : p.n - 1);
    uint4 q[DP / 16];
    win_row<DP>(q, a.q + p.b * a.qs[0] + p.h * a.qs[2], i * a.qs[1], i < p.n, a.D, g);
    const WinTiles tiles = win_keys<T>(a, p);
    RowLoads<DP, T, 4> lk, lv;
    lk.init(a.ks[1], a.D, wave, lane);
    lv.init(a.vs[1], a.D, wave, lane);
    const char *kbase = a.k + p.b * a.ks[0] + p.kv * a.ks[2], *vbase = a.v + p.b * a.vs[0] + p.kv * a.vs[2];
    const uint32_t lds = lds_addr(smem);
    Frags<DP> at;
    at.init(lds, lane);
    const WinSpan span = WinSpan::keys(a, p.mine, last, p.n);
    auto issue = [&](int s) WIN_INLINE {
        if (s == 0 || tiles.leap(s)) {
            lk.seek(kbase, tiles.at(s) * T, p.n);
            lv.seek(vbase, tiles.at(s) * T, p.n);
        }
        const uint32_t to = lds + (s & 1) * 2 * TILE;
        lk.next();
        lv.next();
        lk.issue(to, wave);
        lv.issue(to + TILE, wave);
    };
    const WinMask mask = WinMask::keys(a, i, p.n);
    WinState st;
    float rel;
    floatx16 o[DP / 32];
    win_arrived(q);
    auto run = [&](auto careful) WIN_INLINE {
        constexpr bool FAR = decltype(careful)::value;
        st = {-__builtin_inff(), -__builtin_inff(), 0.0f};
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) o[j] = floatx16{0};
        if (tiles.count) issue(0);
        for (int t = 0; t < tiles.count; ++t) {
            win_sync();
            if (t + 1 < tiles.count) issue(t + 1);
            const int k0 = tiles.at(t) * T, seen = span(k0, k0 + T - 1);
            if (!seen) {
                at.move(t & 1 ? -2 * TILE : 2 * TILE);
                continue;
            }
            constexpr int RB = Rows<DP>::RB, NS = DP / 16, NJ = DP / 32, PD = 4;
            auto read = [&](int e) WIN_INLINE {
                if (e < 2 * NS) return at.rows(e / NS * 32 * RB, e % NS);
                return at.cols(TILE + (e - 2 * NS) / NJ * 16 * RB, (e - 2 * NS) % NJ);
            };
            uint32_t sees[2] = {0xffffu, 0xffffu};  // FAR: of each block's 16 keys of a lane
            auto hide = [&](floatx16& s, int kb) WIN_INLINE {
                if (seen != 1) return;
                if (FAR) sees[kb] = 0;
                mask(k0 + 32 * kb, g, k0 < a.sinks, [&](int v, bool in) WIN_INLINE {
                    s[v] = in ? s[v] : -__builtin_inff();
                    if (FAR) sees[kb] |= (uint32_t)in << v;
                });
            };
            auto anew = [&](float f) WIN_INLINE {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[j][v] *= f;
            };
            uint4 pr, rest;
            floatx16 s[2];
            s[0] = s[1] = floatx16{0};
            float take = 0.0f;
            // The products of one block and the other's softmax side by side: the second
            // block's scores with the first's exponentials, the first's P V with the
            // second's.
            win_stream<2 * NS + 4 * NJ, PD>(read, [&](int e, uint4 f) WIN_INLINE {
                if (e < NS) {
                    s[0] = win_mma<BF>(f, q[e], s[0]);
                    return;
                }
                if (e < 2 * NS) {
                    const int x = e - NS;
                    s[1] = win_mma<BF>(f, q[x], s[1]);
                    if (x == 1) {
                        hide(s[0], 0);
                        take = win_top<BF, FAR>(s[0], st, a.scale2, anew);
                    }
                    constexpr int from = NS > 2 ? 2 : 1;
                    win_exp(s[0], win_piece(x, from, NS), win_piece(x + 1, from, NS), a.scale2, take);
                    return;
                }
                const int y = e - 2 * NS, u = y / NJ, j = y % NJ;
                if (y == NJ)  // what is left of the first block is scaled with the rest
                    take = win_top<BF, FAR>(s[1], st, a.scale2, [&](float f_) WIN_INLINE {
                        anew(f_);
#pragma unroll
                        for (int v = 8; v < 16; ++v) s[0][v] *= f_;
                    });
                if (j == 0) {
                    pr = win_pack8<BF>(s[u >> 1], u & 1);
                    // with one term the sum of the rounded probabilities: their rounding errors
                    // then weigh the values' distance to the output, not the values
                    if (TWO && !FAR) {
                        rest = win_rest8<BF>(s[u >> 1], u & 1, pr);
#pragma unroll
                        for (int v = 0; v < 8; ++v) st.l += s[u >> 1][8 * (u & 1) + v];
                    } else {
                        st.l = win_sum2<BF>(pr.x, win_sum2<BF>(pr.y, win_sum2<BF>(pr.z, win_sum2<BF>(pr.w, st.l))));
                    }
                }
                o[j] = FAR ? win_mma_some<BF>(f, pr, sees[u >> 1] >> 8 * (u & 1), o[j]) : win_mma<BF>(f, pr, o[j]);
                if (TWO && !FAR) o[j] = win_mma<BF>(f, rest, o[j]);
                if (y == 0) hide(s[1], 1);
                if (u == 1 || u == 2) win_exp(s[1], 8 * (y - NJ) / NJ, 8 * (y + 1 - NJ) / NJ, a.scale2, take);
            });
            at.move(t & 1 ? -2 * TILE : 2 * TILE);
        }
        at.move(tiles.count & 1 ? -2 * TILE : 0);  // to the first stage again
        rel = win_rel<BF, FAR>(st, a.scale2);
    };
    run(std::false_type());
    // Scores past 2^20, or a value that is not finite (a product with a probability
    // of 0 in its tile made it everyone's): once more, with care.
    float odd = st.top * a.scale2 > 0x1p20f || (st.top != -__builtin_inff() && st.top * a.scale2 < -0x1p20f) ? 1.0f : st.l * 0.0f;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) odd = fmaf(o[j][v], 0.0f, odd);
    if (__builtin_expect(__syncthreads_or(!(odd == 0.0f)), 0)) run(std::true_type());
    const float l = half_sum(st.l);
    const bool any = l != 0.0f && i < p.n;
    if (a.far.parts && p.unit.tile < a.far.tiles && p.mine < a.far.rows) {
        const int64_t row = (((int64_t)p.b * a.far.rows + i) * a.H + p.h) * (a.far.parts + 1) + p.unit.part;
        if (i < a.far.rows) win_part<DP>(a.part + row * (DP + 8), o, 1.0f, i < p.n, any ? st.top : -__builtin_inff(), i < p.n ? l : 0.0f, rel - win_shift<BF>(), g);
    }
    if (p.unit.part) return;
    const bool joined = a.far.parts && i < a.far.rows;
    if (a.stat && g == 0 && i < a.NP && !joined)
        win_stat<BF>(a.top, a.stat, ((int64_t)p.b * a.H + p.h) * a.NP + i, any, st.top, rel + __builtin_amdgcn_logf(l));
    win_store<DP, BF, TWO>(o, any ? 1.0f / l : 0.0f, !any, i < a.N && !joined, a.out + p.b * a.os[0] + (int64_t)i * a.os[1] + p.h * a.os[2], a.D, g,
                           a.rests + (((int64_t)p.b * a.N + i) * a.H + p.h) * 2 * a.D);
}

// fp16 gradients: dS is carried times a power of two of its column (one query in
// dQ, one key in dK), so that the largest so far lies in [2^14, 2^15): the
// sums are float32 and follow it down where a larger one comes.
__device__ __forceinline__ float win_lower(float c, float mx) {
    const int e = 15 - __builtin_amdgcn_frexp_expf(mx);
    const float to = __builtin_amdgcn_ldexpf(1.0f, e < -126 ? -126 : e > 126 ? 126 : e);
    return to < c ? to : c;
}
template <int DP, bool BF>
__device__ __forceinline__ void win_scale_ds(floatx16& ds, float& c, floatx16 (&o)[DP / 32]) {
    if constexpr (!BF) {
        float mx = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, fabsf(ds[v]));
        mx = half_max(mx);
        if (__any(mx * c > 0x1p15f)) {
            const float to = mx * c > 0x1p15f ? win_lower(c, mx) : c, f = to / c;
            c = to;
#pragma unroll
            for (int j = 0; j < DP / 32; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[j][v] *= f;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) ds[v] *= c;
    }
}

// Gradient of the queries, laid out as the forward: S^T = K Q^T and dP^T = V dO^T
// in one lane's query, dQ^T = K^T dS^T.  Leaves rowsum(dO O) for the other.  Of
// the forward's sizes 120 us (0.95 PFLOP/s) and 42.
template <int DP, bool BF, bool TWO>
__global__ void __launch_bounds__(256, DP > 64 ? 2 : 3) window_grad_q_kernel(WinArgs a) {
    extern __shared__ __align__(256) char smem[];
    constexpr int T = 64, TILE = T * Rows<DP>::RB;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const WinPlace p = win_place(a, wave);
    const int i = p.mine + r, last = (p.mine + 31 < p.n - 1 ? p.mine + 31 : p.n - 1);
    const int64_t row = ((int64_t)p.b * a.H + p.h) * a.NP + i;
    uint4 q[DP / 16], go[DP / 16];
    win_row<DP>(q, a.q + p.b * a.qs[0] + p.h * a.qs[2], i * a.qs[1], i < p.n, a.D, g);
    win_row<DP>(go, a.go + p.b * a.gos[0] + p.h * a.gos[2], i * a.gos[1], i < p.n, a.D, g);
    float delta = 0.0f;
    {
        uint4 out[DP / 16], rest[DP / 16];
        win_row<DP>(out, a.o + p.b * a.os[0] + p.h * a.os[2], i * a.os[1], i < p.n, a.D, g);
        win_row<DP>(rest, a.rests + ((int64_t)p.b * a.N * a.H + p.h) * 2 * a.D, (int64_t)i * a.H * 2 * a.D, i < p.n, a.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) delta = win_dot8<BF>(go[s], rest[s], win_dot8<BF>(go[s], out[s], delta));
        delta = half_sum(delta);
    }
    if (g == 0 && i < a.NP && !p.unit.part) a.delta[row] = delta;
    float top = i < a.NP ? a.top[row] : 0.0f, stat = i < a.NP ? a.stat[row] : __builtin_inff();
    if (!a.gq) return;
    const WinTiles tiles = win_keys<T>(a, p);
    RowLoads<DP, T, 4> lk, lv;
    lk.init(a.ks[1], a.D, wave, lane);
    lv.init(a.vs[1], a.D, wave, lane);
    const char *kbase = a.k + p.b * a.ks[0] + p.kv * a.ks[2], *vbase = a.v + p.b * a.vs[0] + p.kv * a.vs[2];
    const uint32_t lds = lds_addr(smem);
    Frags<DP> at;
    at.init(lds, lane);
    const WinSpan span = WinSpan::keys(a, p.mine, last, p.n);
    auto issue = [&](int s) WIN_INLINE {
        if (s == 0 || tiles.leap(s)) {
            lk.seek(kbase, tiles.at(s) * T, p.n);
            lv.seek(vbase, tiles.at(s) * T, p.n);
        }
        const uint32_t to = lds + (s & 1) * 2 * TILE;
        lk.next();
        lv.next();
        lk.issue(to, wave);
        lv.issue(to + TILE, wave);
    };
    const WinMask mask = WinMask::keys(a, i, p.n);
    floatx16 o[DP / 32];
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) o[j] = floatx16{0};
    float c = BF ? 1.0f : 0x1p126f;
    win_arrived(q);
    win_arrived(go);
    asm volatile("" : "+v"(top), "+v"(stat), "+v"(delta));
    if (tiles.count) issue(0);
    for (int t = 0; t < tiles.count; ++t) {
        win_sync();
        if (t + 1 < tiles.count) issue(t + 1);
        const int k0 = tiles.at(t) * T, seen = span(k0, k0 + T - 1);
        if (!seen) {
            at.move(t & 1 ? -2 * TILE : 2 * TILE);
            continue;
        }
        constexpr int RB = Rows<DP>::RB, NS = DP / 16, NJ = DP / 32, PD = 4;
        // the scores and dP of one block, then the other's, then both blocks' dQ
        auto read = [&](int e) WIN_INLINE {
            if (e < 4 * NS) return at.rows((e / NS & 1) * TILE + e / (2 * NS) * 32 * RB, e % NS);
            return at.cols((e - 4 * NS) / NJ * 16 * RB, (e - 4 * NS) % NJ);
        };
        floatx16 s[2], dp = floatx16{0};
        s[0] = s[1] = floatx16{0};
        uint4 ds, rest;
        auto finish = [&](int kb) WIN_INLINE {  // dS from P and dP
#pragma unroll
            for (int v = 0; v < 16; ++v) s[kb][v] *= dp[v] - delta;
            if (seen == 1)
                mask(k0 + 32 * kb, g, k0 < a.sinks, [&](int v, bool in) WIN_INLINE { s[kb][v] = in ? s[kb][v] : 0.0f; });
            win_scale_ds<DP, BF>(s[kb], c, o);
            dp = floatx16{0};
        };
        win_stream<4 * NS + 4 * NJ, PD>(read, [&](int e, uint4 f) WIN_INLINE {
            const int kb = e / (2 * NS), x = e % NS;
            if (e < 4 * NS) {
                if (e / NS & 1) {
                    dp = win_mma<BF>(f, go[x], dp);
                    win_exp_from(s[kb], win_piece(x, 1, NS), win_piece(x + 1, 1, NS), top, a.scale2, stat);
                } else {
                    s[kb] = win_mma<BF>(f, q[x], s[kb]);
                    if (kb && x == 0) finish(0);
                }
                return;
            }
            const int y = e - 4 * NS, u = y / NJ, j = y % NJ;
            if (y == (BF ? 1 : 2 * NJ)) finish(1);  // fp16: it may scale what was summed, so behind the first's
            if (j == 0) {
                ds = win_pack8<BF>(s[u >> 1], u & 1);
                if (TWO) rest = win_rest8<BF>(s[u >> 1], u & 1, ds);
            }
            o[j] = win_mma<BF>(f, ds, o[j]);
            if (TWO) o[j] = win_mma<BF>(f, rest, o[j]);
        });
        at.move(t & 1 ? -2 * TILE : 2 * TILE);
    }
    const float f = (BF ? 1.0f : 0x1p-15f) / c;
    if (a.far.parts && p.unit.tile < a.far.tiles && p.mine < a.far.rows) {
        const int64_t slot = (((int64_t)p.b * a.far.rows + i) * a.H + p.h) * (a.far.parts + 1) + p.unit.part;
        if (i < a.far.rows) win_part<DP>(a.part + slot * (DP + 8), o, f, i < p.n, 0.0f, 1.0f, 0.0f, g);
    }
    if (p.unit.part) return;
    char* dst = a.gq + (((int64_t)p.b * a.N + i) * a.H + p.h) * 2 * a.D;
    win_store<DP, BF>(o, a.scale * f, i >= p.n, i < a.N && !(a.far.parts && i < a.far.rows), dst, a.D, g);
}

// Gradient of the keys and values: a workgroup of four waves has 64 keys, 32 to a
// wave and its fellow, which take every other 32 of the queries that see them,
// of all heads that share them.  S = Q K^T and dP = dO V^T with a key to a lane:
// P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS.  K stays in
// registers, V in LDS (with both, 128-value heads spill); with two stages of Q
// and dO that is 80 KB, two workgroups a CU.  Heads up to 64: three, with fewer
// fragments ahead (96 heads of 64 over 1,025 tokens 49 us, with two a CU 7 more; a
// few registers spill, outside the products).  The long case of the forward 175 us
// (0.85 PFLOP/s), its sinks' far queries in parts (in their tile's own workgroup
// seven times that).  Statistics come by lane broadcasts: a
// 128-bit LDS read of one address by half a wave took 24 clocks.
constexpr int kWinKeys = 64, kWinStep = 64;
template <int DP>
constexpr int win_grad_lds() {
    const int rows = Rows<DP>::RB * (kWinKeys + 4 * kWinStep), sums = 2 * 32 * (DP + 4) * 4;
    return rows > sums ? rows : sums;
}
// The value of lane E of each 16 lanes in all of them.
template <int E>
__device__ __forceinline__ float win_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + E, 0xf, 0xf, true));
}
// P, and dP - rowsum(dO O), of a lane's key and 16 queries, whose statistics lie in 16 lanes
template <int... E>
__device__ __forceinline__ void win_probs(std::integer_sequence<int, E...>, floatx16& s, float top, float scale2, float stat) {
    ((s[E] = __builtin_amdgcn_exp2f((s[E] - win_lane<E>(top)) * scale2 - win_lane<E>(stat))), ...);
}
template <int... E>
__device__ __forceinline__ void win_diff(std::integer_sequence<int, E...>, floatx16& dp, float delta) {
    ((dp[E] -= win_lane<E>(delta)), ...);
}
template <int DP, bool BF, bool TWO>
__global__ void __launch_bounds__(256, DP > 64 ? 2 : 3) window_grad_kv_kernel(WinArgs a) {
    extern __shared__ __align__(256) char smem[];
    constexpr int RB = Rows<DP>::RB, V = kWinKeys * RB, STAGE = 2 * kWinStep * RB;  // V, two stages of Q and dO
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), block = wave & 1, half = wave >> 1;
    const WinUnit unit = win_unit(a.kfar, a.B * a.KV, (a.N + kWinKeys - 1) / kWinKeys);
    const int b = unit.group / a.KV, kv = unit.group - b * a.KV, group = a.H / a.KV;
    const int n = win_length(a, b, a.N), k0 = unit.tile * kWinKeys, mine = k0 + 32 * block, key = mine + r;
    const int klast = (mine + 31 < n - 1 ? mine + 31 : n - 1), kend = (k0 + kWinKeys < n ? k0 + kWinKeys : n) - 1;
    uint4 kf[DP / 16];
    win_row<DP>(kf, a.k + b * a.ks[0] + kv * a.ks[2], key * a.ks[1], key < n, a.D, g);
    // the queries that see them: first tiles (seeing all), then [t0, t1), for each head
    int lo = a.causal ? k0 : k0 - a.window + 1, hi = kend + a.window;
    if (k0 < a.sinks) hi = n, lo = a.causal ? lo : 0;
    lo = lo < 0 ? 0 : lo;
    hi = hi > n ? n : hi;
    WinTiles q;
    q.first = a.causal ? 0 : ((a.sinks < lo ? a.sinks : lo) + kWinStep - 1) / kWinStep;
    q.t0 = lo / kWinStep > q.first ? lo / kWinStep : q.first;
    const int t1 = (hi + kWinStep - 1) / kWinStep;
    q.count = kend < k0 ? 0 : q.first + (t1 > q.t0 ? t1 - q.t0 : 0);
    q = win_share(a.kfar, unit, q, (k0 + kWinKeys + a.window + kWinStep - 1) / kWinStep, kend < k0 ? 0 : (n + kWinStep - 1) / kWinStep);
    const int steps = q.count * group;

    RowLoads<DP, kWinStep, 4> lq, lo_;
    lq.init(a.qs[1], a.D, wave, lane);
    lo_.init(a.gos[1], a.D, wave, lane);
    const uint32_t lds = lds_addr(smem);
    Frags<DP> at;
    at.init(lds + V + 32 * half * RB, lane);
    // the step that is loaded next: head `head` of query tile qt; heads go round within a tile
    int head = 0, qt = 0, q0 = 0, q0_next = 0;
    float top = 0.0f, stat = 0.0f, delta = 0.0f, top_next = 0.0f, stat_next = 0.0f, delta_next = 0.0f;
    const int mine_q = 32 * half + acc_row(lane & 15, g);  // whose statistics this lane loads
    int64_t row = 0;
    auto place = [&]() WIN_INLINE {
        const int first = q.at(qt) * kWinStep;
        lq.seek(a.q + b * a.qs[0] + kv * group * a.qs[2], first, n);
        lo_.seek(a.go + b * a.gos[0] + kv * group * a.gos[2], first, n);
        row = ((int64_t)b * a.H + kv * group) * a.NP + first;
        q0_next = first + 32 * half;
    };
    auto issue = [&](int s) WIN_INLINE {
        const uint32_t to = lds + V + (s & 1) * STAGE;
        if (head == group) {
            head = 0;
            ++qt;
            place();
        }
        top_next = a.top[row + mine_q];
        stat_next = a.stat[row + mine_q];
        delta_next = a.delta[row + mine_q];
        lq.resource();
        lo_.resource();
        lq.issue(to, wave);
        lo_.issue(to + kWinStep * RB, wave);
        lq.at += a.qs[2];
        lo_.at += a.gos[2];
        row += a.NP;
        ++head;
    };
    if (steps) {
        RowLoads<DP, kWinKeys, 4> lv;
        lv.init(a.vs[1], a.D, wave, lane);
        lv.seek(a.v + b * a.vs[0] + kv * a.vs[2], k0, n);
        lv.resource();
        lv.issue(lds, wave);
        place();
        issue(0);
    }
    floatx16 ok[DP / 32], ov[DP / 32];
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) ok[j] = ov[j] = floatx16{0};
    const WinMask mask = WinMask::queries(a, key);
    const WinSpan span = WinSpan::queries(a, mine, klast);
    float c = BF ? 1.0f : 0x1p126f;
    win_arrived(kf);
    for (int t = 0; t < steps; ++t) {
        win_sync();
        asm volatile("" : "+v"(top_next), "+v"(stat_next), "+v"(delta_next));
        top = top_next, stat = stat_next, delta = delta_next;
        q0 = q0_next;
        if (t + 1 < steps) issue(t + 1);
        const int seen = q0 < n ? span(q0, q0 + 31) : 0;
        if (seen) {
            constexpr int NS = DP / 16, NJ = DP / 32, PD = 2, OUT = kWinStep * RB;
            const uint32_t vt = 32 * (block - half) * RB - V - (t & 1) * STAGE;  // V's rows from Q's
            // Q; dO and V in turn; dO and Q transposed
            auto read = [&](int e) WIN_INLINE {
                if (e < NS) return at.rows(0, e);
                if (e < 3 * NS) return at.rows((e - NS) & 1 ? vt : OUT, (e - NS) / 2);
                const int x = e - 3 * NS;
                return at.cols((x < 2 * NJ ? OUT : 0) + x / NJ % 2 * 16 * RB, x % NJ);
            };
            uint4 pr, was, rest;
            floatx16 s = floatx16{0}, dp = floatx16{0};
            win_stream<3 * NS + 4 * NJ, PD>(read, [&](int e, uint4 f) WIN_INLINE {
                if (e < NS) {
                    s = win_mma<BF>(f, kf[e], s);
                    return;
                }
                if (e < 3 * NS) {
                    if (!((e - NS) & 1)) {
                        was = f;
                        return;
                    }
                    dp = win_mma<BF>(was, f, dp);
                    if (e == 3 * NS - 1) {
                        win_probs(std::make_integer_sequence<int, 16>(), s, top, a.scale2, stat);
                        if (seen == 1)
                            mask(q0, g, !a.causal && q0 < a.sinks, [&](int v, bool in) WIN_INLINE { s[v] = in ? s[v] : 0.0f; });
                    }
                    return;
                }
                const int x = e - 3 * NS, j = x % NJ;
                if (x < 2 * NJ) {
                    if (j == 0) {
                        pr = win_pack8<BF>(s, x / NJ);
                        if (TWO) rest = win_rest8<BF>(s, x / NJ, pr);
                    }
                    ov[j] = win_mma<BF>(f, pr, ov[j]);
                    if (TWO) ov[j] = win_mma<BF>(f, rest, ov[j]);
                    if (x == 1) {
                        win_diff(std::make_integer_sequence<int, 16>(), dp, delta);
#pragma unroll
                        for (int v = 0; v < 16; ++v) dp[v] *= s[v];
                        if (seen == 1) {
                            win_rare();
#pragma unroll
                            for (int v = 0; v < 16; ++v) dp[v] = s[v] == 0.0f ? 0.0f : dp[v];
                        }
                    }
                } else {
                    if (x == 2 * NJ) win_scale_ds<DP, BF>(dp, c, ok);
                    if (j == 0) {
                        pr = win_pack8<BF>(dp, x / NJ % 2);
                        if (TWO) rest = win_rest8<BF>(dp, x / NJ % 2, pr);
                    }
                    ok[j] = win_mma<BF>(f, pr, ok[j]);
                    if (TWO) ok[j] = win_mma<BF>(f, rest, ok[j]);
                }
            });
        }
        at.move(t & 1 ? -STAGE : STAGE);
    }
    // the fellow's sums through LDS, one tensor after the other
    const float fv = BF ? 1.0f : 0x1p-15f;
    float* sums = reinterpret_cast<float*>(smem) + (block * 32 + r) * (DP + 4);
    const bool parted = a.kfar.parts && unit.tile < a.kfar.tiles;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        floatx16(&o)[DP / 32] = w ? ov : ok;
        const float f = w ? 1.0f : 1.0f / c;
        win_sync();
        if (half) {
#pragma unroll
            for (int j = 0; j < DP / 32; ++j)
#pragma unroll
                for (int v = 0; v < 16; v += 4)
                    *reinterpret_cast<f32x4*>(sums + 32 * j + acc_row(v, g)) =
                        (f32x4){o[j][v] * f, o[j][v + 1] * f, o[j][v + 2] * f, o[j][v + 3] * f};
        }
        win_sync();
        if (!half) {
#pragma unroll
            for (int j = 0; j < DP / 32; ++j)
#pragma unroll
                for (int v = 0; v < 16; v += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(sums + 32 * j + acc_row(v, g));
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][v + e] = o[j][v + e] * f + x[e];
                }
            if (parted && key < a.kfar.rows) {
                const int64_t row = ((((int64_t)w * a.B + b) * a.kfar.rows + key) * a.KV + kv) * (a.kfar.parts + 1) + unit.part;
                win_part<DP>(a.kpart + row * (DP + 8), o, fv, key < n, 0.0f, 1.0f, 0.0f, g);
            }
            char* dst = w ? a.gv : a.gk;
            if (dst && !unit.part)
                win_store<DP, BF>(o, w ? fv : fv * a.scale, key >= n, key < a.N && !(parted && key < a.kfar.rows),
                                  dst + (((int64_t)b * a.N + key) * a.KV + kv) * 2 * a.D, a.D, g);
        }
    }
}

// The last tokens over a cache.  A workgroup has one key head of one sequence,
// up to 32 of its rows (queries x heads that share it) and a part of the keys that
// any of the sequence's new tokens sees (so 32 rows of many new tokens go over all
// of theirs: 2,048 with a window of 128, 16 heads of 128 on 4, 0.32 ms, the whole
// form 13 us); its waves take tiles of 32 keys in turn, each through LDS of its
// own, without waiting for each other.  Parts are joined by window_join_kernel.  P goes into P V
// as two 16-bit terms: the matrix units wait for memory here, and with one the
// rounding of P is half of the output's error (bf16 2.3e-3 of it, with two 1.65e-3,
// its own rounding).  Bound by HBM (64 streams, 4 key heads of 128, 4,100 slots,
// bf16: 103 us, 5.2 TB/s, with one term 99), at few heads by a wave's tiles, one
// read's latency behind the other (8 streams, 12 heads of 64, 1,028 slots 9.7 us,
// with one 9.0).
template <int DP>
constexpr int win_waves() { return DP > 64 ? 4 : 8; }  // their rings fill 128 KB of LDS at most
template <int DP, bool BF>
__global__ void __launch_bounds__(64 * win_waves<DP>(), 1) window_cached_kernel(WinArgs a) {
    extern __shared__ __align__(256) char smem[];
    constexpr int W = win_waves<DP>(), T = 32, RB = Rows<DP>::RB, TILE = T * RB, LOADS = T / Rows<DP>::PER;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = a.H / a.KV;
    int u = blockIdx.x;
    const int split = u % a.splits;
    u /= a.splits;
    const int blk = u % a.blocks;
    u /= a.blocks;
    const int kv = u % a.KV, b = u / a.KV;
    const int row = 32 * blk + r, tok = row / group, h = kv * group + row - tok * group;
    const bool inside = row < a.rows;
    const int len = win_length(a, b, a.M), i = len - a.N + tok;
    uint4 q[DP / 16];
    win_row<DP>(q, a.q + b * a.qs[0], tok * a.qs[1] + h * a.qs[2], inside, a.D, g);

    const int lo = len - a.N - a.window + 1 < 0 ? 0 : len - a.N - a.window + 1;
    const int sinks = a.sinks < len ? a.sinks : len;
    const int first = ((sinks < lo ? sinks : lo) + T - 1) / T, t0 = lo / T > first ? lo / T : first;
    const int t1 = (len + T - 1) / T, count = first + (t1 > t0 ? t1 - t0 : 0);
    const int from = (int)((int64_t)count * split / a.splits), to = (int)((int64_t)count * (split + 1) / a.splits);

    const uint32_t lds = lds_addr(smem) + wave * 4 * TILE;  // K, V; twice
    const char *kbase = a.k + b * a.ks[0] + kv * a.ks[2], *vbase = a.v + b * a.vs[0] + kv * a.vs[2];
    // slots that no query sees are not read: what they hold is not to count
    auto issue = [&](int s, int buf) {
        const int j0 = (s < first ? s : t0 + s - first) * T;
        intx4 rk = tile_rsrc(kbase + (int64_t)j0 * a.ks[1]), rv = tile_rsrc(vbase + (int64_t)j0 * a.vs[1]);
#pragma unroll
        for (int p = 0; p < LOADS; ++p) {
            const int x = p * Rows<DP>::PER + lane / Rows<DP>::CH, j = j0 + x;
            const int ch = (lane & (Rows<DP>::CH - 1)) ^ Rows<DP>::swz(x);
            const bool in = 8 * ch < a.D && j < len && (j >= lo || j < sinks);
            dma_buffer(rk, in ? (uint32_t)(x * (int)a.ks[1] + 16 * ch) : kTileOut, lds + buf * 2 * TILE + p * 1024);
            dma_buffer(rv, in ? (uint32_t)(x * (int)a.vs[1] + 16 * ch) : kTileOut, lds + buf * 2 * TILE + TILE + p * 1024);
        }
    };
    Frags<DP> at;
    at.init(lds, lane);
    WinState st = {-__builtin_inff(), -__builtin_inff(), 0.0f};
    floatx16 o[DP / 32];
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) o[j] = floatx16{0};
    const WinMask mask = WinMask::keys(a, i, len);
    int s = from + wave, buf = 0;
    win_arrived(q);
    if (s < to) issue(s, 0);
    for (; s < to; s += W, buf ^= 1) {
        if (s + W < to) {
            issue(s + W, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const int j0 = (s < first ? s : t0 + s - first) * T;
        // whether some row does not see all of it
        const bool some = j0 + T > len - a.N + 1 || (len - 1 - j0 >= a.window && j0 + T > sinks);
        const uint32_t bt = buf * 2 * TILE;
        constexpr int NS = DP / 16, NJ = DP / 32, PD = 8;
        auto read = [&](int e) WIN_INLINE {
            if (e < NS) return at.rows(bt, e);
            return at.cols(bt + TILE + (e - NS) / NJ * 16 * RB, (e - NS) % NJ);
        };
        floatx16 sc = floatx16{0};
        uint4 pr, rest;
        uint32_t sees = 0;
        win_stream<NS + 2 * NJ, PD < NS + 2 * NJ ? PD : NS + 2 * NJ>(read, [&](int e, uint4 f) WIN_INLINE {
            if (e < NS) {
                sc = win_mma<BF>(f, q[e], sc);
                if (e < NS - 1) return;
                if (some)
                    mask(j0, g, j0 < sinks, [&](int v, bool in) WIN_INLINE {
                        sc[v] = in ? sc[v] : -__builtin_inff();
                        sees |= (uint32_t)in << v;
                    });
                const float take = win_top<BF, true>(sc, st, a.scale2, [&](float f_) WIN_INLINE {
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v) o[j][v] *= f_;
                });
                win_exp(sc, 0, 16, a.scale2, take);
                return;
            }
            const int u = (e - NS) / NJ, j = (e - NS) % NJ;
            if (j == 0) {
                pr = win_pack8<BF>(sc, u);
                rest = win_rest8<BF>(sc, u, pr);
#pragma unroll
                for (int v = 0; v < 8; ++v) st.l += sc[8 * u + v];
            }
            if (some && a.N > 1) {
                win_rare();
                o[j] = win_mma_some<BF>(f, pr, sees >> 8 * u, o[j]);
                o[j] = win_mma_some<BF>(f, rest, sees >> 8 * u, o[j]);
            } else {
                o[j] = win_mma<BF>(f, pr, o[j]);
                o[j] = win_mma<BF>(f, rest, o[j]);
            }
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this buffer is free for the next load
    }
    // the waves' sums, in their order
    st.l = half_sum(st.l);
    __syncthreads();
    constexpr int LD = DP + 4;
    float* sums = reinterpret_cast<float*>(smem);  // [wave][row][LD]
    float* ml = sums + W * 32 * LD;                // [wave][row][2]
    if (inside) {
#pragma unroll
        for (int j = 0; j < DP / 32; ++j)
#pragma unroll
            for (int v = 0; v < 16; v += 4)
                *reinterpret_cast<f32x4*>(sums + (wave * 32 + r) * LD + 32 * j + acc_row(v, g)) =
                    (f32x4){o[j][v], o[j][v + 1], o[j][v + 2], o[j][v + 3]};
        if (g == 0) ml[(wave * 32 + r) * 2] = st.top, ml[(wave * 32 + r) * 2 + 1] = st.l;
    }
    __syncthreads();
    const int rows = a.rows - 32 * blk < 32 ? a.rows - 32 * blk : 32;
    for (int e = tid; e < rows * (DP / 8); e += 64 * W) {
        const int x = e / (DP / 8), d = 8 * (e - x * (DP / 8));
        float m = -__builtin_inff(), l = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, ml[(w * 32 + x) * 2]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = ml[(w * 32 + x) * 2], f = mw == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((mw - m) * a.scale2);
            l += f * ml[(w * 32 + x) * 2 + 1];
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = fmaf(f, sums[(w * 32 + x) * LD + d + t], v[t]);
        }
        const int orow = 32 * blk + x, ot = orow / group, oh = kv * group + orow - ot * group;
        if (a.splits > 1) {
            const int64_t at_ = (((int64_t)b * a.N + ot) * a.H + oh) * a.splits + split;
            float* dst = a.part + at_ * (DP + 8);  // as win_part
#pragma unroll
            for (int t = 0; t < 8; t += 4) *reinterpret_cast<f32x4*>(dst + d + t) = (f32x4){v[t], v[t + 1], v[t + 2], v[t + 3]};
            if (d == 0) dst[DP] = m, dst[DP + 1] = l, dst[DP + 2] = 0.0f;
        } else if (d < a.D) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            char* dst = a.out + (((int64_t)b * a.N + ot) * a.H + oh) * 2 * a.D + 2 * d;
            *reinterpret_cast<uint4*>(dst) = make_uint4(win_pack<BF>(v[0] * inv, v[1] * inv), win_pack<BF>(v[2] * inv, v[3] * inv),
                                                        win_pack<BF>(v[4] * inv, v[5] * inv), win_pack<BF>(v[6] * inv, v[7] * inv));
        }
    }
}

// Rows [sequence][token][head] from their slots, a workgroup a row at a time: DP / 4 threads
// hold its values, the others every so many slots (one thread over 49 slots of a
// gradient's 16 rows: 17 us, so 5).  Outputs (a slot as win_part leaves it), or
// plain sums times `factor` (GRAD).  A slot without any has the score -inf and sums
// of 0; one whose scores are all NaN has it too, and a sum of NaN, so no slot is
// passed over for its weight of 0.
constexpr int kWinSlots = 256;
struct WinJoin {
    const float* part;
    char* out[2];         // GRAD: keys and values, rows of one behind the other's; NULL: not wanted
    char* rests;          // of the output, contiguous, or NULL
    float factor[2];
    float *top, *stat;    // [B, heads, NP], or NULL
    float scale2;
    int64_t os[3];
    int64_t rows, all;    // sequences x tokens x heads; of both tensors
    int tokens, heads, slots, D, N, NP;
};
template <int DP, bool BF, bool GRAD>
__global__ void __launch_bounds__(256) window_join_kernel(WinJoin a) {
    constexpr int LD = DP + 8, TD = DP / 4, SG = 256 / TD;  // SG slots at once (DP = 96: 10, and threads to spare)
    __shared__ float weight[kWinSlots], most[4], total[4];
    __shared__ f32x4 sums[SG][TD];
    const int tid = threadIdx.x;
    for (int64_t at = blockIdx.x; at < a.all; at += gridDim.x) {
        const int which = at >= a.rows;
        const int64_t row = at - (which ? a.rows : 0);
        char* out = a.out[which];
        if (!out) continue;
        __syncthreads();  // the row before has been read
        const float* src = a.part + at * a.slots * LD;
        float m = 0.0f, l = 0.0f;
        if (!GRAD) {
            const float e = tid < a.slots ? src[tid * LD + DP] : -__builtin_inff();
            m = group_max<64>(e);
            if ((tid & 63) == 0) most[tid >> 6] = m;
            __syncthreads();
            m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            const float f = e == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(fmaf(e - m, a.scale2, src[tid * LD + DP + 2]));
            weight[tid] = f;
            l = group_sum<64>(tid < a.slots ? f * src[tid * LD + DP + 1] : 0.0f);
            if ((tid & 63) == 0) total[tid >> 6] = l;
            __syncthreads();
            l = total[0] + total[1] + total[2] + total[3];
        }
        const int d = tid % TD, sg = tid / TD;
        f32x4 v = {0, 0, 0, 0};
        if (sg < SG)
#pragma unroll 4
            for (int s = sg; s < a.slots; s += SG) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(src + s * LD + 4 * d);
                const float f = GRAD ? 1.0f : weight[s];
#pragma unroll
                for (int t = 0; t < 4; ++t) v[t] = fmaf(f, x[t], v[t]);
            }
        if (sg < SG) sums[sg][d] = v;
        __syncthreads();
        const int64_t seq = row / ((int64_t)a.tokens * a.heads);
        const int rest = (int)(row - seq * a.tokens * a.heads), tok = rest / a.heads, h = rest - tok * a.heads;
        if (!GRAD && a.stat && tid == 0)
            win_stat<BF>(a.top, a.stat, (seq * a.heads + h) * a.NP + tok, l != 0.0f, m, win_shift<BF>() + __builtin_amdgcn_logf(l));
        if (sg || 4 * d >= a.D) continue;
#pragma unroll
        for (int s = 1; s < SG; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] += sums[s][d][t];
        const float inv = GRAD ? a.factor[which] : l == 0.0f ? 0.0f : 1.0f / l;
        const uint2 x = make_uint2(win_pack<BF>(v[0] * inv, v[1] * inv), win_pack<BF>(v[2] * inv, v[3] * inv));
        *reinterpret_cast<uint2*>(out + seq * a.os[0] + tok * a.os[1] + h * a.os[2] + 8 * d) = x;
        if (!GRAD && a.rests)
            *reinterpret_cast<uint2*>(a.rests + ((seq * a.N + tok) * a.heads + h) * 2 * a.D + 8 * d) =
                make_uint2(win_rest<BF>(v[0] * inv, v[1] * inv, x.x), win_rest<BF>(v[2] * inv, v[3] * inv, x.y));
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static WinArgs win_args(const rpfq_window_desc& d, const void* q, const void* k, const void* v, const int32_t* lengths) {
    WinArgs a = {};
    a.q = reinterpret_cast<const char*>(q), a.k = reinterpret_cast<const char*>(k), a.v = reinterpret_cast<const char*>(v);
    for (int i = 0; i < 3; ++i)
        a.qs[i] = 2 * d.q_stride[i], a.ks[i] = 2 * d.k_stride[i], a.vs[i] = 2 * d.v_stride[i], a.os[i] = 2 * d.out_stride[i],
        a.gos[i] = 2 * d.grad_stride[i];
    a.lengths = lengths;
    a.B = (int)d.B, a.N = (int)d.N, a.H = (int)d.H, a.KV = (int)d.KV, a.D = (int)d.D, a.M = (int)d.M;
    a.NP = (int)window_rows(d.N);
    const int64_t most = d.M > d.N ? d.M : d.N;
    a.window = (int)(d.window < most ? d.window : most);
    a.sinks = (int)(d.sinks < most ? d.sinks : most);
    a.causal = d.causal;
    a.scale = d.scale;
    a.scale2 = d.scale * 1.4426950408889634f;
    a.top = d.top;
    a.rests = reinterpret_cast<char*>(d.rests);
    const int group = a.H / a.KV;
    a.hw = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    a.qw = 4 / a.hw;
    a.tiles = (a.NP + 32 * a.qw - 1) / (32 * a.qw);  // the statistics' rows behind N too
    return a;
}
template <class K>
static hipError_t win_launch(K kernel, std::atomic<uint64_t>& done, const WinArgs& a, int64_t blocks, int threads, int lds, hipStream_t s) {
    const hipError_t e = set_lds_attr_once(reinterpret_cast<const void*>(kernel), lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, a);
    return hipGetLastError();
}
#define WIN_LAUNCH(kernel, a, blocks, threads, lds, s)                         \
    [&] {                                                                      \
        static std::atomic<uint64_t> done{0};                                  \
        return win_launch(&kernel, done, a, blocks, threads, lds, s);          \
    }()

template <int DP, bool BF, bool GRAD>
static hipError_t win_join(WinJoin j, hipStream_t s) {
    j.all = j.rows * (j.out[1] ? 2 : 1);
    const int64_t most = 1 << 20;
    hipLaunchKernelGGL((window_join_kernel<DP, BF, GRAD>), dim3((unsigned)(j.all < most ? j.all : most)), dim3(256), 0, s, j);
    return hipGetLastError();
}
// rows of `tokens` contiguous tokens of n a sequence
static WinJoin win_joined(const WinArgs& a, const float* part, int tokens, int64_t n, int heads, int slots) {
    WinJoin j = {part};
    j.os[0] = n * heads * 2 * a.D, j.os[1] = (int64_t)heads * 2 * a.D, j.os[2] = 2 * a.D;
    j.rows = (int64_t)a.B * tokens * heads;
    j.tokens = tokens, j.heads = heads, j.slots = slots, j.D = a.D, j.N = a.N, j.NP = a.NP;
    j.scale2 = a.scale2;
    return j;
}
struct WinForward {
    const WinArgs& a;
    hipStream_t s;
    template <int DP, bool BF>
    hipError_t run() {
        const int64_t units = win_units(a.far, (int64_t)a.B * (a.H / a.hw), a.tiles);
        const hipError_t e = a.rests ? WIN_LAUNCH((window_forward_kernel<DP, BF, true>), a, units, 256, 4 * 64 * Rows<DP>::RB, s)
                                     : WIN_LAUNCH((window_forward_kernel<DP, BF, false>), a, units, 256, 4 * 64 * Rows<DP>::RB, s);
        if (e != hipSuccess || !a.far.parts) return e;
        WinJoin j = win_joined(a, a.part, a.far.rows, a.N, a.H, a.far.parts + 1);
        for (int i = 0; i < 3; ++i) j.os[i] = a.os[i];
        j.out[0] = a.out, j.rests = a.rests, j.top = a.top, j.stat = a.stat;
        return win_join<DP, BF, false>(j, s);
    }
};
// P and dS go into the gradients' products as one 16-bit term: over many rows what
// that rounds off adds up to as much as the results' own rounding (together 1.41 of
// it).  Over few rows it does not even out, and the results were off by up to 1.7
// of it: up to 8,192 rows (tokens x heads) have a second term each.  With it always,
// 8,192 tokens of 16 heads of 128 on 4 take 474 us forward and backward, with one
// 401; 512 tokens of 12 heads of 64 (6,144 rows) take 53 in a graph and with one 46,
// both less than the host's time without a graph.
constexpr int64_t kWinFewRows = 8192;
struct WinGrad {
    const WinArgs& a;
    hipStream_t s;
    template <int DP, bool BF>
    hipError_t run() {
        return (int64_t)a.B * a.H * a.N <= kWinFewRows ? go<DP, BF, true>() : go<DP, BF, false>();
    }
    template <int DP, bool BF, bool TWO>
    hipError_t go() {
        hipError_t e = WIN_LAUNCH((window_grad_q_kernel<DP, BF, TWO>), a, win_units(a.far, (int64_t)a.B * (a.H / a.hw), a.tiles), 256,
                                  4 * 64 * Rows<DP>::RB, s);
        if (e == hipSuccess && a.gq && a.far.parts) {
            WinJoin j = win_joined(a, a.part, a.far.rows, a.N, a.H, a.far.parts + 1);
            j.out[0] = a.gq, j.factor[0] = a.scale;
            e = win_join<DP, BF, true>(j, s);
        }
        if (e != hipSuccess || (!a.gk && !a.gv)) return e;
        e = WIN_LAUNCH((window_grad_kv_kernel<DP, BF, TWO>), a, win_units(a.kfar, (int64_t)a.B * a.KV, (a.N + kWinKeys - 1) / kWinKeys), 256,
                       win_grad_lds<DP>(), s);
        if (e != hipSuccess || !a.kfar.parts) return e;
        WinJoin j = win_joined(a, a.kpart, a.kfar.rows, a.N, a.KV, a.kfar.parts + 1);
        j.out[0] = a.gk, j.out[1] = a.gv, j.factor[0] = a.scale, j.factor[1] = 1.0f;
        return win_join<DP, BF, true>(j, s);
    }
};
template <int DP>
constexpr int win_cached_lds() {
    constexpr int W = win_waves<DP>();
    const int rings = W * 4 * 32 * Rows<DP>::RB, sums = W * 32 * (DP + 6) * 4;
    return rings > sums ? rings : sums;
}
struct WinCached {
    const WinArgs& a;
    hipStream_t s;
    template <int DP, bool BF>
    hipError_t run() {
        const hipError_t e = WIN_LAUNCH((window_cached_kernel<DP, BF>), a, (int64_t)a.B * a.KV * a.blocks * a.splits, 64 * win_waves<DP>(),
                                        win_cached_lds<DP>(), s);
        if (e != hipSuccess || a.splits == 1) return e;
        WinJoin j = win_joined(a, a.part, a.N, a.N, a.H, a.splits);
        j.out[0] = a.out;
        return win_join<DP, BF, false>(j, s);
    }
};
template <bool BF, class Go>
static hipError_t win_dim(int D, Go go) {
    if (D <= 32) return go.template run<32, BF>();
    if (D <= 64) return go.template run<64, BF>();
    if (D <= 96) return go.template run<96, BF>();
    return go.template run<128, BF>();
}
template <class Go>
static hipError_t win_dispatch(const rpfq_window_desc& d, Go go) {
    return d.dtype == RPFQ_BF16 ? win_dim<true>((int)d.D, go) : win_dim<false>((int)d.D, go);
}

// Whether the tiles with sinks go in parts: where one of them has more steps than
// a CU's share of them all (`slots` workgroups at once), so that the launch would
// wait for it; a part is `share` of a tile's own steps.  `rows`, `steps` a tile.
// Up to 128 sinks: the parts' float32 sums grow with them (16 heads of 128: 72 MB
// then). With more a tile goes over its range alone: 8,192 tokens, 16 heads of 128
// on 4, window 1,024, forward and backward 0.43 ms with 128 and 1.0 with 129.
static WinFar win_far(int64_t sinks, int64_t groups, int64_t tiles, int64_t rows, int64_t window, int64_t N, int heads, int share) {
    WinFar f = {(int)((sinks + rows - 1) / rows), (int)sinks, 0};
    const int64_t all = heads * ((N + 63) / 64), near = heads * ((rows + window) / 64 + 1), slots = 2 * device_cus();
    if (!sinks || sinks > 128 || all <= 2 * near || all * slots <= groups * tiles * near) return f;
    const int64_t step = near / share > 4 ? near / share : 4, parts = (all - near + step - 1) / step;
    f.parts = (int)(parts > 64 ? 64 : parts);
    return f;
}
static void win_fars(WinArgs& a) {
    const int64_t near = 2 * (int64_t)a.window;  // to both sides
    if (!a.causal) a.far = win_far(a.sinks, (int64_t)a.B * (a.H / a.hw), a.tiles, 32 * a.qw, near, a.N, 1, 4);
    a.kfar = win_far(a.sinks, (int64_t)a.B * a.KV, (a.N + kWinKeys - 1) / kWinKeys, kWinKeys, a.causal ? a.window : near, a.N, a.H / a.KV, 8);
}
static size_t win_part_floats(const WinFar& f, int64_t heads, int64_t B, int64_t D) {
    return f.parts ? (size_t)B * f.rows * heads * (f.parts + 1) * ((D + 31) / 32 * 32 + 8) : 0;
}
// The workspace: rowsum(dO O) (gradient), the sinks' sums as queries, as keys.
size_t window_bytes(const rpfq_window_desc& d, bool grad) {
    WinArgs a = win_args(d, nullptr, nullptr, nullptr, nullptr);
    win_fars(a);
    size_t n = win_part_floats(a.far, a.H, a.B, a.D);
    if (grad) n += (size_t)a.B * a.H * a.NP + 2 * win_part_floats(a.kfar, a.KV, a.B, a.D);
    return 4 * n;
}

hipError_t launch_window_attention(const rpfq_window_desc& d, const void* q, const void* k, const void* v, const int32_t* lengths,
                                   void* out, float* stat, void* work, hipStream_t s) {
    WinArgs a = win_args(d, q, k, v, lengths);
    win_fars(a);
    a.out = reinterpret_cast<char*>(out);
    a.stat = stat;
    a.part = reinterpret_cast<float*>(work);
    return win_dispatch(d, WinForward{a, s});
}
hipError_t launch_window_attention_grad(const rpfq_window_desc& d, const void* q, const void* k, const void* v, const int32_t* lengths,
                                        const void* out, const void* grad_out, const float* stat, void* gq, void* gk, void* gv,
                                        void* work, hipStream_t s) {
    WinArgs a = win_args(d, q, k, v, lengths);
    a.o = reinterpret_cast<const char*>(out), a.go = reinterpret_cast<const char*>(grad_out);
    a.stat = const_cast<float*>(stat);
    win_fars(a);
    a.delta = reinterpret_cast<float*>(work);
    a.part = a.delta + (size_t)a.B * a.H * a.NP;
    a.kpart = a.part + win_part_floats(a.far, a.H, a.B, a.D);
    a.gq = reinterpret_cast<char*>(gq), a.gk = reinterpret_cast<char*>(gk), a.gv = reinterpret_cast<char*>(gv);
    return win_dispatch(d, WinGrad{a, s});
}

// Parts of the keys of one key head.  One where a wave has 5 tiles of 32 keys at
// most: a second launch, to join, costs more than its share of them (a token of 8
// streams, 12 heads of 64 over 1,028 slots: 14.8 us in 9 parts, 9.4 in one).
// Else as many as fill the chip's workgroups, two at least for long ones, whose
// lengths differ (64 streams, 4 key heads of 128 over 4,100 slots: 106 us in 2
// parts, 118 in 4, 136 in 9), each of 4 tiles (a tile a wave) or more.  Several
// blocks of rows a key head that fill the chip: one, since every row's float32 sums
// go through memory twice (4 key heads of 128, bf16: 8 x 64 new tokens over 4,096
// slots 60 us in 2 parts, 50 in one; 8 x 2,048 3.2 ms and 2.6, and 0.3 GB less).
int window_splits(const rpfq_window_desc& d) {
    const int64_t blocks = ((d.H / d.KV) * d.N + 31) / 32, units = d.B * d.KV * blocks, waves = d.D > 64 ? win_waves<128>() : win_waves<64>();
    const int64_t window = d.window < d.M ? d.window : d.M, sinks = d.sinks < d.M ? d.sinks : d.M;  // any int64: clamped before they are added
    const int64_t all = window + d.N - 1 + sinks, keys = all < d.M ? all : d.M;
    if (keys <= 5 * 32 * waves) return 1;
    if (blocks > 1 && units >= device_cus()) return 1;
    const int64_t most = (keys + 127) / 128, fill = device_cus() / units, want = fill > 2 ? fill : 2;
    const int64_t s = most < want ? most : want;
    return (int)(s < 1 ? 1 : s > kWinSlots ? kWinSlots : s);
}
// Threads of the largest launch of a call: a grid of 2^32 or more is none.
int64_t window_threads(const rpfq_window_desc& d, bool cached, bool grad) {
    if (cached) return d.B * d.KV * ((d.H / d.KV * d.N + 31) / 32) * window_splits(d) * 64 * (d.D > 64 ? win_waves<128>() : win_waves<64>());
    WinArgs a = win_args(d, nullptr, nullptr, nullptr, nullptr);
    win_fars(a);
    const int64_t q = win_units(a.far, (int64_t)a.B * (a.H / a.hw), a.tiles);
    const int64_t k = grad ? win_units(a.kfar, (int64_t)a.B * a.KV, (a.N + kWinKeys - 1) / kWinKeys) : 0;
    return 256 * (q > k ? q : k);
}
size_t window_cached_bytes(const rpfq_window_desc& d) {
    const int s = window_splits(d);
    if (s == 1) return 0;
    const size_t dp = (size_t)((d.D + 31) / 32 * 32);
    return (size_t)d.B * d.N * d.H * s * (dp + 8) * 4;
}
hipError_t launch_window_attention_cached(const rpfq_window_desc& d, const void* q, const void* k, const void* v, const int32_t* lengths,
                                          void* out, void* work, hipStream_t s) {
    WinArgs a = win_args(d, q, k, v, lengths);
    a.out = reinterpret_cast<char*>(out);
    a.part = reinterpret_cast<float*>(work);
    a.causal = 1;
    a.rows = a.H / a.KV * a.N;
    a.blocks = (a.rows + 31) / 32;
    a.splits = window_splits(d);
    return win_dispatch(d, WinCached{a, s});
}

}  // namespace rpfq
