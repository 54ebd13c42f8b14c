// The matrix product under the unembedding's cross entropy (unembed.hip): 16-bit operands, fp32 accumulation.
//
//   C[i][j] = sum_k A(i, k) * B(j, k)
//
// One workgroup computes a BI x BJ tile in steps of SK k.  Both operand tiles of a step go global -> LDS by
// global_load_lds_dwordx4 (1 KiB a wave and instruction, no registers) into one of NS buffers while another one is
// multiplied; one barrier a step.  Operands come in two layouts:
//   row-major  A(i, k) = A[i * ld + k]: LDS rows of 64 k = 128 bytes, two buffers, a fragment is one ds_read_b128
//   k-major    A(i, k) = A[k * ld + i]: LDS rows of BI elements, four buffers of 32 k, a fragment is two transposing
//              ds_read_b64_tr_b16
// (Four buffers of 32 k give a copy three steps of time instead of three quarters of a longer one: k-major 1209 against 1178
// TFLOP/s on random operands at 768 x 21760 x 16384 and 1854 against 1567 on zeros, which the power limit leaves alone.
// Row-major rows of 32 k are 64 bytes, half a cache line: 1142 against 1195.)
// 16-byte chunks are permuted through the source address of the copy (row-major: chunk ^ (row / 2) % 8; k-major: the
// 64-byte groups ^ k % 4), which spreads the lanes of a fragment read over the banks: no conflict is counted.
// What bounds the loop is power: at 70 % of its issue slots the matrix pipe runs at 1.5-1.6 GHz on real operands, and the
// vendor's own kernel, at 94 %, at 1.44 (1340-1375 TFLOP/s at 8192^3; this loop 1292).
//
// fp32 operands are split into two fp16 planes: v / s = h1 + h2, s a power of two that brings the largest magnitude into
// [2^14, 2^15).  h1 holds 11 bits and h2 the next 11: 22 bits for values down to 2^-17 of the largest, a fixed 2^-39 of it
// below (fp16 ends at 2^-24).  The product is h1 h1' + h1 h2' + h2 h1'; the dropped h2 h2' is 2^-22 of it at most.  Every
// product of two fp16 values is exact in the matrix pipe, sums are fp32: the result carries the error of an fp32 product at
// a third of the 16-bit rate, 5 times the fp32 matrix rate.
// G, whose entries are probabilities and span many more powers of two, is split as h1 + h2 / 2048: 22 bits down to 2^-28 of
// the largest and a fixed 2^-50 of it below; the other operand's h1 is divided by 2048 in registers before it meets that h2.
// The planes of 32 neighbouring elements lie next to each other, element e's h1 at e / 32 * 64 + e % 32 and its h2 32 behind
// it: a cache line holds both, and a step brings both planes of half as many k through LDS for three products, where one
// pass a product would bring each plane three times in two.
#pragma once
#include <type_traits>

#include "tsc_internal.h"

namespace unembed_gemm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(1))) void *gptr_t;
typedef __attribute__((address_space(3))) void *lptr_t;

constexpr int BK = 64;  // k are counted and padded in multiples of this

template <int WI_, int WJ_, int VI_, int VJ_> struct Tile {  // 32 x 32 blocks of a wave, waves of a workgroup
    static constexpr int WI = WI_, WJ = WJ_, VI = VI_, VJ = VJ_, NW = VI * VJ, NT = 64 * NW;
    static constexpr int BI = VI * WI * 32, BJ = VJ * WJ * 32;
    static constexpr int OCC = 2;  // waves a SIMD at least
};
// (LARGE as four waves of 128 x 128, one a SIMD with its 256 sums in accumulator registers, has 2/3 of the LDS reads and a
// loop without a spill; alone it measured 1195 TFLOP/s against 1292 of eight waves of 128 x 64 at 8192^3, and its epilogue
// overlaps with nothing: loss of 65536 rows 6.55 ms against 4.47.  Two workgroups a CU of four waves and 128 x 192, so that one
// multiplies while the other takes exponentials: 4.58 against 4.16 ms, 1178 against 1063 us at 16384 rows -- they move more bytes
// a product, and power is the limit.)
typedef Tile<4, 2, 2, 4> TileLarge;   // 256 x 256, one workgroup a CU
typedef Tile<2, 2, 2, 2> TileMedium;  // 128 x 128, two
typedef Tile<1, 2, 4, 1> TileTall;    // 128 x 64: few tokens, the vocabulary streams
typedef Tile<2, 1, 1, 4> TileWide;    // 64 x 128: the same with the operands exchanged

struct Operand {
    const short *p;
    long long ld;  // 16-bit elements (of both planes) between rows (row-major) or between k (k-major)
    int rows;      // valid i (j); the tile's others read copies of valid ones
};

// 16 bytes a lane, global -> LDS: base + off (of the lane) to LDS address at + 16 * lane.  Written out, and not through the
// builtin, because the compiler would wait for every copy in flight before the next LDS read, whichever buffer that reads;
// Gemm::run waits by itself, once a step.  (m0 is the compiler's only next to an instruction that takes it; none here does.)
__device__ __forceinline__ void copy16(const char *base, unsigned off, unsigned at) {
    const unsigned long long b = (unsigned long long)base;  // (uniform; said again for where the compiler lost sight of it)
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)b), hi = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32));
    const unsigned long long u = (unsigned long long)hi << 32 | lo;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(u));
}

// One tile of a workgroup's stream: first rows of both operands.
struct TileAt {
    int i0, j0;
};

// The product of a stream of tiles.  All steps of all tiles of a workgroup form one stream: step s + 1 is in LDS and steps up
// to s + NS on their way while step s is multiplied, also across the end of a tile, so that only the first tile waits for
// memory.
//
//   step s:  products of all but the last 16 k, each group while the fragments of the next are read
//            wait: own fragments of the last group are in registers, own copies of step s + 1 have landed; barrier
//            products of the last group while the first fragments of step s + 1 are read and the copies of step s + NS issued
//
// Behind the barrier nobody reads the buffer of step s any more and everybody's part of step s + 1 is there.
// SCALED (two planes): the operand whose h2 is held times 2048 -- 0: none, 1: A, 2: B.
template <class C, bool KMAJOR, bool F16, int PLANES, int SCALED = 0> struct Gemm {
    static_assert(PLANES == 1 || F16, "planes are fp16");
    static constexpr int SK = (KMAJOR ? 32 : 64) / PLANES, NS = KMAJOR ? 4 : 2, KK = SK / 16;
    static constexpr int ABYTES = C::BI * SK * PLANES * 2, BBYTES = C::BJ * SK * PLANES * 2, STAGE = ABYTES + BBYTES;
    static constexpr int LDS_BYTES = NS * STAGE;
    static constexpr int PA = ABYTES / 1024 / C::NW, PB = BBYTES / 1024 / C::NW, P = PA + PB;  // 1-KiB pieces of a step and wave
    static_assert(P * C::NW * 1024 == STAGE, "whole pieces a wave");

    // byte offsets of this lane's part of the PIECES 1-KiB pieces of this wave, relative to the tile's base
    template <int ROWS, int PIECES>
    static __device__ __forceinline__ void offsets(const Operand &o, int row0, unsigned (&off)[PIECES]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int piece = wave * PIECES + q;
            if (KMAJOR) {
                constexpr int CH = ROWS * PLANES / 8;  // 16-byte chunks of a k
                const int at = piece * 64 + lane, k = at / CH, c = (at % CH) ^ (((k & 3) << 2) & (CH - 1));
                const int last = (PLANES == 2 ? (o.rows + 31) / 32 * 64 : (o.rows + 7) / 8 * 8) - 8 - row0 * PLANES;
                const int i = c * 8 < last ? c * 8 : last;  // (last >= 0: a tile has at least one row)
                off[q] = (unsigned)(k * (int)o.ld + i) * 2u;
            } else {
                const int r = piece * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
                const int i = row0 + r < o.rows ? r : o.rows - 1 - row0;
                off[q] = (unsigned)(i * (int)o.ld + c * 8) * 2u;
            }
        }
    }
    static __device__ __forceinline__ const char *base(const Operand &o, int row0, int k0) {
        return (const char *)(o.p + (KMAJOR ? (long long)k0 * BK * o.ld + row0 * PLANES : (long long)row0 * o.ld + (long long)k0 * BK * PLANES));
    }
    static __device__ __forceinline__ long long step_bytes(const Operand &o) { return KMAJOR ? 2ll * SK * o.ld : 128; }

    template <int ROWS> struct Frag {  // fragment reads of one operand
        static constexpr int PITCH = ROWS * PLANES * 2;   // k-major: bytes of a k
        unsigned at[KMAJOR ? KK : KK * PLANES];           // LDS address of block 0: of each 16 k, row-major also of each plane
        __device__ __forceinline__ Frag(int row0, int extra) {
            const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
            if constexpr (KMAJOR) {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const int l = lane & 15, g = lane >> 4, k = kk * 16 + (g >> 1) * 8 + (l >> 2);
                    const int i = (g & 1) * 16 + (l & 3) * 4;  // of the block
                    const int chunk = row0 * PLANES / 8 + (i >> 3);
                    at[kk] = extra + k * PITCH + ((chunk ^ (((k & 3) << 2) & (ROWS * PLANES / 8 - 1))) << 4) + (i & 4) * 2;
                }
            } else {
#pragma unroll
                for (int c = 0; c < KK * PLANES; ++c) at[c] = extra + (row0 + li) * 128 + (((c * 2 + lh) ^ ((li >> 1) & 7)) << 4);
            }
        }
        // rows row0 + 32 * b, 16 k number kk, a plane: lane l holds row l % 32, k = 8 * (l / 32) + 0..7
        __device__ __forceinline__ s16x8 read(const char *lds, unsigned buf, int kk, int plane, int b) const {
            if constexpr (KMAJOR) {
                // the chunk permutation acts on the 64-byte groups, so a block's distance, 64 bytes a plane, is an exclusive or too
                typedef __attribute__((address_space(3))) s16x4 *p4;
                const char *p = lds + (at[kk] ^ ((b * PLANES + plane) * 64)) + buf;
                const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)p);
                const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)(p + 4 * PITCH));
                return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                return *(const s16x8 *)(lds + at[plane * KK + kk] + buf + b * 4096);
            }
        }
    };
    static __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        if constexpr (F16)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }

    static __device__ __forceinline__ s16x8 smaller(s16x8 h) {  // h1 / 2048
        return __builtin_bit_cast(s16x8, __builtin_bit_cast(f16x8, h) * (_Float16)(1.f / 2048.f));
    }

    // tiles t = 0 .. n_tiles - 1 at tile(t), k from k0 * BK to k1 * BK.  begin(t, acc) sets a tile's accumulators,
    // done(t, acc) takes its sums.  LDS of the stages: lds[0 .. LDS_BYTES).
    template <class At, class Begin, class Done>
    static __device__ __forceinline__ void run(const Operand &A, const Operand &B, int n_tiles, At tile, int k0, int k1, char *lds,
                                               Begin begin, Done done) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int n = (k1 - k0) * (BK / SK);
        f32x16 acc[C::WI][C::WJ];
        if (n_tiles <= 0) return;
        if (n <= 0) {  // (a part of the k-steps behind their end)
            for (int t = 0; t < n_tiles; ++t) {
                begin(t, acc);
                done(t, acc);
            }
            return;
        }
        const Frag<C::BI> ra((wave / C::VJ) * (C::WI * 32), 0);
        const Frag<C::BJ> rb((wave % C::VJ) * (C::WJ * 32), ABYTES);
        unsigned offa[PA], offb[PB];
        // the producer: the next step to copy
        int pt = 0, ps = 0;
        unsigned pbuf = 0;
        const char *pa, *pb;
        const long long da = step_bytes(A), db = step_bytes(B);
        auto set_tile = [&]() {
            const TileAt at = tile(pt);
            offsets<C::BI, PA>(A, at.i0, offa);
            offsets<C::BJ, PB>(B, at.j0, offb);
            pa = base(A, at.i0, k0);
            pb = base(B, at.j0, k0);
        };
        const unsigned l0 = (unsigned)(size_t)(lptr_t)lds, la = l0 + wave * PA * 1024, lb = l0 + ABYTES + wave * PB * 1024;
        auto piece = [&](int q) {
            if (q < PA) copy16(pa, offa[q < PA ? q : 0], la + pbuf + q * 1024);
            else copy16(pb, offb[q < PA ? 0 : q - PA], lb + pbuf + (q - PA) * 1024);
        };
        auto advance = [&]() {
            pbuf = pbuf + STAGE == LDS_BYTES ? 0 : pbuf + STAGE;
            if (++ps < n) {
                pa += da;
                pb += db;
                return;
            }
            if (pt + 1 < n_tiles) {
                ps = 0;
                ++pt;
                set_tile();
            }  // else: the stream is at its end, its last step is copied again (NS times, unread: no branch in the loop)
        };
        set_tile();
        for (int i = 0; i < NS; ++i) {
#pragma unroll
            for (int q = 0; q < P; ++q) piece(q);
            advance();
        }
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * P) : "memory");
        s16x8 fa[2][C::WI], fb[2][C::WJ];
        unsigned buf = 0;
        constexpr int G = C::WI * C::WJ;
        // all products of fragments x and y, and behind each of them a part of the `reads` fragment reads read(r) and (COPY) of
        // the step's copies, in this order: a burst of either would leave the matrix pipe idle, and so would the compiler's
        // own order.  The reads end with the first half of the products.
        auto group = [&](const s16x8(&x)[C::WI], const s16x8(&y)[C::WJ], auto copy_, auto reads_, auto read) __attribute__((always_inline)) {
            constexpr int R = decltype(reads_)::value;
            constexpr bool COPY = decltype(copy_)::value;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int a = g / C::WJ, b = a & 1 ? C::WJ - 1 - g % C::WJ : g % C::WJ;  // (back and forth: one operand stays)
                acc[a][b] = mfma(x[a], y[b], acc[a][b]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = g * 2 * R / G; r < (g + 1) * 2 * R / G && r < R; ++r) read(r);
                if (COPY)
#pragma unroll
                    for (int q = g * P / G; q < (g + 1) * P / G; ++q) piece(q);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const std::false_type no;
        const std::true_type yes;
        const std::integral_constant<int, C::WI> wi;
        const std::integral_constant<int, C::WJ> wj;
        const std::integral_constant<int, C::WI + C::WJ> both;
        auto next_step = [&]() __attribute__((always_inline)) {  // own reads of this step's buffer are done, the next step is there
            buf = buf + STAGE == LDS_BYTES ? 0 : buf + STAGE;
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * P) : "memory");
        };
        // reads of the 16 k number kk: both operands' h1 into sets sa and sb
        auto first = [&](int kk, int sa, int sb) {
            return [&, kk, sa, sb](int r) __attribute__((always_inline)) {
                if (r < C::WJ) fb[sb][r < C::WJ ? r : 0] = rb.read(lds, buf, kk, 0, r);
                else fa[sa][r < C::WJ ? 0 : r - C::WJ] = ra.read(lds, buf, kk, 0, r - C::WJ);
            };
        };
        // Two planes: the three products of 16 k.  The set that is free before the last product takes the next h1 of its operand,
        // so one operand's h1 changes between the sets from one 16 k to the next (PAR).
        //   SCALED 0, 1: h1 h1', h1 h2', h2 h1' -- B's h1 in set PAR;     SCALED 2: h1 h1', h2 h1', h1 h2' -- A's h1 in set PAR
        auto three = [&](auto par_, auto last_, int kk, int kk_next) __attribute__((always_inline)) {
            constexpr int PAR = decltype(par_)::value;
            constexpr bool LAST = decltype(last_)::value;  // of its step
            if constexpr (SCALED == 2) {
                group(fa[PAR], fb[0], no, wi, [&](int r) __attribute__((always_inline)) { fa[PAR ^ 1][r] = ra.read(lds, buf, kk, 1, r); });
                group(fa[PAR ^ 1], fb[0], no, wj, [&](int r) __attribute__((always_inline)) { fb[1][r] = rb.read(lds, buf, kk, 1, r); });
#pragma unroll
                for (int a = 0; a < C::WI; ++a) fa[PAR][a] = smaller(fa[PAR][a]);
                if constexpr (LAST) next_step();
                group(fa[PAR], fb[1], last_, both, first(kk_next, PAR ^ 1, 0));
            } else {
                group(fa[0], fb[PAR], no, wj, [&](int r) __attribute__((always_inline)) { fb[PAR ^ 1][r] = rb.read(lds, buf, kk, 1, r); });
                group(fa[0], fb[PAR ^ 1], no, wi, [&](int r) __attribute__((always_inline)) { fa[1][r] = ra.read(lds, buf, kk, 1, r); });
                if constexpr (SCALED == 1) {
#pragma unroll
                    for (int b = 0; b < C::WJ; ++b) fb[PAR][b] = smaller(fb[PAR][b]);
                }
                if constexpr (LAST) next_step();
                group(fa[1], fb[PAR], last_, both, first(kk_next, 0, PAR ^ 1));
            }
            if constexpr (LAST) advance();
        };
        const std::integral_constant<int, 0> even;
        const std::integral_constant<int, 1> odd;
#pragma unroll
        for (int r = 0; r < C::WI + C::WJ; ++r) first(0, 0, 0)(r);
        for (int t = 0; t < n_tiles; ++t) {
            begin(t, acc);
            if constexpr (PLANES == 1) {
                for (int s = 0; s < n; ++s) {
                    if constexpr (KK == 4) {
                        group(fa[0], fb[0], no, both, first(1, 1, 1));
                        group(fa[1], fb[1], no, both, first(2, 0, 0));
                    }
                    group(fa[0], fb[0], no, both, first(KK - 1, 1, 1));
                    next_step();
                    group(fa[1], fb[1], yes, both, first(0, 0, 0));  // (behind the last tile's last step these are not used)
                    advance();
                }
            } else if constexpr (KK == 2) {
                for (int s = 0; s < n; ++s) {
                    three(even, no, 0, 1);
                    three(odd, yes, 1, 0);
                }
            } else {
                for (int s = 0; s < n; s += 2) {  // (n is a multiple of 4)
                    three(even, yes, 0, 0);
                    three(odd, yes, 0, 0);
                }
            }
            done(t, acc);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may arrive in LDS that is somebody else's by then
    }
};

// Element r of a 32 x 32 block: row (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), column lane & 31.
__device__ __forceinline__ int block_row(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }

}  // namespace unembed_gemm
