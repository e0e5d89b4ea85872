// Products in 8-bit floating point: P[i, j] = sum_k A(i, k) B(j, k), A and B held as
// e4m3 codes with a power of two for every 128 of k, accumulated in f32.
//
// The scales.  A block's scale is the least power of two with which no magnitude of
// the block passes 448, the largest code: the scaling is exact, so a value is
// rounded once, and v_mfma_scale_f32_16x16x128_f8f6f4 takes the exponents of both
// operands as bytes beside the codes: one instruction is one block of k, and no
// vector instruction is spent on scales.  (A power of two costs at most one bit of
// range below a scale of amax / 448, and none of precision but for codes near the
// smallest.)
//
// The sums.  Of eight adjacent products the instruction cuts off, towards zero, what
// lies below 2^-13 of the largest one's power of two (measured with single products;
// the groups of eight, and the sum with the accumulator, are added as f32 is): an
// error of 2^-16 of the sum of magnitudes at most was seen over 128 random terms, well
// below the rounding of a 16-bit result, which is what such sums go to.  In a training
// step the kept z has it, and with z a few codes of dz in a thousand are the next ones:
// 8192 x 4096 by 8192 bf16 is 2.0e-3 off 64 bits, 1.7e-3 with exact sums.  f32 results
// do without: their operands are made as bf16 values (a code times its power of two
// has four bits) and multiplied by train_gemm.hpp's instructions, at half the rate.
//
// Operands.  Codes have k contiguous, rows padded with zeros to whole blocks.  Scales
// are bytes (the exponent + 127) in words of four blocks: of weights, words of every 128
// rows in turn; of rows made for a product, the rows' words of the same four blocks
// side by side, so that a workgroup that makes the codes of 128 x 128 writes its 128
// bytes into four lines.  All three products of a layer have this layout, as
// the kernel that makes the codes writes them transposed where that is wanted.
//
// Tile.  As train_gemm.hpp's, with the same swizzles: 128 bytes of k are one staged
// width and one instruction per 16 x 16 block; a lane holds the chunks l / 16 and 4 +
// l / 16 of its row, in either operand, which is any order of k as long as a block has
// one scale.  The words of the scales of four staged widths go through LDS too; a lane
// shifts its words down by a byte each width.
#pragma once
#include "train_epilogue.hpp"
#include "train_launch.hpp"

namespace mlrs {
namespace train {

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <>
struct Elem<uint8_t> {
    typedef u32x4 Frag;
};

// Where the scales of an operand are: the word of four blocks of row r, or of 128 rows
// (shift 7), is at s + (r >> shift) * step + word * plane.
struct ScaleRows {
    const uint8_t* s;
    int64_t step, plane, rows;  // bytes, bytes, and how many of r >> shift
    int shift;
};

struct Fp8Args {
    GemmArgs g;
    ScaleRows sa, sb;
};

__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
#else
    (void)a;
    (void)b;
    (void)sa;
    (void)sb;
    return c;
#endif
}

__device__ __forceinline__ i32x8 join_halves(u32x4 lo, u32x4 hi) {
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Panels of either operand that a tile keeps in LDS.
template <int MB>
__host__ __device__ constexpr int fp8_depth() {
    return MB == 2 ? 3 : 2;
}
template <int WM, int WN, int MB, int NB>
__host__ __device__ constexpr int fp8_lds() {
    return fp8_depth<MB>() * (WM * MB + WN * NB) * 16 * kStageBytes + 2 * (WM * MB + WN * NB) * 16 * 4;
}

// A wave's copies of a panel of codes into LDS, in the places of train_gemm.hpp's
// Stager: eight rows an instruction, a lane the chunk that the swizzle of its row puts
// there.  What that adds to an instruction's first row is the same for every second
// instruction, and for both operands, whose rows are as long: two registers a lane,
// where the accumulators leave few.
struct CodeStager {
    const char* base;  // the wave's first row, at k = 0
    int64_t bytes;     // from base to the operand's end
    int64_t pair;      // bytes of sixteen rows
    __device__ __forceinline__ void init(const Operand& o, int32_t row0, int32_t rows, int32_t wave_rows, int wave) {
        const int64_t first = (int64_t)row0 + (int64_t)wave * wave_rows;
        base = reinterpret_cast<const char*>(o.p) + first * o.ld;
        bytes = ((int64_t)rows - first) * o.ld;
        pair = 16 * o.ld;
    }
    // Instruction I of the wave's, at k0; past the end come zeros.
    template <int I>
    __device__ __forceinline__ void load(char* lds, int64_t k0, const uint32_t (&off)[2]) const {
        const int64_t skip = k0 + (I / 2) * pair, left = bytes - skip;
        const uint64_t at = (uint64_t)(base + skip);
        u32x4 rsrc;
        rsrc[0] = (uint32_t)at;
        rsrc[1] = (uint32_t)(at >> 32) & 0xFFFFu;
        rsrc[2] = left < 0x7FFFFFFF ? (left > 0 ? (uint32_t)left : 0u) : 0x7FFFFFFFu;
        rsrc[3] = 0x00027000u;
        copy_to_lds(rsrc, lds + I * 1024, off[I & 1]);
    }
};

// The words of 64 rows' scales into LDS.
struct ScaleCopy {
    const uint8_t* base;  // of the tile's first row (or its 128)
    int64_t plane;
    uint32_t bytes;       // of a plane, from base to its end
    uint32_t off;         // the lane's
    __device__ __forceinline__ void init(const ScaleRows& s, int32_t row0, int32_t row) {
        const int64_t first = row0 >> s.shift, left = (s.rows - first) * s.step;
        base = s.s + first * s.step;
        plane = s.plane;
        bytes = left < 0x7FFFFFFF ? (left > 0 ? (uint32_t)left : 0u) : 0x7FFFFFFFu;
        off = (uint32_t)((((int64_t)row0 + row) >> s.shift) - first) * (uint32_t)s.step;
    }
    // Word w; past the last one zeros.
    __device__ __forceinline__ void load(char* lds, int32_t w, bool past) const {
        const uint64_t from = (uint64_t)(base + w * plane);
        // uniform, which the compiler must see
        const int lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)from);
        const int hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(from >> 32));
        const int records = __builtin_amdgcn_readfirstlane(past ? 0 : (int)bytes);
        u32x4 rsrc;
        rsrc[0] = (uint32_t)lo;
        rsrc[1] = (uint32_t)hi & 0xFFFFu;
        rsrc[2] = (uint32_t)records;
        rsrc[3] = 0x00027000u;
        copy_word_to_lds(rsrc, lds, off);
    }
};

// A workgroup of every product.  8192^3 takes 429 to 437 us, 2.5 PFLOP/s (the library's
// product with one scale a tensor 406), where the matrix instructions alone take 302,
// without copies 333, without LDS reads 405: bound by the chip's power, at a clock near
// 2.0 GHz with the matrix cores busy for 59 % of the cycles, and by the copies.  Copies
// spread between the last part's instructions, and a second barrier that frees a slot
// earlier, were 30 % slower and 1.5 % faster.
// buf: fp8_lds bytes, the kernel's only LDS.
template <int WM, int WN, int MB, int NB, typename Epi>
__device__ __forceinline__ void fp8_workgroup(const Fp8Args& q, const Epi& epi, uint32_t wg, char* buf) {
    constexpr int BM = WM * MB * 16, BN = WN * NB * 16, WAVES = WM * WN;
    constexpr int kA = BM * kStageBytes, kB = BN * kStageBytes, kPair = kA + kB;
    constexpr int kDepth = fp8_depth<MB>();
    constexpr int kScales = (BM + BN) * 4;  // bytes of four widths
    constexpr int kScaleWaves = (BM + BN) / 64;
    static_assert(BM % 64 == 0 && BN % 64 == 0 && kScaleWaves <= WAVES && (kScaleWaves & (kScaleWaves - 1)) == 0,
                  "a wave copies the scales of 64 rows");
    const GemmArgs& g = q.g;
    char* const scales = buf + kDepth * kPair;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const TilePlace t = tile_place(g, wg);
    const int32_t m0 = t.tm * BM, n0 = t.tn * BN;
    const int32_t k_lo = t.split * g.k_split;
    const int32_t k_hi = g.k - k_lo < g.k_split ? g.k : k_lo + g.k_split;
    const int32_t widths = (k_hi - k_lo) / kStageBytes;

    static_assert(BM == BN, "both operands' panels alike");
    constexpr int kInstr = BM / 8 / WAVES, kCopies = 2 * kInstr;  // of an operand, of both
    static_assert(kInstr % 2 == 0, "sixteen rows at a time");
    CodeStager sa, sb;
    sa.init(g.a, m0, g.m, kInstr * 8, wave);
    sb.init(g.b, n0, g.n, kInstr * 8, wave);
    uint32_t off[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 8 * i + (lane >> 3);
        off[i] = (uint32_t)r * (uint32_t)g.a.ld + 16u * (uint32_t)((lane & 7) ^ k_swizzle(r));
    }
    char* const panel = buf + wave * kInstr * 1024;  // the wave's part of a panel
    ScaleCopy sc;
    const int part = wave & (kScaleWaves - 1);  // of the words; small tiles have more waves
    if (part < BM / 64)
        sc.init(q.sa, m0, part * 64 + lane);
    else
        sc.init(q.sb, n0, (part - BM / 64) * 64 + lane);
    Reader<uint8_t, true, BM, MB> ra;
    Reader<uint8_t, true, BN, NB> rb;
    ra.init(wm * MB * 16, lane);
    rb.init(wn * NB * 16, lane);

    // A width's code is one block without branches, four of them in turn: what it
    // does with the scales goes by its place U = p % 4.
    // Copies of width p, the scales of four before them: they are the older ones
    // where it is waited for all but the last.
    // Instructions I of them alone, FROM <= I < TO of either operand.
    auto copy_some = [&](int32_t p, int at, auto from, auto to) {
        const int64_t k0 = p < widths ? k_lo + p * kStageBytes : (int64_t)1 << 40;  // past the end: zeros
        auto one = [&](auto i) {
            if constexpr (decltype(i)::v >= decltype(from)::v && decltype(i)::v < decltype(to)::v) {
                sa.template load<decltype(i)::v>(panel + at, k0, off);
                sb.template load<decltype(i)::v>(panel + at + kA, k0, off);
            }
        };
        one(Set<0>{});
        one(Set<1>{});
        one(Set<2>{});
        one(Set<3>{});
    };
    static_assert(kInstr <= 4, "four are spelled out");
    auto copy_scales = [&](int32_t p, auto u) {
        if constexpr ((decltype(u)::v & 3) == 0)
            sc.load(scales + __builtin_amdgcn_readfirstlane(((p >> 2) & 1) * kScales + part * 256),
                    (k_lo >> 9) + (p >> 2), p >= widths);
    };
    auto copy = [&](int32_t p, int at, auto u) {
        copy_scales(p, u);
        copy_some(p, at, Set<0>{}, Set<kInstr>{});
    };
    auto next = [&](int at) { return at + kPair >= kDepth * kPair ? 0 : at + kPair; };
    auto frag_a = [&](const char* from, int i) { return join_halves(ra.get(from, 0, i), ra.get(from, 1, i)); };
    auto frag_b = [&](const char* from, int j) { return join_halves(rb.get(from + kA, 0, j), rb.get(from + kA, 1, j)); };

    f32x4 acc[MB][NB] = {};
    uint32_t wa[MB], wb[NB];  // scales, the width's in the low byte
    const int ra0 = (wm * MB * 16 + (lane & 15)) * 4, rb0 = (BM + wn * NB * 16 + (lane & 15)) * 4;
    // the scales of width p
    auto turn_scales = [&](int32_t p, auto u) {
        if constexpr ((decltype(u)::v & 3) != 0) {
#pragma unroll
            for (int i = 0; i < MB; ++i) wa[i] >>= 8;
#pragma unroll
            for (int j = 0; j < NB; ++j) wb[j] >>= 8;
        } else {
            const char* from = scales + ((p >> 2) & 1) * kScales;
#pragma unroll
            for (int i = 0; i < MB; ++i) wa[i] = *reinterpret_cast<const uint32_t*>(from + ra0 + i * 64);
#pragma unroll
            for (int j = 0; j < NB; ++j) wb[j] = *reinterpret_cast<const uint32_t*>(from + rb0 + j * 64);
        }
    };
    // every wave has width p in registers; width p + 1 is in LDS
    auto publish = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        wait_copies<(kDepth - 2) * kCopies>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    int cur = 0;
    auto all_widths = [&](auto width) {
        for (int32_t p = 0;;) {
            width(p, Set<0>{});
            if (++p == widths) break;
            width(p, Set<1>{});
            if (++p == widths) break;
            width(p, Set<2>{});
            if (++p == widths) break;
            width(p, Set<3>{});
            if (++p == widths) break;
        }
    };

    copy(0, 0, Set<0>{});
#pragma unroll
    for (int p = 1; p < kDepth; ++p) copy(p, p * kPair, Set<1>{});
    wait_copies<(kDepth - 1) * kCopies>();
    __builtin_amdgcn_s_barrier();
    if constexpr (MB == 2) {
        i32x8 fa[2][MB], fb[2][NB];
        auto fetch = [&](const char* from, int set) {
#pragma unroll
            for (int i = 0; i < MB; ++i) fa[set][i] = frag_a(from, i);
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[set][j] = frag_b(from, j);
        };
        fetch(buf, 0);
        turn_scales(0, Set<0>{});
        all_widths([&](int32_t p, auto u) {
            constexpr int U = decltype(u)::v, kSet = U & 1;
            publish();
            copy(p + kDepth, cur, Set<U + kDepth>{});
            cur = next(cur);
            fetch(buf + cur, kSet ^ 1);
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    acc[i][j] = mfma_fp8(fa[kSet][i], fb[kSet][j], acc[i][j], wa[i], wb[j]);
            turn_scales(p + 1, Set<U + 1>{});
        });
    } else {
        // Parts of two blocks of rows, their fragments read a part ahead, across the
        // widths too: the barrier that publishes width p + 1 stands before the last
        // part of width p.  After it width p + 2 is copied where p was.
        constexpr int kParts = MB / 2;
        static_assert(NB == 4, "four steps of the last part");
        i32x8 fa[2][2], fb[NB];
        auto fetch_a = [&](const char* from, int part) {
#pragma unroll
            for (int i = 0; i < 2; ++i) fa[part & 1][i] = frag_a(from, part * 2 + i);
        };
        fetch_a(buf, 0);
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j] = frag_b(buf, j);
        turn_scales(0, Set<0>{});
        all_widths([&](int32_t p, auto u) {
            constexpr int U = decltype(u)::v;
            const char* here = buf + cur;
#pragma unroll
            for (int part = 0; part + 1 < kParts; ++part) {
                __builtin_amdgcn_sched_barrier(0);
                fetch_a(here, part + 1);
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        acc[part * 2 + i][j] =
                            mfma_fp8(fa[part & 1][i], fb[j], acc[part * 2 + i][j], wa[part * 2 + i], wb[j]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // LDS reads and matrix instructions in turn
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, NB / 2, 0);
                }
            }
            publish();
            copy(p + kDepth, cur, Set<U + kDepth>{});
            cur = next(cur);
            fetch_a(buf + cur, 0);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[MB - 2 + i][j] = mfma_fp8(fa[1][i], fb[j], acc[MB - 2 + i][j], wa[MB - 2 + i], wb[j]);
                fb[j] = frag_b(buf + cur, j);
            }
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            turn_scales(p + 1, Set<U + 1>{});
        });
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    wait_copies<0>();  // copies past the end may still write their zeros

    Place p;
    p.m0 = m0 + wm * MB * 16;
    p.n0 = n0 + wn * NB * 16;
    p.m = g.m;
    p.n = g.n;
    p.split = t.split;
    p.tile_m = t.tm;
    p.lane = lane;
    p.wave = wave;
    p.wm = wm;
    p.wn = wn;
    epi.template run<WM, WN, MB, NB>(acc, p, buf);
}

template <int WM, int WN, int MB, int NB, typename Epi>
__global__ __launch_bounds__(WM* WN * 64, 2) void fp8_kernel(Fp8Args q, Epi epi) {
    __shared__ __attribute__((aligned(1024))) char buf[fp8_lds<WM, WN, MB, NB>()];
    fp8_workgroup<WM, WN, MB, NB, Epi>(q, epi, blockIdx.x, buf);
}

}  // namespace train
}  // namespace mlrs
