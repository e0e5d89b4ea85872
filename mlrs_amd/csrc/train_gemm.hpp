// The matrix product under the training operators: P[i, j] = sum_k A(i, k) B(j, k)
// for f32, f16 and bf16 operands, accumulated in f32 on the matrix cores, and
// handed to an epilogue while it is still in registers.
//
// Operands.  Either operand is stored with its contraction index contiguous
// ("K layout", ptr[row * ld + k]) or with its row index contiguous ("R
// layout", ptr[k * ld + row]), so the three products of a layer need no
// transposed copies: x w^T is K x K, dz w is R x K, dz^T x is R x R.  Pointers
// are 16-byte aligned and ld is a multiple of 16 bytes; what is not the host
// packs, or f32 operands are copied word by word (BYTES 4, 64 x 64 tiles: their
// matrix instructions take longer than four times as many copies).
//
// Tile.  A workgroup computes BM x BN of P, its waves a WM x WN grid of parts
// of MB x NB blocks of 16 x 16 (v_mfma_f32_16x16x32 for 16-bit types, four
// v_mfma_f32_16x16x4 for f32).  A large product is bound by the chip's power,
// and register-only chains of the 16 x 16 instruction reach 2,080 TFLOP/s where
// those of 32 x 32 x 16 reach 1,830.  A is the operand whose index runs along
// the output's rows in memory: a lane then holds four consecutive elements of
// one output row.  128 bytes of the contraction axis are staged at a time,
// straight from HBM into a ring of LDS slots; out-of-range elements come back as
// zeros from the buffer descriptor's bounds check.
//
// LDS layout.  K operand: a row's 128 bytes as eight 16-byte chunks, chunk c
// kept at c ^ ((row >> 1) & 7), so that sixteen rows read at one c (a pass of
// a 16-byte read: 64 banks) touch all banks.  R
// operand: the tile's elements of one k back to back, their 16-byte chunks
// kept at c ^ r_swizzle(k): the eight k of half a wave's transposing read
// (16-bit types) and the four of a wave's read (f32) then lie in different
// banks.  The swizzle
// is applied to the global address of each lane, as the copy into LDS is
// linear.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace mlrs {
namespace train {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// The element types by what the kernels need of them.  Conversions to 16 bits
// round to nearest even.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    typedef f32x4 Frag;  // 16 bytes of the contraction axis
    typedef f32x4 Vec4;
};
template <>
struct Elem<_Float16> {
    typedef f16x8 Frag;
    typedef f16x4 Vec4;
};
template <>
struct Elem<__bf16> {
    typedef bf16x8 Frag;
    typedef bf16x4 Vec4;
};

struct Operand {
    const void* p;
    int64_t ld;  // elements
};

struct GemmArgs {
    Operand a, b;
    int32_t m, n, k;       // P is m x n (a's rows, b's rows)
    int32_t tiles_m, tiles_n;
    int32_t splits;        // parts of the contraction axis, a grid's worth of tiles each
    int32_t k_split;       // elements of k in a part (a multiple of the staged width)
    int32_t band;          // tiles of m that are walked together (L2 reuse)
    const uint32_t* flag;  // null, or: run only where (*flag == mark) == wanted
    uint32_t mark;
    bool wanted;
};

// Whether another kernel does this launch's work.
__device__ __forceinline__ bool skipped(const uint32_t* flag, uint32_t mark, bool wanted) {
    return flag && (*flag == mark) != wanted;
}
__device__ __forceinline__ bool skipped(const GemmArgs& g) { return skipped(g.flag, g.mark, g.wanted); }

constexpr int kStageBytes = 128;  // of the contraction axis, per buffer

template <typename T>
__host__ __device__ constexpr int stage_elems() {
    return kStageBytes / (int)sizeof(T);
}

#if defined(__HIP_DEVICE_COMPILE__)
#define MLRS_LDS __attribute__((address_space(3)))
#else
#define MLRS_LDS
#endif

template <typename T>
__device__ __forceinline__ f32x4 mfma_step(typename Elem<T>::Frag a, typename Elem<T>::Frag b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    } else if constexpr (__is_same(T, _Float16)) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
#else
    (void)a;
    (void)b;
#endif
    return c;
}

// K layout: what the chunk index of a row is exclusive-ored with.
__device__ __forceinline__ int k_swizzle(int row) { return (row >> 1) & 7; }

// R layout: what the chunk index of step k is exclusive-ored with.
template <typename T, int ROWS>
__device__ __forceinline__ int r_swizzle(int k) {
    if (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
    return (ROWS * 2 >= 256 ? (k & 3) << 2 : ((k >> 1) & 1) << 2) ^ (((k >> 3) & 1) << 1);
}

// 16 bytes per lane from a buffer straight into LDS, lane i's at lds + 16 i; lds
// and the descriptor are uniform over the wave.  Counted by vmcnt, which the
// caller waits for: written as an instruction because the compiler would wait
// for every copy under way at each transposing LDS read, not knowing that they
// touch other slots.  It has no result register; the wait state between writing
// M0 and the copy is written too, as the compiler does not look into the block.
__device__ __forceinline__ void copy_to_lds(u32x4 rsrc, char* lds, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"((uint32_t)(uintptr_t)(MLRS_LDS void*)lds), "v"(offset), "s"(rsrc)
                 : "memory");
#else
    (void)rsrc;
    (void)lds;
    (void)offset;
#endif
}

// The same with four bytes per lane, for f32 operands in place whose rows are no
// multiple of 16 bytes: lane i's are at lds + 4 i.
__device__ __forceinline__ void copy_word_to_lds(u32x4 rsrc, char* lds, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"((uint32_t)(uintptr_t)(MLRS_LDS void*)lds), "v"(offset), "s"(rsrc)
                 : "memory");
#else
    (void)rsrc;
    (void)lds;
    (void)offset;
#endif
}

// One operand's copy into LDS: the bytes of ROWS rows (or columns) of one
// staged width, 64 BYTES per wave and instruction.
template <typename T, bool KC, int ROWS, int WAVES, int BYTES = 16>
struct Stager {
    static constexpr int kInstr = ROWS * kStageBytes / (64 * BYTES) / WAVES;
    static constexpr int kPlaces = BYTES == 16 ? 2 : 8;  // of a lane in a row, K layout: by the copy
    static constexpr int kChunks = ROWS * (int)sizeof(T) / 16;  // of one k (R layout)
    static_assert(kInstr >= 1, "a wave copies at least one kilobyte");
    const char* base;   // the tile's first element at k = 0
    int64_t bytes;      // from base to the operand's end
    int64_t step;       // bytes per element of k
    int32_t chunk[kPlaces];  // K layout: where in the row the lane's bytes are
    uint32_t off[kInstr];

    __device__ __forceinline__ void init(const Operand& o, int32_t row0, int32_t rows, int32_t k, int wave, int lane) {
        const int64_t es = (int64_t)sizeof(T);
        // whole rows: the bounds check works by the lanes' bytes, which end at ld
        const int64_t total = (KC ? (int64_t)rows : (int64_t)k) * o.ld * es;
        const int64_t at = KC ? (int64_t)row0 * o.ld * es : (int64_t)row0 * es;
        base = reinterpret_cast<const char*>(o.p) + at;
        bytes = total - at;
        step = KC ? es : o.ld * es;
        const uint32_t ldb = (uint32_t)(o.ld * es);
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) chunk[i] = 0;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const int q = ((wave * kInstr + i) * 64 + lane) / (16 / BYTES);  // the chunk's place in LDS
            const uint32_t in = BYTES == 16 ? 0u : 4u * (uint32_t)(lane & 3);
            if constexpr (KC) {
                static_assert(kInstr % kPlaces == 0, "which chunk a lane copies goes by the copy");
                const int r = q >> 3, c = (q & 7) ^ k_swizzle(r);
                chunk[i % kPlaces] = 16 * c + (int)in;
                off[i] = (uint32_t)r * ldb + 16u * (uint32_t)c + in;
            } else {
                const int kk = q / kChunks;
                const int c = (q % kChunks) ^ r_swizzle<T, ROWS>(kk);
                off[i] = (uint32_t)kk * ldb + 16u * (uint32_t)c + in;
            }
        }
    }

    // Part PART of PARTS of the copies of elements k0 .. k0 + the staged width;
    // k is the end of the contraction, past which come zeros.
    template <int PART, int PARTS>
    __device__ __forceinline__ void load(char* lds, int32_t k0, int32_t k, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int64_t skip = (int64_t)k0 * step;
        const int64_t left = bytes - skip;
        const uint32_t records = left < 0x7FFFFFFF ? (left > 0 ? (uint32_t)left : 0u) : 0x7FFFFFFFu;
        const uint64_t at = (uint64_t)(base + skip);
        u32x4 rsrc;
        rsrc[0] = (uint32_t)at;
        rsrc[1] = (uint32_t)(at >> 32) & 0xFFFFu;
        rsrc[2] = records;
        rsrc[3] = 0x00027000u;
        // chunks past the end of a row would be the next row's
        bool out[kPlaces];
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) out[i] = KC && chunk[i] >= (k - k0) * (int)sizeof(T);
#pragma unroll
        for (int i = PART * kInstr / PARTS; i < (PART + 1) * kInstr / PARTS; ++i) {
            const uint32_t from = out[i % kPlaces] ? 0x80000000u : off[i];
            if constexpr (BYTES == 16)
                copy_to_lds(rsrc, lds + (wave * kInstr + i) * 1024, from);
            else
                copy_word_to_lds(rsrc, lds + (wave * kInstr + i) * 256, from);
        }
#else
        (void)lds;
        (void)k0;
        (void)k;
        (void)wave;
#endif
    }
};

// One operand's fragments out of LDS: BLOCKS blocks of 16 rows from row
// `first`; step s of the two in a staged width.  Lane l holds sixteen bytes of
// row l % 16 along k, the (l / 16)-th of the step.
template <typename T, bool KC, int ROWS, int BLOCKS>
struct Reader {
    int at[KC ? 2 : BLOCKS];

    __device__ __forceinline__ void init(int first, int lane) {
        const int g = lane >> 4, r = lane & 15;
        if constexpr (KC) {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = (first + r) * kStageBytes + (((4 * s + g) ^ k_swizzle(r)) << 4);
        } else if constexpr (sizeof(T) == 2) {
            // lane 4 q + p of sixteen addresses four elements of step q of
            // four; the transposing read hands lane i column i of them
            const int q = r >> 2, p = lane & 3;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int c = ((first >> 4) + b) * 2 + (p >> 1);
                at[b] = (8 * g + q) * (ROWS * 2) + ((c ^ r_swizzle<T, ROWS>(8 * g + q)) << 4) + (p & 1) * 8;
            }
        } else {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int c = ((first >> 4) + b) * 4 + (r >> 2);
                at[b] = 4 * g * (ROWS * 4) + ((c ^ r_swizzle<T, ROWS>(4 * g)) << 4) + (r & 3) * 4;
            }
        }
    }

    __device__ __forceinline__ typename Elem<T>::Frag get(const char* lds, int s, int b) const {
        typedef typename Elem<T>::Frag Frag;
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (KC) {
            return *reinterpret_cast<const Frag*>(lds + at[s] + b * 16 * kStageBytes);
        } else if constexpr (sizeof(T) == 2) {
            // the swizzle of k + 4 and of k + 32 is that of k
            const char* q = lds + at[b] + s * 32 * (ROWS * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLRS_LDS s16x4*)q);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLRS_LDS s16x4*)(q + 4 * (ROWS * 2)));
            return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const char* q = lds + at[b] + s * 16 * (ROWS * 4);
            Frag f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float*>(q + i * (ROWS * 4));
            return f;
        }
#else
        (void)lds;
        (void)s;
        (void)b;
        return Frag{};
#endif
    }
};

// What an epilogue is told about the wave's part of the tile.
struct Place {
    int32_t m0, n0;    // first row (of a) and column (of b) of the wave's blocks
    int32_t m, n;      // the extents of P
    int32_t split;
    int32_t tile_m;    // the workgroup's tile index along m
    int lane, wave;
    int wm, wn;        // the wave's place in the workgroup's grid
};

// Workgroups go to the eight XCDs in turn; give each XCD a contiguous run of
// tiles, so that its L2 holds the operand panels that its workgroups share.
__device__ __forceinline__ int32_t xcd_tile(int32_t wg, int32_t total) {
    const int32_t per = total >> 3, extra = total & 7;
    const int32_t x = wg & 7, i = wg >> 3;
    return x * per + (x < extra ? x : extra) + i;
}

// The tile of a workgroup: bands of `band` tiles of m, walked along n.
struct TilePlace {
    int32_t tm, tn, split;
};
__device__ __forceinline__ TilePlace tile_place(const GemmArgs& g, uint32_t wg) {
    const int32_t tiles = g.tiles_m * g.tiles_n;
    TilePlace p;
    p.split = wg / tiles;
    const int32_t t = xcd_tile(wg - p.split * tiles, tiles);
    const int32_t per_band = g.band * g.tiles_n;
    const int32_t bnd = t / per_band, in = t - bnd * per_band;
    const int32_t width = g.tiles_m - bnd * g.band < g.band ? g.tiles_m - bnd * g.band : g.band;
    p.tm = bnd * g.band + in % width;
    p.tn = in / width;
    return p;
}

// A number as a type: which of two sets of fragments.
template <int V>
struct Set {
    static constexpr int v = V;
};

// Waits until at most N of the wave's copies are under way.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N < 64, "six bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// Panels that a tile keeps in LDS, and their bytes.
template <int MB, int NB>
__host__ __device__ constexpr int gemm_slots() {
    return MB * NB == 4 ? 6 : 5;
}
template <int WM, int MB, int NB>
__host__ __device__ constexpr int gemm_lds() {
    return gemm_slots<MB, NB>() * WM * MB * 16 * kStageBytes;
}

// A workgroup of every product.  8192 x 8192 x 8192 in bf16: 729 us forwards (K x
// K), 764 for dx (R x K), 740 for dw (R x R) on one card, 744, 827 and 799 on
// another, 1330 to 1508 TFLOP/s, where the matrix instructions alone would do 2080
// at the clock that the chip's power allows; with the copies left out it was 1576
// in 32 x 32 blocks.  In 256 x 256 tiles eight waves of 128 x 64 read 192 KB of
// fragments and copy 64 KB for 2048 cycles of matrix work a staged width, the LDS
// being busy for as long; one workgroup fills a CU.  Four waves of 128 x 128 read a
// third less and are no faster (756 us), as a wave alone on its SIMD waits for
// itself.
// buf: gemm_lds bytes, the kernel's only LDS.
template <typename T, bool AKC, bool BKC, int WM, int WN, int MB, int NB, typename Epi, int BYTES = 16>
__device__ __forceinline__ void gemm_workgroup(const GemmArgs& g, const Epi& epi, uint32_t wg, char* buf) {
    constexpr int BM = WM * MB * 16, BN = WN * NB * 16, WAVES = WM * WN;
    constexpr int kA = BM * kStageBytes, kB = BN * kStageBytes;
    constexpr int BK = stage_elems<T>();
    static_assert(kA == kB, "panels of either operand take the same slots");
    constexpr bool kSmall = MB * NB == 4;
    constexpr int kAhead = 3;  // staged widths under way, of a small tile
    constexpr int kSlots = gemm_slots<MB, NB>();
    static_assert(!kSmall || kSlots == 2 * kAhead, "two panels a width");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    const TilePlace t = tile_place(g, wg);
    const int32_t m0 = t.tm * BM, n0 = t.tn * BN;
    const int32_t k_lo = t.split * g.k_split;
    const int32_t k_hi = g.k - k_lo < g.k_split ? g.k : k_lo + g.k_split;

    Stager<T, AKC, BM, WAVES, BYTES> sa;
    Stager<T, BKC, BN, WAVES, BYTES> sb;
    sa.init(g.a, m0, g.m, k_hi, wave, lane);
    sb.init(g.b, n0, g.n, k_hi, wave, lane);
    Reader<T, AKC, BM, MB> ra;
    Reader<T, BKC, BN, NB> rb;
    ra.init(wm * MB * 16, lane);
    rb.init(wn * NB * 16, lane);

    f32x4 acc[MB][NB] = {};

    if constexpr (kSmall) {
        // A small tile has too little to multiply in a step to hide an LDS read
        // behind: the fragments of a whole staged width are read while those of
        // the one before are multiplied.  At the barrier of width p its fragments
        // are in registers, width p + 1 is published, and width p + kAhead goes
        // where p was.  4096 x 256 x 4096 in bf16: 33.1 us a step at a time with
        // five slots, 20.2 so.
        typename Elem<T>::Frag fa[2][2][MB], fb[2][2][NB];
        constexpr int IA = decltype(sa)::kInstr, IB = decltype(sb)::kInstr;
        auto fetch = [&](const char* from, auto set) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < MB; ++i) fa[set.v][s][i] = ra.get(from, s, i);
#pragma unroll
                for (int j = 0; j < NB; ++j) fb[set.v][s][j] = rb.get(from + kA, s, j);
            }
        };
        int cur = 0;
        auto next = [&](int at) { return at + 2 * kA >= kAhead * 2 * kA ? 0 : at + 2 * kA; };
        auto width = [&](int32_t k0, auto set, auto other) {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            wait_copies<(kAhead - 2) * (IA + IB)>();
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            sa.template load<0, 1>(buf + cur, k0 + kAhead * BK, k_hi, wave);
            sb.template load<0, 1>(buf + cur + kA, k0 + kAhead * BK, k_hi, wave);
            cur = next(cur);
            fetch(buf + cur, other);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        acc[i][j] = mfma_step<T>(fa[set.v][s][i], fb[set.v][s][j], acc[i][j]);
        };
#pragma unroll
        for (int p = 0; p < kAhead; ++p) {
            sa.template load<0, 1>(buf + 2 * p * kA, k_lo + p * BK, k_hi, wave);
            sb.template load<0, 1>(buf + (2 * p + 1) * kA, k_lo + p * BK, k_hi, wave);
        }
        wait_copies<(kAhead - 1) * (IA + IB)>();
        __builtin_amdgcn_s_barrier();
        fetch(buf, Set<0>{});
        // an even number of widths: past the end come zeros
        for (int32_t k0 = k_lo; k0 < k_hi; k0 += 2 * BK) {
            width(k0, Set<0>{}, Set<1>{});
            width(k0 + BK, Set<1>{}, Set<0>{});
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
        wait_copies<0>();
    } else {
        // Panels A0 B0 A1 B1 ... go round five slots of LDS.  A staged width is
        // multiplied in four parts, the lower and the upper half of the wave's rows
        // in each of its two steps, and fragments are read a part ahead, across the
        // widths too: the barrier that publishes width p + 1 stands before the last
        // part of width p, whose fragments are in registers by then.  After it
        // nothing reads A_p and B_p any more; B_{p+2} and A_{p+3} are copied over
        // them, a quarter of the copies in every part, so that neither the matrix
        // nor the memory pipeline sees a burst.
        constexpr int HB = MB / 2;
        typename Elem<T>::Frag fa[2][HB], fb[2][NB];
        auto fetch_a = [&](const char* from, int s, int half) {
#pragma unroll
            for (int i = 0; i < HB; ++i) fa[half][i] = ra.get(from, s, half * HB + i);
        };
        auto fetch_b = [&](const char* from, int s) {
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[s][j] = rb.get(from, s, j);
        };
        auto multiply = [&](int half, int s) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int i = 0; i < HB; ++i)
                    acc[half * HB + i][j] = mfma_step<T>(fa[half][i], fb[s][j], acc[half * HB + i][j]);
        };
        // LDS reads and matrix instructions in turn
        auto interleave = [&](auto with_b) {
            constexpr int kA1 = AKC ? 1 : sizeof(T) == 2 ? 2 : 4, kB1 = BKC ? 1 : sizeof(T) == 2 ? 2 : 4;
            constexpr int kReads = HB * kA1 + (decltype(with_b)::v ? NB * kB1 : 0);
            constexpr int kMath = HB * NB * (sizeof(T) == 4 ? 4 : 1);
            constexpr int kPer = (kReads + kMath - 1) / kMath, kEvery = kMath / kReads > 1 ? kMath / kReads : 1;
#pragma unroll
            for (int i = 0; i < kMath / kEvery; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, kEvery, 0);
            }
        };
        // `ahead` slots past the one at `at`
        auto slot = [&](int at, int ahead) {
            const int to = at + ahead * kA;
            return buf + (to >= kSlots * kA ? to - kSlots * kA : to);
        };
        constexpr int IA = decltype(sa)::kInstr, IB = decltype(sb)::kInstr;

        sa.template load<0, 1>(buf, k_lo, k_hi, wave);
        sb.template load<0, 1>(buf + kA, k_lo, k_hi, wave);
        sa.template load<0, 1>(buf + 2 * kA, k_lo + BK, k_hi, wave);
        sb.template load<0, 2>(buf + 3 * kA, k_lo + BK, k_hi, wave);
        wait_copies<IA + IB / 2>();
        __builtin_amdgcn_s_barrier();
        fetch_a(buf, 0, 0);
        fetch_b(buf + kA, 0);
        int cur = 0;  // of A_p
        for (int32_t k0 = k_lo; k0 < k_hi; k0 += BK) {
            const char *pa = buf + cur, *pb = slot(cur, 1);
            __builtin_amdgcn_sched_barrier(0);
            sb.template load<1, 2>(slot(cur, 3), k0 + BK, k_hi, wave);
            fetch_a(pa, 0, 1);
            multiply(0, 0);
            interleave(Set<0>{});
            __builtin_amdgcn_sched_barrier(0);
            sa.template load<0, 2>(slot(cur, 4), k0 + 2 * BK, k_hi, wave);
            fetch_a(pa, 1, 0);
            fetch_b(pb, 1);
            multiply(1, 0);
            interleave(Set<1>{});
            __builtin_amdgcn_sched_barrier(0);
            sa.template load<1, 2>(slot(cur, 4), k0 + 2 * BK, k_hi, wave);
            fetch_a(pa, 1, 1);
            multiply(0, 1);
            interleave(Set<0>{});
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the last fragments of p
            wait_copies<IA>();
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            sb.template load<0, 2>(buf + cur, k0 + 2 * BK, k_hi, wave);
            fetch_a(slot(cur, 2), 0, 0);
            fetch_b(slot(cur, 3), 0);
            multiply(1, 1);
            interleave(Set<1>{});
            cur = cur + 2 * kA >= kSlots * kA ? cur - (kSlots - 2) * kA : cur + 2 * kA;
        }
        // copies past the end of the contraction may still write their zeros
        wait_copies<0>();
    }

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

// A product of operands in K layout.
template <typename T, int WM, int WN, int MB, int NB, typename Epi, int BYTES = 16>
__global__ __launch_bounds__(WM* WN * 64, 2) void gemm_kernel(GemmArgs g, Epi epi) {
    __shared__ __attribute__((aligned(1024))) char buf[gemm_lds<WM, MB, NB>()];
    if (skipped(g)) return;
    gemm_workgroup<T, true, true, WM, WN, MB, NB, Epi, BYTES>(g, epi, blockIdx.x, buf);
}

}  // namespace train
}  // namespace mlrs
