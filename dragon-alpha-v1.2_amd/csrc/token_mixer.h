// Shared by the kernels that mix the tokens of a sequence (windowed attention, linear attention with a decay).
//
// All of them multiply with v_mfma_f32_32x32x2_f32 and let a wavefront own 32 rows of the one operand as COLUMNS of the
// result: lane (r, h) holds column r, result register v is row 8*(v/4) + 4*h + v%4.  A first product's result is then, register
// for register, the B operand of a second product whose MFMA step v consumes row 8*(v/4) + 4*h + v%4 from lane half h.
//
// A tile of ROWS sequence rows sits in LDS as [row][DW]; a row is read in two ways:
//   chunk-wise (4 consecutive floats of row r per lane: the A operand of a product along the head dimension), from a
//              tile whose 16-byte chunk c of row r lies at position c ^ kin_swizzle<DW>(r);
//   column-wise (lane r takes float 32b + r: the A operand of a product along the sequence).
// A tile that is read in both ways is stored with the swizzle: 32 lanes that read 32 consecutive floats of one row touch
// the same eight chunks in another order, still every bank once.
#pragma once
#include "gemm_mfma_kernel.h"

namespace dragon {
namespace {

constexpr float MIX_LOG2E = 1.44269504088896340736f;
constexpr float MIX_LN2 = 0.69314718055994530942f;

// the values that lane r of either half holds, in both: {of half 0, of half 1}
struct MixHalves { float a, b; };
__device__ __forceinline__ MixHalves mix_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return {__builtin_bit_cast(float, (unsigned)y[0]), __builtin_bit_cast(float, (unsigned)y[1])};
}

// the sequence row that result register v of lane half h stands for
__device__ __forceinline__ constexpr int mix_row(int v, int h) { return 8 * (v / 4) + 4 * h + (v % 4); }

__device__ __forceinline__ int mix_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// the byte address of LDS memory, for transfers
__device__ __forceinline__ unsigned mix_lds(const float* lds) {
    return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const float*)lds;
}
// this wavefront's transfers have landed
__device__ __forceinline__ void mix_wait() { __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); }

// One [ROWS][DW] tile from memory straight into LDS by THREADS threads of a workgroup (whole wavefronts): no staging registers, no vector
// instructions (which the matrix pipe would wait for).  The hardware puts lane l's 16 bytes at the wave's base + 16 * l, so
// the swizzle moves to the global side: the lane at slot c of row r fetches chunk c ^ swizzle(r).  A lane's byte offset
// never changes; the tile's first row goes into the descriptor's base and the rows that exist into its size, so rows beyond
// them and chunks beyond the row's d4 floats arrive as zeros.  Everything but the offsets has to be uniform.
template <int DW, int ROWS, bool SWIZZLE, int THREADS = NTHREADS>
struct MixTile {
    static constexpr int CPR = DW / 4, WAVES = THREADS / 64, BLOCKS = ROWS * DW / 256;   // blocks of 1 KiB, one transfer each
    static constexpr int PASSES = (BLOCKS + WAVES - 1) / WAVES;
    static constexpr bool EVEN = BLOCKS % WAVES == 0;
    int off[PASSES];
    __device__ __forceinline__ void init(int t, int pitch, int d4) {
#pragma unroll
        for (int s = 0; s < PASSES; s++) {
            const int at = s * THREADS + t, row = at / CPR, slot = at % CPR, chunk = SWIZZLE ? (slot ^ kin_swizzle<DW>(row)) : slot;
            off[s] = chunk * 4 < d4 ? (row * pitch + chunk * 4) * 4 : OOB_OFFSET;
        }
    }
    // rows [0, left) of the tile that starts at `base` into the LDS tile whose address for wavefront `wave` is `lds`
    // (mix_lds of the tile + 1024 * wavefront); left < 1: zeros
    __device__ __forceinline__ void fetch(const float* base, int left, int pitch, unsigned lds, int wave = 0) const {
        const int rows = left < 0 ? 0 : (left < ROWS ? left : ROWS);
        const unsigned long long b = (unsigned long long)base;
        const v4u rsrc = {(unsigned)mix_uniform((int)b), (unsigned)mix_uniform((int)(b >> 32)) & 0xffffu,
                          (unsigned)mix_uniform(rows * pitch * 4), (unsigned)RSRC_FLAGS};
        const unsigned to = (unsigned)mix_uniform((int)lds);
        static_for<PASSES>([&](auto sc) {
            constexpr int s = decltype(sc)::value;
            if (EVEN || s * WAVES + wave < BLOCKS) dma_f4_lean<s * THREADS * 16>(rsrc, to, off[s]);
        });
    }
};

// The order in which a product's LDS reads and matrix instructions are issued: READS reads first, then always one read behind
// MFMAS matrix instructions.  Left alone the compiler reads an operand just before it is needed and the matrix pipe waits
// for LDS between any two uses.
// (The barriers around a product keep other reads out of the count.)
template <int READS, int TOTAL, int MFMAS>
__device__ __forceinline__ void mix_order() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    static_for<TOTAL - READS>([&](auto) {
        __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    });
    __builtin_amdgcn_sched_group_barrier(0x8, READS * MFMAS, 0);
    __builtin_amdgcn_sched_barrier(0);
}

// result[row of the tile][column] += tile . cols^T over the head dimension: cols[g] holds d = 8g + 4h .. +3 of the lane's
// column; the tile is swizzled
template <int DW, int NG>
__device__ __forceinline__ void mix_rows_product(v16f& s, const float* tile, const v4f (&cols)[NG], int r, int h) {
    // Chunk 2g + h of row r lies at (2g + h) ^ swizzle: the lane's place of chunk h, with 2g exchanged into its low four bits
    // (a row begins at a multiple of 2^(number of its chunks) of them, so nothing else is touched).
    const unsigned at = mix_lds(tile) + r * (DW * 4) + 16 * (h ^ kin_swizzle<DW>(r));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < NG; g++) {
        typedef const __attribute__((address_space(3))) v4f* lds_v4f;
        const v4f a = *(lds_v4f)(size_t)((at ^ (32 * (g & 7))) + 256 * (g >> 3));
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, cols[g].x, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, cols[g].y, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, cols[g].z, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, cols[g].w, s, 0, 0, 0);
    }
    mix_order<2, NG, 4>();
}

// Where lane (r, h) finds float 32b + r of tile row mix_row(v, h): one lane's part, exchanged with a constant of two bits
// where the tile is swizzled, plus a constant.  (Tiles are aligned to 1 KiB, so an exchange stays inside a row.)
template <int DW, bool SWIZZLE>
struct MixColumns {
    int base;
    __device__ __forceinline__ void init(int r, int h) {
        base = 16 * h * DW + (SWIZZLE ? 16 * ((r >> 2) ^ (DW > 32 ? 4 * h : 2 * h)) + 4 * (r & 3) : 4 * r);
    }
    static constexpr int variant(int v) { return !SWIZZLE ? 0 : DW > 32 ? v % 4 : 2 * ((v / 4) & 1) + ((v % 4) >> 1); }
    static constexpr int exchange(int c) { return !SWIZZLE ? 0 : 16 * (DW > 32 ? c : 4 * (c >> 1) + (c & 1)); }
    static constexpr int place(int v, int b) {
        return (8 * (v / 4) + v % 4) * DW * 4 + 16 * ((8 * b) ^ (SWIZZLE && DW > 32 ? 8 * ((v / 4) & 1) : 0));
    }
};

// out^T[d][column] += sum over the tile's rows of tile[row][d] * p[row][column]
template <int DW, int DC, bool SWIZZLE>
__device__ __forceinline__ void mix_columns_product(v16f (&o)[DC], const float* tile, const v16f& p, const MixColumns<DW, SWIZZLE>& cols) {
    typedef MixColumns<DW, SWIZZLE> C;
    typedef const __attribute__((address_space(3))) float* lds_float;
    unsigned at[4];
#pragma unroll
    for (int c = 0; c < 4; c++) at[c] = (mix_lds(tile) + cols.base) ^ C::exchange(c);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int v = 0; v < 16; v++) {
#pragma unroll
        for (int b = 0; b < DC; b++)
            o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(lds_float)(size_t)(at[C::variant(v)] + C::place(v, b)), p[v], o[b], 0, 0, 0);
    }
    mix_order<4, 16 * DC / 2, 2>();                       // the compiler reads two values at a time
}

// a lane's column of a result, times f: float 32b + 8g + 4h .. +3 of the row at `row`
template <int DC>
__device__ __forceinline__ void mix_store_row(float* row, const v16f (&o)[DC], float f, int d4, int h) {
    d4 = fresh(d4);     // or the tests' results, 4 * DC of them, sit in scalar registers all through the kernel
#pragma unroll
    for (int b = 0; b < DC; b++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int d = 32 * b + 8 * g + 4 * h;
            if (d < d4) *(v4f*)(row + d) = (v4f){o[b][4 * g] * f, o[b][4 * g + 1] * f, o[b][4 * g + 2] * f, o[b][4 * g + 3] * f};
        }
}

// the lane's column of an operand: 4 consecutive floats per group of 8, zeros where the row does not exist
template <int NG>
__device__ __forceinline__ void mix_load_cols(v4f (&c)[NG], const float* row, bool exists, int d4, int h) {
    d4 = fresh(d4);
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const int d = 8 * g + 4 * h;
        c[g] = (exists && d < d4) ? *(const v4f*)(row + d) : (v4f)(0.0f);
    }
}

inline bool mix_aligned16(int64_t a) { return (a & 15) == 0; }
// HIP takes fewer than 2^32 threads along a grid's dimension
inline bool mix_launch_fits(long long workgroups, int threads) { return workgroups * threads < 0x100000000LL; }

// element strides of a tensor [N, L, head, d4] (head_inner) or [N, head, L, d4]
struct MixLayout {
    long long n, h;
    int l;
};
inline MixLayout mix_layout(int head_inner, int head, int L, int d4) {
    MixLayout x;
    x.l = head_inner ? head * d4 : d4;
    x.h = head_inner ? (long long)d4 : (long long)L * d4;
    x.n = (long long)head * L * d4;
    return x;
}

}  // namespace
}  // namespace dragon
