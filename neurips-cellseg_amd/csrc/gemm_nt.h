// C[m][n] = sum_k A[m][k] B[n][k], both operands with k contiguous: the matrix product under the head losses and the 4-bit linear layer.
//
// All operand types share one byte layout.  A slab is 128 bytes of k per row (64 bf16 / fp16, 32 fp32, 256 e2m1), eight 16-byte chunks;
// a matrix instruction's operand is ONE chunk per lane (row lane % 16, chunk lane / 16), so the staging below never looks at the type:
//   bf16, fp16  v_mfma_f32_16x16x32: a lane holds 8 consecutive k
//   fp32        v_mfma_f32_16x16x4: element j of the chunk goes to the j-th of four instructions (the same k order in A and B)
//   e2m1        v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds 32 consecutive k, one e8m0 scale each
// Slabs go from global memory to LDS without registers (global_load_lds_dwordx4: 64 lanes x 16 bytes land at consecutive LDS addresses).
// Chunk c of row r is stored at place c ^ (r & 7) - by choosing what each lane fetches - so the 16 rows that a fragment read touches fall
// on all banks.  A chunk behind the end of k is fetched from a page of zeros, a row behind the last one from the last row (the epilogue
// drops it), so no access leaves the operands.
#pragma once
#include "cs_common.h"

#include <type_traits>

namespace cs {
namespace nt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Kind { BF16 = 0, FP16 = 1, FP32 = 2, E2M1 = 3 };

struct Operand {
    const char* ptr;       // row 0
    int64_t pitch;         // bytes between rows: a multiple of 16, below 2^23 (256 rows then fit a 32-bit offset)
    int64_t rows;          // >= 1
};

struct Problem {
    Operand a, b;
    int kbytes;            // bytes of k per row, a multiple of 16
    // e2m1: scales of A's and B's rows in tile order, a 32-bit word per (pair of slabs, row, chunk column g): byte 2 s + h is the e8m0 scale
    // of chunk 4 h + g of slab s of the pair.  rows_a / rows_b rows per pair, multiples of 256.
    const unsigned *scales_a, *scales_b;
    int64_t rows_a, rows_b;
    int tiles_m, tiles_n;
    int splits, slabs_per_split;       // k is cut into `splits` runs of slabs (1: no cut); each is a tile of its own for the epilogue
};

static __device__ __attribute__((aligned(16))) const unsigned zero_page[4] = {0u, 0u, 0u, 0u};

// 64 lanes x 16 bytes: what lane l's address points to -> LDS address dst + 16 l (dst: the same in all lanes).  dst is a number, not a
// pointer into the array that is read below: the compiler would else wait for every load before every LDS read; wait_loads() waits.
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;
__device__ __forceinline__ void dma16(unsigned dst, const char* from) {
    __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(size_t)dst, 16, 0, 0);
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(size_t)(const __attribute__((address_space(3))) void*)p;
}
// waits until at most N of this wave's loads are under way and its LDS reads are done
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// c += a b over one chunk per lane; e2m1: byte SEL of the lanes' scale words (an immediate of the instruction)
template <int KIND, int SEL>
__device__ __forceinline__ f32x4 mma(i32x4 a, i32x4 b, f32x4 c, int scale_a, int scale_b) {
    if constexpr (KIND == BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (KIND == FP16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else if constexpr (KIND == FP32) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else {
        const i32x8 x = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, y = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, SEL, scale_a, SEL, scale_b);   // 4: both operands e2m1
    }
}

// block id -> (tile_m, tile_n, split).  Blocks go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, walked in groups of
// 8 tile rows, so the tiles that run together on an XCD share their operands' slabs in its L2.
struct Tile { int m, n, split; };
__device__ __forceinline__ Tile tile_of(int id, const Problem& p) {
    const int per = p.tiles_m * p.tiles_n, total = per * p.splits;
    const int q = total >> 3, r = total & 7, xcd = id & 7, at = id >> 3;
    int t = xcd < r ? xcd * (q + 1) + at : r * (q + 1) + (xcd - r) * q + at;
    const int split = t / per;
    t -= split * per;
    const int group = t / (8 * p.tiles_n), first = group * 8, height = min(p.tiles_m - first, 8);
    t -= group * 8 * p.tiles_n;
    return {first + t % height, t / height, split};
}

// What one block multiplies: BM x BN outputs, WM x WN waves, STAGES slabs of both operands in LDS.
template <int KIND, int BM, int BN, int WM, int WN, int STAGES>
struct Ring {
    static constexpr int KIND_ = KIND, TILE_M = BM, TILE_N = BN, WAVES_M = WM, WAVES_N = WN;
    static constexpr int THREADS = WM * WN * 64, MF = BM / WM / 16, NF = BN / WN / 16;
    static constexpr int STAGE_BYTES = (BM + BN) * 128, LDS_BYTES = STAGES * STAGE_BYTES;
    static constexpr int LOADS = (BM + BN) / 8 / (WM * WN);             // 1 KB loads per wave and slab
    static_assert((BM + BN) % (8 * WM * WN) == 0 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "");

    // first output row / column of fragment i / j of this wave inside the tile; a lane holds rows + 4 * (lane / 16) + 0..3, column + lane % 16
    static __device__ __forceinline__ int row0(int wm, int i) { return wm * (BM / WM) + i * 16; }
    static __device__ __forceinline__ int col0(int wn, int j) { return wn * (BN / WN) + j * 16; }

    static __device__ __forceinline__ void run(const Problem& p, Tile t, char* lds, f32x4 (&acc)[MF][NF]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        const int slabs = (p.kbytes + 127) >> 7, first = t.split * p.slabs_per_split, last = min(slabs, first + p.slabs_per_split) - 1;
        const bool tail = (p.kbytes & 127) != 0;
        const int64_t m0 = (int64_t)t.m * BM, n0 = (int64_t)t.n * BN;
        const char* base[LOADS];
        unsigned off[LOADS];
        const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 3)) * 16u;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = (wave * LOADS + i) * 8;                      // of the A rows followed by the B rows; BM is a multiple of 8
            const bool in_a = row < BM;
            const Operand& o = in_a ? p.a : p.b;
            const int64_t r0 = in_a ? m0 + row : n0 + (row - BM);
            const int64_t from = r0 < o.rows ? r0 : o.rows - 1;
            const int64_t mine = r0 + (lane >> 3) < o.rows ? r0 + (lane >> 3) : o.rows - 1;
            base[i] = o.ptr + from * o.pitch;
            off[i] = (unsigned)((mine - from) * o.pitch) + chunk;
        }
        const unsigned to = lds_address(lds) + (unsigned)(wave * LOADS) * 1024u;
        auto load = [&](int slab, int slot) {
            slab = min(slab, last);                                      // the ring runs on behind the last slab: what it fetches is never read
            const unsigned dst = to + (unsigned)(slot * STAGE_BYTES);
            const int64_t k = (int64_t)slab * 128;
            if (tail && slab == slabs - 1) {
                const bool in = k + chunk < p.kbytes;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) dma16(dst + i * 1024, in ? base[i] + off[i] + k : (const char*)zero_page);
            } else {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) dma16(dst + i * 1024, base[i] + k + off[i]);
            }
        };
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        int place[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) place[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ (lane & 7)) * 16);
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) load(first + s, s);
        // scale words of a pair of slabs, one pair ahead; `first` is even
        int scale_a[MF], scale_b[NF], next_a[MF], next_b[NF];
        auto load_scales = [&](int slab) {
            const int64_t pair = min(slab, last) >> 1;
#pragma unroll
            for (int i = 0; i < MF; ++i) next_a[i] = (int)p.scales_a[(pair * p.rows_a + m0 + row0(wm, i)) * 4 + (lane & 15) * 4 + (lane >> 4)];
#pragma unroll
            for (int j = 0; j < NF; ++j) next_b[j] = (int)p.scales_b[(pair * p.rows_b + n0 + col0(wn, j)) * 4 + (lane & 15) * 4 + (lane >> 4)];
        };
        if constexpr (KIND == E2M1) load_scales(first);
        int slot = 0, fill = STAGES - 1;
        auto step = [&](int k, auto odd) {
            wait_loads<(STAGES - 2) * LOADS>();                          // this slab is there ...
            barrier();                                                   // ... for every wave, and nobody reads the previous one any more
            load(k + STAGES - 1, fill);
            if constexpr (KIND == E2M1 && !odd.value) {
#pragma unroll
                for (int i = 0; i < MF; ++i) scale_a[i] = next_a[i];
#pragma unroll
                for (int j = 0; j < NF; ++j) scale_b[j] = next_b[j];
                load_scales(k + 2);
            }
            const char* sa = lds + slot * STAGE_BYTES + row0(wm, 0) * 128;
            const char* sb = lds + slot * STAGE_BYTES + (BM + col0(wn, 0)) * 128;
            auto half = [&](auto h) {
                constexpr int SEL = 2 * decltype(odd)::value + decltype(h)::value;
                i32x4 b[NF];
#pragma unroll
                for (int j = 0; j < NF; ++j) b[j] = *(const i32x4*)(sb + place[h.value] + j * 2048);
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    const i32x4 a = *(const i32x4*)(sa + place[h.value] + i * 2048);
#pragma unroll
                    for (int j = 0; j < NF; ++j) acc[i][j] = mma<KIND, SEL>(a, b[j], acc[i][j], scale_a[i], scale_b[j]);
                }
            };
            half(std::integral_constant<int, 0>());
            half(std::integral_constant<int, 1>());
            slot = slot + 1 == STAGES ? 0 : slot + 1;
            fill = fill + 1 == STAGES ? 0 : fill + 1;
        };
        if constexpr (KIND == E2M1) {
            for (int k = first; k <= last; k += 2) {
                step(k, std::integral_constant<int, 0>());
                if (k < last) step(k + 1, std::integral_constant<int, 1>());
            }
        } else {
            for (int k = first; k <= last; ++k) step(k, std::integral_constant<int, 0>());
        }
        wait_loads<0>();
        barrier();                                                       // LDS is the epilogue's
    }
};

}  // namespace nt
}  // namespace cs
