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
#include <utility>

namespace cs {
namespace nt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 bytes at the address of any value: one instruction, as fast as an aligned one where the address is aligned
typedef i32x4 Loose __attribute__((aligned(2)));
typedef f32x4 LooseSum __attribute__((aligned(4)));

enum Kind { BF16 = 0, FP16 = 1, FP32 = 2, E2M1 = 3 };

struct Operand {
    const char* ptr;       // row 0
    int64_t pitch;         // bytes between rows: a multiple of 16, below 2^25 (128 rows then fit a 32-bit offset)
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

// a barrier behind this wave's LDS accesses, with its global loads and stores left under way
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    barrier();
}

// between a wave's LDS writes and its reads of what other lanes of it wrote, and back: the wave's LDS accesses run in order, but the compiler
// sees one lane and may exchange those that do not meet in it
__device__ __forceinline__ void wave_sync() { asm volatile("" ::: "memory"); }

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

// The same with the sum in place in accumulation registers (the compiler else moves the 256 of a large tile about between its uses).  One
// instruction (fp32: of element `element`); no other of the next few may touch the same sum, and a reader of the sum waits for the pipe.
template <int KIND, int SEL>
__device__ __forceinline__ void mma_in_place(f32x4& c, i32x4 a, i32x4 b, int element, int scale_a, int scale_b) {
    if constexpr (KIND == BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else if constexpr (KIND == FP16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else if constexpr (KIND == FP32) asm volatile("v_mfma_f32_16x16x4_f32 %0, %1, %2, %0" : "+a"(c) : "v"(a[element]), "v"(b[element]));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
                     : "+a"(c) : "v"(a), "v"(b), "v"(scale_a), "v"(scale_b), "n"(SEL & 1), "n"(SEL >> 1));
}

// block id -> (tile_m, tile_n, split).  Blocks go to the 8 XCDs in turn and about 256 run at a time.  Of every 256 consecutive tiles an
// XCD gets 32 in a row; tiles are walked in groups of 8 tile rows, so an XCD's 32 share 8 + 4 operand panels in its L2 and all 256 share
// 8 + 32 in the memory-side cache.
struct Tile { int m, n, split; };
__device__ __forceinline__ Tile tile_of(int id, const Problem& p) {
    const int per = p.tiles_m * p.tiles_n, whole = per * p.splits & ~255;
    int t = id < whole ? (id & ~255) + (id & 7) * 32 + ((id & 255) >> 3) : id;
    const int split = t / per;
    t -= split * per;
    const int group = t / (8 * p.tiles_n), first = group * 8, height = min(p.tiles_m - first, 8);
    t -= group * 8 * p.tiles_n;
    return {first + t % height, t / height, split};
}

// a value that the compiler does not carry through a loop in a dozen forms (it spills them): computed again where it is used
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

template <class F, int... N>
__device__ __forceinline__ void each(std::integer_sequence<int, N...>, F f) { (f(std::integral_constant<int, N>()), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F f) { each(std::make_integer_sequence<int, N>(), f); }

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

// The same from rows at any address and of any length in values (k need not end with 16 bytes): through registers, two slabs ahead, since the direct
// way into LDS wants 16-byte chunks.  For products that the bytes of A bound: a copy of A to aligned rows would cost two more passes over it.
template <int KIND, int BM, int BN, int WM, int WN>
struct AnyRow : Ring<KIND, BM, BN, WM, WN, 2> {
    typedef Ring<KIND, BM, BN, WM, WN, 2> Base;
    static constexpr int MF = Base::MF, NF = Base::NF, LOADS = Base::LOADS, STAGE_BYTES = Base::STAGE_BYTES, VALUE = KIND == FP32 ? 4 : 2;
    static_assert(KIND != E2M1, "");

    // the first `left` bytes, zeros behind them
    static __device__ __forceinline__ i32x4 part(const char* from, int left) {
        if (left >= 16) return *(const Loose*)from;
        i32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < 16; b += VALUE)
            if (b < left) {
                if constexpr (VALUE == 4) v[b / 4] = *(const int*)(from + b);
                else v[b / 4] |= (int)((unsigned)*(const unsigned short*)(from + b) << (b % 4 * 8));
            }
        return v;
    }
    static __device__ __forceinline__ void run(const Problem& p, Tile t, char* lds, f32x4 (&acc)[MF][NF]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        const int slabs = (p.kbytes + 127) >> 7, first = t.split * p.slabs_per_split, last = min(slabs, first + p.slabs_per_split) - 1;
        const int64_t m0 = (int64_t)t.m * BM, n0 = (int64_t)t.n * BN;
        const char* row_at[LOADS];
        const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = (wave * LOADS + i) * 8;
            const Operand& o = row < BM ? p.a : p.b;
            const int64_t mine = (row < BM ? m0 + row : n0 + (row - BM)) + (lane >> 3);
            row_at[i] = o.ptr + (mine < o.rows ? mine : o.rows - 1) * o.pitch + chunk;
        }
        auto fetch = [&](int slab, i32x4 (&to)[LOADS]) {
            slab = min(slab, last);
            const int64_t k = (int64_t)slab * 128;
            if (k + 128 <= p.kbytes) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) to[i] = *(const Loose*)(row_at[i] + k);
            } else {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) to[i] = part(row_at[i] + k, (int)(p.kbytes - k) - chunk);
            }
        };
        auto put = [&](int slot, const i32x4 (&from)[LOADS]) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) *(i32x4*)(lds + slot * STAGE_BYTES + (wave * LOADS + i) * 1024 + lane * 16) = from[i];
        };
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        int place[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) place[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ (lane & 7)) * 16);
        i32x4 x[LOADS], y[LOADS];
        fetch(first, x);
        fetch(first + 1, y);
        put(0, x);
        fetch(first + 2, x);
        auto step = [&](int k, int slot, i32x4 (&next)[LOADS]) {
            lds_barrier();                                               // this slab is there for every wave, and nobody reads the previous one any more
            put(slot ^ 1, next);
            fetch(k + 3, next);
            const char* sa = lds + slot * STAGE_BYTES + Base::row0(wm, 0) * 128;
            const char* sb = lds + slot * STAGE_BYTES + (BM + Base::col0(wn, 0)) * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                i32x4 b[NF];
#pragma unroll
                for (int j = 0; j < NF; ++j) b[j] = *(const i32x4*)(sb + place[h] + j * 2048);
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    const i32x4 a = *(const i32x4*)(sa + place[h] + i * 2048);
#pragma unroll
                    for (int j = 0; j < NF; ++j) acc[i][j] = mma<KIND, 0>(a, b[j], acc[i][j], 0, 0);
                }
            }
        };
        for (int k = first; k <= last; k += 2) {
            step(k, 0, y);
            if (k < last) step(k + 1, 1, x);
        }
        lds_barrier();                                                   // LDS is the epilogue's
    }
};

// The large tile: 256 x 256 outputs on 4 waves of 128 x 128, one wave per SIMD.  Against 8 waves of 128 x 64 it reads 128 instead of
// 192 KB of LDS per slab (a CU reads 128 bytes per clock and needs 2048 clocks of matrix instructions per slab), so LDS stays behind the
// matrix pipe.  A wave multiplies a half slab (64 products, 16 clocks each) while it reads the fragments of the next:
//   first half of a slab    reads the second half's fragments; FREE: all waves have them, the slab after the next starts over this one
//   second half             LANDED: the next slab is there for all waves; reads its first half's fragments
// What bounds this loop is the way from L2 to LDS and the issue of anything between two products: one fetch in front of every fourth
// product and a read in front of two of five take 1.39 us a slab (the products alone 0.91); all fetches of a slab in a row 1.49, one wait for
// everything per slab 1.55 (bf16, 4096 x 8192 x 8192: 1545 TFLOP/s).
// A block takes its tiles one after the other as one stream of slabs: while the epilogue of a tile runs, the first two slabs of the next
// are under way or there.  The epilogue has the LDS behind LDS_BYTES; it must not wait for the loads in flight.
template <int KIND, bool TAIL = false>
struct Wide {
    static constexpr int KIND_ = KIND, TILE_M = 256, TILE_N = 256, WAVES_M = 2, WAVES_N = 2, THREADS = 256, MF = 8, NF = 8;
    static constexpr int STAGE_BYTES = 512 * 128, LDS_BYTES = 2 * STAGE_BYTES + (KIND == E2M1 ? 2 * 8192 : 0), LOADS = 16;
    static constexpr int FREE = 44, LANDED = 23;                // products of a half in front of which the two barriers stand
    static constexpr int OUT = (64 - FREE + LANDED) / 4;         // of a slab's fetches: how many are out when LANDED is reached
    static_assert(FREE >= 3 + 38 && LANDED + 38 <= 64 && (64 - FREE) % 4 == 0 && LANDED % 4 == 3 && OUT < LOADS, "");
    // of a half's 16 reads: how many stand in front of product n, 2 in 5 from product `from` on
    static __device__ constexpr int reads(int n, int from) { return n <= from ? 0 : ((n - from) * 2 + 3) / 5 > 16 ? 16 : ((n - from) * 2 + 3) / 5; }
    static_assert(reads(FREE, 3) == 16 && reads(64, LANDED) == 16, "");
    static __device__ __forceinline__ int row0(int wm, int i) { return wm * 128 + i * 16; }
    static __device__ __forceinline__ int col0(int wn, int j) { return wn * 128 + j * 16; }

    template <class EPI>
    static __device__ __forceinline__ void run(const Problem& p, char* lds, const EPI& epi) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave >> 1, wn = wave & 1;
        const int tiles = p.tiles_m * p.tiles_n * p.splits, stride = gridDim.x;
        const int slabs = (p.kbytes + 127) >> 7, pairs = (slabs + 1) >> 1;
        const std::integral_constant<int, 0> zero;
        const std::integral_constant<int, 1> one;
        auto first_of = [&](const Tile& t) { return t.split * p.slabs_per_split; };
        auto last_of = [&](const Tile& t) { return KIND == E2M1 ? 2 * pairs - 1 : min(slabs, (t.split + 1) * p.slabs_per_split) - 1; };   // e2m1: whole pairs

        // ---- the stream of slabs: waves 0 and 1 fetch A, 2 and 3 B: 128 rows each, 8 rows a fetch
        const Operand& o = wave < 2 ? p.a : p.b;
        const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 3)) * 16u;
        const unsigned to = lds_address(lds) + (unsigned)wave * 16384u;
        int fetch_tile = blockIdx.x, fetch_slab = first_of(tile_of(fetch_tile, p)), fetch_last;
        const char* base;
        unsigned off[LOADS];
        auto point = [&](auto again) {                                   // at fetch_tile
            const Tile t = tile_of(fetch_tile, p);
            fetch_last = last_of(t);
            const int64_t r0 = (wave < 2 ? (int64_t)t.m * 256 : (int64_t)t.n * 256) + (wave & 1) * 128;
            const int64_t from = r0 < o.rows ? r0 : o.rows - 1;
            const int left = (int)min((int64_t)128, o.rows - from);      // rows that exist
            base = o.ptr + from * o.pitch;
            const int row = fresh(lane >> 3);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const unsigned v = (unsigned)min(i * 8 + row, left - 1) * (unsigned)o.pitch + chunk;
                if constexpr (again.value) asm volatile("v_mov_b32 %0, %1" : "+v"(off[i]) : "v"(v));   // in place: the loop would else copy all 16 every time
                else off[i] = v;
            }
        };
        auto advance = [&]() {                                           // behind the last tile the last slab comes again, unread
            if (fetch_slab < fetch_last) ++fetch_slab;
            else if (fetch_tile + stride < tiles) {
                fetch_tile += stride;
                fetch_slab = first_of(tile_of(fetch_tile, p));
                point(one);
            }
        };
        // TAIL: k does not end with a slab; where this lane's chunk of the last one lies behind the end it fetches the page of zeros.  A build of
        // its own, since the branch around each fetch costs 10 %.
        const char* at;
        auto aim = [&]() { at = base + (int64_t)fetch_slab * 128; };
        auto load = [&](int slot, int i) {
            const unsigned dst = to + (unsigned)(slot * STAGE_BYTES + i * 1024);
            if (TAIL && fetch_slab * 128 + 128 > p.kbytes) dma16(dst, fetch_slab * 128 + (int)chunk < p.kbytes ? at + off[i] : (const char*)zero_page);
            else dma16(dst, at + off[i]);
        };

        // ---- e2m1: the scale words of a pair of slabs, 16 bytes a row, fetched one pair ahead into LDS behind the slabs; 16 words a lane go to
        // registers before the pair begins
        int scale[16], scale_tile = blockIdx.x, scale_pair = 0, scale_slot = 0;
        const int64_t scale_pitch = (wave < 2 ? p.rows_a : p.rows_b) * 16;      // bytes of a pair
        auto scales_of = [&](int id) {
            const Tile t = tile_of(id, p);
            return (const char*)(wave < 2 ? p.scales_a + (int64_t)t.m * 1024 : p.scales_b + (int64_t)t.n * 1024) + (wave & 1) * 2048;
        };
        const char* scale_at = KIND == E2M1 ? scales_of(scale_tile) : nullptr;
        auto load_scales = [&]() {
            const unsigned dst = lds_address(lds) + (unsigned)(2 * STAGE_BYTES + scale_slot * 8192 + wave * 2048);
            dma16(dst, scale_at + lane * 16);
            dma16(dst + 1024, scale_at + lane * 16 + 1024);
            scale_slot ^= 1;
            if (++scale_pair < pairs) {
                scale_at += scale_pitch;
            } else if (scale_tile + stride < tiles) {
                scale_pair = 0;
                scale_tile += stride;
                scale_at = scales_of(scale_tile);
            }                                                            // behind the last tile the last pair comes again, unread
        };
        auto read_scales = [&]() {                                       // of the pair that was fetched last
            const char* from = lds + 2 * STAGE_BYTES + (scale_slot ^ 1) * 8192 + (lane & 15) * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int n = 0; n < 16; ++n) scale[n] = *(const int*)(from + (n < NF ? 4096 + wn * 2048 + n * 256 : wm * 2048 + (n - NF) * 256));
        };

        int place[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) place[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ (lane & 7)) * 16);
        const char* sa = lds + wm * 16384;
        const char* sb = lds + 32768 + wn * 16384;
        i32x4 a[2][MF], b[2][NF];
        auto read = [&](int slot, auto h, int n) {                      // the n-th of a half slab's 16 fragments
            if (n < NF) b[h.value][n] = *(const i32x4*)(sb + slot * STAGE_BYTES + place[h.value] + n * 2048);
            else a[h.value][n - NF] = *(const i32x4*)(sa + slot * STAGE_BYTES + place[h.value] + (n - NF) * 2048);
        };
        f32x4 acc[MF][NF];
        // 64 products of a half, with before(n) in front of the n-th; the order is kept as it is written
        auto multiply = [&](auto odd, auto h, auto before) {
            constexpr int PER = KIND == FP32 ? 4 : 1;                    // fp32: an instruction per element, all 64 products between two of them
            each<64>([&](auto n) {
                before(n);
                __builtin_amdgcn_sched_barrier(0);
                each<PER>([&](auto q) {
                    constexpr int N = n.value * PER + q.value, E = N >> 6, I = (N & 63) >> 3, J = I & 1 ? 7 - (N & 7) : N & 7;
                    mma_in_place<KIND, 2 * odd.value + h.value>(acc[I][J], a[h.value][I], b[h.value][J], E, scale[NF + I], scale[J]);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        int slot = 0;
        auto step = [&](auto odd) {
            constexpr bool SCALES = KIND == E2M1 && odd.value == 0;      // 2 more loads in flight when LANDED is reached
            multiply(odd, zero, [&](auto n) {
                constexpr int N = n.value, I = (N - FREE) / 4;
                if constexpr (reads(N + 1, 3) > reads(N, 3)) read(slot, one, reads(N, 3));
                if constexpr (SCALES && N == 1) load_scales();
                if constexpr (N == 2) advance();
                if constexpr (N == FREE - 1) aim();
                if constexpr (N == FREE) lds_barrier();
                if constexpr (N > FREE && (N - FREE) % 4 == 3) load(slot, I);
            });
            multiply(odd, one, [&](auto n) {
                constexpr int N = n.value, I = (N + 64 - FREE) / 4;
                if constexpr ((N + 64 - FREE) % 4 == 3 && I < LOADS) load(slot, I);
                if constexpr (N == LANDED) {
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OUT + (SCALES ? 2 : 0)) : "memory");
                    barrier();
                }
                if constexpr (reads(N + 1, LANDED) > reads(N, LANDED)) read(slot ^ 1, zero, reads(N, LANDED));
            });
            if constexpr (KIND == E2M1 && odd.value == 1) read_scales();
            slot ^= 1;
        };

        if constexpr (KIND == E2M1) load_scales();
        point(zero);
        aim();
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(0, i);
        advance();
        aim();
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(1, i);
        wait_loads<LOADS>();
        barrier();
        for (int id = blockIdx.x; id < tiles; id += stride) {
            point(zero);                                                 // again, and the first fragments too: no register but the sums lives through an epilogue
#pragma unroll
            for (int n = 0; n < 16; ++n) read(slot, zero, n);
            if constexpr (KIND == E2M1) read_scales();
            const Tile t = tile_of(id, p);
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const auto ahead = epi.template ahead<Wide>(t, tid);
            int left = last_of(t) - first_of(t) + 1;
            do {
                step(zero);
                if constexpr (KIND == E2M1) step(one);
                left -= KIND == E2M1 ? 2 : 1;
                if (left == 0) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");    // the last sums leave the pipe before anything reads them
            } while (left);
            epi.template operator()<Wide>(p, t, lds + LDS_BYTES, acc, ahead);
        }
        wait_loads<0>();
    }
};

// the sums of columns `from` on stay in accumulation registers up to here: over branches the compiler else takes all of them out at once and
// spills (a third of the time of an epilogue)
template <class R>
__device__ __forceinline__ void hold(f32x4 (&acc)[R::MF][R::NF], int from) {
    if constexpr (R::MF * R::NF > 32)
#pragma unroll
        for (int i = 0; i < R::MF; ++i)
#pragma unroll
            for (int j = 0; j < R::NF; ++j)
                if (j >= from) asm volatile("" : "+a"(acc[i][j]));
}

// a sum out of its accumulation registers, here and not earlier: 256 of them read ahead of their use would not fit beside what is live
__device__ __forceinline__ f32x4 take(const f32x4& sum) {
    f32x4 v;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "=v"(v) : "0"(sum));
    return v;
}

__device__ __forceinline__ void give(f32x4& sum, f32x4 v) { asm volatile("" : "=a"(sum) : "0"(v)); }

// A wave's tile to out[n][m] (m contiguous, `ld` elements between rows), n < rows, m < width: 16-bit rows 16 at a time, 32-bit rows 8 at a time
// through LDS, so that a store covers whole lines (from registers it would cover runs of 32 or 64 bytes), and past the caches: written the plain
// way the 33 MB that 256 tiles leave at once push the operands out of L2 (50176 x 4096 x 2048: 1180 TFLOP/s, with whole lines 1260, past the
// caches 1440).  `value`: sum -> what is stored; `add`: onto what is there.
template <class T, int N> struct Stage {         // rows of N elements; chunk c of 16 bytes of row r lies at c ^ r: rows written together meet on no bank
    static constexpr int ROWS = 32 / (int)sizeof(T), LANES = N * (int)sizeof(T) / 16, BYTES = ROWS * N * (int)sizeof(T);
    static __device__ __forceinline__ int at(int row, int byte) { return (row * LANES + ((byte >> 4) ^ (row & (LANES - 1)))) * 16 + (byte & 15); }
};
template <class R, class T>
constexpr int stage_bytes() { return R::WAVES_M * R::WAVES_N * Stage<T, R::TILE_M / R::WAVES_M>::BYTES; }

template <class R, class T, class VALUE>
__device__ __forceinline__ void store_tile(Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], T* out, int64_t ld, int rows, int width, bool add, VALUE value) {
    typedef Stage<T, R::TILE_M / R::WAVES_M> S;
    struct alignas(4 * sizeof(T)) Four { T v[4]; };
    struct alignas(16) Chunk { T v[16 / sizeof(T)]; };
    const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / R::WAVES_N, wn = wave % R::WAVES_N;
    const int m = t.m * R::TILE_M + R::row0(wm, 0) + (lane % S::LANES) * (16 / (int)sizeof(T)), g4 = (lane >> 4) * 4, col = lane & 15;
    char* stage = lds + wave * S::BYTES;
#pragma unroll
    for (int j = 0; j < R::NF; ++j)
#pragma unroll
        for (int part = 0; part < 16; part += S::ROWS) {
            hold<R>(acc, j);
#pragma unroll
            for (int i = 0; i < R::MF; ++i) {
                const f32x4 v = take(acc[i][j]);
                const Four f = {{(T)value(v[0]), (T)value(v[1]), (T)value(v[2]), (T)value(v[3])}};
                if (S::ROWS == 16 || (col & ~(S::ROWS - 1)) == part) *(Four*)(stage + S::at(col & (S::ROWS - 1), (i * 16 + g4) * (int)sizeof(T))) = f;
            }
            wave_sync();
#pragma unroll
            for (int r = 0; r < S::ROWS; r += 64 / S::LANES) {
                const int row = r + lane / S::LANES, n = t.n * R::TILE_N + R::col0(wn, j) + part + row;
                if (row >= S::ROWS || n >= rows || m >= width) continue;
                Chunk c = *(const Chunk*)(stage + S::at(row, (lane % S::LANES) * 16));
                T* to = out + (int64_t)n * ld + m;
                if (m + 16 / (int)sizeof(T) <= width) {
                    if (add) {
                        const Chunk old = __builtin_bit_cast(Chunk, *(const Loose*)to);
#pragma unroll
                        for (int e = 0; e < 16 / (int)sizeof(T); ++e) c.v[e] = (T)((float)c.v[e] + (float)old.v[e]);
                    }
                    __builtin_nontemporal_store(__builtin_bit_cast(i32x4, c), (Loose*)to);
                } else {
#pragma unroll
                    for (int e = 0; e < 16 / (int)sizeof(T); ++e)
                        if (m + e < width) to[e] = add ? (T)((float)c.v[e] + (float)to[e]) : c.v[e];
                }
            }
            wave_sync();
        }
}

// What an epilogue loads before its tile's products, which hide it: EPI::ahead.  This one: nothing.
struct NoAhead {};

// A kernel's body: the LDS that it needs, and its tile (Ring) or tiles (Wide)
template <class R> struct Persistent { static constexpr bool value = false; };
template <int KIND, bool TAIL> struct Persistent<Wide<KIND, TAIL>> { static constexpr bool value = true; };
template <class R, class EPI>
constexpr int lds_bytes() {
    return Persistent<R>::value ? R::LDS_BYTES + EPI::template lds<R>() : R::LDS_BYTES > EPI::template lds<R>() ? R::LDS_BYTES : EPI::template lds<R>();
}
template <class R, class EPI>
__device__ __forceinline__ void product(const Problem& p, char* lds, const EPI& epi) {
    if constexpr (Persistent<R>::value) {
        R::run(p, lds, epi);
    } else {
        const Tile t = tile_of(blockIdx.x, p);
        f32x4 acc[R::MF][R::NF];
        const auto ahead = epi.template ahead<R>(t, threadIdx.x);
        R::run(p, t, lds, acc);
        epi.template operator()<R>(p, t, lds, acc, ahead);
    }
}

constexpr int CUS = 256;                     // of an MI355X: one block of large tiles each

// Blocks of a launch.  Long tiles go to a block each: they are dealt out as CUs come free, and 1 % of a tile is saved by chaining them (16 tiles of
// 64 slabs: 1.60 against 1.64 ms chained; 2 tiles of 510 slabs: 1.63 against 1.49 ms, the slowest CU's two).
constexpr int64_t MOST_BLOCKS = (int64_t)1 << 24;      // of 256 threads in a launch, whose threads are counted in 32 bits: these excluded
template <class R>
unsigned grid_of(const Problem& p) {
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    return (unsigned)(Persistent<R>::value && (p.slabs_per_split < 128 || tiles >= MOST_BLOCKS) && tiles > CUS ? CUS : tiles);
}

}  // namespace nt
}  // namespace cs
