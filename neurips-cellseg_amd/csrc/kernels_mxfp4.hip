// gfx950 (MI355X): the microscaled 4-bit format (OCP MX, MXFP4) - quantisation, dequantisation and the linear layer on it.
// 32 consecutive values along the inner axis share one scale 2^(s - 127), s = floor(log2 max|x|) - 2 + 127 clamped at 0 (one e8m0 byte);
// each value is x / scale rounded to e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), ties to the even code, above 6 to 6.  A block
// with an infinity or NaN has the scale byte 0xff, which stands for NaN.  Two codes a byte, the even one in the low half; a row that ends
// inside a block is filled up with zeros.
// Quantisation and its inverse are bound by memory: 8192 x 8192, bf16, 26 and 25 us for 170 MB each (6.6 TB/s).  The product: 4096 x 4096 -> 16384
// 136 us (4.0 PFLOP/s), its scales and x prepared in 10 us; both 135 to 143 us in a row of calls.
#include "gemm_nt.h"

namespace cs {
namespace {
using namespace nt;

template <int TYPE> struct Value;
template <> struct Value<CS_TYPE_BF16> { typedef __bf16 T; };
template <> struct Value<CS_TYPE_FP16> { typedef _Float16 T; };
template <> struct Value<CS_TYPE_FP32> { typedef float T; };

// 8 values from column c of a row of `width`
template <class T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t width, float (&v)[8]) {
    if (c + 8 <= width) {
        struct alignas(16) Sixteen { T v[16 / sizeof(T)]; };
        struct { Sixteen part[sizeof(T) / 2]; __device__ T at(int i) const { return part[i * sizeof(T) / 16].v[i % (16 / sizeof(T))]; } } e;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.part[i] = __builtin_bit_cast(Sixteen, ((const Loose*)(row + c))[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)e.at(i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < width ? (float)row[c + i] : 0.f;
    }
}

// 8 values of a lane, 4 lanes a block -> their codes; `scale`: the block's byte, the same in the 4 lanes
__device__ __forceinline__ unsigned encode8(const float (&v)[8], unsigned* scale) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu);
    most = max(most, (unsigned)__shfl_xor((int)most, 1));
    most = max(most, (unsigned)__shfl_xor((int)most, 2));
    const int field = (int)(most >> 23);                                 // the exponent's field of the largest
    if (field == 255) {
        *scale = 255u;
        return 0u;
    }
    const int s = field > 2 ? field - 2 : 0;
    *scale = (unsigned)s;
    const float by = __builtin_bit_cast(float, (unsigned)(254 - s) << 23);   // 2^(127 - s): s <= 252, a normal number
    // v_cvt_scalef32_pk_fp4_f32 with scale 1: two values to the nearest code, ties to even, above 6 to 6 (a comparison per border costs 14
    // instructions a value and as much time as the memory)
    unsigned out = 0;
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[0] * by, v[1] * by, 1.f, 0);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[2] * by, v[3] * by, 1.f, 1);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[4] * by, v[5] * by, 1.f, 2);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[6] * by, v[7] * by, 1.f, 3);
    return out;
}

// place of the scale byte of (row, block) in the order that the product reads (gemm_nt.h: a word per pair of slabs, row and chunk column)
__device__ __forceinline__ int64_t tile_place(int64_t row, int64_t block, int64_t rows) {
    return (((block >> 4) * rows + row) * 4 + (block & 3)) * 4 + ((block >> 2) & 3);
}

// Rows over thread blocks: one row or, where a row has fewer than 256 / 4 blocks of 32, several.  -> the thread's row and item (4 a block of 32)
struct Place { int64_t row; int item; };
__device__ __forceinline__ Place place_of(int64_t block, int items) {
    if (items >= 256) return {block, (int)threadIdx.x};
    const int rows = 256 / items, r = (int)threadIdx.x / items;
    return {r < rows ? block * rows + r : (int64_t)1 << 62, (int)threadIdx.x - r * items};
}
unsigned row_blocks(int64_t rows, int64_t items) {
    const int64_t per = items >= 256 ? 1 : 256 / items;
    return (unsigned)((rows + per - 1) / per);
}

template <class T>
__global__ __launch_bounds__(256) void quantise_kernel(const T* x, int64_t pitch, int64_t rows, int64_t width, int blocks, uint8_t* codes, uint8_t* scales) {
    const Place p = place_of(blockIdx.x, blocks * 4);
    if (p.row >= rows) return;                                           // a block's 4 lanes go together
    for (int i = p.item; i < blocks * 4; i += 256) {
        float v[8];
        load8(x + p.row * pitch, (int64_t)i * 8, width, v);
        unsigned scale;
        *(unsigned*)(codes + (p.row * blocks * 4 + i) * 4) = encode8(v, &scale);
        if ((i & 3) == 0) scales[p.row * blocks + (i >> 2)] = (uint8_t)scale;
    }
}

// What the product reads: x quantised, and both operands' scales in its order (gemm_nt.h) over rows_x / rows_w rows, blocks up to a multiple of
// 16, with scale 1 where there is no row or block.  The first `x_blocks` thread blocks take x, the others 64 rows of a pair of the weight's scales.
template <class T>
__global__ __launch_bounds__(256) void prepare_kernel(const T* x, int64_t pitch, int64_t rows, int64_t width, int blocks, uint8_t* codes, uint8_t* scales_x,
                                                      int64_t rows_x, const uint8_t* scales, int64_t outputs, uint8_t* scales_w, int64_t rows_w, unsigned x_blocks) {
    const int padded = (blocks + 15) / 16 * 16;
    if (blockIdx.x < x_blocks) {
        const Place p = place_of(blockIdx.x, padded * 4);
        if (p.row >= rows_x) return;
        for (int i = p.item; i < padded * 4; i += 256) {
            const bool in = p.row < rows && (i >> 2) < blocks;           // the same in a block's 4 lanes
            float v[8];
            if (in) load8(x + p.row * pitch, (int64_t)i * 8, width, v);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = 0.f;
            unsigned scale;
            const unsigned code = encode8(v, &scale);
            if (in) *(unsigned*)(codes + (p.row * blocks * 4 + i) * 4) = code;
            if ((i & 3) == 0) scales_x[tile_place(p.row, i >> 2, rows_x)] = (uint8_t)(in ? scale : 127u);
        }
        return;
    }
    const unsigned at = blockIdx.x - x_blocks, groups = (unsigned)(rows_w / 64), pair = at / groups;
    const int64_t row = (int64_t)(at - pair * groups) * 64 + (threadIdx.x >> 2);
    const int g = threadIdx.x & 3;
    unsigned word = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const int block = (int)pair * 16 + h * 4 + g;
        word |= (row < outputs && block < blocks ? (unsigned)scales[row * blocks + block] : 127u) << (8 * h);
    }
    ((unsigned*)scales_w)[(pair * rows_w + row) * 4 + g] = word;
}

template <class T>
__global__ __launch_bounds__(256) void dequantise_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t width, int blocks, T* out) {
    const Place p = place_of(blockIdx.x, blocks * 4);
    if (p.row >= rows) return;
    for (int i = p.item; i < blocks * 4; i += 256) {
        const unsigned code = *(const unsigned*)(codes + (p.row * blocks * 4 + i) * 4), s = scales[p.row * blocks + (i >> 2)];
        const float by = s == 255u ? __builtin_nanf("") : s == 0u ? __builtin_bit_cast(float, 1u << 22) : __builtin_bit_cast(float, s << 23);     // 2^(s - 127)
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.f, 3)};
        struct alignas(16) Eight { T v[8]; } e;
#pragma unroll
        for (int k = 0; k < 8; ++k) e.v[k] = (T)(v[k >> 1][k & 1] * by);
        const int64_t c = (int64_t)i * 8;
        T* to = out + p.row * width + c;
        if (c + 8 <= width) {
            if constexpr (sizeof(T) == 2) __builtin_nontemporal_store(__builtin_bit_cast(i32x4, e), (Loose*)to);
            else __builtin_memcpy(to, &e, sizeof(e));
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < width) to[k] = e.v[k];
    }
}

// ---- the linear layer: y[n][m] = sum_k x[n][k] w[m][k], m the outputs ------------------------------------------------------------------
template <class T>
struct LinearEpi {
    T* out;            // [rows][outputs]
    int rows, outputs;
    template <class R> static constexpr int lds() { return stage_bytes<R, T>(); }
    template <class R> __device__ __forceinline__ NoAhead ahead(Tile, int) const { return {}; }
    template <class R>
    __device__ __forceinline__ void operator()(const Problem& p, Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], NoAhead) const {
        store_tile<R>(t, lds, acc, out, outputs, rows, outputs, false, [](float v) { return v; });
    }
};

template <class R, class EPI>
__global__ __launch_bounds__(R::THREADS) void linear_kernel(Problem p, EPI epi) {
    __shared__ __attribute__((aligned(1024))) char lds[lds_bytes<R, EPI>()];
    product<R>(p, lds, epi);
}

typedef Ring<E2M1, 128, 128, 2, 2, 2> Middle;
typedef Ring<E2M1, 128, 32, 4, 1, 4> Flat;

// Up to 16 rows, as a server decodes: the weights are read once and nothing else counts.  A block has 16 outputs; its 4 waves take runs of 8 blocks
// of k (128 bytes of a weight row) in turn, straight from memory into the matrix instruction, and join their sums in LDS.  Every thread block
// quantises the few rows for itself, into LDS: one launch instead of three, and x is in L2.  1 x 4096 -> 16384: 13.1 us, 13.4 us from call to call (26.4 us in
// three launches); 36 MB would take 6.4 us.
constexpr int FEW_LDS = 40 << 10;                 // 4 blocks a CU
__host__ __device__ inline int few_pitch(int blocks) { return (blocks + 3) / 4 * 64 + 16; }      // bytes of a row's codes, off the powers of two
int few_lds(int64_t rows, int64_t blocks) { return blocks > 4096 ? FEW_LDS + 1 : (int)(rows * (few_pitch((int)blocks) + (blocks + 3) / 4 * 4)); }

bool few_rows(int64_t rows, int64_t blocks) { return rows <= 16 && few_lds(rows, blocks) <= FEW_LDS; }

template <class T>
__global__ __launch_bounds__(256) void few_rows_kernel(const T* x, int64_t pitch, int rows, int64_t width, int blocks, const uint8_t* codes, const uint8_t* scales,
                                                       int outputs, T* y) {
    extern __shared__ __attribute__((aligned(16))) char few[];
    __shared__ f32x4 join[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, steps = (blocks + 3) >> 2, cp = few_pitch(blocks), sp = steps * 4;
    char* const xs = few + rows * cp;                                    // scales of x [rows][sp]
    // 4 runs of weights go out before x is quantised, and always 4 runs ahead of the products
    const int g = lane >> 4, m0 = blockIdx.x * 16, m = min(m0 + (lane & 15), outputs - 1), n = (lane & 15) < rows ? lane & 15 : 0;
    const uint8_t* wc = codes + (int64_t)m * blocks * 16;
    const uint8_t* ws = scales + (int64_t)m * blocks;
    i32x4 a[8];
    int sa[8];
    auto fetch = [&](int unit, int to) {                                 // run `unit`: steps 2 unit and 2 unit + 1 of 4 blocks; zeros behind the last
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int block = (2 * unit + h) * 4 + g, in = min(block, blocks - 1);
            a[to * 2 + h] = *(const i32x4*)(wc + (int64_t)in * 16);
            sa[to * 2 + h] = ws[in];
            if (block >= blocks) a[to * 2 + h] = i32x4{0, 0, 0, 0}, sa[to * 2 + h] = 127;
        }
    };
#pragma unroll
    for (int c = 0; c < 4; ++c) fetch(wave + 4 * c, c);
    for (int i = tid; i < rows * sp * 4; i += 256) {
        const int row = rows == 1 ? 0 : i / (sp * 4), block = (i >> 2) - row * sp;
        float v[8];
        load8(x + row * pitch, (int64_t)block * 32 + (i & 3) * 8, width, v);   // zeros behind the width
        unsigned scale;
        *(unsigned*)(few + row * cp + block * 16 + (i & 3) * 4) = encode8(v, &scale);
        if ((i & 3) == 0) xs[row * sp + block] = (char)scale;
    }
    __syncthreads();
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int u = wave; 2 * u < steps; u += 16)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int unit = u + 4 * c;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int block = (2 * unit + h) * 4 + g;
                i32x4 b = {0, 0, 0, 0};
                int sb = 127;
                if (block < blocks) {
                    b = *(const i32x4*)(few + n * cp + block * 16);
                    sb = (uint8_t)xs[n * sp + block];
                }
                acc = mma<E2M1, 0>(a[c * 2 + h], b, acc, sa[c * 2 + h], sb);
            }
            if (2 * (unit + 16) < steps) fetch(unit + 16, c);
        }
    join[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && (lane & 15) < rows) {
        acc = (join[0][lane] + join[1][lane]) + (join[2][lane] + join[3][lane]);
        T* to = y + (int64_t)(lane & 15) * outputs;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m0 + g * 4 + r < outputs) to[m0 + g * 4 + r] = (T)acc[r];
    }
}

template <class R, class T>
int launch_linear(hipStream_t st, Problem p, LinearEpi<T> epi) {
    p.tiles_m = (int)((p.a.rows + R::TILE_M - 1) / R::TILE_M);
    p.tiles_n = (int)((p.b.rows + R::TILE_N - 1) / R::TILE_N);
    p.splits = 1;
    p.slabs_per_split = (p.kbytes + 127) / 128;
    CS_REQUIRE((int64_t)p.tiles_m * p.tiles_n < (Persistent<R>::value ? (int64_t)1 << 30 : MOST_BLOCKS), "mxfp4 linear: too many tiles");
    linear_kernel<R, LinearEpi<T>><<<dim3(grid_of<R>(p)), R::THREADS, 0, st>>>(p, epi);
    CS_HIP(hipGetLastError());
    return CS_OK;
}

struct LinearPlan {
    size_t bytes;
    uint8_t *codes, *scales_x, *scales_w;
    int64_t blocks, rows_x, rows_w;
};
LinearPlan make_plan(int64_t rows, int64_t width, int64_t outputs, void* base) {
    LinearPlan p{};
    p.blocks = (width + 31) / 32;
    p.rows_x = (rows + 255) / 256 * 256;
    p.rows_w = (outputs + 255) / 256 * 256;
    const int64_t tiled = (p.blocks + 15) / 16 * 16;
    if (few_rows(rows, p.blocks)) return p;
    size_t at = 0;
    auto take = [&](int64_t n) {
        uint8_t* q = base ? (uint8_t*)base + at : nullptr;
        at += ((size_t)n + 255) & ~(size_t)255;
        return q;
    };
    p.codes = take(rows * p.blocks * 16);
    p.scales_x = take(p.rows_x * tiled);
    p.scales_w = take(p.rows_w * tiled);
    p.bytes = at;
    return p;
}

int check_sizes(int64_t rows, int64_t width, int type, const char* what) {
    CS_REQUIRE(rows >= 0 && rows < (int64_t)1 << 30 && width >= 1 && width < (int64_t)1 << 24, "%s: rows %lld, width %lld out of range", what, (long long)rows,
               (long long)width);
    CS_REQUIRE(type >= CS_TYPE_BF16 && type <= CS_TYPE_FP32, "%s: unknown type %d", what, type);
    return CS_OK;
}

constexpr int64_t LAUNCH_ROWS = MOST_BLOCKS / 2;       // rows of a launch, a block each at most

template <class T>
int quantise(const void* x, int64_t pitch, int64_t rows, int64_t width, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const int64_t blocks = (width + 31) / 32;
    for (int64_t r = 0; r < rows; r += LAUNCH_ROWS) {
        const int64_t some = rows - r < LAUNCH_ROWS ? rows - r : LAUNCH_ROWS;
        quantise_kernel<T><<<row_blocks(some, blocks * 4), 256, 0, st>>>((const T*)x + r * pitch, pitch, some, width, (int)blocks,
                                                                       codes + r * blocks * 16, scales + r * blocks);
    }
    CS_HIP(hipGetLastError());
    return CS_OK;
}
template <class T>
int dequantise(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t width, void* out, hipStream_t st) {
    const int64_t blocks = (width + 31) / 32;
    for (int64_t r = 0; r < rows; r += LAUNCH_ROWS) {
        const int64_t some = rows - r < LAUNCH_ROWS ? rows - r : LAUNCH_ROWS;
        dequantise_kernel<T><<<row_blocks(some, blocks * 4), 256, 0, st>>>(codes + r * blocks * 16, scales + r * blocks, some, width, (int)blocks,
                                                                         (T*)out + r * width);
    }
    CS_HIP(hipGetLastError());
    return CS_OK;
}
template <class T>
int linear(const void* x, int64_t pitch, int64_t rows, int64_t width, const uint8_t* codes, const uint8_t* scales, int64_t outputs, void* y, const LinearPlan& p,
           hipStream_t st) {
    if (few_rows(rows, p.blocks)) {
        CS_REQUIRE((outputs + 15) / 16 < MOST_BLOCKS, "mxfp4 linear: too many outputs");
        few_rows_kernel<T><<<dim3((unsigned)((outputs + 15) / 16)), 256, few_lds(rows, p.blocks), st>>>((const T*)x, pitch, (int)rows, width, (int)p.blocks,
                                                                                                   codes, scales, (int)outputs, (T*)y);
        CS_HIP(hipGetLastError());
        return CS_OK;
    }
    const int64_t padded = (p.blocks + 15) / 16 * 16;
    const int64_t x_blocks = row_blocks(p.rows_x, padded * 4), w_blocks = p.rows_w / 64 * (padded / 16);
    CS_REQUIRE(x_blocks + w_blocks < MOST_BLOCKS, "mxfp4 linear: too many outputs");
    prepare_kernel<T><<<dim3((unsigned)(x_blocks + w_blocks)), 256, 0, st>>>((const T*)x, pitch, rows, width, (int)p.blocks, p.codes, p.scales_x,
                                                                             p.rows_x, scales, outputs, p.scales_w, p.rows_w, (unsigned)x_blocks);
    CS_HIP(hipGetLastError());
    Problem q{};
    q.a = Operand{(const char*)codes, p.blocks * 16, outputs};
    q.b = Operand{(const char*)p.codes, p.blocks * 16, rows};
    q.kbytes = (int)(p.blocks * 16);
    q.scales_a = (const unsigned*)p.scales_w;
    q.scales_b = (const unsigned*)p.scales_x;
    q.rows_a = p.rows_w;
    q.rows_b = p.rows_x;
    const LinearEpi<T> epi{(T*)y, (int)rows, (int)outputs};
    if (rows <= 64) return launch_linear<Flat>(st, q, epi);
    if (((outputs + 255) / 256) * ((rows + 255) / 256) >= 192) {
        // whole pairs of slabs, or zeros behind the end
        if (q.kbytes % 256) return launch_linear<Wide<E2M1, true>>(st, q, epi);
        return launch_linear<Wide<E2M1, false>>(st, q, epi);
    }
    return launch_linear<Middle>(st, q, epi);
}

}  // namespace
}  // namespace cs

extern "C" {
using namespace cs;

int cs_mxfp4_quantize(const void* x, int64_t pitch, int64_t rows, int64_t width, int type, uint8_t* codes, uint8_t* scales, void* stream) {
    if (int rc = check_sizes(rows, width, type, "mxfp4 quantize")) return rc;
    if (!rows) return CS_OK;
    CS_REQUIRE(x && codes && scales, "mxfp4 quantize: NULL pointer");
    CS_REQUIRE(((uintptr_t)codes & 3) == 0, "mxfp4 quantize: codes start at a multiple of 4 bytes");
    ProfScope prof(K_MXFP4, (hipStream_t)stream, 0, (double)rows * width * (type == CS_TYPE_FP32 ? 4.53 : 2.53));
    if (type == CS_TYPE_BF16) return quantise<__bf16>(x, pitch, rows, width, codes, scales, (hipStream_t)stream);
    if (type == CS_TYPE_FP16) return quantise<_Float16>(x, pitch, rows, width, codes, scales, (hipStream_t)stream);
    return quantise<float>(x, pitch, rows, width, codes, scales, (hipStream_t)stream);
}

int cs_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t width, int type, void* out, void* stream) {
    if (int rc = check_sizes(rows, width, type, "mxfp4 dequantize")) return rc;
    if (!rows) return CS_OK;
    CS_REQUIRE(out && codes && scales, "mxfp4 dequantize: NULL pointer");
    CS_REQUIRE(((uintptr_t)codes & 3) == 0, "mxfp4 dequantize: codes start at a multiple of 4 bytes");
    ProfScope prof(K_MXFP4, (hipStream_t)stream, 0, (double)rows * width * (type == CS_TYPE_FP32 ? 4.53 : 2.53));
    if (type == CS_TYPE_BF16) return dequantise<__bf16>(codes, scales, rows, width, out, (hipStream_t)stream);
    if (type == CS_TYPE_FP16) return dequantise<_Float16>(codes, scales, rows, width, out, (hipStream_t)stream);
    return dequantise<float>(codes, scales, rows, width, out, (hipStream_t)stream);
}

size_t cs_mxfp4_linear_workspace_bytes(int64_t rows, int64_t width, int64_t outputs) {
    if (check_sizes(rows, width, CS_TYPE_BF16, "mxfp4 linear") || check_sizes(outputs, width, CS_TYPE_BF16, "mxfp4 linear")) return 0;
    return make_plan(rows, width, outputs, nullptr).bytes;
}

int cs_mxfp4_linear(const void* x, int64_t pitch, int64_t rows, int64_t width, int type, const uint8_t* codes, const uint8_t* scales, int64_t outputs, void* y,
                    void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes(rows, width, type, "mxfp4 linear")) return rc;
    if (int rc = check_sizes(outputs, width, type, "mxfp4 linear")) return rc;
    if (!rows || !outputs) return CS_OK;
    CS_REQUIRE(x && y && codes && scales && (workspace || !cs_mxfp4_linear_workspace_bytes(rows, width, outputs)), "mxfp4 linear: NULL pointer");
    CS_REQUIRE(((uintptr_t)codes & 15) == 0 && ((uintptr_t)y & 15) == 0, "mxfp4 linear: codes and output start at a multiple of 16 bytes");
    const LinearPlan p = make_plan(rows, width, outputs, workspace);
    if (workspace_bytes < p.bytes) {
        set_error("mxfp4 linear: workspace of %zu bytes, %zu are needed", workspace_bytes, p.bytes);
        return CS_ERR_WORKSPACE;
    }
    const double size = type == CS_TYPE_FP32 ? 4.0 : 2.0;
    ProfScope prof(K_MXFP4, (hipStream_t)stream, 2.0 * rows * width * outputs, size * rows * (width + outputs) + 0.53 * outputs * width);
    if (type == CS_TYPE_BF16) return linear<__bf16>(x, pitch, rows, width, codes, scales, outputs, y, p, (hipStream_t)stream);
    if (type == CS_TYPE_FP16) return linear<_Float16>(x, pitch, rows, width, codes, scales, outputs, y, p, (hipStream_t)stream);
    return linear<float>(x, pitch, rows, width, codes, scales, outputs, y, p, (hipStream_t)stream);
}

}  // extern "C"
