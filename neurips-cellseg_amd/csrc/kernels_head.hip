// gfx950 (MI355X): losses of a linear head over a large vocabulary, whose logits come in pieces where they are large - the cross entropy and the
// distillation from a teacher's top logits.  Both are one computation: row i has a sparse target distribution q_i over a few ids (the
// cross entropy: one id, q = 1) and, with u = z / T, z = H W^T, lse_i = log sum_j exp(u_ij), p = exp(u - lse):
//   loss_i = T^2 (sum_k q_ik log q_ik + lse_i - sum_k q_ik u_i[id_ik]),   d loss_i / d z = T (p_i - q_i)
// Forward: one matrix product whose epilogue leaves, per row and tile of the vocabulary, the maximum and the sum of exponentials, and the
// few z that the loss names; a wave per row joins them.  Backward, in pieces of the vocabulary: the same product again, its epilogue
// writes G = p - q of the piece (and its transpose), then dH += G W and dW = G^T H as two products of the same kernel.  Where z is small or dear it is
// kept instead (Saved::scores, Saved::kept).
// Large calls are bound by the matrix pipe, which is busy 0.49 (G) to 0.68 (dH) of the time, at the clock that power leaves, 1.8 to 2.0 GHz.  8192 x 4096 over
// 131072 words, bf16: forward 7.1 ms (1240 TFLOP/s), G 7.7 ms, dH and dW 6.8 ms each (1290).
// Rows are the tokens; in every product the m axis is the one that is contiguous in what the epilogue writes (a lane holds 4 consecutive m).
#include "gemm_nt.h"

#include <math.h>

namespace cs {
namespace {
using namespace nt;

constexpr int KD_MAX_TOP = 1024;
constexpr int NO_ID = 0x7fffffff;
// c z - M is the exact c z less a float: where |c z| passes 2^31 the rounding of M alone, half its last place, leaves the range of 2^x.  From this
// temperature on that takes logits of 14 000 and more.
constexpr double MIN_TEMPERATURE = 1e-5;
constexpr int FEW_ROWS = 64;
enum RowState { ROW_SKIP = 0, ROW_COUNT = 1, ROW_BAD = 2 };

template <int KIND> struct Elem;
template <> struct Elem<BF16> { typedef __bf16 T; static constexpr float G_SCALE = 1.f; };
// fp16 holds 2^-24 at least: G, whose entries are p (down to 1 / vocab) and p - q, in [-1, 1], is kept times 2^14
template <> struct Elem<FP16> { typedef _Float16 T; static constexpr float G_SCALE = 16384.f; };
template <> struct Elem<FP32> { typedef float T; static constexpr float G_SCALE = 1.f; };

// what the forward pass leaves for the backward pass
struct Saved {
    float2* norm;      // [rows] M, 1 / sum_j 2^(c z_j - M);  c = log2(e) / T, M = the largest c z_j rounded up
    int* state;        // [rows] RowState
    float* inv_count;  // [1]
    int* ids;          // [rows][top] ascending, each id once, NO_ID behind the last (a target that does not count: NO_ID)
    float* q;          // [rows][top] (distillation)
    float* z;          // [rows][top]
    uint16_t* starts;  // [rows][starts_pitch] distillation: how many ids of the row lie below 128 t
    int64_t starts_pitch;
    float* scores;     // up to FEW_ROWS rows: z of the whole vocabulary, 1 KB a run of 32 ids and 16 rows: lane l's ids run + 4 (l / 16) + {0..3, 16..19}, row l % 16; else NULL
    float* kept;       // fp32, more rows: z [rows][kept_pitch], or NULL
    int64_t kept_pitch;
};

__device__ __forceinline__ int64_t id_at(const void* ids, int bits, int64_t i) {
    return bits == 64 ? ((const int64_t*)ids)[i] : (int64_t)((const int*)ids)[i];
}
struct Targets {       // of the cross entropy, as the caller has them
    const void* ids;
    int bits;
    int64_t pitch, ignore;
};

// The listed ids of a row that fall into a tile's from .. from + size: positions x .. y of its ascending list, from the table beside the list, so
// that no tile searches.  One thread per row looks them up before the tile's products and puts them, with what belongs to the first, into LDS:
// a wave that met them one fragment after the other would wait for each (a row of 64 ids has one in a tile of 50 000 / 256 every third time,
// seldom a second).
__device__ __forceinline__ int2 listed_of(const Saved& s, int64_t n, int from, int size) {
    const uint16_t* at = s.starts + n * s.starts_pitch + (from >> 7);
    return make_int2(at[0], at[size >> 7]);
}

// ---- forward: of a tile's rows M, the largest c z rounded up, and the sum of 2^(c z - M); and the listed z ----------------------------
// Bound by its products; the epilogue of a large tile takes 6 us of exponentials, during which the next tile's first slabs arrive (65536 words, 2048 x
// 1024: 258 us, 1070 TFLOP/s).  M is a whole number: c z - M is one rounding from exact, and sums of different M join by exact powers of two
// (|c z| up to 2^31: beyond 2^24 the largest lies above or below its M by half of M's last place, which 2^x still holds).
template <bool LIST>
struct NormEpi {
    float2* part;      // [rows][tiles_m]
    Saved s;
    Targets targets;   // cross entropy
    int rows, vocab, top;
    float c;           // log2(e) / T
    static constexpr bool ANY_ROW = true;      // reads the caller's rows
    struct Row { int lo, hi, first, none; };
    template <class R> static constexpr int lds() { return R::TILE_N * (int)sizeof(Row) + R::WAVES_M * R::TILE_N * 8; }
    template <class R>
    __device__ __forceinline__ Row ahead(Tile t, int tid) const {
        Row r{};
        if (tid < R::TILE_N) {
            const int n = t.n * R::TILE_N + tid, in = min(n, rows - 1), m0 = t.m * R::TILE_M;
            if constexpr (LIST) {
                const int2 at = listed_of(s, in, m0, R::TILE_M);
                r = {at.x, n < rows ? at.y : at.x, 0, 0};
            } else {
                const int64_t id = id_at(targets.ids, targets.bits, in * targets.pitch);
                r = {0, n < rows && id >= m0 && id < m0 + R::TILE_M ? 1 : 0, (int)id, 0};
            }
        }
        return r;
    }
    template <class R>
    __device__ __forceinline__ void operator()(const Problem& p, Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], Row mine) const {
        static_assert(R::TILE_N <= R::THREADS, "");
        const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / R::WAVES_N, wn = wave % R::WAVES_N;
        const int m0 = t.m * R::TILE_M, n0 = t.n * R::TILE_N;
        Row* info = (Row*)lds;                                           // [TILE_N]
        float2* join = (float2*)(lds + R::TILE_N * sizeof(Row));         // [WAVES_M][TILE_N]
        const int g4 = (lane >> 4) * 4;
        hold<R>(acc, 0);
        if (tid < R::TILE_N) {
            if (LIST && mine.lo < mine.hi) mine.first = s.ids[(int64_t)(n0 + tid) * top + mine.lo];
            info[tid] = mine;
        }
        if (m0 + R::TILE_M > vocab) {                                    // behind the last word
#pragma unroll
            for (int j = 0; j < R::NF; ++j)
#pragma unroll
                for (int i = 0; i < R::MF; ++i) {
                    f32x4 v = take(acc[i][j]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = m0 + R::row0(wm, i) + g4 + r < vocab ? v[r] : -INFINITY;
                    give(acc[i][j], v);
                }
        }
        lds_barrier();
#pragma unroll
        for (int j = 0; j < R::NF; ++j) {
            f32x4 v[R::MF];
            hold<R>(acc, j);
#pragma unroll
            for (int i = 0; i < R::MF; ++i) v[i] = take(acc[i][j]);
            if constexpr (R::TILE_N == 32) {                             // few rows: a lane holds what one of their gradients' products takes
                const int block = (n0 + R::col0(wn, j)) >> 4, blocks = (rows + 15) >> 4;
                if (s.scores && block < blocks) {
                    float* const to = s.scores + ((((int64_t)m0 + R::row0(wm, 0)) >> 5) * blocks + block) * 512 + lane * 8;
                    *(f32x4*)to = v[0];
                    *(f32x4*)(to + 4) = v[1];
                }
            }
            if constexpr (R::KIND_ == FP32 && R::TILE_N != 32) {
                const int n = n0 + R::col0(wn, j) + (lane & 15);
                if (s.kept && n < rows) {
                    float* const to = s.kept + n * s.kept_pitch + m0 + R::row0(wm, 0) + g4;
#pragma unroll
                    for (int i = 0; i < R::MF; ++i) *(f32x4*)(to + i * 16) = v[i];
                }
            }
            float m = -INFINITY, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < R::MF; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = fmaxf(m, v[i][r]);
            m = fmaxf(m, __shfl_xor(m, 16));
            m = ceilf(fmaxf(m, __shfl_xor(m, 32)) * c);
            const float at = m == -INFINITY ? 0.f : m;                   // no value above -inf: the sum is 0, not NaN
#pragma unroll
            for (int i = 0; i < R::MF; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] += __builtin_amdgcn_exp2f(fmaf(v[i][r], c, -at));
            sum[0] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            sum[0] += __shfl_xor(sum[0], 16);
            sum[0] += __shfl_xor(sum[0], 32);
            if (lane < 16) join[wm * R::TILE_N + R::col0(wn, j) + lane] = make_float2(m, sum[0]);
            const Row listed = info[R::col0(wn, j) + (lane & 15)];
            const int64_t row = (int64_t)(n0 + R::col0(wn, j) + (lane & 15)) * top;
            for (int e = listed.lo; e < listed.hi; ++e) {
                const int want = (e == listed.lo ? listed.first : s.ids[row + e]) - m0 - g4;
                float z = 0.f;
                bool here = false;
#pragma unroll
                for (int i = 0; i < R::MF; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (want == R::row0(wm, i) + r) {
                            z = v[i][r];
                            here = true;
                        }
                if (here) s.z[row + e] = z;
            }
        }
        lds_barrier();
        if (tid < R::TILE_N && n0 + tid < rows) {
            float m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < R::WAVES_M; ++w) m = fmaxf(m, join[w * R::TILE_N + tid].x);
            const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < R::WAVES_M; ++w) {
                const float2 v = join[w * R::TILE_N + tid];
                sum += v.x == -INFINITY ? v.y : v.y * __builtin_amdgcn_exp2f(v.x - at);
            }
            part[(int64_t)(n0 + tid) * p.tiles_m + t.m] = make_float2(m, sum);
        }
    }
};

// ---- backward: G = p - q of a piece of the vocabulary, and its transpose ----------------------------------------------------------
// 50000 words, 4096 x 2048: 929 us against 809 us of the same product in the forward pass.
// The listed entries come from the z of the forward pass, p - q in fp32 before the one rounding.  That rounding, in 16 bits, is of the size of the gradients' own:
// bf16, 4096 x 2048, 50000 words, each 1.66e-3 of the gradient (root mean square), both 1.92e-3 (cross entropy, whose targets' values are mostly exact) and
// 2.33e-3 (distillation, sqrt(2) x 1.66e-3).  Two 16-bit parts, as up to 64 rows, would be 4 N V D operations on top of 8.  Both matrices leave through LDS, 16 rows (fp32: 8)
// of a wave's tile at a time, as whole lines and past the caches: see store_tile.
template <class T> struct alignas(4 * sizeof(T)) Four { T v[4]; };
// 4 values rounded to T, or zeros whatever they are where `keep` is 0
template <class T>
__device__ __forceinline__ Four<T> pack(f32x4 v, unsigned keep) {
    if constexpr (sizeof(T) == 2) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef T Tx2 __attribute__((ext_vector_type(2)));
        const uint2 w = make_uint2(__builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){v[0], v[1]}, Tx2)) & keep,
                                   __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){v[2], v[3]}, Tx2)) & keep);
        return __builtin_bit_cast(Four<T>, w);
    } else {
        i32x4 w = __builtin_bit_cast(i32x4, v);
        w &= i32x4{(int)keep, (int)keep, (int)keep, (int)keep};
        return __builtin_bit_cast(Four<T>, w);
    }
}

// SCALED (16 bits, a gradient per row): G^T holds G times the row's factor, rounded once.  A copy of h times the factor would be one rounding more, and
// leaves the range of fp16 where a row's gradient is below 2^-14 of the largest; G, kept times 2^14, has 2^14 more of it.  (4096 x 2048, 50000 words, fp16: the
// backward pass 2.34 ms, as with one gradient for all rows.)
template <int KIND, bool LIST, bool SCALED>
struct GradEpi {
    typedef typename Elem<KIND>::T T;
    T* g;              // [padded rows][pitch_g]
    T* gt;             // [piece][pitch_gt] or NULL
    int64_t pitch_g, pitch_gt;
    Saved s;
    int rows, from, size, top;     // this piece: ids from .. from + size
    float c;
    const float* in_w;             // SCALED
    static constexpr bool ANY_ROW = true;
    // fragment columns that go together: 64 rows are a line of a 16-bit G^T, and all 128 at once do not fit the registers
    template <class R> static constexpr int group() { return R::NF < 4 ? R::NF : 4; }
    template <class R> static constexpr int wave_lds() {
        return Stage<T, (R::TILE_M / R::WAVES_M > 16 * group<R>() ? R::TILE_M / R::WAVES_M : 16 * group<R>())>::BYTES;
    }
    struct alignas(16) Row { float m, inv; unsigned keep; int lo, hi, first; float d, w; };   // keep: 0 for a row that does not count, else ~0; d: G at the first listed id; w: SCALED
    template <class R> static constexpr int lds() { return R::TILE_N * (int)sizeof(Row) + R::WAVES_M * R::WAVES_N * wave_lds<R>(); }
    // p - q of a listed entry
    __device__ __forceinline__ float grad_at(float m, float inv, int64_t entry) const {
        return (__builtin_amdgcn_exp2f(fmaf(s.z[entry], c, -m)) * inv - (LIST ? s.q[entry] : 1.f)) * Elem<KIND>::G_SCALE;
    }
    // staged rows of N elements -> memory
    template <int N>
    __device__ __forceinline__ static void put(const char* stage, T* to, int64_t pitch, int lane) {
        typedef Stage<T, N> S;
        struct alignas(16) Chunk { T v[16 / sizeof(T)]; };               // what was staged as T is read as T
        wave_sync();
#pragma unroll
        for (int r = 0; r < S::ROWS; r += 64 / S::LANES) {
            const int row = r + lane / S::LANES, at = (lane % S::LANES) * 16;
            if (64 / S::LANES <= S::ROWS || row < S::ROWS) __builtin_nontemporal_store(__builtin_bit_cast(i32x4, *(const Chunk*)(stage + S::at(row, at))), (i32x4*)((char*)(to + row * pitch) + at));
        }
        wave_sync();
    }
    template <class R>
    __device__ __forceinline__ Row ahead(Tile t, int tid) const {
        Row r{};
        if (tid < R::TILE_N) {
            const int n = t.n * R::TILE_N + tid, in = min(n, rows - 1), m0 = t.m * R::TILE_M;
            const float2 norm = s.norm[in];
            const int state = n < rows ? s.state[in] : ROW_SKIP;
            int2 at;
            if constexpr (LIST) {
                at = listed_of(s, in, from + m0, R::TILE_M);
            } else {
                r.first = s.ids[in];
                r.d = s.z[in];                                           // z so far
                at = make_int2(0, (unsigned)(r.first - from - m0) < (unsigned)R::TILE_M ? 1 : 0);
            }
            r.m = norm.x;
            r.inv = state == ROW_BAD ? __builtin_nanf("") : norm.y;
            r.keep = state == ROW_SKIP ? 0u : ~0u;
            r.lo = at.x;
            r.hi = state == ROW_COUNT ? at.y : at.x;
            if constexpr (SCALED) r.w = in_w[in];
        }
        return r;
    }
    template <class R>
    __device__ __forceinline__ void operator()(const Problem& p, Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], Row mine) const {
        constexpr int TM = R::TILE_M / R::WAVES_M, JG = group<R>(), TN = 16 * JG;
        static_assert(R::TILE_N <= R::THREADS, "");
        const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / R::WAVES_N, wn = wave % R::WAVES_N;
        const int m0 = t.m * R::TILE_M, n0 = t.n * R::TILE_N, g4 = (lane >> 4) * 4, col = lane & 15;
        Row* info = (Row*)lds;                                           // [TILE_N]
        char* stage = lds + R::TILE_N * sizeof(Row) + wave * wave_lds<R>();
        hold<R>(acc, 0);
        if (tid < R::TILE_N) {
            const int64_t first = (int64_t)(n0 + tid) * top + mine.lo;
            if constexpr (LIST) {
                if (mine.lo < mine.hi) {
                    mine.first = s.ids[first];
                    mine.d = grad_at(mine.m, mine.inv, first);
                }
            } else {
                mine.d = (__builtin_amdgcn_exp2f(fmaf(mine.d, c, -mine.m)) * mine.inv - 1.f) * Elem<KIND>::G_SCALE;
            }
            mine.inv *= Elem<KIND>::G_SCALE;
            info[tid] = mine;
        }
        lds_barrier();
        typedef Stage<T, TM> SG;
        typedef Stage<T, TN> ST;
#pragma unroll
        for (int j0 = 0; j0 < R::NF; j0 += JG) {
            Four<T> packed[R::MF][JG];                                   // for G^T
#pragma unroll
            for (int jj = 0; jj < JG; ++jj) {
                const int j = j0 + jj;
                f32x4 v[R::MF];
                hold<R>(acc, j);
                const Row info_j = info[R::col0(wn, j) + col];
#pragma unroll
                for (int i = 0; i < R::MF; ++i) v[i] = take(acc[i][j]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < R::MF; ++i) v[i][r] = __builtin_amdgcn_exp2f(fmaf(v[i][r], c, -info_j.m));
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < R::MF; ++i) v[i][r] *= info_j.inv;
                const int64_t row = (int64_t)(n0 + R::col0(wn, j) + col) * top;
                for (int e = info_j.lo; e < info_j.hi; ++e) {
                    const int want = (e == info_j.lo ? info_j.first : s.ids[row + e]) - from - m0 - g4;
                    const float d = e == info_j.lo ? info_j.d : grad_at(info_j.m, info_j.inv * (1.f / Elem<KIND>::G_SCALE), row + e);
#pragma unroll
                    for (int i = 0; i < R::MF; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[i][r] = want == R::row0(wm, i) + r ? d : v[i][r];
                }
                T* to = g + (int64_t)(n0 + R::col0(wn, j)) * pitch_g + m0 + R::row0(wm, 0);
#pragma unroll
                for (int i = 0; i < R::MF; ++i) packed[i][jj] = pack<T>(v[i], info_j.keep);
                if (m0 + R::TILE_M > size)                               // behind the piece's last id
#pragma unroll
                    for (int i = 0; i < R::MF; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m0 + R::row0(wm, i) + g4 + r >= size) packed[i][jj].v[r] = (T)0.f;
                Four<T> unscaled[R::MF];
                if constexpr (SCALED) {
#pragma unroll
                    for (int i = 0; i < R::MF; ++i) {
                        unscaled[i] = packed[i][jj];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[i][r] *= info_j.w;
                        packed[i][jj] = pack<T>(v[i], info_j.keep);
                    }
                    if (m0 + R::TILE_M > size)
#pragma unroll
                        for (int i = 0; i < R::MF; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (m0 + R::row0(wm, i) + g4 + r >= size) packed[i][jj].v[r] = (T)0.f;
                }
#pragma unroll
                for (int part = 0; part < 16; part += SG::ROWS) {
#pragma unroll
                    for (int i = 0; i < R::MF; ++i)
                        if (SG::ROWS == 16 || (col & ~(SG::ROWS - 1)) == part) *(Four<T>*)(stage + SG::at(col & (SG::ROWS - 1), (i * 16 + g4) * (int)sizeof(T))) = SCALED ? unscaled[i] : packed[i][jj];
                    put<TM>(stage, to + part * pitch_g, pitch_g, lane);
                }
            }
            if (!gt) continue;
#pragma unroll
            for (int i = 0; i < R::MF; ++i) {
                T* to = gt + (int64_t)(m0 + R::row0(wm, i)) * pitch_gt + n0 + R::col0(wn, j0);
#pragma unroll
                for (int part = 0; part < 16; part += ST::ROWS) {
#pragma unroll
                    for (int j = 0; j < JG; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (ST::ROWS == 16 || (g4 & ~(ST::ROWS - 1)) == part) *(T*)(stage + ST::at((g4 + r) & (ST::ROWS - 1), (j * 16 + col) * (int)sizeof(T))) = packed[i][j].v[r];
                    put<TN>(stage, to + part * pitch_gt, pitch_gt, lane);
                }
            }
        }
    }
};

// fp32: the same from a kept z.  To compute z again costs 7 times the time of its way through memory (width 768: 2 x 768 / 152 TFLOP/s against
// 8 bytes / 5.5 TB/s for each of its values).  In 16 bits (1450 TFLOP/s) it costs as much as that way at a width of about 1050, 3.9 times as much at 4096; z is not
// kept there above 64 rows, whatever the width: it would be twice the size of G, or more.  64 rows x 64 ids a block; 1024 rows, 16384 words: 31 us for 201 MB,
// z partly from the caches, against 232 us of the product.
template <bool LIST>
__global__ __launch_bounds__(256) void kept_grad_kernel(Saved s, int rows, int vocab, int top, float c, float* g, float* gt, int64_t pitch_g, int64_t pitch_gt) {
    __shared__ float tile[64 * 65];                                      // a column's 4 rows of 16 lanes, and 4 columns, on 64 banks
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64, at = threadIdx.x & 15, m = m0 + at * 4;
#pragma unroll
    for (int part = 0; part < 64; part += 16) {
        const int row = part + (threadIdx.x >> 4), n = n0 + row;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        const int state = n < rows ? s.state[n] : ROW_SKIP;
        if (state != ROW_SKIP) {
            const float2 norm = s.norm[n];
            const float inv = state == ROW_BAD ? __builtin_nanf("") : norm.y;
            const f32x4 z = *(const f32x4*)(s.kept + n * s.kept_pitch + m);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_exp2f(fmaf(z[e], c, -norm.x)) * inv;
            if (state == ROW_COUNT) {
                int2 listed = make_int2(0, 1);
                if constexpr (LIST) listed = listed_of(s, n, m0 & ~127, 128);
                for (int e = listed.x; e < listed.y; ++e) {
                    const int64_t entry = (int64_t)n * top + e;
                    const int want = s.ids[entry] - m;
                    const float target = LIST ? s.q[entry] : 1.f;
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] -= want == x ? target : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = m + e < vocab ? v[e] : 0.f;
        }
        *(f32x4*)(g + n * pitch_g + m) = v;
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[row * 65 + at * 4 + e] = v[e];
    }
    if (!gt) return;
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 64; part += 16) {
        const int col = part + (threadIdx.x >> 4);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = tile[(at * 4 + e) * 65 + col];
        *(f32x4*)(gt + (m0 + col) * pitch_gt + n0 + at * 4) = v;
    }
}

// ---- the factor of every row.  dH of row n is hidden(n) (G W)_n; dW sums weight_row(n) G_n h_n and is multiplied by weight().  A gradient per row is
// divided by the largest, so that 16-bit products of it keep their range (row_scale_kernel).  Rows that do not count get 0 by selection.
struct Factors {
    const float *grad, *inv_count;     // one gradient for all rows
    const int* state;
    const float *to_h, *in_w, *w_scale;    // one per row; else NULL
    float f;                           // T / Elem::G_SCALE
    __device__ __forceinline__ float hidden(int64_t n) const { return to_h ? to_h[n] : state[n] != ROW_SKIP ? *grad * *inv_count * f : 0.f; }
    __device__ __forceinline__ float weight_row(int64_t n) const { return in_w ? in_w[n] : state[n] != ROW_SKIP ? 1.f : 0.f; }
    __device__ __forceinline__ float weight() const { return w_scale ? *w_scale : *grad * *inv_count * f; }
};

// ---- dH: fp32 sums over the pieces ------------------------------------------------------------------------------------------------
struct SumEpi {
    static constexpr bool ANY_ROW = false;
    float* out;        // [splits][rows][width]
    int rows, width;
    bool add;
    template <class R> static constexpr int lds() { return stage_bytes<R, float>(); }
    template <class R> __device__ __forceinline__ NoAhead ahead(Tile, int) const { return {}; }
    template <class R>
    __device__ __forceinline__ void operator()(const Problem& p, Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], NoAhead) const {
        store_tile<R>(t, lds, acc, out + (int64_t)t.split * rows * width, width, rows, width, add, [](float v) { return v; });
    }
};

// ---- dW: one rounding ---------------------------------------------------------------------------------------------------------------
template <int KIND>
struct OutEpi {
    static constexpr bool ANY_ROW = false;
    typedef typename Elem<KIND>::T T;
    T* out;            // [rows of n][width]
    int rows, width;
    Factors factors;
    template <class R> static constexpr int lds() { return stage_bytes<R, T>(); }
    template <class R> __device__ __forceinline__ NoAhead ahead(Tile, int) const { return {}; }
    template <class R>
    __device__ __forceinline__ void operator()(const Problem& p, Tile t, char* lds, f32x4 (&acc)[R::MF][R::NF], NoAhead) const {
        const float f = factors.weight();
        store_tile<R>(t, lds, acc, out, width, rows, width, false, [f](float v) { return v * f; });
    }
};

template <int KIND> using AnyMiddle = AnyRow<KIND, 128, 128, 2, 2>;
template <int KIND> using AnyFlat = AnyRow<KIND, 128, 32, 4, 1>;

template <class R, class EPI>
__global__ __launch_bounds__(R::THREADS) void product_kernel(Problem p, EPI epi) {
    __shared__ __attribute__((aligned(1024))) char lds[lds_bytes<R, EPI>()];
    product<R>(p, lds, epi);
}

template <int KIND> using Middle = Ring<KIND, 128, 128, 2, 2, 2>;
template <int KIND> using Flat = Ring<KIND, 128, 32, 4, 1, 4>;

enum Shape { LARGE, MIDDLE, FLAT };
struct ShapeSize { int m, n; };
constexpr ShapeSize SHAPES[3] = {{256, 256}, {128, 128}, {128, 32}};

// Rounds over the 256 CUs, in units of a middle tile's products at full rate.  A large tile runs at that rate; fp32 middle tiles at 0.87 of it, two
// on a CU or one, 16-bit ones at 0.7 and, alone on their CU, at 0.53 (16384 x 4096 with 65..1000 rows: a large tile 943 / 104 us, middle tiles 278 / 50
// us for one on each CU, 536 / 73 us for two).  So 100 rows of a large vocabulary, which leave most of a 256 x 256 tile empty, go to middle
// tiles and 200 go to large ones.  splits: into how many runs of 32 slabs k may be cut, 8 times as many for middle tiles.
Shape shape_for(int64_t m, int64_t n, int size, int64_t splits = 1) {
    if (n <= 64) return FLAT;
    const int64_t tl = ((m + 255) / 256) * ((n + 255) / 256), tm = ((m + 127) / 128) * ((n + 127) / 128);
    int64_t sl = 1, sm = 1;
    if (splits > 1) {
        sl = tl >= 192 ? 1 : CUS / tl < splits ? CUS / tl : splits;
        sm = tm >= 256 ? 1 : (512 + tm - 1) / tm < splits * 8 ? (512 + tm - 1) / tm : splits * 8;
    }
    const double large = 4.0 * (double)((tl * sl + CUS - 1) / CUS) / (double)sl, rounds = (double)((tm * sm + CUS - 1) / CUS) / (double)sm;
    return tm >= MOST_BLOCKS || large <= rounds * (size == 4 ? 1.15 : tm * sm <= CUS ? 1.9 : 1.4) ? LARGE : MIDDLE;
}

struct Cut { int splits, per; };
// k in so many runs that the tiles fill the 256 CUs (large tiles once, small ones twice), of 4 slabs at least
Cut cut_for(int64_t m, int64_t n, int kbytes, Shape sh, int most) {
    const int64_t tiles = ((m + SHAPES[sh].m - 1) / SHAPES[sh].m) * ((n + SHAPES[sh].n - 1) / SHAPES[sh].n);
    const int slabs = (kbytes + 127) / 128;
    int64_t splits = sh == LARGE ? (tiles >= 192 ? 1 : CUS / tiles) : tiles >= 256 ? 1 : (512 + tiles - 1) / tiles;
    if (splits > slabs / 4) splits = slabs / 4;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    const int per = (int)((slabs + splits - 1) / splits);
    return {(slabs + per - 1) / per, per};
}

template <int KIND, class EPI>
int launch_product(hipStream_t st, Shape sh, const Operand& a, const Operand& b, int kbytes, Cut cut, const EPI& epi, bool any_row = false) {
    Problem p{a, b, kbytes, nullptr, nullptr, 0, 0, (int)((a.rows + SHAPES[sh].m - 1) / SHAPES[sh].m), (int)((b.rows + SHAPES[sh].n - 1) / SHAPES[sh].n), cut.splits, cut.per};
    CS_REQUIRE((int64_t)p.tiles_m * p.tiles_n * p.splits < (sh == LARGE ? (int64_t)1 << 30 : MOST_BLOCKS), "head loss: too many tiles");
    if (sh == LARGE && p.kbytes % 128) product_kernel<Wide<KIND, true>, EPI><<<dim3(grid_of<Wide<KIND, true>>(p)), 256, 0, st>>>(p, epi);
    else if (sh == LARGE) product_kernel<Wide<KIND, false>, EPI><<<dim3(grid_of<Wide<KIND, false>>(p)), 256, 0, st>>>(p, epi);
    else if (any_row) {
        if constexpr (EPI::ANY_ROW) {
            if (sh == MIDDLE) product_kernel<AnyMiddle<KIND>, EPI><<<dim3(grid_of<AnyMiddle<KIND>>(p)), 256, 0, st>>>(p, epi);
            else product_kernel<AnyFlat<KIND>, EPI><<<dim3(grid_of<AnyFlat<KIND>>(p)), 256, 0, st>>>(p, epi);
        }
    } else if (sh == MIDDLE) product_kernel<Middle<KIND>, EPI><<<dim3(grid_of<Middle<KIND>>(p)), 256, 0, st>>>(p, epi);
    else product_kernel<Flat<KIND>, EPI><<<dim3(grid_of<Flat<KIND>>(p)), 256, 0, st>>>(p, epi);
    CS_HIP(hipGetLastError());
    return CS_OK;
}

// ---- rows ---------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float teacher_at(const void* p, int type, int64_t i) {
    if (type == CS_TYPE_BF16) return (float)((const __bf16*)p)[i];
    if (type == CS_TYPE_FP16) return (float)((const _Float16*)p)[i];
    return ((const float*)p)[i];
}

// One block per row: q = softmax(teacher / T) and sum q log q in 64 bits, the ids sorted, the mass of an id that comes twice joined.
// Bound by the sort in LDS: 4096 rows of 64 entries 41 us, 16 rows of 16 entries 11 us.
__global__ __launch_bounds__(256) void teacher_rows_kernel(const void* ids, int bits, int64_t ids_pitch, const void* teacher, int type, int64_t teacher_pitch,
                                                           int top, int64_t vocab, double inv_t, double* entropy, Saved s) {
    __shared__ unsigned long long key[KD_MAX_TOP];       // id, place in the row
    __shared__ float mass[KD_MAX_TOP];                   // by place in the row
    __shared__ int head[2][KD_MAX_TOP];                  // how many different ids up to here
    __shared__ double sums[4][2];
    __shared__ float most[4];
    __shared__ int bad;
    const int64_t n = blockIdx.x;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
    int size = 1;
    while (size < top) size *= 2;
    if (tid == 0) bad = 0;
    __syncthreads();
    float m = -INFINITY;
    for (int i = tid; i < size; i += threads) {
        const int64_t id = i < top ? id_at(ids, bits, n * ids_pitch + i) : -1;
        const float l = i < top ? teacher_at(teacher, type, n * teacher_pitch + i) : 0.f;
        const bool live = id >= 0 && l != -INFINITY;
        if (live && id >= vocab) bad = 1;
        key[i] = live ? ((unsigned long long)(id < vocab ? id : vocab) << 32) | (unsigned)i : ~0ull;
        if (i < top) mass[i] = live ? l : -INFINITY;
        if (live) m = fmaxf(m, l);
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    if (lane == 0) most[wave] = m;
    __syncthreads();
    m = most[0];
    for (int w = 1; w < waves; ++w) m = fmaxf(m, most[w]);
    double total = 0.0, cross = 0.0;                     // sum e, sum e log e;  e = exp((l - m) / T)
    for (int i = tid; i < top; i += threads) {
        const float l = mass[i];
        if (l == -INFINITY) continue;
        const double x = ((double)l - (double)m) * inv_t, e = exp(x);
        total += e;
        cross += e > 0.0 ? e * x : e;                    // e log e -> 0 with e
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
        total += __shfl_xor(total, x);
        cross += __shfl_xor(cross, x);
    }
    if (lane == 0) {
        sums[wave][0] = total;
        sums[wave][1] = cross;
    }
    __syncthreads();
    total = cross = 0.0;
    for (int w = 0; w < waves; ++w) {
        total += sums[w][0];
        cross += sums[w][1];
    }
    const bool some = total != 0.0;                      // NaN counts
    if (tid == 0) {
        s.state[n] = bad ? ROW_BAD : some ? ROW_COUNT : ROW_SKIP;
        entropy[n] = some ? cross / total - log(total) : 0.0;
    }
    for (int i = tid; i < top; i += threads) {
        const float l = mass[i];
        mass[i] = l == -INFINITY ? 0.f : (float)(exp(((double)l - (double)m) * inv_t) / total);
    }
    for (int width = 2; width <= size; width *= 2)       // bitonic
        for (int step = width >> 1; step; step >>= 1) {
            __syncthreads();
            for (int i = tid; i < size; i += threads) {
                const int o = i ^ step;
                if (o > i) {
                    const unsigned long long a = key[i], b = key[o];
                    if ((a > b) == ((i & width) == 0)) {
                        key[i] = b;
                        key[o] = a;
                    }
                }
            }
        }
    __syncthreads();
    for (int i = tid; i < size; i += threads) head[0][i] = key[i] != ~0ull && (i == 0 || (key[i - 1] >> 32) != (key[i] >> 32)) ? 1 : 0;
    int from = 0;
    for (int step = 1; step < size; step *= 2, from ^= 1) {
        __syncthreads();
        for (int i = tid; i < size; i += threads) head[from ^ 1][i] = head[from][i] + (i >= step ? head[from][i - step] : 0);
    }
    __syncthreads();
    const int used = head[from][size - 1];
    for (int i = tid; i < size; i += threads) {
        const bool first = key[i] != ~0ull && (i == 0 || (key[i - 1] >> 32) != (key[i] >> 32));
        if (!first) continue;
        float q = 0.f;
        const unsigned id = (unsigned)(key[i] >> 32);
        for (int k = i; k < size && (unsigned)(key[k] >> 32) == id; ++k) q += mass[(unsigned)key[k]];
        const int64_t to = n * top + head[from][i] - 1;
        s.ids[to] = (int64_t)id < vocab ? (int)id : NO_ID;
        s.q[to] = q;
        s.z[to] = 0.f;
    }
    __syncthreads();
    for (int64_t i = tid; i < s.starts_pitch; i += threads) {            // ids below 128 i among the ascending ones: a search of what was just written
        const int64_t below = i * 128;
        int lo = 0, hi = size;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)(key[mid] >> 32) < below) lo = mid + 1;         // a place behind the last has id 2^32 - 1
            else hi = mid;
        }
        s.starts[n * s.starts_pitch + i] = (uint16_t)(lo ? head[from][lo - 1] : 0);
    }
    for (int i = tid; i < top; i += threads)
        if (i >= used) {
            s.ids[n * top + i] = NO_ID;
            s.q[n * top + i] = 0.f;
            s.z[n * top + i] = 0.f;
        }
}

// One row by one wave: joins the tiles' maxima and sums, in 64 bits, into the row's loss -> in lane 0: the loss, and what the backward pass needs
template <bool LIST>
__device__ __forceinline__ double row_loss(int64_t n, int lane, const float2* part, int tiles, int top, int64_t vocab, float c, double t, const double* entropy,
                                           const Targets& targets, const Saved& s, int* counted) {
    const float2* row = part + n * tiles;
    int state;
    if constexpr (LIST) {
        state = s.state[n];
    } else {
        const int64_t id = id_at(targets.ids, targets.bits, n * targets.pitch);
        state = id == targets.ignore ? ROW_SKIP : id >= 0 && id < vocab ? ROW_COUNT : ROW_BAD;
        if (lane == 0) {
            s.state[n] = state;
            s.ids[n] = state == ROW_COUNT ? (int)id : NO_ID;
        }
    }
    float m = -INFINITY;
    for (int i = lane; i < tiles; i += 64) m = fmaxf(m, row[i].x);
#pragma unroll
    for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    const float at = m == -INFINITY ? 0.f : m;
    double sum = 0.0, named = 0.0;
    for (int i = lane; i < tiles; i += 64) {
        const float2 v = row[i];
        sum += v.x == -INFINITY ? (double)v.y : ldexp((double)v.y, (int)fmaxf(v.x - at, -2000.f));
    }
    if constexpr (LIST) {
        for (int i = lane; i < top; i += 64)
            if (s.ids[n * top + i] != NO_ID) {
                const float q = s.q[n * top + i];
                if (q > 0.f || q != q) named += (double)q * (double)s.z[n * top + i];
            }
    } else if (lane == 0 && state == ROW_COUNT) {
        named = (double)s.z[n];
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
        sum += __shfl_xor(sum, x);
        named += __shfl_xor(named, x);
    }
    // in units of 1 / T as the kernels have it, c ln 2
    double loss = t * t * ((LIST ? entropy[n] : 0.0) + log(sum) + ((double)m - named * (double)c) * 0.69314718055994531);
    if (state == ROW_SKIP) loss = 0.0;
    if (state == ROW_BAD) loss = (double)__builtin_nanf("");
    if (lane == 0) s.norm[n] = make_float2(m, (float)(1.0 / sum));
    *counted = state != ROW_SKIP;
    return loss;
}

// the sum over a block's 16 waves, in their order
__device__ __forceinline__ void reduce_block(double sum, int count, bool mean, float* loss, float* inv_count) {
    __shared__ double sums[16];
    __shared__ int counts[16];
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = sum;
        counts[threadIdx.x >> 6] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        count = 0;
        for (int w = 0; w < 16; ++w) {
            sum += sums[w];
            count += counts[w];
        }
        const double inv = mean ? 1.0 / (double)(count > 0 ? count : 1) : 1.0;
        if (loss) *loss = (float)(sum * inv);
        *inv_count = (float)inv;
    }
}

template <bool LIST>
__global__ __launch_bounds__(256) void row_loss_kernel(const float2* part, int tiles, int64_t rows, int top, int64_t vocab, float c, double t, const double* entropy,
                                                       Targets targets, Saved s, double* losses, float* out) {
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= rows) return;
    int counted;
    const double loss = row_loss<LIST>(n, threadIdx.x & 63, part, tiles, top, vocab, c, t, entropy, targets, s, &counted);
    if ((threadIdx.x & 63) == 0) {
        losses[n] = loss;
        if (out) out[n] = (float)loss;
    }
}

// one block: the sum over the rows in a fixed order
__global__ __launch_bounds__(1024) void reduce_loss_kernel(const double* losses, const int* state, int64_t rows, bool mean, float* loss, float* inv_count) {
    double sum = 0.0;
    int count = 0;
    for (int64_t n = threadIdx.x; n < rows; n += 1024) {
        sum += losses[n];
        count += state[n] != ROW_SKIP;
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
        sum += __shfl_xor(sum, x);
        count += __shfl_xor(count, x);
    }
    reduce_block(sum, count, mean, loss, inv_count);
}

// both for few rows, in one launch of one block
template <bool LIST>
__global__ __launch_bounds__(1024) void few_losses_kernel(const float2* part, int tiles, int rows, int top, int64_t vocab, float c, double t, const double* entropy,
                                                          Targets targets, Saved s, float* out, bool mean, float* loss, float* inv_count) {
    double sum = 0.0;
    int count = 0;
    for (int n = threadIdx.x >> 6; n < rows; n += 16) {
        int counted;
        const double one = row_loss<LIST>(n, threadIdx.x & 63, part, tiles, top, vocab, c, t, entropy, targets, s, &counted);
        if (out && (threadIdx.x & 63) == 0) out[n] = (float)one;
        sum += one;
        count += counted;
    }
    reduce_block(sum, count, mean, loss, inv_count);
}

// One block: the factors where every row has a gradient of its own
__global__ __launch_bounds__(1024) void row_scale_kernel(const float* grad, int64_t stride, const int* state, int64_t rows, float f, float* to_h, float* in_w, float* w_scale) {
    __shared__ float most[16];
    const int tid = threadIdx.x;
    float big = 0.f;
    for (int64_t n = tid; n < rows; n += 1024)
        if (state[n] != ROW_SKIP) big = fmaxf(big, fabsf(grad[n * stride]));
#pragma unroll
    for (int x = 32; x; x >>= 1) big = fmaxf(big, __shfl_xor(big, x));
    if ((tid & 63) == 0) most[tid >> 6] = big;
    __syncthreads();
    big = most[0];
    for (int w = 1; w < 16; ++w) big = fmaxf(big, most[w]);
    for (int64_t n = tid; n < rows; n += 1024) {
        const bool live = state[n] != ROW_SKIP;
        const float g = grad[n * stride];
        to_h[n] = live ? g * f : 0.f;
        in_w[n] = !live ? 0.f : big == 0.f ? g : g / big;
    }
    if (tid == 0) *w_scale = (big == 0.f ? 1.f : big) * f;
}

// src [rows][cols] (element pitch) -> dst [cols][pitch], columns of dst behind the rows zero up to `padded`; SCALED: row n times its factor (0 selects 0).
// 16 bytes a lane on both sides (50000 x 2048, 16 bits: 42 us, against 79 us with single values); the tile of 8 x 8 chunks lies in LDS with chunk c of row r at c ^ (r / E), so that a column is read from all banks.
template <class T, bool SCALED>
__global__ __launch_bounds__(256) void transpose_kernel(const T* src, int64_t src_pitch, int64_t rows, int64_t cols, T* dst, int64_t dst_pitch, int64_t padded,
                                                        Factors factors) {
    constexpr int E = 16 / (int)sizeof(T), SIDE = 8 * E, CHUNKS = SIDE * 8;
    struct alignas(16) Chunk { T v[E]; };
    __shared__ Chunk tile[CHUNKS];
    const int64_t r0 = (int64_t)blockIdx.x * SIDE, c0 = (int64_t)blockIdx.y * SIDE;
#pragma unroll
    for (int i = threadIdx.x; i < CHUNKS; i += 256) {
        const int r = i >> 3, ch = i & 7;
        const int64_t row = r0 + r, col = c0 + ch * E;
        Chunk v{};
        if (row < rows && col < cols) {
            const T* from = src + row * src_pitch + col;
            if (col + E <= cols) v = __builtin_bit_cast(Chunk, *(const Loose*)from);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (col + e < cols) v.v[e] = from[e];
            if constexpr (SCALED) {
                const float f = factors.weight_row(row);
                if (f != 1.f)
#pragma unroll
                    for (int e = 0; e < E; ++e) v.v[e] = f == 0.f ? (T)0.f : (T)((float)v.v[e] * f);
            }
        }
        tile[r * 8 + (ch ^ (r / E))] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = threadIdx.x; i < CHUNKS; i += 256) {
        const int c = i >> 3, ch = i & 7;                                // column c, rows ch * E ..
        const int64_t col = c0 + c, row = r0 + ch * E;
        Chunk v;
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[e] = tile[(ch * E + e) * 8 + ((c / E) ^ ch)].v[c % E];
        if (col < cols && row < padded) *(Chunk*)(dst + col * dst_pitch + row) = v;
    }
}

// src [rows][cols] -> dst [rows][pitch] of whole 16 bytes, zeros behind the columns
template <class T>
__global__ __launch_bounds__(256) void copy_rows_kernel(const T* src, int64_t src_pitch, int64_t rows, int64_t cols, T* dst, int64_t pitch) {
    constexpr int E = 16 / (int)sizeof(T);
    struct alignas(16) Chunk { T v[E]; };
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4)          // a wave takes a row
        for (int64_t c = (threadIdx.x & 63) * E; c < pitch; c += 64 * E) {
            const T* from = src + r * src_pitch + c;
            Chunk v{};
            if (c + E <= cols) v = __builtin_bit_cast(Chunk, *(const Loose*)from);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (c + e < cols) v.v[e] = from[e];
            *(Chunk*)(dst + r * pitch + c) = v;
        }
}

// the sums of all runs of k, in their order, times the row's factor; 4 columns a lane
template <class T>
__global__ __launch_bounds__(256) void hidden_grad_kernel(const float* sums, int splits, int64_t rows, int64_t width, Factors factors, T* out) {
    const int64_t n = blockIdx.x, run = rows * width;
    const float f = factors.hidden(n);
    const float* from = sums + n * width;
    for (int64_t c = (int64_t)threadIdx.x * 4; c < width; c += 1024) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        const int left = (int)min((int64_t)4, width - c);
        if (left == 4) {
#pragma unroll 8
            for (int s = 0; s < splits; ++s) v += *(const LooseSum*)(from + s * run + c);
        } else {
            for (int s = 0; s < splits; ++s)
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (e < left) v[e] += from[s * run + c + e];
        }
        T to[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = (T)(f == 0.f ? 0.f : v[e] * f);
        if (left == 4) __builtin_memcpy(out + n * width + c, to, sizeof(to));
        else
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) out[n * width + c + e] = to[e];
    }
}

template <class T>
__global__ __launch_bounds__(256) void zero_kernel(T* out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (T)0.f;
}

// ---- the gradients of few rows -------------------------------------------------------------------------------------------------------------
// Up to 64 rows are bound by the weight's bytes: the forward pass keeps z (no more bytes than the weight), and the weight is read, and its gradient
// written, once more: no transposes, no second product.  G = p - q, kept as the sum of two 16-bit values (with few rows the rounding of one would
// be the largest of the gradient's errors: nothing averages it), costs two instructions where one would do, which the memory hides.
// The order of k inside an instruction is free as long as both operands share it:
//   dH[n][d] = sum_v G[n][v] W[v][d]   k-slot (lane / 16, e) is id 4 (lane / 16) + e, e < 4, and 16 + 4 (lane / 16) + e - 4 of a run of 32 ids: what
//                                      a lane holds of z
//   dW[v][d] = sum_n G[v][n] H[n][d]   k-slot (lane / 16, e) is row 8 (lane / 16) + e of a run of 32
// W and H come straight from memory, 16 bytes of 8 rows a lane, and are turned in registers into one operand per column.
// A piece (1 KB twice) holds, per lane, 8 values: 16 bits: the high parts, the low parts; fp32: four and four.
template <int KIND>
__device__ __forceinline__ void put_piece(char* to, int lane, const float (&v)[8]) {
    typedef typename Elem<KIND>::T T;
    if constexpr (sizeof(T) == 2) {
        struct alignas(16) Chunk { T v[8]; } high, low;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            high.v[e] = (T)v[e];
            low.v[e] = (T)(v[e] - (float)high.v[e]);
        }
        *(Chunk*)(to + lane * 16) = high;
        *(Chunk*)(to + 1024 + lane * 16) = low;
    } else {
        *(f32x4*)(to + lane * 16) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)(to + 1024 + lane * 16) = f32x4{v[4], v[5], v[6], v[7]};
    }
}

// Bound by z and G, 4 + 8 bytes a value; 5 us for 32 rows of 8192 words.  z -> pieces of G for dH, [run of 32 ids][16 rows], and, times the row's factor, for dW, [run of 32 ids][32 rows][16 ids].  A wave takes a run.
template <int KIND, bool LIST>
__global__ __launch_bounds__(256) void few_scores_kernel(Saved s, Factors factors, int rows, int64_t from, int64_t runs, int top, float c, char* g_h, char* g_w) {
    __shared__ float turn[4][32 * 36];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, col = lane & 15, blocks = (rows + 15) >> 4;
    const int64_t run = (int64_t)blockIdx.x * 4 + wave;
    if (run >= runs) return;
    const int64_t id0 = from + run * 32;
    float* const mine = turn[wave];
    for (int b32 = 0; b32 * 2 < blocks; ++b32) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int block = b32 * 2 + j, n = block * 16 + col, in = min(n, rows - 1);
            float v[8] = {};
            if (block < blocks) {
                const float* z = s.scores + ((from >> 5) + run) * blocks * 512 + block * 512 + lane * 8;
                const f32x4 z0 = *(const f32x4*)z, z1 = *(const f32x4*)(z + 4);
                const float2 norm = s.norm[in];
                const int state = n < rows ? s.state[in] : ROW_SKIP;
                const float inv = state == ROW_BAD ? __builtin_nanf("") : norm.y;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_exp2f(fmaf(e < 4 ? z0[e & 3] : z1[e & 3], c, -norm.x)) * inv;
                int2 at = make_int2(0, 1);
                if constexpr (LIST) at = listed_of(s, in, (int)(id0 & ~(int64_t)127), 128);
                if (state != ROW_COUNT) at.y = at.x;
                for (int e = at.x; e < at.y; ++e) {
                    const int64_t entry = (int64_t)in * top + e;
                    const int want = s.ids[entry] - (int)id0;
                    const float target = LIST ? s.q[entry] : 1.f;
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] -= want == (x < 4 ? 0 : 12) + 4 * q + x ? target : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = state == ROW_SKIP ? 0.f : v[e] * Elem<KIND>::G_SCALE;
                if (g_h) put_piece<KIND>(g_h + (run * blocks + block) * 2048, lane, v);
                const float f = n < rows ? factors.weight_row(n) : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = f == 0.f ? 0.f : v[e] * f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mine[((e < 4 ? 0 : 12) + 4 * q + e) * 36 + j * 16 + col] = v[e];
        }
        wave_sync();
        if (g_w)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x4 a = *(const f32x4*)(mine + (i * 16 + col) * 36 + q * 8), b = *(const f32x4*)(mine + (i * 16 + col) * 36 + q * 8 + 4);
                const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                put_piece<KIND>(g_w + ((run * ((blocks + 1) >> 1) + b32) * 2 + i) * 2048, lane, v);
            }
        wave_sync();
    }
}

// 8 rows of 16 bytes -> one operand of 8 values per column
template <int KIND> struct Turned;
template <int KIND>
struct Turned16 {
    static constexpr int COLS = 8;
    i32x4 v[8];
    __device__ __forceinline__ void set(const i32x4 (&r)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = (int)__builtin_amdgcn_perm((unsigned)r[2 * e + 1][j >> 1], (unsigned)r[2 * e][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
    }
    // sum += (high + low) x column j
    __device__ __forceinline__ f32x4 times(i32x4 high, i32x4 low, int j, f32x4 sum) const {
        return mma<KIND, 0>(low, v[j], mma<KIND, 0>(high, v[j], sum, 0, 0), 0, 0);
    }
};
template <> struct Turned<BF16> : Turned16<BF16> {};
template <> struct Turned<FP16> : Turned16<FP16> {};
template <>
struct Turned<FP32> {
    static constexpr int COLS = 4;
    i32x4 v[8];
    __device__ __forceinline__ void set(const i32x4 (&r)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r[e];
    }
    __device__ __forceinline__ f32x4 times(i32x4 a, i32x4 b, int j, f32x4 sum) const {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(e < 4 ? x[e & 3] : y[e & 3], __builtin_bit_cast(f32x4, v[e])[j], sum, 0, 0, 0);
        return sum;
    }
};

// past the caches, unless rows start anywhere: their lines are then written in parts, which the caches join (4 rows, 123517 x 1311, bf16: a step
// 341 us past the caches, 313 us through them; 65536 x 2048: 172 and 183 us)
__device__ __forceinline__ void store_line(i32x4 v, void* to, bool aligned) {
    if (aligned) {                                                       // the compiler would join both stores into one through the caches
        asm volatile("; past the caches");
        __builtin_nontemporal_store(v, (Loose*)to);
        asm volatile("; are the whole lines");
    } else {
        asm volatile("; through the caches");
        *(Loose*)to = v;
        asm volatile("; are the parts");
    }
}

struct FewGrads {
    const char *hidden, *weight;           // of the first id here
    int64_t hidden_pitch, weight_pitch;    // bytes, any
    const char *g_h, *g_w;                 // pieces, NULL where that gradient is not wanted
    float* sums;                           // [splits][rows][width] of dH
    char* out;                             // dW of the first id here, rows of `width`
    int rows, width, groups, splits;
    int64_t ids, runs, runs_per_split;
    bool add;
    Factors factors;
};

// A wave takes 16 bytes of 16 lanes = 256 bytes of columns and a run of ids; the four waves of a block lie side by side and share G in the caches,
// the blocks of one run of ids lie in one XCD.  65536 x 2048, bf16, 16 rows: about 110 us for the 537 MB that are read and written (4.9 TB/s).  Behind the last column a lane
// computes the last whole 16 bytes again: of dW it stores the same values, of the sums of dH only the columns that no other lane has.
template <int KIND, int BLOCKS>
__global__ __launch_bounds__(256, BLOCKS == 1 ? 2 : 1) void few_grads_kernel(FewGrads p) {
    typedef typename Elem<KIND>::T T;
    typedef Turned<KIND> Op;
    constexpr int COLS = Op::COLS, PAIRS = (BLOCKS + 1) / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, col = lane & 15;
    const int id = blockIdx.x, split = (id / (8 * p.groups)) * 8 + id % 8, chunk = (id / 8 % p.groups) * 4 + wave;
    if (split >= p.splits || chunk * 16 * COLS >= p.width) return;
    const int d = min((chunk * 16 + col) * COLS, p.width - COLS);
    const int64_t first = split * p.runs_per_split, last = min(first + p.runs_per_split, p.runs) - 1;
    Op h[PAIRS];
    if (p.g_w) {
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
            i32x4 r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int n = k * 32 + q * 8 + e, in = min(n, p.rows - 1);
                const bool counts = p.factors.in_w ? p.factors.in_w[in] != 0.f : p.factors.state[in] != ROW_SKIP;
                const int keep = n < p.rows && counts ? ~0 : 0;
                r[e] = *(const Loose*)(p.hidden + in * p.hidden_pitch + (int64_t)d * sizeof(T)) & i32x4{keep, keep, keep, keep};
            }
            h[k].set(r);
        }
    }
    f32x4 sum[BLOCKS][COLS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int j = 0; j < COLS; ++j) sum[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float f = p.g_w ? p.factors.weight() : 0.f;
    i32x4 next[8];
    auto load = [&](int64_t run) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t v = min(run * 32 + (e < 4 ? 0 : 12) + 4 * q + e, p.ids - 1);
            next[e] = *(const Loose*)(p.weight + v * p.weight_pitch + (int64_t)d * sizeof(T));
        }
    };
    if (p.g_h) load(first);
#pragma unroll 1
    for (int64_t run = first; run <= last; ++run) {
        i32x4 gh[BLOCKS][2], gw[PAIRS][2][2];
        if (p.g_w)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x) gw[k][i][x] = *(const i32x4*)(p.g_w + ((run * PAIRS + k) * 2 + i) * 2048 + x * 1024 + lane * 16);
        if (p.g_h) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int x = 0; x < 2; ++x) gh[b][x] = *(const i32x4*)(p.g_h + (run * BLOCKS + b) * 2048 + x * 1024 + lane * 16);
            Op w;
            w.set(next);
            load(min(run + 1, last));
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int j = 0; j < COLS; ++j) sum[b][j] = w.times(gh[b][0], gh[b][1], j, sum[b][j]);
        }
        if (p.g_w)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f32x4 dw[COLS];
#pragma unroll
                for (int j = 0; j < COLS; ++j) {
                    dw[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) dw[j] = h[k].times(gw[k][i][0], gw[k][i][1], j, dw[j]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    struct alignas(16) Chunk { T v[COLS]; } to;
#pragma unroll
                    for (int j = 0; j < COLS; ++j) to.v[j] = (T)(dw[j][r] * f);
                    const int64_t v = run * 32 + i * 16 + q * 4 + r;
                    if (v < p.ids) store_line(__builtin_bit_cast(i32x4, to), p.out + (v * p.width + d) * (int64_t)sizeof(T), p.width * sizeof(T) % 16 == 0);
                }
            }
    }
    if (!p.g_h) return;
    const int others = (chunk * 16 + col) * COLS - d;                    // how many of this lane's columns are another lane's: each is added to once
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = b * 16 + q * 4 + r;
            if (n >= p.rows) continue;
            float* to = p.sums + ((int64_t)split * p.rows + n) * p.width + d;
#pragma unroll
            for (int j = 0; j < COLS; j += 4) {
                f32x4 v = {sum[b][j][r], sum[b][j + 1][r], sum[b][j + 2][r], sum[b][j + 3][r]};
                if (j >= others) {
                    if (p.add) v += *(const LooseSum*)(to + j);
                    *(LooseSum*)(to + j) = v;
                } else {
#pragma unroll
                    for (int e = 1; e < 4; ++e)
                        if (j + e >= others) to[j + e] = p.add ? to[j + e] + v[e] : v[e];
                }
            }
        }
}

// the sums of all runs of ids, 16 waves a block, 64 columns of a row
template <class T>
__global__ __launch_bounds__(1024) void few_hidden_kernel(const float* sums, int splits, int64_t rows, int64_t width, Factors factors, T* out) {
    __shared__ float part[16][64];
    const int64_t n = blockIdx.y, c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), run = rows * width;
    const int group = threadIdx.x >> 6;
    float v = 0.f;
    if (c < width)
#pragma unroll 4
        for (int s = group; s < splits; s += 16) v += sums[s * run + n * width + c];
    part[group][threadIdx.x & 63] = v;
    __syncthreads();
    if (group || c >= width) return;
#pragma unroll
    for (int g = 1; g < 16; ++g) v += part[g][threadIdx.x];
    const float f = factors.hidden(n);
    out[n * width + c] = (T)(f == 0.f ? 0.f : v * f);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
struct Arena {
    char* base;
    size_t at = 0;
    template <class T> T* take(size_t count) {
        T* p = base ? (T*)(base + at) : nullptr;
        at += (count * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
};
constexpr int64_t PIECE_BYTES = (int64_t)512 << 20;      // of G
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int type_bytes(int type) { return type == CS_TYPE_FP32 ? 4 : 2; }

// whether the forward pass keeps z and few_grads_kernel makes the gradients: few rows, and z takes no more than the weight
bool few(const cs_head_loss& h) {
    const int size = type_bytes(h.type);
    return h.keep_scores && h.rows && h.rows <= FEW_ROWS && h.width * size >= 16 && up(h.rows, 16) * 4 <= h.width * size;
}

// whether the forward pass keeps z whole in fp32: where it is one piece of G, which the backward pass makes room for anyway
bool kept(const cs_head_loss& h) {
    return h.keep_scores && h.type == CS_TYPE_FP32 && h.rows > FEW_ROWS && up(h.rows, 256) * up(h.vocab, 256) * 4 <= PIECE_BYTES;
}

Saved carve_saved(const cs_head_loss& h, void* base, size_t* bytes) {
    Arena a{(char*)base};
    Saved s;
    const size_t n = (size_t)h.rows, k = (size_t)h.top;
    s.norm = a.take<float2>(n);
    s.state = a.take<int>(n);
    s.inv_count = a.take<float>(1);
    s.ids = a.take<int>(n * k);
    s.z = a.take<float>(n * k);
    const bool kd = h.kind == CS_HEAD_DISTILLATION;
    s.q = a.take<float>(kd ? n * k : 0);
    s.starts_pitch = (h.vocab + 255) / 256 * 2 + 1;
    s.starts = a.take<uint16_t>(kd ? n * (size_t)s.starts_pitch : 0);
    if (!kd) s.starts = nullptr;
    s.scores = few(h) ? a.take<float>((size_t)(up(h.vocab, 128) * up(h.rows, 16))) : nullptr;
    s.kept_pitch = up(h.vocab, 256) + 32;
    s.kept = kept(h) ? a.take<float>((size_t)(h.rows * s.kept_pitch)) : nullptr;
    *bytes = a.at;
    return s;
}

// whether the product can read an operand where it lies
bool in_place(const void* p, int64_t pitch, int64_t width, int size) {
    return ((uintptr_t)p & 15) == 0 && (pitch * size) % 16 == 0 && (width * size) % 16 == 0 && pitch * size < ((int64_t)1 << 25);
}

struct Plan {
    size_t bytes;
    char *hidden, *weight;                 // padded copies, NULL where the tensor is read in place
    bool any_row;                          // both are read in place whatever their alignment
    int64_t hidden_pitch, weight_pitch;    // bytes
    float2* part;
    double *losses, *entropy;
    int64_t padded, piece;                 // rows and vocabulary of a piece, rounded up to 256
    // elements between the rows of G, W^T (piece_pitch), G^T and H^T (row_pitch): 128 bytes more than the rows, since rows a power of two apart
    // meet in few memory channels (a product over 65 536-byte rows: 1100 instead of 1450 TFLOP/s)
    int64_t piece_pitch, row_pitch;
    Cut cut;                               // of the sums of dH over the first piece; a shorter last piece adds to fewer of them
    Shape dh_shape;
    char *g, *gt, *wt, *ht;
    float *sums, *to_h, *in_w, *w_scale;
    int64_t runs, runs_per_split;          // few rows: of 32 ids, in a piece and for a block; blocks side by side and along the ids
    int groups, splits;
};

Plan make_plan(const cs_head_loss& h, int backward, void* base) {
    Plan p{};
    Arena a{(char*)base};
    const int size = type_bytes(h.type);
    const int64_t width_pitch = up(h.width * size, 128);
    bool hin = in_place(h.hidden, h.hidden_pitch, h.width, size), win = in_place(h.weight, h.weight_pitch, h.width, size);
    p.hidden_pitch = hin ? h.hidden_pitch * size : width_pitch;
    p.weight_pitch = win ? h.weight_pitch * size : width_pitch;
    if (backward && few(h)) {
        const int64_t runs = up(h.vocab, 32) / 32, run_bytes = up(h.rows, 16) * 128, most = PIECE_BYTES / run_bytes / 4 * 4;
        const int blocks = (int)(up(h.rows, 16) / 16);
        p.runs = runs < most ? runs : most;
        p.groups = (int)((h.width * size + 1023) / 1024);
        const int64_t want = blocks == 1 ? 2 * CUS : CUS;                // blocks that run at a time; 4 runs of ids at least
        int64_t splits = p.groups < want ? want / p.groups : 1;
        if (splits > p.runs / 4) splits = p.runs / 4 > 0 ? p.runs / 4 : 1;
        p.runs_per_split = (p.runs + splits - 1) / splits;
        p.splits = (int)((p.runs + p.runs_per_split - 1) / p.runs_per_split);
        p.to_h = a.take<float>((size_t)h.rows);
        p.in_w = a.take<float>((size_t)h.rows);
        p.w_scale = a.take<float>(1);
        if (backward & 1) {
            p.g = a.take<char>((size_t)(p.runs * run_bytes));
            p.sums = a.take<float>((size_t)p.splits * h.rows * h.width);
        }
        if (backward & 2) p.gt = a.take<char>((size_t)(p.runs * up(h.rows, 32) * 128));
        p.bytes = a.at;
        return p;
    }
    const bool products = !backward || !kept(h);           // of hidden and weight themselves
    // a weight whose rows start anywhere is read as it lies where it is read once (one column of tiles) or the products take long anyway (fp32);
    // else it is copied (50001 x 777, bf16, the forward pass of 100 rows: 46 us against 57 copied, of 300 rows: 99 against 83)
    int64_t some = backward && h.rows ? PIECE_BYTES / (up(h.rows, 256) * size) / 256 * 256 : h.vocab;     // words of a product
    if (some < 256) some = 256;
    if (some > h.vocab) some = h.vocab;
    if (products && !win && h.rows && (h.rows <= 128 || size == 4) && shape_for(some, h.rows, size) != LARGE && h.hidden_pitch * size < (int64_t)1 << 40 && h.weight_pitch * size < (int64_t)1 << 32) {
        p.any_row = hin = win = true;
        p.hidden_pitch = h.hidden_pitch * size;
        p.weight_pitch = h.weight_pitch * size;
    }
    if (!hin && products) p.hidden = a.take<char>((size_t)(h.rows * width_pitch));
    if (!win && products) p.weight = a.take<char>((size_t)(h.vocab * width_pitch));
    if (!backward) {
        const Shape sh = shape_for(h.vocab, h.rows, size);
        p.part = a.take<float2>((size_t)(h.rows * ((h.vocab + SHAPES[sh].m - 1) / SHAPES[sh].m)));
        p.losses = a.take<double>((size_t)h.rows);
        p.entropy = a.take<double>((size_t)(h.kind == CS_HEAD_DISTILLATION ? h.rows : 0));
    } else if (h.rows) {
        p.padded = up(h.rows, 256);
        p.piece = PIECE_BYTES / (p.padded * size) / 256 * 256;
        if (p.piece < 256) p.piece = 256;
        if (p.piece > up(h.vocab, 256)) p.piece = up(h.vocab, 256);
        p.piece_pitch = p.piece + 128 / size;
        p.row_pitch = p.padded + 128 / size;
        p.g = a.take<char>((size_t)(p.padded * p.piece_pitch * size));
        p.to_h = a.take<float>((size_t)h.rows);
        p.in_w = a.take<float>((size_t)h.rows);
        p.w_scale = a.take<float>(1);
        if (backward & 1) {
            const int kbytes = (int)((p.piece < h.vocab ? p.piece : up(h.vocab, 64)) * size);
            p.dh_shape = shape_for(h.width, h.rows, size, kbytes / 128 / 32);  // runs of 32 slabs at least for large tiles
            p.cut = cut_for(h.width, h.rows, kbytes, p.dh_shape, 64);
            p.wt = a.take<char>((size_t)(h.width * p.piece_pitch * size));
            p.sums = a.take<float>((size_t)p.cut.splits * h.rows * h.width);
        }
        if (backward & 2) {
            p.gt = a.take<char>((size_t)(p.piece * p.row_pitch * size));
            p.ht = a.take<char>((size_t)(h.width * p.row_pitch * size));
        }
    }
    p.bytes = a.at;
    return p;
}

template <class T>
void copy_rows(hipStream_t st, const void* src, int64_t pitch, int64_t rows, int64_t cols, void* dst, int64_t dst_pitch_bytes) {
    copy_rows_kernel<T><<<dim3((unsigned)(rows < (1 << 22) ? (rows + 3) / 4 : 1 << 20)), 256, 0, st>>>((const T*)src, pitch, rows, cols, (T*)dst, dst_pitch_bytes / (int64_t)sizeof(T));
}
template <class T, bool SCALED>
void transpose(hipStream_t st, const void* src, int64_t pitch, int64_t rows, int64_t cols, void* dst, int64_t dst_pitch, int64_t padded, const Factors& factors) {
    constexpr int SIDE = 128 / (int)sizeof(T);
    transpose_kernel<T, SCALED><<<dim3((unsigned)((padded + SIDE - 1) / SIDE), (unsigned)((cols + SIDE - 1) / SIDE)), 256, 0, st>>>((const T*)src, pitch, rows, cols, (T*)dst,
                                                                                                                                   dst_pitch, padded, factors);
}

int check_head(const cs_head_loss* h) {
    CS_REQUIRE(h, "head loss: NULL descriptor");
    CS_REQUIRE(h->rows >= 0 && h->rows < MOST_BLOCKS && h->vocab >= 1 && h->vocab < (int64_t)1 << 30 && h->width >= 1 && h->width < (int64_t)1 << 21,
               "head loss: rows %lld, vocab %lld, width %lld out of range", (long long)h->rows, (long long)h->vocab, (long long)h->width);
    CS_REQUIRE(h->type >= CS_TYPE_BF16 && h->type <= CS_TYPE_FP32, "head loss: unknown type %d", h->type);
    CS_REQUIRE(h->kind == CS_HEAD_CROSS_ENTROPY || h->kind == CS_HEAD_DISTILLATION, "head loss: unknown kind %d", h->kind);
    CS_REQUIRE(h->reduction >= CS_REDUCE_NONE && h->reduction <= CS_REDUCE_SUM, "head loss: unknown reduction %d", h->reduction);
    CS_REQUIRE(h->ids_bits == 32 || h->ids_bits == 64, "head loss: ids of %d bits", h->ids_bits);
    if (h->kind == CS_HEAD_DISTILLATION) {
        CS_REQUIRE(h->top >= 1 && h->top <= KD_MAX_TOP, "head loss: %d teacher logits per row: 1..%d are supported", h->top, KD_MAX_TOP);
        CS_REQUIRE(h->teacher_type >= CS_TYPE_BF16 && h->teacher_type <= CS_TYPE_FP32, "head loss: unknown teacher type %d", h->teacher_type);
        CS_REQUIRE(h->temperature >= MIN_TEMPERATURE && h->temperature < 1e30, "head loss: temperature %g: %g and more are supported", h->temperature, MIN_TEMPERATURE);
    } else {
        CS_REQUIRE(h->top == 1 && h->temperature == 1.0, "head loss: the cross entropy has top = 1 and temperature = 1");
    }
    CS_REQUIRE(h->hidden_pitch >= h->width || h->rows <= 1, "head loss: hidden rows overlap (pitch %lld < width %lld)", (long long)h->hidden_pitch, (long long)h->width);
    CS_REQUIRE(h->weight_pitch >= h->width || h->vocab <= 1, "head loss: weight rows overlap (pitch %lld < width %lld)", (long long)h->weight_pitch, (long long)h->width);
    return CS_OK;
}

template <int KIND>
int forward(const cs_head_loss& h, const Plan& p, const Saved& s, float* row_losses, float* loss, hipStream_t st) {
    typedef typename Elem<KIND>::T T;
    const int size = sizeof(T);
    const bool kd = h.kind == CS_HEAD_DISTILLATION;
    if (h.rows) {
        const Targets targets{h.ids, h.ids_bits, h.ids_pitch, h.ignore_index};
        if (kd) {
            const int threads = h.top <= 64 ? 64 : h.top <= 128 ? 128 : 256;
            teacher_rows_kernel<<<dim3((unsigned)h.rows), threads, 0, st>>>(h.ids, h.ids_bits, h.ids_pitch, h.teacher, h.teacher_type, h.teacher_pitch, h.top, h.vocab,
                                                                           1.0 / h.temperature, p.entropy, s);
        }
        if (p.hidden) copy_rows<T>(st, h.hidden, h.hidden_pitch, h.rows, h.width, p.hidden, p.hidden_pitch);
        if (p.weight) copy_rows<T>(st, h.weight, h.weight_pitch, h.vocab, h.width, p.weight, p.weight_pitch);
        const Operand a{p.weight ? p.weight : (const char*)h.weight, p.weight_pitch, h.vocab}, b{p.hidden ? p.hidden : (const char*)h.hidden, p.hidden_pitch, h.rows};
        const int kbytes = (int)(p.hidden || p.weight ? up(h.width * size, 16) : h.width * size);
        const float c = (float)(1.4426950408889634 / h.temperature);
        const Shape sh = shape_for(h.vocab, h.rows, size);
        const int tiles = (int)((h.vocab + SHAPES[sh].m - 1) / SHAPES[sh].m);
        const Cut whole{1, (kbytes + 127) / 128};
        if (int rc = kd ? launch_product<KIND>(st, sh, a, b, kbytes, whole, NormEpi<true>{p.part, s, targets, (int)h.rows, (int)h.vocab, h.top, c}, p.any_row)
                        : launch_product<KIND>(st, sh, a, b, kbytes, whole, NormEpi<false>{p.part, s, targets, (int)h.rows, (int)h.vocab, h.top, c}, p.any_row))
            return rc;
        const bool mean = h.reduction == CS_REDUCE_MEAN;
        if (h.rows <= FEW_ROWS) {
            if (kd) few_losses_kernel<true><<<1, 1024, 0, st>>>(p.part, tiles, (int)h.rows, h.top, h.vocab, c, h.temperature, p.entropy, targets, s, row_losses, mean, loss, s.inv_count);
            else few_losses_kernel<false><<<1, 1024, 0, st>>>(p.part, tiles, (int)h.rows, h.top, h.vocab, c, h.temperature, p.entropy, targets, s, row_losses, mean, loss, s.inv_count);
            CS_HIP(hipGetLastError());
            return CS_OK;
        }
        const dim3 grid((unsigned)((h.rows + 3) / 4));
        if (kd) row_loss_kernel<true><<<grid, 256, 0, st>>>(p.part, tiles, h.rows, h.top, h.vocab, c, h.temperature, p.entropy, targets, s, p.losses, row_losses);
        else row_loss_kernel<false><<<grid, 256, 0, st>>>(p.part, tiles, h.rows, h.top, h.vocab, c, h.temperature, p.entropy, targets, s, p.losses, row_losses);
        if (h.reduction == CS_REDUCE_NONE) {                             // nothing to reduce: the backward pass has a gradient per row
            CS_HIP(hipGetLastError());
            return CS_OK;
        }
    }
    reduce_loss_kernel<<<1, 1024, 0, st>>>(p.losses, s.state, h.rows, h.reduction == CS_REDUCE_MEAN, loss, s.inv_count);
    CS_HIP(hipGetLastError());
    return CS_OK;
}

template <int KIND>
int backward(const cs_head_loss& h, const Plan& p, const Saved& s, const float* grad, int64_t grad_stride, void* gh, void* gw, hipStream_t st) {
    typedef typename Elem<KIND>::T T;
    const int size = sizeof(T);
    if (!h.rows) {
        if (gw) zero_kernel<T><<<1024, 256, 0, st>>>((T*)gw, h.vocab * h.width);
        CS_HIP(hipGetLastError());
        return CS_OK;
    }
    const bool kd = h.kind == CS_HEAD_DISTILLATION;
    const float c = (float)(1.4426950408889634 / h.temperature);
    Factors factors{grad, s.inv_count, s.state, nullptr, nullptr, nullptr, (float)(h.temperature / (double)Elem<KIND>::G_SCALE)};
    if (h.reduction == CS_REDUCE_NONE) {
        row_scale_kernel<<<1, 1024, 0, st>>>(grad, grad_stride, s.state, h.rows, factors.f, p.to_h, p.in_w, p.w_scale);
        factors.to_h = p.to_h, factors.in_w = p.in_w, factors.w_scale = p.w_scale;
    }
    if (s.scores) {
        for (int64_t from = 0; from < h.vocab; from += p.runs * 32) {
            const int64_t len = h.vocab - from < p.runs * 32 ? h.vocab - from : p.runs * 32, runs = (len + 31) / 32;
            const dim3 scores_grid((unsigned)((runs + 3) / 4));
            char *const g_h = gh ? p.g : nullptr, *const g_w = gw ? p.gt : nullptr;
            if (kd) few_scores_kernel<KIND, true><<<scores_grid, 256, 0, st>>>(s, factors, (int)h.rows, from, runs, h.top, c, g_h, g_w);
            else few_scores_kernel<KIND, false><<<scores_grid, 256, 0, st>>>(s, factors, (int)h.rows, from, runs, h.top, c, g_h, g_w);
            const FewGrads few{(const char*)h.hidden, (const char*)h.weight + from * h.weight_pitch * size, h.hidden_pitch * size, h.weight_pitch * size, g_h, g_w, p.sums,
                               (char*)gw + from * h.width * size, (int)h.rows, (int)h.width, p.groups, (int)((runs + p.runs_per_split - 1) / p.runs_per_split), len, runs,
                               p.runs_per_split, from != 0, factors};
            const dim3 grid((unsigned)(up(few.splits, 8) * p.groups));
            if (h.rows <= 16) few_grads_kernel<KIND, 1><<<grid, 256, 0, st>>>(few);
            else if (h.rows <= 32) few_grads_kernel<KIND, 2><<<grid, 256, 0, st>>>(few);
            else if (h.rows <= 48) few_grads_kernel<KIND, 3><<<grid, 256, 0, st>>>(few);
            else few_grads_kernel<KIND, 4><<<grid, 256, 0, st>>>(few);
        }
        if (gh) few_hidden_kernel<T><<<dim3((unsigned)((h.width + 63) / 64), (unsigned)h.rows), 1024, 0, st>>>(p.sums, p.splits, h.rows, h.width, factors, (T*)gh);
        CS_HIP(hipGetLastError());
        return CS_OK;
    }
    if (p.hidden) copy_rows<T>(st, h.hidden, h.hidden_pitch, h.rows, h.width, p.hidden, p.hidden_pitch);
    if (p.weight) copy_rows<T>(st, h.weight, h.weight_pitch, h.vocab, h.width, p.weight, p.weight_pitch);
    const int kbytes = (int)(p.hidden || p.weight ? up(h.width * size, 16) : h.width * size);
    const bool scaled = KIND != nt::FP32 && gw && factors.in_w;         // the row's factor is in G^T, else in the copy of h
    Factors of_h = factors;
    if (scaled) of_h.in_w = nullptr;
    if (gw) transpose<T, true>(st, h.hidden, h.hidden_pitch, h.rows, h.width, p.ht, p.row_pitch, up(h.rows, 32), of_h);
    for (int64_t from = 0; from < h.vocab; from += p.piece) {
        const int64_t len = h.vocab - from < p.piece ? h.vocab - from : p.piece, klen = up(len, 64);
        const Operand a{(p.weight ? p.weight : (const char*)h.weight) + from * p.weight_pitch, p.weight_pitch, len};
        const Operand b{p.hidden ? p.hidden : (const char*)h.hidden, p.hidden_pitch, h.rows};
        const Cut whole{1, (kbytes + 127) / 128};
        T* const g = (T*)p.g;
        T* const gt = gw ? (T*)p.gt : nullptr;
        const Shape sh = p.any_row && h.rows > 64 ? MIDDLE : shape_for(len, h.rows, size);
        if (s.kept) {
            const dim3 grid((unsigned)((len + 63) / 64), (unsigned)((h.rows + 63) / 64));
            if (kd) kept_grad_kernel<true><<<grid, 256, 0, st>>>(s, (int)h.rows, (int)len, h.top, c, (float*)g, (float*)gt, p.piece_pitch, p.row_pitch);
            else kept_grad_kernel<false><<<grid, 256, 0, st>>>(s, (int)h.rows, (int)len, h.top, c, (float*)g, (float*)gt, p.piece_pitch, p.row_pitch);
        } else {
            auto grads = [&](auto list, auto with_factor) {
                return launch_product<KIND>(st, sh, a, b, kbytes, whole, GradEpi<KIND, list.value, with_factor.value>{g, gt, p.piece_pitch, p.row_pitch, s, (int)h.rows, (int)from, (int)len, h.top, c,
                                                                                                                      factors.in_w}, p.any_row);
            };
            int rc;
            if constexpr (KIND != nt::FP32) {
                if (scaled) rc = kd ? grads(std::true_type(), std::true_type()) : grads(std::false_type(), std::true_type());
                else rc = kd ? grads(std::true_type(), std::false_type()) : grads(std::false_type(), std::false_type());
            } else {
                rc = kd ? grads(std::true_type(), std::false_type()) : grads(std::false_type(), std::false_type());
            }
            if (rc) return rc;
        }
        if (gh) {
            transpose<T, false>(st, (const T*)h.weight + from * h.weight_pitch, h.weight_pitch, len, h.width, p.wt, p.piece_pitch, klen, factors);
            const int kb = (int)(klen * size), slabs = (kb + 127) / 128;
            const Cut cut{(slabs + p.cut.per - 1) / p.cut.per, p.cut.per};
            const SumEpi epi{p.sums, (int)h.rows, (int)h.width, from != 0};
            if (int rc = launch_product<KIND>(st, p.dh_shape, Operand{p.wt, p.piece_pitch * size, h.width}, Operand{p.g, p.piece_pitch * size, h.rows}, kb, cut, epi)) return rc;
        }
        if (gw) {
            const int kb = (int)(up(h.rows, 32) * size);
            const OutEpi<KIND> epi{(T*)gw + from * h.width, (int)len, (int)h.width, factors};
            if (int rc = launch_product<KIND>(st, shape_for(h.width, len, size), Operand{p.ht, p.row_pitch * size, h.width}, Operand{p.gt, p.row_pitch * size, len}, kb,
                                              Cut{1, (kb + 127) / 128}, epi))
                return rc;
        }
    }
    if (gh) hidden_grad_kernel<T><<<dim3((unsigned)h.rows), 256, 0, st>>>(p.sums, p.cut.splits, h.rows, h.width, factors, (T*)gh);
    CS_HIP(hipGetLastError());
    return CS_OK;
}

}  // namespace
}  // namespace cs

extern "C" {
using namespace cs;

size_t cs_head_loss_saved_bytes(const cs_head_loss* h) {
    if (check_head(h) != CS_OK) return 0;
    size_t bytes;
    carve_saved(*h, nullptr, &bytes);
    return bytes;
}

size_t cs_head_loss_workspace_bytes(const cs_head_loss* h, int backward) {
    if (check_head(h) != CS_OK) return 0;
    return make_plan(*h, backward, nullptr).bytes;
}

int cs_head_loss_forward(const cs_head_loss* h, float* row_losses, float* loss, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_head(h)) return rc;
    CS_REQUIRE((h->hidden || !h->rows) && h->weight && (h->ids || !h->rows) && (h->teacher || !h->rows || h->kind == CS_HEAD_CROSS_ENTROPY) && saved && workspace,
               "head loss: NULL pointer");
    size_t need;
    const Saved s = carve_saved(*h, saved, &need);
    const Plan p = make_plan(*h, 0, workspace);
    if (saved_bytes < need || workspace_bytes < p.bytes) {
        set_error("head loss: workspace of %zu / %zu bytes, %zu / %zu are needed", saved_bytes, workspace_bytes, need, p.bytes);
        return CS_ERR_WORKSPACE;
    }
    const double nvd = 2.0 * (double)h->rows * (double)h->vocab * (double)h->width;
    ProfScope prof(K_HEAD_LOSS, (hipStream_t)stream, nvd, (double)(h->rows + h->vocab) * h->width * type_bytes(h->type));
    if (h->type == CS_TYPE_BF16) return forward<nt::BF16>(*h, p, s, row_losses, loss, (hipStream_t)stream);
    if (h->type == CS_TYPE_FP16) return forward<nt::FP16>(*h, p, s, row_losses, loss, (hipStream_t)stream);
    return forward<nt::FP32>(*h, p, s, row_losses, loss, (hipStream_t)stream);
}

int cs_head_loss_backward(const cs_head_loss* h, const void* saved, size_t saved_bytes, const float* grad, int64_t grad_stride, void* grad_hidden, void* grad_weight,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_head(h)) return rc;
    const int want = (grad_hidden ? 1 : 0) | (grad_weight ? 2 : 0);
    if (!want) return CS_OK;
    CS_REQUIRE(((uintptr_t)grad_hidden & 15) == 0 && ((uintptr_t)grad_weight & 15) == 0, "head loss: gradients are written at 16-byte aligned addresses");
    CS_REQUIRE((h->hidden || !h->rows) && h->weight && saved && (grad || !h->rows) && workspace, "head loss: NULL pointer");
    size_t need;
    const Saved s = carve_saved(*h, const_cast<void*>(saved), &need);
    const Plan p = make_plan(*h, want, workspace);
    if (saved_bytes < need || workspace_bytes < p.bytes) {
        set_error("head loss: workspace of %zu / %zu bytes, %zu / %zu are needed", saved_bytes, workspace_bytes, need, p.bytes);
        return CS_ERR_WORKSPACE;
    }
    const double nvd = 2.0 * (double)h->rows * (double)h->vocab * (double)h->width;
    ProfScope prof(K_HEAD_LOSS, (hipStream_t)stream, nvd * ((want & 1) + (want >> 1)), 2.0 * (double)(h->rows + h->vocab) * h->width * type_bytes(h->type));
    if (h->type == CS_TYPE_BF16) return backward<nt::BF16>(*h, p, s, grad, grad_stride, grad_hidden, grad_weight, (hipStream_t)stream);
    if (h->type == CS_TYPE_FP16) return backward<nt::FP16>(*h, p, s, grad, grad_stride, grad_hidden, grad_weight, (hipStream_t)stream);
    return backward<nt::FP32>(*h, p, s, grad, grad_stride, grad_hidden, grad_weight, (hipStream_t)stream);
}

}  // extern "C"
