// Low-rank adapters of many requests at once, beside a shared projection: out[t] = y[t] + scale[a] B[a] (A[a] x[t]) with
// a the adapter of token t.  Tokens are grouped by adapter with the layer's own dispatch (an adapter takes the place of an
// expert); the plan that comes of it holds for every projection of the batch.
//
// Two kernels: v = A x, d_in shared out over blocks whose sums go through a workspace and are added in a fixed order, then
// y + scale B v, which starts under the first and fetches y and B meanwhile.  A token costs 2 r (d_in + d_out) products for its
// (d_in + 2 d_out) elements, so memory bounds large batches and the latency of two kernels small ones.  Device time and what
// the bytes take at the copy rate, us: 64 tokens and as many adapters of rank 16, 4096 x 4096, BF16 7.5 and 1.9; 4096 tokens, 8 of
// rank 16 21.9 and 15.3; 777 tokens of up to rank 24, 1000 x 2724, FP32 13.9 and 3.2; 16384 tokens of rank 64, 4096 x 10240, FP16
// 182 and 129.  As one kernel, with clusters and distributed shared memory, the second of these took 25.3.
#include <cfloat>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace infmoe {

namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int APPLY_THREADS = 256;
constexpr int APPLY_WARPS = APPLY_THREADS / 32;
constexpr int MAX_WIDTH = 1 << 24;   // of x and y: places in a row are counted in bytes in 32 bits

// A plan cuts the tokens into tiles, all of whose rows have the same adapter, twice: tiles of at most FEW and of at most MANY rows.
// Which of them a call takes goes by its own sizes.
constexpr int FEW = 16, MANY = 128;

// Tiles of a batch: whole tiles of every adapter and what is left of each, and those of the tokens without one.
long long max_tiles(long long T, int n, int rows) {
    const long long kinds = (long long)n + 1;
    return T / rows + (T < kinds ? T : kinds);
}

struct Tiling {
    size_t tiles, rows;      // int4 [max_tiles], int [max_tiles][FEW or MANY]
};
struct PlanLayout {
    size_t pos, offset, count;
    Tiling few, many;
    size_t total;
};
PlanLayout plan_layout(long long T, int n) {
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    PlanLayout p{};
    p.offset = up(sizeof(int) * (size_t)T);
    p.count = p.offset + up(sizeof(int) * ((size_t)n + 1));
    p.total = p.count + up(sizeof(int) * (size_t)n);
    const auto add = [&](Tiling* t, int rows) {
        const size_t tiles = (size_t)max_tiles(T, n, rows);
        t->tiles = p.total;
        t->rows = t->tiles + up(sizeof(int4) * tiles);
        p.total = t->rows + up(sizeof(int) * tiles * (size_t)rows);
    };
    add(&p.few, FEW);
    add(&p.many, MANY);
    return p;
}

// tiles[i] = {adapter (-1: none), first row of expert order, rows, 0}; rows = 0 behind the last tile.  Block 0 makes the tiles of FEW
// rows, block 1 those of MANY.
__global__ void __launch_bounds__(PLAN_THREADS)
adapter_tiles_kernel(long long T, int n, const int* offset, int4* __restrict__ few, int few_capacity, int4* __restrict__ many,
                     int many_capacity) {
    pdl_trigger();
    pdl_wait();
    __shared__ int s_sum[32];
    __shared__ int s_base;
    int4* const tiles = blockIdx.x == 0 ? few : many;
    const int tile_rows = blockIdx.x == 0 ? FEW : MANY, capacity = blockIdx.x == 0 ? few_capacity : many_capacity;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) s_base = 0;
    __syncthreads();
    for (int a0 = 0; a0 <= n; a0 += PLAN_THREADS) {
        const int a = a0 + (int)threadIdx.x;
        int begin = 0, rows = 0;
        if (a <= n) {
            begin = offset[a];
            rows = (a < n ? offset[a + 1] : (int)T) - begin;
        }
        const int mine = (rows + tile_rows - 1) / tile_rows;
        int incl = mine;
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int at = s_base + incl - mine;
        for (int w = 0; w < warp; ++w) at += s_sum[w];
        for (int i = 0; i < mine; ++i)
            if (at + i < capacity)
                tiles[at + i] = make_int4(a < n ? a : -1, begin + i * tile_rows, min(tile_rows, rows - i * tile_rows), 0);
        __syncthreads();
        if (threadIdx.x == PLAN_THREADS - 1) s_base = at + mine;
        __syncthreads();
    }
    for (int i = s_base + (int)threadIdx.x; i < capacity; i += PLAN_THREADS) tiles[i] = make_int4(-1, 0, 0, 0);
}

// rows[i][r] = token of row r of tile i: found without looking at the tile, so that a block of the products has both at once.
// Blocks of MANY threads: MANY / FEW of the first tiling's tiles, or one of the second's.
__global__ void __launch_bounds__(MANY)
adapter_rows_kernel(const int* pos, const int4* few, int* __restrict__ few_rows, int few_tiles, const int4* many,
                    int* __restrict__ many_rows, int few_blocks) {
    pdl_trigger();
    pdl_wait();
    const bool first = (int)blockIdx.x < few_blocks;
    const int tile_rows = first ? FEW : MANY;
    const int i = first ? (int)blockIdx.x * (MANY / FEW) + (int)threadIdx.x / FEW : (int)blockIdx.x - few_blocks, r = (int)threadIdx.x % tile_rows;
    if (first && i >= few_tiles) return;
    const int4 tile = first ? few[i] : many[i];
    if (r < tile.z) (first ? few_rows : many_rows)[i * tile_rows + r] = pos[tile.y + r];
}

struct ApplyArgs {
    const void *x, *y, *a, *b;
    void* out;
    long long ldx, ldy, ldo;
    int rank, d_in, d_out;
    const float* scale;       // [adapters] or NULL: 1
    const int* rank_of;       // [adapters] or NULL: all `rank`
    const int4* tiles;
    const int* rows;          // [tiles][FEW or MANY]: tokens
    int x_grain, a_grain, b_grain, y_grain;   // bytes of one copy to shared memory: 16, 8, 4, or 2 (ordinary loads)
    int out_vec;              // out is written 16 bytes at a time
    float* sums;              // [k_split][tiles][FEW or MANY][RP]: shares of A x
    int tile_count, k_split, col_split;      // tiles, and blocks that share out d_in, and d_out, of a tile
    int* status;
};

// The 16 bytes at dst come from src, those from byte `left` on are zero.  src is a multiple of grain.  FAST: it is one of 16, and
// so is left, or (not WHOLE) that lies in 0..16.
template <bool FAST, bool WHOLE = true>
__device__ __forceinline__ void copy_piece(uint32_t dst, const char* src, int left, int grain) {
    if (FAST) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(WHOLE ? (left > 0 ? 16 : 0) : left) : "memory");
    } else if (grain == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(min(16, max(0, left))) : "memory");
    } else if (grain == 8) {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i), "l"(src + i), "r"(min(8, max(0, left - i))) : "memory");
    } else if (grain == 4) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i), "l"(src + i), "r"(min(4, max(0, left - i))) : "memory");
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(src) + 2 * i;
            const uint32_t lo = 4 * i < left ? p[0] : 0, hi = 4 * i + 2 < left ? p[1] : 0;
            w[i] = lo | hi << 16;
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Four 8 x 16-byte matrices: lanes 0-7, 8-15, ... give their rows; a lane gets word (lane % 4) of row lane / 4 of each.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// c += a b over 32 bytes of K: 16 values of 16 bits, or 8 of TF32.
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if constexpr (std::is_same_v<T, __nv_bfloat16>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An FP32 value as two of 11 significant bits: rounded to the first, and what that leaves rounded to the second.  Of a value in [1, 2) the
// first leaves at most 2^-11 in steps of 2^-23, so at most 2^-23 is lost.  The product of two second parts, at most 2^-22 of the whole, is left
// out: a product is off by at most 2^-21, to either side (a first part that is cut off made it 2^-20 and always too small).  With that product
// rank 32 takes 131 us for 119 and the error of sums of 4 to 4096 terms is the same within 10 %: it is that of sums in the tensor cores' 32 bits.
// An infinity, NaN, and what the first part rounds to an infinity have no such parts: the second is NaN or the opposite infinity, and
// every sum that it enters is NaN (plain_sum).
__device__ __forceinline__ void split_tf32(const uint32_t v, uint32_t& hi, uint32_t& lo) {
    hi = (v + 0x1000u) & 0xffffe000u;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(__fsub_rn(__uint_as_float(v), __uint_as_float(hi))));
}
// sum_i a[i] b[i] in FP32: stands in the place of a sum of parts that is no finite number.
__device__ __forceinline__ float plain_sum(const float* a, const float* b, int n) {
    float sum = 0.f;
#pragma unroll 1
    for (int i = 0; i < n && sum == sum; ++i) sum = fmaf(a[i], b[i], sum);
    return sum;
}

// What is left of v after its rounding to T (0 where that is no finite value).
template <typename T>
__device__ __forceinline__ float rest_of(float v) {
    const float h = to_float(from_float<T>(v));
    return fabsf(h) <= FLT_MAX ? __fsub_rn(v, h) : 0.f;
}

// ---- tiles of FEW rows: mma.sync --------------------------------------------------------------------
// First kernel, A x: stages of M rows of x and RP rows of A, 256 bytes of K each, so that each of the warps has a 32-byte step of K.
// Second kernel, y + scale B v: stages of COLUMNS columns, M rows of y and COLUMNS rows of B, so that each of the warps has a unit of
// 16 rows and 32 columns (or every other time).

// Blocks an SM has room for: small ranks leave room for more, and each of them has little in flight (4096 tokens of rank 16: four
// 21.8 us, three 25.8, two 27.3).
constexpr int few_per_sm(int padded_rank) { return padded_rank == 16 ? 4 : padded_rank == 32 ? 3 : 2; }

template <typename T, int RP>
struct ApplyShape {
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr int SIZE = (int)sizeof(T), M = FEW;
    static constexpr int clamp_stages(int n) { return n < 2 ? 2 : n > 8 ? 8 : n; }
    static constexpr int larger(int a, int b) { return a > b ? a : b; }

    static constexpr int SUBS = 2, K_CHUNK = SUBS * 128 / SIZE;     // 128-byte parts of K in a stage
    static constexpr int STAGE1 = SUBS * (M + RP) * 128;
    static constexpr int S1 = clamp_stages((RP == 16 ? 40 : RP == 32 ? 64 : RP == 64 ? 84 : 110) * 1024 / STAGE1);
    static constexpr int PART = APPLY_WARPS * 16 * RP * 4;          // the warps' sums, in the place of the stages
    static constexpr int SMEM1 = larger(PART, S1 * STAGE1);

    static constexpr int UNITS = RP * SIZE >= 128 ? 4 : 8;          // FP32, rank 16, 1024 tokens, 1024 x 1024: eight 8.8 us, four 9.5
    static constexpr int COLUMNS = UNITS * 32;
    static constexpr int Y_PIECES = COLUMNS * SIZE / 16, B_PIECES = RP * SIZE / 16;   // 16-byte pieces of a row of y, of B
    static constexpr int Y_BYTES = M * Y_PIECES * 16;
    static constexpr int STAGE2 = Y_BYTES + COLUMNS * B_PIECES * 16;
    static_assert(M * Y_PIECES >= APPLY_THREADS && SUBS * M * 8 >= APPLY_THREADS, "a copy of x and of y for every thread");
    static constexpr int S2 = clamp_stages((RP == 16 ? 48 : RP == 32 ? 72 : RP == 64 ? 84 : 110) * 1024 / STAGE2);
    static constexpr int PER_SM = few_per_sm(RP);
    static constexpr int V_ROW = RP * SIZE + 16;                    // bytes of a row of A x; the padding spreads rows over the banks
    static constexpr int V_BYTES = M * V_ROW;                       // 16 bits: once more for the second parts
    static constexpr int SMEM2 = S2 * STAGE2 + (WIDE ? 1 : 2) * V_BYTES;

    // Place (in units of 16 bytes) of a piece of row `col` of B.  A matrix of the second product has columns 2j, 2j + 1, 2j + 8,
    // 2j + 9, ... 2j + 25 of a unit (see there): bits 0, 3 and 4 of the column have to tell eight banks of 16 bytes apart.
    static __device__ __forceinline__ uint32_t b_place(int col, int piece) {
        const int c0 = col & 1, c3 = (col >> 3) & 1, c4 = (col >> 4) & 1;
        const int z = B_PIECES == 2 ? c3 + 4 * c4 : B_PIECES == 4 ? c3 + 2 * c4 : c0 + 2 * c3 + 4 * c4;
        return (uint32_t)((col * B_PIECES + piece) ^ z);
    }
    // Of a row of y: a warp's 16-byte accesses take four neighbouring pieces (FP32: every other one) of two rows at a time.
    static __device__ __forceinline__ uint32_t y_place(int row, int piece) {
        return (uint32_t)(row * Y_PIECES + (piece ^ ((row & 1) * (WIDE ? 1 : 4))));
    }
};

// out = y in these columns of `rows` rows.
template <typename T>
__device__ __forceinline__ void copy_rows(const ApplyArgs& p, int rows, const int* s_pos, int col_begin, int col_end) {
    constexpr int N = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    const bool vec = p.out_vec && p.y_grain == 16;
    for (int r = threadIdx.x >> 5; r < rows; r += APPLY_WARPS) {
        const T* src = static_cast<const T*>(p.y) + s_pos[r] * p.ldy;
        T* dst = static_cast<T*>(p.out) + s_pos[r] * p.ldo;
        if (vec)
            for (int c = col_begin + lane * N; c < col_end; c += 32 * N)
                *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
        else
            for (int c = col_begin + lane; c < col_end; c += 32) dst[c] = src[c];
    }
}

// FAST: x, A, B and y are copied, and out written, in whole pieces of 16 bytes.
template <typename T, int RP, bool FAST>
__global__ void __launch_bounds__(APPLY_THREADS, ApplyShape<T, RP>::PER_SM) adapter_down_kernel(const ApplyArgs p) {
    using S = ApplyShape<T, RP>;
    constexpr bool WIDE = S::WIDE;
    constexpr int SIZE = S::SIZE, M = S::M;
    extern __shared__ __align__(128) char smem[];
    __shared__ int s_pos[M];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile_index = blockIdx.x / p.k_split, share = blockIdx.x % p.k_split;
    pdl_wait();
    pdl_trigger();
    const int4 tile = p.tiles[tile_index];
    const int token = tid < M ? p.rows[tile_index * M + tid] : 0;
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    if (tile.z <= 0 || rank == 0) return;
    if (tid < tile.z) s_pos[tid] = token;
    __syncthreads();
    const T* const A = static_cast<const T*>(p.a) + (long long)tile.x * p.rank * p.d_in;
    const uint32_t ring = smem_u32(smem);

    const int stages_all = (p.d_in + S::K_CHUNK - 1) / S::K_CHUNK;
    const int stage_begin = (int)((long long)stages_all * share / p.k_split);
    const int stages = (int)((long long)stages_all * (share + 1) / p.k_split) - stage_begin;
    // a thread copies the same 16 bytes of every stage: piece tid % 8 of row tid / 8 and of those 32 further on
    constexpr int X_COPIES = S::SUBS * M * 8 / APPLY_THREADS, A_COPIES = (S::SUBS * RP * 8 + APPLY_THREADS - 1) / APPLY_THREADS;
    const int piece = tid & 7, row0 = tid >> 3;
    const char *x_at[X_COPIES], *a_at[A_COPIES];
    int x_left[X_COPIES], a_left[A_COPIES];                         // bytes of the row from there on, none for a row that is not there
#pragma unroll
    for (int i = 0; i < X_COPIES; ++i) {
        const int n = row0 + 32 * i, r = n % M, k = stage_begin * S::K_CHUNK * SIZE + (n / M) * 128 + piece * 16;
        x_left[i] = r < tile.z ? p.d_in * SIZE - k : 0;
        x_at[i] = reinterpret_cast<const char*>(static_cast<const T*>(p.x) + s_pos[min(r, tile.z - 1)] * p.ldx) + k;
    }
#pragma unroll
    for (int i = 0; i < A_COPIES; ++i) {
        const int n = row0 + 32 * i, r = n % RP, sub = n / RP, k = stage_begin * S::K_CHUNK * SIZE + sub * 128 + piece * 16;
        a_left[i] = r < rank && sub < S::SUBS ? p.d_in * SIZE - k : INT_MIN / 2;
        a_at[i] = reinterpret_cast<const char*>(A + (long long)min(r, rank - 1) * p.d_in) + k;
    }
    const uint32_t piece_at = (uint32_t)((piece ^ (row0 & 7)) << 4);
    const auto fetch = [&](int n, int slot) {
        if (n < stages) {
            const uint32_t to = ring + (uint32_t)slot * S::STAGE1 + piece_at;
            const long long at = (long long)n * (S::SUBS * 128);
            const int gone = n * (S::SUBS * 128);
#pragma unroll
            for (int i = 0; i < X_COPIES; ++i) {
                const int row = row0 + 32 * i;
                copy_piece<FAST>(to + (row % M + row / M * (M + RP)) * 128, x_at[i] + at, x_left[i] - gone, p.x_grain);
            }
#pragma unroll
            for (int i = 0; i < A_COPIES; ++i) {
                const int row = row0 + 32 * i;
                if (a_left[i] > INT_MIN / 4)
                    copy_piece<FAST>(to + (M + row % RP + row / RP * (M + RP)) * 128, a_at[i] + at, a_left[i] - gone, p.a_grain);
            }
        }
        copies_commit();
    };
    const int n_pairs = (rank + 15) / 16;
    float acc[RP / 8][4];
#pragma unroll
    for (int j = 0; j < RP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
#pragma unroll
    for (int c = 0; c < S::S1 - 1; ++c) fetch(c, c);
    const int xr = lane & 15, wr = (lane & 7) + ((lane >> 4) << 3);
    const auto multiply = [&](uint32_t stage, int s) {
        uint32_t x[4];
        load_matrices(x, stage + xr * 128 + (((2 * s + (lane >> 4)) ^ (xr & 7)) << 4));
        uint32_t x_lo[4];
        if constexpr (WIDE)
#pragma unroll
            for (int i = 0; i < 4; ++i) split_tf32(x[i], x[i], x_lo[i]);
        const uint32_t w_at = stage + (M + wr) * 128 + (((2 * s + ((lane >> 3) & 1)) ^ (wr & 7)) << 4);
        constexpr int GROUP = RP / 16 < 4 ? RP / 16 : WIDE ? 2 : 4;   // pairs of n tiles whose loads are in flight together
#pragma unroll
        for (int n0 = 0; n0 < RP / 16; n0 += GROUP) {
            if (n0 >= n_pairs) break;
            uint32_t w[GROUP][4];
#pragma unroll
            for (int n = 0; n < GROUP; ++n) load_matrices(w[n], w_at + (n0 + n) * 2048);
            if constexpr (WIDE) {
                uint32_t w_lo[GROUP][4];
#pragma unroll
                for (int n = 0; n < GROUP; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(w[n][i], w[n][i], w_lo[n][i]);
#pragma unroll
                for (int h = 0; h < 2 * GROUP; ++h) mma<T>(acc[2 * n0 + h], x_lo, w[h / 2][2 * (h & 1)], w[h / 2][2 * (h & 1) + 1]);
#pragma unroll
                for (int h = 0; h < 2 * GROUP; ++h) mma<T>(acc[2 * n0 + h], x, w_lo[h / 2][2 * (h & 1)], w_lo[h / 2][2 * (h & 1) + 1]);
            }
#pragma unroll
            for (int h = 0; h < 2 * GROUP; ++h) mma<T>(acc[2 * n0 + h], x, w[h / 2][2 * (h & 1)], w[h / 2][2 * (h & 1) + 1]);
        }
    };
    int read = 0, fill = S::S1 - 1;                                 // slots of the ring
    for (int c = 0; c < stages; ++c) {
        copies_wait<S::S1 - 2>();
        __syncthreads();               // the stage is complete, and everybody is done with the one that is filled next
        fetch(c + S::S1 - 1, fill);
        const uint32_t stage = ring + (uint32_t)read * S::STAGE1;
        multiply(stage + (warp >> 2) * (M + RP) * 128, warp & 3);
        read = read + 1 == S::S1 ? 0 : read + 1;
        fill = fill + 1 == S::S1 ? 0 : fill + 1;
    }
    copies_wait<0>();
    __syncthreads();

    // sums over the warps
    float* const part = reinterpret_cast<float*>(smem);             // [warps][M][RP]
#pragma unroll
    for (int j = 0; j < RP / 8; ++j) {
        float* at = part + (warp * M + (lane >> 2)) * RP + j * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(at + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    float* const sums = p.sums + (size_t)(share * p.tile_count + tile_index) * (M * RP);
    for (int i = tid * 4; i < tile.z * RP; i += APPLY_THREADS * 4) {
        float4 sum = *reinterpret_cast<const float4*>(part + i);
#pragma unroll
        for (int g = 1; g < APPLY_WARPS; ++g) {
            const float4 o = *reinterpret_cast<const float4*>(part + g * M * RP + i);
            sum = make_float4(sum.x + o.x, sum.y + o.y, sum.z + o.z, sum.w + o.w);
        }
        if constexpr (WIDE) {
            const int from = stage_begin * S::K_CHUNK, n = min(p.d_in - from, stages * S::K_CHUNK);
            const T* const x = static_cast<const T*>(p.x) + s_pos[i / RP] * p.ldx + from;
            const T* const w = A + (long long)(i % RP) * p.d_in + from;
            const int left = rank - i % RP;
            if (!(fabsf(sum.x) <= FLT_MAX) && 0 < left) sum.x = plain_sum(x, w, n);
            if (!(fabsf(sum.y) <= FLT_MAX) && 1 < left) sum.y = plain_sum(x, w + p.d_in, n);
            if (!(fabsf(sum.z) <= FLT_MAX) && 2 < left) sum.z = plain_sum(x, w + 2ll * p.d_in, n);
            if (!(fabsf(sum.w) <= FLT_MAX) && 3 < left) sum.w = plain_sum(x, w + 3ll * p.d_in, n);
        }
        *reinterpret_cast<float4*>(sums + i) = sum;
    }
}

// Starts under adapter_down_kernel, which triggers behind its own wait: what was there before that one, y among it, may be read
// before this one's wait, and the first stages are under way then.
template <typename T, int RP, bool FAST>
__global__ void __launch_bounds__(APPLY_THREADS, ApplyShape<T, RP>::PER_SM) adapter_up_kernel(const ApplyArgs p) {
    using S = ApplyShape<T, RP>;
    constexpr bool WIDE = S::WIDE;
    constexpr int SIZE = S::SIZE, M = S::M;
    extern __shared__ __align__(128) char smem[];
    __shared__ float s_unscale[M];
    __shared__ int s_pos[M];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile_index = blockIdx.x / p.col_split, share = blockIdx.x % p.col_split;
    const int4 tile = p.tiles[tile_index];
    const int token = tid < M ? p.rows[tile_index * M + tid] : 0;
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    const float scale = tile.x >= 0 && p.scale ? p.scale[tile.x] : 1.f;
    if (tile.z <= 0 || (rank == 0 && p.out == p.y)) {
        pdl_wait();
        return;
    }
    if (tid < tile.z) s_pos[tid] = token;
    __syncthreads();

    // this block's columns
    const int col_stages_all = (p.d_out + S::COLUMNS - 1) / S::COLUMNS;
    const int col_begin = (int)((long long)col_stages_all * share / p.col_split) * S::COLUMNS;
    const int col_end = min(p.d_out, (int)((long long)col_stages_all * (share + 1) / p.col_split) * S::COLUMNS);
    const T* const y_base = static_cast<const T*>(p.y);
    T* const out_base = static_cast<T*>(p.out);
    if (rank == 0) {                                                // no adapter, or none of its columns
        pdl_wait();
        pdl_trigger();
        copy_rows<T>(p, tile.z, s_pos, col_begin, col_end);
        return;
    }
    const T* const B = static_cast<const T*>(p.b) + (long long)tile.x * p.d_out * p.rank;
    const uint32_t ring = smem_u32(smem);

    constexpr int Y_COPIES = M * S::Y_PIECES / APPLY_THREADS;
    constexpr int B_COPIES = (S::COLUMNS * S::B_PIECES + APPLY_THREADS - 1) / APPLY_THREADS;
    constexpr int Y_ROWS = APPLY_THREADS / S::Y_PIECES, B_ROWS = APPLY_THREADS / S::B_PIECES;   // rows between a thread's copies
    const char* y_at[Y_COPIES];
    const int y_row = tid / S::Y_PIECES, y_piece = tid % S::Y_PIECES, b_row = tid / S::B_PIECES, b_piece = tid % S::B_PIECES;
#pragma unroll
    for (int i = 0; i < Y_COPIES; ++i)
        y_at[i] = reinterpret_cast<const char*>(y_base + s_pos[min(y_row + i * Y_ROWS, tile.z - 1)] * p.ldy + col_begin) + y_piece * 16;
    const int y_left = (p.d_out - col_begin) * SIZE - y_piece * 16;
    const int b_left = min(16, max(0, rank * SIZE - b_piece * 16));  // past the adapter's rank there are zeros
    const char* const b_at = reinterpret_cast<const char*>(B + (long long)(col_begin + b_row) * p.rank) + (b_left > 0 ? b_piece * 16 : 0);
    const int row_size = p.rank * SIZE;
    const int col_stages = (col_end - col_begin + S::COLUMNS - 1) / S::COLUMNS;
    const auto fetch_columns = [&](int n, int slot) {
        if (n < col_stages) {
            const uint32_t to = ring + (uint32_t)slot * S::STAGE2;
            const int left = y_left - n * (S::COLUMNS * SIZE), cols = p.d_out - col_begin - n * S::COLUMNS - b_row;
            if (left > 0)
#pragma unroll
                for (int i = 0; i < Y_COPIES; ++i)
                    if (y_row + i * Y_ROWS < tile.z)
                        copy_piece<FAST>(to + S::y_place(y_row + i * Y_ROWS, y_piece) * 16, y_at[i] + (long long)n * (S::COLUMNS * SIZE), left, p.y_grain);
            const char* from = b_at + (long long)n * (S::COLUMNS * row_size);
#pragma unroll
            for (int i = 0; i < B_COPIES; ++i)
                if (i * B_ROWS < cols && (S::COLUMNS * S::B_PIECES >= APPLY_THREADS || b_row < S::COLUMNS))
                    copy_piece<FAST, false>(to + S::Y_BYTES + S::b_place(b_row + i * B_ROWS, b_piece) * 16, from + i * B_ROWS * row_size, b_left, p.b_grain);
        }
        copies_commit();
    };
#pragma unroll
    for (int c = 0; c < S::S2 - 1; ++c) fetch_columns(c, c);
    pdl_wait();
    pdl_trigger();

    // A x: the shares of all blocks.  A thread has four columns of a row, and of rows ROWS further on.
    char* const v_smem = smem + S::S2 * S::STAGE2;
    {
        constexpr int LANES = RP / 4, ROWS = APPLY_THREADS / LANES, PASSES = (M + ROWS - 1) / ROWS;
        const int col = tid % LANES * 4, r0 = tid / LANES;
        const float* const from = p.sums + (size_t)tile_index * (M * RP) + r0 * RP + col;
        const size_t stride = (size_t)p.tile_count * (M * RP);
        float4 v[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int TOGETHER = PASSES <= 1 ? 8 : PASSES <= 2 ? 4 : PASSES <= 4 ? 2 : 1;
#pragma unroll TOGETHER
        for (int q = 0; q < p.k_split; ++q) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                if (r0 + i * ROWS >= tile.z) continue;
                const float4 o = __ldcg(reinterpret_cast<const float4*>(from + q * stride + i * ROWS * RP));
                v[i] = make_float4(v[i].x + o.x, v[i].y + o.y, v[i].z + o.z, v[i].w + o.w);
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = r0 + i * ROWS;
            if (col >= rank) v[i].x = 0.f;
            if (col + 1 >= rank) v[i].y = 0.f;
            if (col + 2 >= rank) v[i].z = 0.f;
            if (col + 3 >= rank) v[i].w = 0.f;
            if constexpr (std::is_same_v<T, __half>) {              // FP16 has neither BF16's range nor A x a bound
                float most = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
                for (int off = LANES / 2; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                const int e = row_exponent(most);
                const float up = exp2_int(e);
                if (col == 0 && r < tile.z) s_unscale[r] = exp2_int(-e);
                v[i] = make_float4(v[i].x * up, v[i].y * up, v[i].z * up, v[i].w * up);
            }
            if (r >= tile.z) continue;
            char* const to = v_smem + r * S::V_ROW + col * SIZE;
            if constexpr (WIDE) {
                *reinterpret_cast<float4*>(to) = v[i];
            } else {
                *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<T>(v[i].x, v[i].y), pack_pair<T>(v[i].z, v[i].w));
                *reinterpret_cast<uint2*>(to + S::V_BYTES) = make_uint2(pack_pair<T>(rest_of<T>(v[i].x), rest_of<T>(v[i].y)),
                                                                        pack_pair<T>(rest_of<T>(v[i].z), rest_of<T>(v[i].w)));
            }
        }
    }
    __syncthreads();

    // this block's columns, a warp a unit of every stage, or of every other one
    constexpr int STEPS = RP * SIZE / 32;                           // 32-byte steps of K
    constexpr bool HOLD = STEPS <= 4;                               // A x stays in registers
    const int g = lane >> 2, q = lane & 3;
    T* out_row[2];
    bool row_ok[2];
    float factor[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        row_ok[h] = r < tile.z;
        out_row[h] = out_base + (long long)s_pos[row_ok[h] ? r : 0] * p.ldo + col_begin + q * 8;
        factor[h] = std::is_same_v<T, __half> && row_ok[h] ? s_unscale[r] * scale : scale;
    }
    const uint32_t v_addr = smem_u32(v_smem) + (lane & 15) * S::V_ROW + ((lane >> 4) << 4);
    uint32_t v[HOLD ? STEPS : 1][4], v_lo[HOLD ? STEPS : 1][4];
    const auto load_v = [&](int s, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        load_matrices(hi, v_addr + s * 32);
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) split_tf32(hi[i], hi[i], lo[i]);
        } else {
            load_matrices(lo, v_addr + S::V_BYTES + s * 32);
        }
    };
    if constexpr (HOLD)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) load_v(s, v[s], v_lo[s]);
    // Accumulator columns 2q, 2q + 1 of product j stand for columns 8q + 2j, 8q + 2j + 1 of the unit, so that a lane holds eight
    // neighbours: row i of matrix j of B is its row (i / 2) 8 + 2j + i % 2.  Four columns or four steps further on the place is
    // that many rows or 128 bytes further on (b_place).
    const int b_first = ((lane & 7) >> 1) * 8 + (lane & 1) + 2 * (lane >> 4);
    uint32_t b_step_at[STEPS < 4 ? STEPS : 4];
#pragma unroll
    for (int s = 0; s < (STEPS < 4 ? STEPS : 4); ++s) b_step_at[s] = ring + S::Y_BYTES + S::b_place(b_first, 2 * s + ((lane >> 3) & 1)) * 16;
    constexpr int N = 16 / SIZE;
    const int u = warp % S::UNITS;
    uint32_t cell[2][8 / N];                                        // its pieces of y
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) cell[h][i] = S::y_place(g + 8 * h, u * (32 / N) + q * (8 / N) + i) * 16;
#pragma unroll
    for (int s = 0; s < (STEPS < 4 ? STEPS : 4); ++s) b_step_at[s] += (uint32_t)u * (32 * S::B_PIECES * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) out_row[h] += u * 32;
    int read = 0, fill = S::S2 - 1;                                 // slots of the ring
    for (int c = 0; c < col_stages; ++c) {
        copies_wait<S::S2 - 2>();
        __syncthreads();
        fetch_columns(c + S::S2 - 1, fill);
        const uint32_t slot = (uint32_t)read * S::STAGE2;
        read = read + 1 == S::S2 ? 0 : read + 1;
        fill = fill + 1 == S::S2 ? 0 : fill + 1;
        if (S::UNITS == APPLY_WARPS || (c & 1) == warp / S::UNITS) {
            float sum[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[j][i] = 0.f;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                if constexpr (!HOLD) load_v(s, v[0], v_lo[0]);
                const uint32_t(&hi)[4] = v[HOLD ? s : 0];
                const uint32_t(&lo)[4] = v_lo[HOLD ? s : 0];
                uint32_t w[2][4];
#pragma unroll
                for (int jp = 0; jp < 2; ++jp) load_matrices(w[jp], b_step_at[s & 3] + slot + jp * (4 * S::B_PIECES * 16) + s / 4 * 128);
                if constexpr (WIDE) {
                    uint32_t w_lo[2][4];
#pragma unroll
                    for (int i = 0; i < 8; ++i) split_tf32(w[i / 4][i & 3], w[i / 4][i & 3], w_lo[i / 4][i & 3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma<T>(sum[j], hi, w_lo[j / 2][2 * (j & 1)], w_lo[j / 2][2 * (j & 1) + 1]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) mma<T>(sum[j], lo, w[j / 2][2 * (j & 1)], w[j / 2][2 * (j & 1) + 1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) mma<T>(sum[j], hi, w[j / 2][2 * (j & 1)], w[j / 2][2 * (j & 1) + 1]);
            }
            const int left = p.d_out - (col_begin + c * S::COLUMNS + u * 32 + q * 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!row_ok[h]) continue;
                if constexpr (WIDE) {
                    float all = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) all += fabsf(sum[k / 2][2 * h + (k & 1)]);
                    if (!(all <= FLT_MAX))
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float& o = sum[k / 2][2 * h + (k & 1)];
                            if (!(fabsf(o) <= FLT_MAX) && k < left)
                                o = plain_sum(reinterpret_cast<const float*>(v_smem + (g + 8 * h) * S::V_ROW),
                                              reinterpret_cast<const float*>(B) + (long long)(p.d_out - left + k) * p.rank, rank);
                        }
                }
#pragma unroll
                for (int i = 0; i < 8 / N; ++i) {
                    uint4* const at = reinterpret_cast<uint4*>(smem + slot + cell[h][i]);
                    float e[N];
                    unpack16<T>(*at, e);
#pragma unroll
                    for (int k = 0; k < N; ++k) e[k] = fmaf(sum[(i * N + k) / 2][2 * h + (k & 1)], factor[h], e[k]);
                    const uint4 raw = pack16<T>(e);
                    if (!FAST && !p.out_vec)
                        *at = raw;
                    else if (i * N < left)
                        *reinterpret_cast<uint4*>(out_row[h] + c * S::COLUMNS + i * N) = raw;
                }
            }
        }
        if (!FAST && !p.out_vec) {
            // rows that cannot be written 16 bytes at a time: from shared memory, element by element, neighbours by neighbours
            __syncthreads();
            const int first = col_begin + c * S::COLUMNS, width = min(S::COLUMNS, p.d_out - first);
            for (int r = warp; r < tile.z; r += APPLY_WARPS) {
                T* dst = out_base + (long long)s_pos[r] * p.ldo + first;
                for (int e = lane; e < width; e += 32)
                    dst[e] = *reinterpret_cast<const T*>(smem + slot + S::y_place(r, e / N) * 16 + e % N * SIZE);
            }
        }
    }
    copies_wait<0>();
}

// ---- 16-bit types, tiles of 128 rows: tcgen05 ------------------------------------------------------
// The same two kernels with the 128 rows on the M side of tcgen05.mma and sums in tensor memory: one thread issues a stage's MMAs,
// so the warps' work is copies and the last step alone (16384 tokens of rank 64, 4096 x 10240: 182 us, where tiles of 16 rows and
// mma.sync, whose ldmatrix and accumulators keep the SMs busier than the memory, take 265; the bytes are 129 us at the copy
// rate).  Stages are rows of 128 bytes, 16-byte pieces exchanged within eight rows, which is both what cp.async writes without
// conflicts and the 128-byte swizzle that the MMAs read.  Rows of a tile that are not there are not copied: whatever stands in their
// place only makes their own rows of the sums.
constexpr int TC_ROWS = MANY, MANY_PER_SM = 2;                      // of the first kernel

template <int RP>
struct TcShape {
    static constexpr int K_CHUNK = 64, COLUMNS = 64;
    static constexpr int STAGE1 = (TC_ROWS + RP) * 128;
    static constexpr int S1 = RP == 128 ? 3 : 4;
    static constexpr int SMEM1 = S1 * STAGE1 + 1024;                // + slack for 1024-byte alignment
    static constexpr int ATOMS = (RP + 63) / 64;                    // 128-byte parts of a row of B
    static constexpr int Y_BYTES = TC_ROWS * 128;
    static constexpr int STAGE2 = Y_BYTES + ATOMS * COLUMNS * 128;
    static constexpr int S2 = 3;
    static constexpr int SMEM2 = S2 * STAGE2 + 1024;
    static constexpr int PER_SM1 = MANY_PER_SM, PER_SM2 = RP == 128 ? 2 : 3;   // blocks an SM has room for
    // Columns of tensor memory: sums, and in the second kernel A x, two values to a column, first parts and second parts.
    static constexpr uint32_t TMEM1 = RP, TMEM2 = COLUMNS + RP <= 128 ? 128 : 256;
    static_assert(RP >= 32, "the least that can be allocated");
};

template <typename T>
__device__ __forceinline__ constexpr uint32_t operand_format() { return std::is_same_v<T, __half> ? 0u : 1u; }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T: 16-bit operands, a row of A to a lane, two values of K to a column; B K-major; K = 16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A lane's four columns of tensor memory.
__device__ __forceinline__ void tmem_st4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A x of a tile.  Tensor memory is allocated before the next kernel may start: blocks that hold some of it never wait for one that
// still needs some.
template <typename T, int RP, bool FAST>
__global__ void __launch_bounds__(APPLY_THREADS) adapter_down_tc_kernel(const ApplyArgs p) {
    using S = TcShape<RP>;
    extern __shared__ __align__(128) char smem_raw[];
    __shared__ __align__(8) uint64_t s_done[S::S1];                 // a stage's MMAs are complete
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_pos[TC_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int tile_index = blockIdx.x / p.k_split, share = blockIdx.x % p.k_split;
    if (warp == 0) tmem_alloc(&s_tmem, S::TMEM1);
    if (tid == 0) {
        for (int i = 0; i < S::S1; ++i) mbar_init(smem_u32(&s_done[i]), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int4 tile = p.tiles[tile_index];
    const int token = tid < TC_ROWS ? p.rows[tile_index * TC_ROWS + tid] : 0;
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    if (tid < tile.z) s_pos[tid] = token;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = s_tmem;
    if (tile.z > 0 && rank > 0) {
        const T* const A = static_cast<const T*>(p.a) + (long long)tile.x * p.rank * p.d_in;
        const int stages_all = (p.d_in + S::K_CHUNK - 1) / S::K_CHUNK;
        const int stage_begin = (int)((long long)stages_all * share / p.k_split);
        const int stages = (int)((long long)stages_all * (share + 1) / p.k_split) - stage_begin;
        // a thread copies piece tid % 8 of row tid / 8 and of those 32 further on
        constexpr int X_COPIES = TC_ROWS / 32, A_COPIES = (RP + 31) / 32;
        const int piece = tid & 7, row0 = tid >> 3, k = stage_begin * 128 + piece * 16, left0 = p.d_in * 2 - k;
        const char *x_at[X_COPIES], *a_at[A_COPIES];
#pragma unroll
        for (int i = 0; i < X_COPIES; ++i)
            x_at[i] = reinterpret_cast<const char*>(static_cast<const T*>(p.x) + s_pos[min(row0 + 32 * i, tile.z - 1)] * p.ldx) + k;
#pragma unroll
        for (int i = 0; i < A_COPIES; ++i)
            a_at[i] = reinterpret_cast<const char*>(A + (long long)min(row0 + 32 * i, rank - 1) * p.d_in) + k;
        const uint32_t place = (uint32_t)(row0 * 128 + ((piece ^ (row0 & 7)) << 4));
        const auto fetch = [&](int n, int slot) {
            if (n < stages) {
                const uint32_t to = ring + (uint32_t)slot * S::STAGE1 + place;
#pragma unroll
                for (int i = 0; i < X_COPIES; ++i)
                    if (row0 + 32 * i < tile.z) copy_piece<FAST>(to + 4096 * i, x_at[i] + (long long)n * 128, left0 - n * 128, p.x_grain);
#pragma unroll
                for (int i = 0; i < A_COPIES; ++i)
                    if (row0 + 32 * i < rank)
                        copy_piece<FAST>(to + TC_ROWS * 128 + 4096 * i, a_at[i] + (long long)n * 128, left0 - n * 128, p.a_grain);
            }
            copies_commit();
        };
#pragma unroll
        for (int c = 0; c < S::S1 - 1; ++c) fetch(c, c);
        const uint32_t idesc = make_idesc(TC_ROWS, RP, operand_format<T>());
        bool ok = true;
        int slot = 0, before = S::S1 - 1;
        uint32_t phase = 1;                                         // of the slot before: its last use's
        for (int c = 0; c < stages; ++c) {
            copies_wait<S::S1 - 2>();
            fence_async();                                          // what this thread copied is there for the MMAs
            __syncthreads();
            if (warp == 0 && ok && elect_one()) {
                const uint64_t dx = make_smem_desc(ring + (uint32_t)slot * S::STAGE1);
                const uint64_t da = make_smem_desc(ring + (uint32_t)slot * S::STAGE1 + TC_ROWS * 128);
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_f16_ss(tmem, dx + 2 * j, da + 2 * j, idesc, c + j > 0);
                umma_commit(smem_u32(&s_done[slot]));
            }
            // the stage before this one is free once its MMAs are complete
            if (c > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_done[before]), phase, &s_abort));
            if (ok) fetch(c + S::S1 - 1, before);
            else copies_commit();
            before = slot;
            if (slot == 0) phase ^= 1;
            if (++slot == S::S1) slot = 0;
        }
        if (ok) ok = mbar_wait(smem_u32(&s_done[before]), phase, &s_abort);
        copies_wait<0>();
        ok = __syncthreads_and(ok);
        tc_fence_after();
        if (ok) {
            // lanes of tensor memory are rows; four warps have 32 each, the other four the second half of the columns
            constexpr int WIDTH = RP / 2;
            const int row = (warp & 3) * 32 + lane, half = warp >> 2;
            float* to = p.sums + ((size_t)(share * p.tile_count + tile_index) * TC_ROWS + row) * RP + half * WIDTH;
#pragma unroll
            for (int c = 0; c < WIDTH; c += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * WIDTH + c, v);
                tmem_ld_wait();
                if (row < tile.z)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(to + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            }
        } else if (tid == 0 && p.status) {
            atomicOr(p.status, STATUS_WAIT_TIMEOUT);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_free(tmem, S::TMEM1);
}

// y + scale B v of a tile's share of the columns.  Starts under adapter_down_tc_kernel, like adapter_up_kernel.  A x is an operand
// from tensor memory: the shared memory that it took, 32 KB, holds a third block's stages.
template <typename T, int RP, bool FAST>
__global__ void __launch_bounds__(APPLY_THREADS, TcShape<RP>::PER_SM2) adapter_up_tc_kernel(const ApplyArgs p) {
    using S = TcShape<RP>;
    extern __shared__ __align__(128) char smem_raw[];
    __shared__ __align__(8) uint64_t s_done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_pos[TC_ROWS];
    __shared__ float s_unscale[TC_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    char* const ring_ptr = smem_raw + (ring - smem_u32(smem_raw));
    const int tile_index = blockIdx.x / p.col_split, share = blockIdx.x % p.col_split;
    const int4 tile = p.tiles[tile_index];
    const int token = tid < TC_ROWS ? p.rows[tile_index * TC_ROWS + tid] : 0;
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    const float scale = tile.x >= 0 && p.scale ? p.scale[tile.x] : 1.f;
    if (tile.z <= 0 || (rank == 0 && p.out == p.y)) {
        pdl_wait();
        return;
    }
    const int col_stages_all = (p.d_out + S::COLUMNS - 1) / S::COLUMNS;
    const int col_begin = (int)((long long)col_stages_all * share / p.col_split) * S::COLUMNS;
    const int col_end = min(p.d_out, (int)((long long)col_stages_all * (share + 1) / p.col_split) * S::COLUMNS);
    if (tid < tile.z) s_pos[tid] = token;
    if (rank == 0) {                                                // no adapter, or none of its columns
        __syncthreads();
        pdl_wait();
        pdl_trigger();
        copy_rows<T>(p, tile.z, s_pos, col_begin, col_end);
        return;
    }
    if (warp == 0) tmem_alloc(&s_tmem, S::TMEM2);
    if (tid == 0) {
        mbar_init(smem_u32(&s_done), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    constexpr int Y_COPIES = TC_ROWS / 32, B_PIECES = RP / 8, B_ROWS = APPLY_THREADS / B_PIECES;
    constexpr int B_COPIES = (S::COLUMNS + B_ROWS - 1) / B_ROWS;
    const T* const B = static_cast<const T*>(p.b) + (long long)tile.x * p.d_out * p.rank;
    const int piece = tid & 7, row0 = tid >> 3, b_row = tid / B_PIECES, b_piece = tid % B_PIECES;
    const char* y_at[Y_COPIES];
#pragma unroll
    for (int i = 0; i < Y_COPIES; ++i)
        y_at[i] = reinterpret_cast<const char*>(static_cast<const T*>(p.y) + s_pos[min(row0 + 32 * i, tile.z - 1)] * p.ldy + col_begin) + piece * 16;
    const uint32_t y_place = (uint32_t)(row0 * 128 + ((piece ^ (row0 & 7)) << 4));
    const int y_left = (p.d_out - col_begin) * 2 - piece * 16, row_size = p.rank * 2;
    const int b_left = min(16, max(0, rank * 2 - b_piece * 16));    // past the adapter's rank there are zeros
    const char* const b_at = reinterpret_cast<const char*>(B + (long long)(col_begin + b_row) * p.rank) + (b_left > 0 ? b_piece * 16 : 0);
    const int col_stages = (col_end - col_begin + S::COLUMNS - 1) / S::COLUMNS;
    const auto fetch = [&](int n, int slot) {
        if (n < col_stages) {
            const uint32_t to = ring + (uint32_t)slot * S::STAGE2;
            const int left = y_left - n * 128, cols = p.d_out - col_begin - n * S::COLUMNS - b_row;
            if (left > 0)
#pragma unroll
                for (int i = 0; i < Y_COPIES; ++i)
                    if (row0 + 32 * i < tile.z) copy_piece<FAST>(to + y_place + 4096 * i, y_at[i] + (long long)n * 128, left, p.y_grain);
            const char* from = b_at + (long long)n * (S::COLUMNS * row_size);
#pragma unroll
            for (int i = 0; i < B_COPIES; ++i) {
                const int r = b_row + i * B_ROWS;
                if (i * B_ROWS < cols && r < S::COLUMNS)
                    copy_piece<FAST, false>(to + S::Y_BYTES + (b_piece >> 3) * (S::COLUMNS * 128) + r * 128 + (((b_piece & 7) ^ (r & 7)) << 4),
                                            from + i * B_ROWS * row_size, b_left, p.b_grain);
            }
        }
        copies_commit();
    };
#pragma unroll
    for (int c = 0; c < S::S2 - 1; ++c) fetch(c, c);
    pdl_wait();
    pdl_trigger();

    // A x: the shares of all blocks, as first and second parts, through the ring's last slot, which the loop's first turn fills.  The
    // sums by neighbours (a thread has four columns of a row, and of rows ROWS further on), then to tensor memory by rows: a thread
    // half of a row, the one whose lane is its warp's to write.
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    {
        constexpr int PART_ROWS = RP == 128 ? 32 : 64, PITCH = RP * 2 + 16;     // rows at a time, and bytes of a row
        static_assert(2 * PART_ROWS * PITCH <= S::STAGE2, "both parts fit into a slot");
        constexpr int LANES = RP / 4, ROWS = APPLY_THREADS / LANES, PASSES = PART_ROWS / ROWS;
        char* const staged = ring_ptr + (S::S2 - 1) * S::STAGE2;
        const int col = tid % LANES * 4, r0 = tid / LANES;
        const size_t stride = (size_t)p.tile_count * (TC_ROWS * RP);
#pragma unroll 1
        for (int part = 0; part < TC_ROWS; part += PART_ROWS) {
            if (part >= tile.z) break;
            const float* const from = p.sums + ((size_t)tile_index * TC_ROWS + part + r0) * RP + col;
            float4 v[PASSES];
#pragma unroll
            for (int i = 0; i < PASSES; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int q = 0; q < p.k_split; ++q) {
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
                    if (part + r0 + i * ROWS >= tile.z) continue;
                    const float4 o = __ldcg(reinterpret_cast<const float4*>(from + q * stride + i * ROWS * RP));
                    v[i] = make_float4(v[i].x + o.x, v[i].y + o.y, v[i].z + o.z, v[i].w + o.w);
                }
            }
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int r = r0 + i * ROWS;
                if (col >= rank) v[i].x = 0.f;
                if (col + 1 >= rank) v[i].y = 0.f;
                if (col + 2 >= rank) v[i].z = 0.f;
                if (col + 3 >= rank) v[i].w = 0.f;
                if constexpr (std::is_same_v<T, __half>) {          // FP16 has neither BF16's range nor A x a bound
                    float most = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
                    for (int off = LANES / 2; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                    const int e = row_exponent(most);
                    const float up = exp2_int(e);
                    if (col == 0) s_unscale[part + r] = exp2_int(-e);
                    v[i] = make_float4(v[i].x * up, v[i].y * up, v[i].z * up, v[i].w * up);
                }
                char* const to = staged + r * PITCH + col * 2;
                *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<T>(v[i].x, v[i].y), pack_pair<T>(v[i].z, v[i].w));
                *reinterpret_cast<uint2*>(to + PART_ROWS * PITCH) = make_uint2(pack_pair<T>(rest_of<T>(v[i].x), rest_of<T>(v[i].y)),
                                                                               pack_pair<T>(rest_of<T>(v[i].z), rest_of<T>(v[i].w)));
            }
            __syncthreads();
            if ((warp & 3) * 32 / PART_ROWS == part / PART_ROWS) {
#pragma unroll
                for (int c = 0; c < RP; c += 16) {                  // 16 bytes, eight columns of this half
                    const char* at = staged + (row - part) * PITCH + half * RP + c;
                    const uint4 hi = *reinterpret_cast<const uint4*>(at), lo = *reinterpret_cast<const uint4*>(at + PART_ROWS * PITCH);
                    const uint32_t to = lanes + S::COLUMNS + half * (RP / 4) + c / 4;
                    tmem_st4(to, hi.x, hi.y, hi.z, hi.w);
                    tmem_st4(to + RP / 2, lo.x, lo.y, lo.z, lo.w);
                }
                tmem_st_wait();
            }
            __syncthreads();
        }
    }
    const float factor = std::is_same_v<T, __half> && row < tile.z ? scale * s_unscale[row] : scale;
    // the loop's first fences and barrier hand A x to the MMAs

    const uint32_t idesc = make_idesc(TC_ROWS, S::COLUMNS, operand_format<T>());
    bool ok = true;
    int slot = 0, before = S::S2 - 1;
    T* const out_base = static_cast<T*>(p.out);
    for (int c = 0; c < col_stages; ++c) {
        copies_wait<S::S2 - 2>();
        fence_async();
        tc_fence_before();                                          // the sums of the stage before have been read
        __syncthreads();
        tc_fence_after();
        const uint32_t stage = ring + (uint32_t)slot * S::STAGE2;
        if (warp == 0 && ok && elect_one()) {
#pragma unroll
            for (int part = 1; part >= 0; --part)                   // the second parts first
#pragma unroll
                for (int j = 0; j < RP / 16; ++j) {
                    const uint64_t db = make_smem_desc(stage + S::Y_BYTES + j / 4 * (S::COLUMNS * 128)) + 2 * (j & 3);
                    umma_f16_ts(tmem, tmem + S::COLUMNS + part * (RP / 2) + 8 * j, db, idesc, part == 0 || j > 0);
                }
            umma_commit(smem_u32(&s_done));
        }
        if (ok) fetch(c + S::S2 - 1, before);
        else copies_commit();
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_done), c & 1, &s_abort));
        tc_fence_after();
        char* const tile_y = ring_ptr + (stage - ring);
        if (ok) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t sum[16];
                tmem_ld16(lanes + half * 32 + h * 16, sum);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint4* const cell = reinterpret_cast<uint4*>(tile_y + row * 128 + (((half * 4 + h * 2 + i) ^ (row & 7)) << 4));
                    float e[8];
                    unpack16<T>(*cell, e);
#pragma unroll
                    for (int k = 0; k < 8; ++k) e[k] = fmaf(__uint_as_float(sum[i * 8 + k]), factor, e[k]);
                    *cell = pack16<T>(e);
                }
            }
            // Out of shared memory a warp's 32 rows of 64 bytes go to memory four lanes a row (whole sectors), where a lane's own row
            // would be 32 sectors written half.
            __syncwarp();
            const int col0 = col_begin + c * S::COLUMNS + half * 32;
            if (FAST || p.out_vec) {
                const int col = col0 + (lane & 3) * 8;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (warp & 3) * 32 + i * 8 + (lane >> 2);
                    if (r < tile.z && col < p.d_out)
                        *reinterpret_cast<uint4*>(out_base + (long long)s_pos[r] * p.ldo + col) =
                            *reinterpret_cast<const uint4*>(tile_y + r * 128 + (((half * 4 + (lane & 3)) ^ (r & 7)) << 4));
                }
            } else {
                for (int i = 0; i < 32; ++i) {
                    const int r = (warp & 3) * 32 + i;
                    if (r < tile.z && col0 + lane < p.d_out)
                        out_base[(long long)s_pos[r] * p.ldo + col0 + lane] =
                            *reinterpret_cast<const T*>(tile_y + r * 128 + (((half * 4 + lane / 8) ^ (r & 7)) << 4) + lane % 8 * 2);
                }
            }
        }
        before = slot;
        if (++slot == S::S2) slot = 0;
    }
    copies_wait<0>();
    if (!__syncthreads_and(ok) && tid == 0 && p.status) atomicOr(p.status, STATUS_WAIT_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_free(tmem, S::TMEM2);
}

constexpr int SMS = 148;
constexpr int FEW_SHARES = 8, MANY_SHARES = 4;                      // of A x, at most: every block of the second kernel adds them up

// Blocks to a tile: as many as run at once, none with less than a stage.
int split(int tiles, int per_sm, int stages, int most) {
    int n = SMS * per_sm / tiles;
    n = n < most ? n : most;
    n = n < stages ? n : stages;
    return n > 1 ? n : 1;
}

template <typename Down, typename Up>
int launch_pair(Down down, Up up, const ApplyArgs& a, size_t smem1, size_t smem2, cudaStream_t stream) {
    INFMOE_CUDA_TRY(cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem1));
    INFMOE_CUDA_TRY(cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem2));
    INFMOE_CUDA_TRY(launch_chained(down, (unsigned)(a.tile_count * a.k_split), APPLY_THREADS, smem1, 1, stream, a));
    INFMOE_CUDA_TRY(launch_chained(up, (unsigned)(a.tile_count * a.col_split), APPLY_THREADS, smem2, 1, stream, a));
    note_launch(2);
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

template <typename T, int RP, bool FAST>
int launch_few(ApplyArgs a, cudaStream_t stream) {
    using S = ApplyShape<T, RP>;
    a.k_split = split(a.tile_count, S::PER_SM, (a.d_in + S::K_CHUNK - 1) / S::K_CHUNK, FEW_SHARES);
    a.col_split = split(a.tile_count, S::PER_SM, (a.d_out + S::COLUMNS - 1) / S::COLUMNS, 1 << 20);
    return launch_pair(adapter_down_kernel<T, RP, FAST>, adapter_up_kernel<T, RP, FAST>, a, S::SMEM1, S::SMEM2, stream);
}

template <typename T, int RP, bool FAST>
int launch_many(ApplyArgs a, cudaStream_t stream) {
    using S = TcShape<RP>;
    a.k_split = split(a.tile_count, S::PER_SM1, (a.d_in + S::K_CHUNK - 1) / S::K_CHUNK, MANY_SHARES);
    a.col_split = split(a.tile_count, S::PER_SM2, (a.d_out + S::COLUMNS - 1) / S::COLUMNS, 1 << 20);
    return launch_pair(adapter_down_tc_kernel<T, RP, FAST>, adapter_up_tc_kernel<T, RP, FAST>, a, S::SMEM1, S::SMEM2, stream);
}

template <typename T, int RP>
int launch_apply_rank(const ApplyArgs& a, bool many, bool fast, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2 && RP > 16)
        if (many) return fast ? launch_many<T, RP, true>(a, stream) : launch_many<T, RP, false>(a, stream);
    return fast ? launch_few<T, RP, true>(a, stream) : launch_few<T, RP, false>(a, stream);
}

// Tiles of MANY rows or of FEW.  In 16 bits, with many tokens to an adapter, the wide ranks keep mma.sync busier than the memory.
// Measured, FEW and MANY, us, 4096 x 4096 in BF16: rank 16, 16384 tokens 74 and 89; rank 32, 2048 tokens 18 and 26, 4096 tokens
// 36 and 34, 16384 tokens 105 and 91; rank 64, 1024 tokens 21 and 22, 2048 tokens 32 and 30, 4096 tokens 43 and 39.  FP32 has
// three TF32 products to each and stays with FEW.  These lines hold for all widths and go by the adapters that are loaded, not by those that a
// batch uses: 16384 tokens of rank 64 with 1000 loaded and one used stay with FEW.
bool takes_many(long long T, int n, int rank, int dtype) {
    return dtype != INFMOE_F32 && T >= 32ll * n && rank > 16 && T >= (rank > 32 ? 2048 : 4096);
}

int grain_of(const void* p, long long stride_bytes) {
    for (int g = 16; g > 2; g /= 2)
        if ((uintptr_t)p % g == 0 && stride_bytes % g == 0) return g;
    return 2;
}

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Shares of A x: of every tile one, or as many in all as blocks run at once (split).  Does not fall as batches grow, so the workspace of
// the largest serves the others.
size_t workspace_bytes(long long T, int n, int rank, int dtype) {
    const bool many = takes_many(T, n, rank, dtype);
    const int rows = many ? MANY : FEW, rp = padded_rank(rank);
    const long long tiles = max_tiles(T, n, rows), at_once = SMS * (many ? MANY_PER_SM : few_per_sm(rp));
    const long long all = tiles * (many ? MANY_SHARES : FEW_SHARES), most = tiles > at_once ? tiles : at_once;
    return sizeof(float) * (size_t)(all < most ? all : most) * (size_t)rows * (size_t)rp;
}

template <typename T>
int launch_apply(ApplyArgs a, bool many, cudaStream_t stream) {
    const int size = (int)sizeof(T);
    a.x_grain = grain_of(a.x, a.ldx * size);
    a.a_grain = grain_of(a.a, (long long)a.d_in * size);
    a.b_grain = grain_of(a.b, (long long)a.rank * size);
    a.y_grain = grain_of(a.y, a.ldy * size);
    a.out_vec = (long long)a.d_out * size % 16 == 0 && grain_of(a.out, a.ldo * size) == 16;
    const bool fast = a.x_grain == 16 && a.a_grain == 16 && a.b_grain == 16 && a.y_grain == 16 && a.out_vec &&
                      (long long)a.d_in * size % 16 == 0;
    const int rp = padded_rank(a.rank);
    if (rp == 16) return launch_apply_rank<T, 16>(a, many, fast, stream);
    if (rp == 32) return launch_apply_rank<T, 32>(a, many, fast, stream);
    if (rp == 64) return launch_apply_rank<T, 64>(a, many, fast, stream);
    return launch_apply_rank<T, 128>(a, many, fast, stream);
}

int check_plan_size(const char* what, int64_t T, int32_t n) {
    if (T < 0 || n <= 0) {
        set_error("%s: bad argument (T=%lld adapters=%d)", what, (long long)T, n);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    // places in the tables of rows (adapter_rows_kernel and the products) are counted in 32 bits
    if (T > INT_MAX || max_tiles(T, n, MANY) > INT_MAX / MANY || !dispatch_supported(n)) {
        set_error("%s: %lld tokens or %d adapters are more than a plan can hold", what, (long long)T, n);
        return INFMOE_ERR_UNSUPPORTED;
    }
    return INFMOE_OK;
}

}  // namespace

}  // namespace infmoe

using namespace infmoe;

extern "C" {

int infmoe_adapter_plan_bytes(int64_t T, int32_t adapter_count, size_t* bytes) {
    INFMOE_TRY(check_plan_size("adapter_plan_bytes", T, adapter_count));
    if (!bytes) {
        set_error("adapter_plan_bytes: bad argument");
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    *bytes = plan_layout(T, adapter_count).total;
    return INFMOE_OK;
}

int infmoe_adapter_plan(int64_t T, int32_t adapter_count, const int32_t* d_adapter_of_token, void* d_plan, size_t plan_bytes,
                        void* stream) {
    INFMOE_TRY(check_plan_size("adapter_plan", T, adapter_count));
    if (T == 0) return INFMOE_OK;
    const PlanLayout l = plan_layout(T, adapter_count);
    if (!d_adapter_of_token || !d_plan || plan_bytes < l.total || (uintptr_t)d_plan % 16 != 0) {
        set_error("adapter_plan: the plan needs %zu bytes, 16-byte aligned, and the adapter of every token", l.total);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    char* p = static_cast<char*>(d_plan);
    int* offset = reinterpret_cast<int*>(p + l.offset);
    INFMOE_TRY(launch_dispatch(d_adapter_of_token, T, adapter_count, reinterpret_cast<int*>(p),
                               reinterpret_cast<int*>(p + l.count), offset, nullptr, (cudaStream_t)stream));
    const int few = (int)max_tiles(T, adapter_count, FEW), many = (int)max_tiles(T, adapter_count, MANY);
    const auto tiles = [&](const Tiling& t) { return reinterpret_cast<int4*>(p + t.tiles); };
    const auto rows = [&](const Tiling& t) { return reinterpret_cast<int*>(p + t.rows); };
    INFMOE_CUDA_TRY(launch_chained(adapter_tiles_kernel, 2, PLAN_THREADS, 0, 1, (cudaStream_t)stream, T, adapter_count, offset,
                                   tiles(l.few), few, tiles(l.many), many));
    const int few_blocks = (few + MANY / FEW - 1) / (MANY / FEW);
    INFMOE_CUDA_TRY(launch_chained(adapter_rows_kernel, (unsigned)(few_blocks + many), MANY, 0, 1, (cudaStream_t)stream,
                                   reinterpret_cast<const int*>(p), tiles(l.few), rows(l.few), few, tiles(l.many), rows(l.many),
                                   few_blocks));
    note_launch(2);
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

static int check_set(const char* what, const infmoe_adapter_set* set, int64_t T) {
    if (!set || !known_dtype(set->dtype) || set->rank <= 0 || set->d_in <= 0 || set->d_out <= 0 || !set->d_a || !set->d_b) {
        set_error("%s: bad adapter set", what);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    INFMOE_TRY(check_plan_size(what, T, set->adapter_count));
    if (set->rank > INFMOE_ADAPTER_MAX_RANK) {
        set_error("%s: rank %d is larger than %d", what, set->rank, INFMOE_ADAPTER_MAX_RANK);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (set->d_in > MAX_WIDTH || set->d_out > MAX_WIDTH) {
        set_error("%s: rows of %d and %d elements are longer than %d", what, set->d_in, set->d_out, MAX_WIDTH);
        return INFMOE_ERR_UNSUPPORTED;
    }
    return INFMOE_OK;
}

int infmoe_adapter_workspace_bytes(const infmoe_adapter_set* set, int64_t T, size_t* bytes) {
    INFMOE_TRY(check_set("adapter_workspace_bytes", set, T));
    if (!bytes) {
        set_error("adapter_workspace_bytes: bad argument");
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    *bytes = workspace_bytes(T, set->adapter_count, set->rank, set->dtype);
    return INFMOE_OK;
}

int infmoe_adapter_apply(const infmoe_adapter_set* set, int64_t T, const void* d_x, int64_t ldx, const void* d_y, int64_t ldy,
                         void* d_out, int64_t ldo, const void* d_plan, void* d_workspace, size_t ws_bytes, int32_t* d_status,
                         void* stream) {
    INFMOE_TRY(check_set("adapter_apply", set, T));
    if (T == 0) return INFMOE_OK;
    const size_t need = workspace_bytes(T, set->adapter_count, set->rank, set->dtype);
    if (!d_workspace || ws_bytes < need || (uintptr_t)d_workspace % 16 != 0) {
        set_error("adapter_apply: the workspace needs %zu bytes, 16-byte aligned", need);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    if (!d_x || !d_y || !d_out || !d_plan || ldx < set->d_in || ldy < set->d_out || ldo < set->d_out || d_x == d_out ||
        (d_y == d_out && ldy != ldo) || (uintptr_t)d_plan % 16 != 0) {
        set_error("adapter_apply: bad argument (row strides %lld, %lld, %lld; d_out may be d_y, with its stride, but not d_x)",
                  (long long)ldx, (long long)ldy, (long long)ldo);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    const PlanLayout l = plan_layout(T, set->adapter_count);
    const char* plan = static_cast<const char*>(d_plan);
    ApplyArgs a{};
    a.x = d_x;
    a.y = d_y;
    a.a = set->d_a;
    a.b = set->d_b;
    a.out = d_out;
    a.ldx = ldx;
    a.ldy = ldy;
    a.ldo = ldo;
    a.rank = set->rank;
    a.d_in = set->d_in;
    a.d_out = set->d_out;
    a.scale = set->d_scale;
    a.rank_of = set->d_rank;
    const bool many = takes_many(T, set->adapter_count, set->rank, set->dtype);
    const Tiling& tiling = many ? l.many : l.few;
    a.tiles = reinterpret_cast<const int4*>(plan + tiling.tiles);
    a.rows = reinterpret_cast<const int*>(plan + tiling.rows);
    a.tile_count = (int)max_tiles(T, set->adapter_count, many ? MANY : FEW);
    a.sums = static_cast<float*>(d_workspace);
    a.status = d_status;
    if (set->dtype == INFMOE_F32) return launch_apply<float>(a, many, (cudaStream_t)stream);
    if (set->dtype == INFMOE_F16) return launch_apply<__half>(a, many, (cudaStream_t)stream);
    return launch_apply<__nv_bfloat16>(a, many, (cudaStream_t)stream);
}

}  // extern "C"
