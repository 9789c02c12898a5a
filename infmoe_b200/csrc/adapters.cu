// Low-rank adapters of many requests at once, beside a shared projection: out[t] = y[t] + scale[a] B[a] (A[a] x[t]) with
// a the adapter of token t.  Tokens are grouped by adapter with the layer's own dispatch (an adapter takes the place of an
// expert); the plan that comes of it holds for every projection of the batch.
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace infmoe {

namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int APPLY_THREADS = 256;
constexpr int APPLY_WARPS = APPLY_THREADS / 32;
constexpr int MAX_WIDTH = 1 << 24;   // of x and y: places in a row are counted in bytes in 32 bits

// Most rows of a tile, all of which have the same adapter: 16 where tokens are few next to the adapters, which generating
// batches are, else 64.
int tile_rows(long long T, int n) { return T < 32ll * n ? 16 : 64; }
// Tiles of a batch: whole tiles of every adapter and what is left of each, and those of the tokens without one.
long long max_tiles(long long T, int n) {
    const long long kinds = (long long)n + 1;
    return T / tile_rows(T, n) + (T < kinds ? T : kinds);
}

struct PlanLayout {
    size_t pos, offset, count, tiles, total;
};
PlanLayout plan_layout(long long T, int n) {
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    PlanLayout p{};
    p.offset = up(sizeof(int) * (size_t)T);
    p.count = p.offset + up(sizeof(int) * ((size_t)n + 1));
    p.tiles = p.count + up(sizeof(int) * (size_t)n);
    p.total = p.tiles + up(sizeof(int4) * (size_t)max_tiles(T, n));
    return p;
}

// tiles[i] = {adapter (-1: none), first row of expert order, rows, 0}; rows = 0 behind the last tile.
__global__ void __launch_bounds__(PLAN_THREADS)
adapter_tiles_kernel(long long T, int n, int tile_rows, const int* offset, int4* __restrict__ tiles, int capacity) {
    pdl_trigger();
    pdl_wait();
    __shared__ int s_sum[32];
    __shared__ int s_base;
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

struct ApplyArgs {
    const void *x, *y, *a, *b;
    void* out;
    long long ldx, ldy, ldo;
    int rank, d_in, d_out;
    const float* scale;       // [adapters] or NULL: 1
    const int* rank_of;       // [adapters] or NULL: all `rank`
    const int* pos;
    const int4* tiles;
    int x_grain, a_grain, b_grain, y_grain;   // bytes of one copy to shared memory: 16, 8, 4, or 2 (ordinary loads)
    int out_vec;              // out is written 16 bytes at a time
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// The 16 bytes at dst come from src, those from byte `left` on are zero.  src is a multiple of grain.  FAST: it is one of 16, and
// so is left.
template <bool FAST>
__device__ __forceinline__ void copy_piece(uint32_t dst, const char* src, int left, int grain) {
    if (FAST) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(left > 0 ? 16 : 0) : "memory");
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

// An FP32 value as two of 11 significant bits, the second of which the tensor core cuts off behind the eleventh: 2^-21 of the
// value is left out at most.  An infinity has no second part.
__device__ __forceinline__ void split_tf32(const uint32_t v, uint32_t& hi, uint32_t& lo) {
    hi = v & 0xffffe000u;
    const float rest = __fsub_rn(__uint_as_float(v), __uint_as_float(hi));      // NaN for NaN
    lo = (v & 0x7fffffffu) == 0x7f800000u ? 0u : __float_as_uint(rest);
}

// What is left of v after its rounding to T (0 where that is no finite value).
template <typename T>
__device__ __forceinline__ float rest_of(float v) {
    const float h = to_float(from_float<T>(v));
    return fabsf(h) <= FLT_MAX ? __fsub_rn(v, h) : 0.f;
}

// Shared memory of a block is one ring, used twice.  First product: stages of M rows of x and RP rows of A, 128 bytes of K each,
// for M = 16 twice that, so that each of the warps has a 32-byte step (or two) of K.  Second product: stages of COLUMNS columns,
// M rows of y and COLUMNS rows of B, so that each of the warps has a unit of 16 rows and 32 columns (or every other time).
template <typename T, int RP, int M>
struct ApplyShape {
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr int SIZE = (int)sizeof(T);
    static constexpr int M_TILES = M / 16, K_GROUPS = APPLY_WARPS / M_TILES;
    static constexpr int SUBS = M == 16 ? 2 : 1;                    // 128-byte parts of K in a stage
    static constexpr int K_CHUNK = SUBS * 128 / SIZE;
    static constexpr int STAGE1 = SUBS * (M + RP) * 128;
    static constexpr int UNITS = M == 64 ? 2 : RP * SIZE >= 128 ? 4 : 8;
    static constexpr int COLUMNS = UNITS * 32;
    static constexpr int Y_PIECES = COLUMNS * SIZE / 16, B_PIECES = RP * SIZE / 16;   // 16-byte pieces of a row of y, of B
    static constexpr int Y_BYTES = M * Y_PIECES * 16;
    static constexpr int STAGE2 = Y_BYTES + COLUMNS * B_PIECES * 16;
    static constexpr int PART = APPLY_WARPS * 16 * RP * 4;          // the warps' sums of the first product, at the ring's end
    static constexpr int BUDGET = (M == 16 && RP <= 32 ? 48 : RP <= 32 ? 64 : RP == 64 ? 84 : WIDE ? 144 : 72) * 1024;
    static constexpr int clamp_stages(int n) { return n < 2 ? 2 : n > 8 ? 8 : n; }
    static constexpr int S1 = clamp_stages(BUDGET / STAGE1), S2 = clamp_stages(BUDGET / STAGE2);
    static constexpr int larger(int a, int b) { return a > b ? a : b; }
    static constexpr int RING = larger(PART, larger(S1 * STAGE1, S2 * STAGE2));
    static constexpr int EARLY = (RING - PART) / STAGE2 < S2 - 1 ? (RING - PART) / STAGE2 : S2 - 1;   // stages of the second
                                                                    // product that are fetched while the first one's are summed up
    static constexpr int V_ROW = RP * SIZE + 16;                    // bytes of a row of A x; the padding spreads rows over the banks
    static constexpr int V_BYTES = M * V_ROW;                       // 16 bits: once more for the second parts
    static constexpr int SMEM = RING + (WIDE ? 1 : 2) * V_BYTES;

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

// FAST: x, A, B and y are copied, and out written, in whole pieces of 16 bytes.
template <typename T, int RP, int M, bool FAST>
__global__ void __launch_bounds__(APPLY_THREADS, M == 16 && RP <= 32 ? 3 : 1) adapter_apply_kernel(const ApplyArgs p) {
    using S = ApplyShape<T, RP, M>;
    constexpr bool WIDE = S::WIDE;
    constexpr int SIZE = S::SIZE;
    extern __shared__ __align__(128) char smem[];
    __shared__ float s_unscale[M];
    __shared__ int s_pos[M];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank_in_cluster = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    const int4 tile = p.tiles[blockIdx.x / C];
    if (tile.z == 0 || (tile.x < 0 && p.out == p.y)) return;        // all blocks of the cluster alike
    if (tid < tile.z) s_pos[tid] = p.pos[tile.y + tid];
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    const float scale = tile.x >= 0 && p.scale ? p.scale[tile.x] : 1.f;
    __syncthreads();

    // this block's columns of y
    const int col_stages_all = (p.d_out + S::COLUMNS - 1) / S::COLUMNS;
    const int col_begin = (int)((long long)col_stages_all * rank_in_cluster / C) * S::COLUMNS;
    const int col_end = min(p.d_out, (int)((long long)col_stages_all * (rank_in_cluster + 1) / C) * S::COLUMNS);
    const T* const y_base = static_cast<const T*>(p.y);
    T* const out_base = static_cast<T*>(p.out);
    if (rank == 0) {                                                // no adapter, or none of its columns
        if (p.out == p.y) return;
        constexpr int N = 16 / SIZE;
        const bool vec = p.out_vec && p.y_grain == 16;
        for (int r = warp; r < tile.z; r += APPLY_WARPS) {
            const T* src = y_base + s_pos[r] * p.ldy;
            T* dst = out_base + s_pos[r] * p.ldo;
            if (vec)
                for (int c = col_begin + lane * N; c < col_end; c += 32 * N)
                    *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
            else
                for (int c = col_begin + lane; c < col_end; c += 32) dst[c] = src[c];
        }
        return;
    }
    const T* const A = static_cast<const T*>(p.a) + (long long)tile.x * p.rank * p.d_in;
    const T* const B = static_cast<const T*>(p.b) + (long long)tile.x * p.d_out * p.rank;
    const uint32_t ring = smem_u32(smem);
    const int m = warp % S::M_TILES, k_group = warp / S::M_TILES;   // a warp's 16 rows, and its share of K and of the units
    const bool has_rows = m * 16 < tile.z;

    // ---- A x: this block's part of d_in ----
    const int stages_all = (p.d_in + S::K_CHUNK - 1) / S::K_CHUNK;
    const int stage_begin = (int)((long long)stages_all * rank_in_cluster / C);
    const int stages = (int)((long long)stages_all * (rank_in_cluster + 1) / C) - stage_begin;
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
    // the first of what the second product needs is on its way to L2 meanwhile: a warp takes rows of y, the block the part of B
    {
        const int columns = min(col_end - col_begin, 1024 / SIZE);
        const char* b0 = reinterpret_cast<const char*>(B + (long long)col_begin * p.rank);
        const int bytes = columns * p.rank * SIZE;
        for (int i = tid * 128; i < bytes; i += APPLY_THREADS * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(b0 + i));
        for (int r = warp; r < tile.z; r += APPLY_WARPS) {
            const char* y0 = reinterpret_cast<const char*>(y_base + s_pos[r] * p.ldy + col_begin);
            if (lane * 128 < columns * SIZE) asm volatile("prefetch.global.L2 [%0];" ::"l"(y0 + lane * 128));
        }
    }
    const int xr = m * 16 + (lane & 15), wr = (lane & 7) + ((lane >> 4) << 3);
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
        if (has_rows) {
            if constexpr (M == 64) {
                multiply(stage, k_group);
                multiply(stage, k_group + 2);
            } else {
                multiply(stage + (k_group >> 2) * (M + RP) * 128, k_group & 3);
            }
        }
        read = read + 1 == S::S1 ? 0 : read + 1;
        fill = fill + 1 == S::S1 ? 0 : fill + 1;
    }
    copies_wait<0>();
    __syncthreads();

    // the second product's stages, fetched like the first one's
    constexpr int Y_COPIES = M * S::Y_PIECES / APPLY_THREADS;
    constexpr int B_COPIES = (S::COLUMNS * S::B_PIECES + APPLY_THREADS - 1) / APPLY_THREADS;
    constexpr int Y_ROWS = APPLY_THREADS / S::Y_PIECES, B_ROWS = APPLY_THREADS / S::B_PIECES;   // rows between a thread's copies
    const char* y_at[Y_COPIES];
    const int y_row = tid / S::Y_PIECES, y_piece = tid % S::Y_PIECES, b_row = tid / S::B_PIECES, b_piece = tid % S::B_PIECES;
#pragma unroll
    for (int i = 0; i < Y_COPIES; ++i)
        y_at[i] = reinterpret_cast<const char*>(y_base + s_pos[min(y_row + i * Y_ROWS, tile.z - 1)] * p.ldy + col_begin) + y_piece * 16;
    const int y_left = (p.d_out - col_begin) * SIZE - y_piece * 16;
    const int b_left = rank * SIZE - b_piece * 16;                  // past the adapter's rank there are zeros
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
                    copy_piece<FAST>(to + S::Y_BYTES + S::b_place(b_row + i * B_ROWS, b_piece) * 16, from + i * B_ROWS * row_size, b_left, p.b_grain);
        }
        copies_commit();
    };
#pragma unroll
    for (int c = 0; c < S::EARLY; ++c) fetch_columns(c, c);

    // ---- sums over the warps of an m tile, then over the cluster ----
    float* const part = reinterpret_cast<float*>(smem + S::RING - S::PART);             // [K_GROUPS][M][RP]
#pragma unroll
    for (int j = 0; j < RP / 8; ++j) {
        float* at = part + (k_group * M + m * 16 + (lane >> 2)) * RP + j * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(at + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = tid; i < tile.z * RP; i += APPLY_THREADS) {
        float sum = part[i];
#pragma unroll
        for (int g = 1; g < S::K_GROUPS; ++g) sum += part[g * M * RP + i];
        part[i] = sum;
    }
    cluster.sync();
    char* const v_smem = smem + S::RING;
    for (int r = rank_in_cluster + C * warp; r < tile.z; r += C * APPLY_WARPS) {
        // a warp sums up a row and gives it to all blocks: lane l has columns 2 l, 2 l + 1 (and 64 more each)
        constexpr int STEPS = (RP / 2 + 31) / 32;
        float2 v[STEPS];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int col = 2 * (lane + 32 * i);
            v[i] = make_float2(0.f, 0.f);
            if (col < RP) {
                float2 o[8];                                        // of the blocks, all in flight
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < C) o[q] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, q) + r * RP + col);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < C) {
                        v[i].x += o[q].x;
                        v[i].y += o[q].y;
                    }
                if (col >= rank) v[i].x = 0.f;
                if (col + 1 >= rank) v[i].y = 0.f;
            }
            most = fmaxf(most, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        }
        float unscale = 1.f;
        if constexpr (std::is_same_v<T, __half>) {                  // FP16 has neither BF16's range nor A x a bound
            const int e = row_exponent(warp_max(most));
            unscale = exp2_int(-e);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                v[i].x *= exp2_int(e);
                v[i].y *= exp2_int(e);
            }
        }
        for (int q = 0; q < C; ++q) {
            char* to = cluster.map_shared_rank(v_smem, q) + r * S::V_ROW;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int col = 2 * (lane + 32 * i);
                if (col >= RP) continue;
                if constexpr (WIDE) {
                    *reinterpret_cast<float2*>(to + 4 * col) = v[i];
                } else {
                    *reinterpret_cast<uint32_t*>(to + 2 * col) = pack_pair<T>(v[i].x, v[i].y);
                    *reinterpret_cast<uint32_t*>(to + S::V_BYTES + 2 * col) = pack_pair<T>(rest_of<T>(v[i].x), rest_of<T>(v[i].y));
                }
            }
            if (lane == 0) cluster.map_shared_rank(s_unscale, q)[r] = unscale;
        }
    }
    cluster.sync();                    // behind it no block touches another's memory

    // ---- y + scale B v: this block's columns, a warp one m tile of every K_GROUPS-th unit ----
#pragma unroll
    for (int c = S::EARLY; c < S::S2 - 1; ++c) fetch_columns(c, c);
    constexpr int STEPS = RP * SIZE / 32;                           // 32-byte steps of K
    constexpr bool HOLD = STEPS <= 4;                               // A x stays in registers
    const int g = lane >> 2, q = lane & 3;
    T* out_row[2];
    bool row_ok[2];
    float factor[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = m * 16 + g + 8 * h;
        row_ok[h] = r < tile.z;
        out_row[h] = out_base + (long long)s_pos[row_ok[h] ? r : 0] * p.ldo + col_begin + q * 8;
        factor[h] = std::is_same_v<T, __half> && row_ok[h] ? s_unscale[r] * scale : scale;
    }
    const uint32_t v_addr = smem_u32(v_smem) + xr * S::V_ROW + ((lane >> 4) << 4);
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
    const int u = k_group % S::UNITS;                               // the warp's unit of every stage, or of every other one
    uint32_t cell[2][8 / N];                                        // its pieces of y
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) cell[h][i] = S::y_place(m * 16 + g + 8 * h, u * (32 / N) + q * (8 / N) + i) * 16;
#pragma unroll
    for (int s = 0; s < (STEPS < 4 ? STEPS : 4); ++s) b_step_at[s] += (uint32_t)u * (32 * S::B_PIECES * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) out_row[h] += u * 32;
    read = 0;
    fill = S::S2 - 1;
    for (int c = 0; c < col_stages; ++c) {
        copies_wait<S::S2 - 2>();
        __syncthreads();
        fetch_columns(c + S::S2 - 1, fill);
        const uint32_t slot = (uint32_t)read * S::STAGE2;
        read = read + 1 == S::S2 ? 0 : read + 1;
        fill = fill + 1 == S::S2 ? 0 : fill + 1;
        if (has_rows && (S::UNITS == S::K_GROUPS || (c & 1) == k_group / S::UNITS)) {
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

template <typename T, int RP, int M, bool FAST>
int launch_apply_kernel(const ApplyArgs& a, long long tiles, cudaStream_t stream) {
    using S = ApplyShape<T, RP, M>;
    const auto kernel = adapter_apply_kernel<T, RP, M, FAST>;
    INFMOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    // Blocks of a cluster share out K, then the columns of y: as many as run at once, up to 8, and none without work.
    const int k_stages = (a.d_in + S::K_CHUNK - 1) / S::K_CHUNK, col_stages = (a.d_out + S::COLUMNS - 1) / S::COLUMNS;
    const long long at_once = 148ll * (S::SMEM <= 55 * 1024 ? 4 : S::SMEM <= 74 * 1024 ? 3 : S::SMEM <= 112 * 1024 ? 2 : 1);
    unsigned cluster = 1;
    while (cluster < 8 && tiles * cluster * 2 <= at_once && (int)cluster * 2 <= (k_stages > col_stages ? k_stages : col_stages))
        cluster *= 2;
    INFMOE_CUDA_TRY(launch_chained(kernel, (unsigned)tiles * cluster, APPLY_THREADS, S::SMEM, cluster, stream, a));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

template <typename T, int RP>
int launch_apply_rank(const ApplyArgs& a, int rows, bool fast, long long tiles, cudaStream_t stream) {
    if (rows == 16)
        return fast ? launch_apply_kernel<T, RP, 16, true>(a, tiles, stream) : launch_apply_kernel<T, RP, 16, false>(a, tiles, stream);
    return fast ? launch_apply_kernel<T, RP, 64, true>(a, tiles, stream) : launch_apply_kernel<T, RP, 64, false>(a, tiles, stream);
}

int grain_of(const void* p, long long stride_bytes) {
    for (int g = 16; g > 2; g /= 2)
        if ((uintptr_t)p % g == 0 && stride_bytes % g == 0) return g;
    return 2;
}

template <typename T>
int launch_apply(ApplyArgs a, int rows, long long tiles, cudaStream_t stream) {
    const int size = (int)sizeof(T);
    a.x_grain = grain_of(a.x, a.ldx * size);
    a.a_grain = grain_of(a.a, (long long)a.d_in * size);
    a.b_grain = grain_of(a.b, (long long)a.rank * size);
    a.y_grain = grain_of(a.y, a.ldy * size);
    a.out_vec = (long long)a.d_out * size % 16 == 0 && grain_of(a.out, a.ldo * size) == 16;
    const bool fast = a.x_grain == 16 && a.a_grain == 16 && a.b_grain == 16 && a.y_grain == 16 && a.out_vec &&
                      (long long)a.d_in * size % 16 == 0 && !a.rank_of;
    if (a.rank <= 16) return launch_apply_rank<T, 16>(a, rows, fast, tiles, stream);
    if (a.rank <= 32) return launch_apply_rank<T, 32>(a, rows, fast, tiles, stream);
    if (a.rank <= 64) return launch_apply_rank<T, 64>(a, rows, fast, tiles, stream);
    return launch_apply_rank<T, 128>(a, rows, fast, tiles, stream);
}

int check_plan_size(const char* what, int64_t T, int32_t n) {
    if (T < 0 || n <= 0) {
        set_error("%s: bad argument (T=%lld adapters=%d)", what, (long long)T, n);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    if (T > INT_MAX || !dispatch_supported(n)) {
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
    INFMOE_CUDA_TRY(launch_chained(adapter_tiles_kernel, 1, PLAN_THREADS, 0, 1, (cudaStream_t)stream, T, adapter_count,
                                   tile_rows(T, adapter_count), offset, reinterpret_cast<int4*>(p + l.tiles), (int)max_tiles(T, adapter_count)));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

int infmoe_adapter_apply(const infmoe_adapter_set* set, int64_t T, const void* d_x, int64_t ldx, const void* d_y, int64_t ldy,
                         void* d_out, int64_t ldo, const void* d_plan, void* stream) {
    if (!set || !known_dtype(set->dtype) || set->rank <= 0 || set->d_in <= 0 || set->d_out <= 0 || !set->d_a || !set->d_b) {
        set_error("adapter_apply: bad adapter set");
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    INFMOE_TRY(check_plan_size("adapter_apply", T, set->adapter_count));
    if (set->rank > INFMOE_ADAPTER_MAX_RANK) {
        set_error("adapter_apply: rank %d is larger than %d", set->rank, INFMOE_ADAPTER_MAX_RANK);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (set->d_in > MAX_WIDTH || set->d_out > MAX_WIDTH) {
        set_error("adapter_apply: rows of %d and %d elements are longer than %d", set->d_in, set->d_out, MAX_WIDTH);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (T == 0) return INFMOE_OK;
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
    a.pos = reinterpret_cast<const int*>(plan + l.pos);
    a.tiles = reinterpret_cast<const int4*>(plan + l.tiles);
    const long long tiles = max_tiles(T, set->adapter_count);
    const int rows = tile_rows(T, set->adapter_count);
    if (set->dtype == INFMOE_F32) return launch_apply<float>(a, rows, tiles, (cudaStream_t)stream);
    if (set->dtype == INFMOE_F16) return launch_apply<__half>(a, rows, tiles, (cudaStream_t)stream);
    return launch_apply<__nv_bfloat16>(a, rows, tiles, (cudaStream_t)stream);
}

}  // extern "C"
