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

constexpr int TILE_ROWS = 64;      // most rows of a tile; all rows of a tile have the same adapter
constexpr int PLAN_THREADS = 1024;
constexpr int APPLY_THREADS = 256;

// Tiles of a batch: whole tiles of every adapter and what is left of each, and those of the tokens without one.
long long max_tiles(long long T, int n) {
    const long long kinds = (long long)n + 1;
    return T / TILE_ROWS + (T < kinds ? T : kinds);
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
adapter_tiles_kernel(long long T, int n, const int* offset, int4* __restrict__ tiles, int capacity) {
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
        const int mine = (rows + TILE_ROWS - 1) / TILE_ROWS;
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
                tiles[at + i] = make_int4(a < n ? a : -1, begin + i * TILE_ROWS, min(TILE_ROWS, rows - i * TILE_ROWS), 0);
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
    int x_grain, a_grain;     // bytes of one copy of x and of A: 16, 8, 4, or 2 (ordinary loads)
    int b_vec, y_vec;         // B is read, and y and out are accessed, 16 bytes (B of rank 16 in FP16 / BF16: 8) at a time
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// `bytes` of the 16 at dst come from src, the others are zero; src is a multiple of grain.
__device__ __forceinline__ void copy_piece(uint32_t dst, const char* src, int bytes, int grain) {
    if (grain == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    } else if (grain == 8) {
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            const int n = min(8, max(0, bytes - i));
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i), "l"(src + (n ? i : 0)), "r"(n) : "memory");
        }
    } else if (grain == 4) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int n = min(4, max(0, bytes - i));
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i), "l"(src + (n ? i : 0)), "r"(n) : "memory");
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(src) + 2 * i;
            const uint32_t lo = 4 * i < bytes ? p[0] : 0, hi = 4 * i + 2 < bytes ? p[1] : 0;
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
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if constexpr (std::is_same_v<T, __nv_bfloat16>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An FP32 value as two of 11 significant bits; what does not fit into the first one's range has no second.
__device__ __forceinline__ void split_tf32(uint32_t v, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(v)));
    const float h = __uint_as_float(hi);
    const float rest = fabsf(h) <= FLT_MAX ? __fsub_rn(__uint_as_float(v), h) : 0.f;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    union {
        T e[2];
        uint32_t w;
    } u;
    u.e[0] = from_float<T>(a);
    u.e[1] = from_float<T>(b);
    return u.w;
}
// What is left of v after its rounding to T (0 where that is no finite value).
template <typename T>
__device__ __forceinline__ float rest_of(float v) {
    const float h = to_float(from_float<T>(v));
    return fabsf(h) <= FLT_MAX ? __fsub_rn(v, h) : 0.f;
}

template <typename T, int RP>
struct ApplyShape {
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr int CHUNK = 128 / (int)sizeof(T);              // values of K in a stage
    static constexpr int STAGES = RP >= 128 ? 4 : RP >= 64 ? 4 : 6;
    static constexpr int STAGE_BYTES = (TILE_ROWS + RP) * 128;
    static constexpr int V_ROW = RP * (int)sizeof(T) + 16;          // bytes of a row of A x; the padding spreads rows over the banks
    static constexpr int V_BYTES = TILE_ROWS * V_ROW;               // 16 bits: once more for the second parts
    static constexpr int SMEM = STAGES * STAGE_BYTES + (WIDE ? 1 : 2) * V_BYTES;
    static constexpr int GROUP = RP / 4;                            // consecutive values of a B row that a lane reads
    static_assert(512 * RP <= STAGES * STAGE_BYTES, "the warps' sums take the place of the stages");
};

template <typename T, int RP>
__global__ void __launch_bounds__(APPLY_THREADS) adapter_apply_kernel(const ApplyArgs p) {
    using S = ApplyShape<T, RP>;
    constexpr bool WIDE = S::WIDE;
    extern __shared__ __align__(128) char smem[];
    __shared__ float s_unscale[TILE_ROWS];
    __shared__ int s_pos[TILE_ROWS];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank_in_cluster = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    const int4 tile = p.tiles[blockIdx.x / C];
    if (tile.z == 0 || (tile.x < 0 && p.out == p.y)) return;        // all blocks of the cluster alike
    if (tid < tile.z) s_pos[tid] = p.pos[tile.y + tid];
    __syncthreads();

    // this block's columns of y: whole units of 32
    const int units = (p.d_out + 31) / 32;
    const int unit_begin = (int)((long long)units * rank_in_cluster / C), unit_end = (int)((long long)units * (rank_in_cluster + 1) / C);
    const T* const y_base = static_cast<const T*>(p.y);
    T* const out_base = static_cast<T*>(p.out);
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    if (rank == 0) {                                                // no adapter, or none of its columns
        if (p.out == p.y) return;
        const int c0 = unit_begin * 32, c1 = min(p.d_out, unit_end * 32);
        constexpr int N = 16 / (int)sizeof(T);
        for (int r = warp; r < tile.z; r += APPLY_THREADS / 32) {
            const T* src = y_base + s_pos[r] * p.ldy;
            T* dst = out_base + s_pos[r] * p.ldo;
            if (p.y_vec)
                for (int c = c0 + lane * N; c < c1; c += 32 * N)
                    *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
            else
                for (int c = c0 + lane; c < c1; c += 32) dst[c] = src[c];
        }
        return;
    }
    const T* const A = static_cast<const T*>(p.a) + (long long)tile.x * p.rank * p.d_in;
    const T* const B = static_cast<const T*>(p.b) + (long long)tile.x * p.d_out * p.rank;

    // ---- A x: this block's part of d_in ----
    const int chunks_all = (p.d_in + S::CHUNK - 1) / S::CHUNK;
    const int chunk_begin = (int)((long long)chunks_all * rank_in_cluster / C), chunks = (int)((long long)chunks_all * (rank_in_cluster + 1) / C) - chunk_begin;
    const uint32_t stages = smem_u32(smem);
    // a thread copies the same 16 bytes of every stage's rows tid / 8, tid / 8 + 32, ...
    const int piece = tid & 7, row0 = tid >> 3;
    const auto fetch = [&](int chunk) {
        if (chunk < chunks) {
            const uint32_t stage = stages + (uint32_t)(chunk % S::STAGES) * S::STAGE_BYTES;
            const long long k = (long long)(chunk_begin + chunk) * S::CHUNK + piece * (16 / (int)sizeof(T));
            const int bytes = (int)min(16ll, max(0ll, (p.d_in - k) * (long long)sizeof(T)));
            const long long at = bytes ? k : 0;
#pragma unroll
            for (int i = 0; i < TILE_ROWS / 32; ++i) {
                const int r = row0 + 32 * i;
                if (r < tile.z)
                    copy_piece(stage + r * 128 + ((piece ^ (r & 7)) << 4),
                               reinterpret_cast<const char*>(static_cast<const T*>(p.x) + s_pos[r] * p.ldx + at), bytes, p.x_grain);
            }
#pragma unroll
            for (int i = 0; i < (RP + 31) / 32; ++i) {
                const int r = row0 + 32 * i;
                if (r < rank)
                    copy_piece(stage + (TILE_ROWS + r) * 128 + ((piece ^ (r & 7)) << 4),
                               reinterpret_cast<const char*>(A + (long long)r * p.d_in + at), bytes, p.a_grain);
            }
        }
        copies_commit();
    };
    // warps: m tiles of 16 rows, and for each of them a share of the 32-byte steps of K
    const int m_tiles = tile.z > 32 ? 4 : tile.z > 16 ? 2 : 1, k_groups = 8 / m_tiles;
    const int m = warp % m_tiles, k_group = warp / m_tiles;
    const int n_pairs = (rank + 15) / 16;
    float acc[RP / 8][4];
#pragma unroll
    for (int j = 0; j < RP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
#pragma unroll
    for (int c = 0; c < S::STAGES - 1; ++c) fetch(c);
    // what the second product needs is on its way to L2 meanwhile
    {
        const char* b0 = reinterpret_cast<const char*>(B + (long long)unit_begin * 32 * p.rank);
        const long long bytes = ((long long)min(p.d_out, unit_end * 32) - unit_begin * 32) * p.rank * (long long)sizeof(T);
        for (long long i = (long long)tid * 128; i < bytes; i += APPLY_THREADS * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(b0 + i));
        const int row_bytes = (min(p.d_out, unit_end * 32) - unit_begin * 32) * (int)sizeof(T), lines = (row_bytes + 127) / 128;
        for (int i = tid; i < lines * tile.z; i += APPLY_THREADS) {
            const int r = i / lines, l = i - r * lines;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(y_base + s_pos[r] * p.ldy + unit_begin * 32) + l * 128));
        }
    }
    for (int c = 0; c < chunks; ++c) {
        copies_wait<S::STAGES - 2>();
        __syncthreads();               // the stage is complete, and everybody is done with the one that is filled next
        fetch(c + S::STAGES - 1);
        const uint32_t stage = stages + (uint32_t)(c % S::STAGES) * S::STAGE_BYTES;
        const bool mine = m * 16 < tile.z;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (!mine || ((c * 4 + s) & (k_groups - 1)) != k_group) continue;
            uint32_t x[4];
            const int xr = m * 16 + (lane & 15);
            load_matrices(x, stage + xr * 128 + (((2 * s + (lane >> 4)) ^ (xr & 7)) << 4));
            uint32_t x_hi[4], x_lo[4];
            if constexpr (WIDE)
#pragma unroll
                for (int i = 0; i < 4; ++i) split_tf32(x[i], x_hi[i], x_lo[i]);
#pragma unroll
            for (int n = 0; n < RP / 16; ++n) {
                if (n >= n_pairs) break;
                uint32_t w[4];
                const int wr = n * 16 + (lane & 7) + ((lane >> 4) << 3);
                load_matrices(w, stage + (TILE_ROWS + wr) * 128 + (((2 * s + ((lane >> 3) & 1)) ^ (wr & 7)) << 4));
                if constexpr (WIDE) {
                    uint32_t w_hi[4], w_lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(w[i], w_hi[i], w_lo[i]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma<T>(acc[2 * n + h], x_lo, w_hi[2 * h], w_hi[2 * h + 1]);
                        mma<T>(acc[2 * n + h], x_hi, w_lo[2 * h], w_lo[2 * h + 1]);
                        mma<T>(acc[2 * n + h], x_hi, w_hi[2 * h], w_hi[2 * h + 1]);
                    }
                } else {
                    mma<T>(acc[2 * n], x, w[0], w[1]);
                    mma<T>(acc[2 * n + 1], x, w[2], w[3]);
                }
            }
        }
    }
    copies_wait<0>();
    __syncthreads();

    // ---- sums over the warps of an m tile, then over the cluster ----
    float* const part = reinterpret_cast<float*>(smem);             // [k_groups][m_tiles * 16][RP]
    const int part_rows = m_tiles * 16;
#pragma unroll
    for (int j = 0; j < RP / 8; ++j) {
        float* at = part + ((size_t)k_group * part_rows + m * 16 + (lane >> 2)) * RP + j * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(at + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = tid; i < tile.z * RP; i += APPLY_THREADS) {
        float sum = part[i];
        for (int g = 1; g < k_groups; ++g) sum += part[(size_t)g * part_rows * RP + i];
        part[i] = sum;
    }
    cluster.sync();
    char* const v_smem = smem + S::STAGES * S::STAGE_BYTES;
    for (int r = rank_in_cluster + C * warp; r < tile.z; r += C * (APPLY_THREADS / 32)) {
        // a warp sums up a row and gives it to all blocks: lane l has columns 2 l, 2 l + 1 (and 64 more each)
        constexpr int PAIRS = RP / 2, STEPS = (PAIRS + 31) / 32;
        float2 v[STEPS];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int col = 2 * (lane + 32 * i);
            v[i] = make_float2(0.f, 0.f);
            if (col < RP) {
                for (int q = 0; q < C; ++q) {
                    const float2 o = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, q) + r * RP + col);
                    v[i].x += o.x;
                    v[i].y += o.y;
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
                // the place at which the product over K finds column col (see the loads of B)
                const int t = col / S::GROUP, o = col % S::GROUP;
                if constexpr (WIDE) {
                    const int at = (o / 2) * 8 + t;
                    *reinterpret_cast<float*>(to + 4 * at) = v[i].x;
                    *reinterpret_cast<float*>(to + 4 * (at + 4)) = v[i].y;
                } else {
                    const int at = (o / 4) * 16 + (o % 4 < 2 ? 2 * t : 8 + 2 * t);
                    *reinterpret_cast<uint32_t*>(to + 2 * at) = pack_pair<T>(v[i].x, v[i].y);
                    *reinterpret_cast<uint32_t*>(to + S::V_BYTES + 2 * at) = pack_pair<T>(rest_of<T>(v[i].x), rest_of<T>(v[i].y));
                }
            }
            if (lane == 0) cluster.map_shared_rank(s_unscale, q)[r] = unscale;
        }
    }
    cluster.sync();                    // behind it no block touches another's memory

    // ---- y + scale B v: this block's columns ----
    constexpr int STEPS = RP * (int)sizeof(T) / 32;                 // 32-byte steps of K
    constexpr int BLOCK = STEPS > (WIDE ? 4 : 8) ? 4 : STEPS, BLOCKS = STEPS / BLOCK;   // those whose B a lane holds at a time
    const float scale = p.scale ? p.scale[tile.x] : 1.f;
    const int g = lane >> 2, q = lane & 3;
    const uint32_t v_addr = smem_u32(v_smem);
    for (int u = unit_begin + warp; u < unit_end; u += APPLY_THREADS / 32) {
        // Accumulator columns 2q, 2q + 1 of product j stand for columns 8q + 2j, 8q + 2j + 1 of the unit, so that a lane
        // stores eight neighbours; along K a lane holds GROUP consecutive values of a row of B, at the places that the
        // product gives it.
        uint32_t w[4][BLOCK][2];
        const auto load_b = [&](int block) {
            constexpr int RUN = S::GROUP / BLOCKS;
            const int first = q * S::GROUP + block * RUN;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = u * 32 + (g >> 1) * 8 + 2 * j + (g & 1);
                union {
                    T e[RUN];
                    uint32_t w[RUN * sizeof(T) / 4];
                    uint2 v2[RUN * sizeof(T) / 8];
                    uint4 v4[(RUN * sizeof(T) + 15) / 16];
                } in;
                const T* row = B + (long long)col * p.rank + first;
                const int there = col < p.d_out ? rank - first : 0;
                if (p.b_vec && there >= RUN) {
                    if constexpr (RUN * sizeof(T) == 8) {
                        in.v2[0] = *reinterpret_cast<const uint2*>(row);
                    } else {
#pragma unroll
                        for (int i = 0; i < (int)(RUN * sizeof(T) / 16); ++i) in.v4[i] = reinterpret_cast<const uint4*>(row)[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < RUN; ++i) in.e[i] = i < there ? row[i] : from_float<T>(0.f);
                }
#pragma unroll
                for (int s = 0; s < BLOCK; ++s) {
                    w[j][s][0] = in.w[2 * s];
                    w[j][s][1] = in.w[2 * s + 1];
                }
            }
        };
        if constexpr (BLOCKS == 1) load_b(0);
        const int col = u * 32 + q * 8;
        for (int mt = 0; mt * 16 < tile.z; ++mt) {
            float y[2][8];
            bool row_ok[2];
            long long at_out[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = mt * 16 + g + 8 * h;
                row_ok[h] = r < tile.z;
                const long long t = s_pos[row_ok[h] ? r : 0];
                at_out[h] = t * p.ldo + col;
                const T* src = y_base + t * p.ldy + col;
                if (p.y_vec) {
                    if (row_ok[h] && col < p.d_out) {
#pragma unroll
                        for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) {
                            float e[16 / sizeof(T)];
                            load_elems<T, 16 / (int)sizeof(T)>(src + i, e);
#pragma unroll
                            for (int k = 0; k < 16 / (int)sizeof(T); ++k) y[h][i + k] = e[k];
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[h][i] = row_ok[h] && col + i < p.d_out ? to_float(src[i]) : 0.f;
                }
            }
            float sum[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[j][i] = 0.f;
#pragma unroll
            for (int step = 0; step < STEPS; ++step) {
                const int s = step % BLOCK;
                if (BLOCKS > 1 && s == 0) load_b(step / BLOCK);
                uint32_t v[4];
                const uint32_t at = v_addr + (mt * 16 + (lane & 15)) * S::V_ROW + step * 32 + ((lane >> 4) << 4);
                load_matrices(v, at);
                uint32_t v_lo[4];
                if constexpr (WIDE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(v[i], v[i], v_lo[i]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t hi[2], lo[2];
                        split_tf32(w[j][s][0], hi[0], lo[0]);
                        split_tf32(w[j][s][1], hi[1], lo[1]);
                        mma<T>(sum[j], v_lo, hi[0], hi[1]);
                        mma<T>(sum[j], v, lo[0], lo[1]);
                        mma<T>(sum[j], v, hi[0], hi[1]);
                    }
                } else {
                    load_matrices(v_lo, at + S::V_BYTES);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma<T>(sum[j], v_lo, w[j][s][0], w[j][s][1]);
                        mma<T>(sum[j], v, w[j][s][0], w[j][s][1]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!row_ok[h]) continue;
                const float unscale = s_unscale[mt * 16 + g + 8 * h];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        y[h][2 * j + e] = fmaf(sum[j][2 * h + e] * unscale, scale, y[h][2 * j + e]);
                T* dst = out_base + at_out[h];
                if (p.y_vec) {
                    if (col < p.d_out) {
#pragma unroll
                        for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) {
                            float e[16 / sizeof(T)];
#pragma unroll
                            for (int k = 0; k < 16 / (int)sizeof(T); ++k) e[k] = y[h][i + k];
                            store_elems<T, 16 / (int)sizeof(T)>(dst + i, e);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i < p.d_out) dst[i] = from_float<T>(y[h][i]);
                }
            }
        }
    }
}

template <typename T, int RP>
int launch_apply_rank(const ApplyArgs& a, long long tiles, cudaStream_t stream) {
    using S = ApplyShape<T, RP>;
    const auto kernel = adapter_apply_kernel<T, RP>;
    INFMOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    // Blocks of a cluster share out K, then the columns of y: as many as give every SM a few blocks, up to 8, and none without work.
    const int chunks = (a.d_in + S::CHUNK - 1) / S::CHUNK, units = (a.d_out + 31) / 32;
    unsigned cluster = 1;
    while (cluster < 8 && tiles * cluster < 148 * 4 && (int)cluster * 2 <= (chunks > units ? chunks : units)) cluster *= 2;
    INFMOE_CUDA_TRY(launch_chained(kernel, (unsigned)tiles * cluster, APPLY_THREADS, S::SMEM, cluster, stream, a));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

int grain_of(const void* p, long long stride_bytes) {
    for (int g = 16; g > 2; g /= 2)
        if ((uintptr_t)p % g == 0 && stride_bytes % g == 0) return g;
    return 2;
}

template <typename T>
int launch_apply(ApplyArgs a, long long tiles, cudaStream_t stream) {
    const int size = (int)sizeof(T);
    const int padded = a.rank <= 16 ? 16 : a.rank <= 32 ? 32 : a.rank <= 64 ? 64 : 128;
    const int group = padded / 4 * size, b_bytes = group < 16 ? group : 16;
    a.x_grain = grain_of(a.x, a.ldx * size);
    a.a_grain = grain_of(a.a, (long long)a.d_in * size);
    a.b_vec = (uintptr_t)a.b % b_bytes == 0 && (long long)a.rank * size % b_bytes == 0;
    a.y_vec = a.d_out % 8 == 0 && grain_of(a.y, a.ldy * size) == 16 && grain_of(a.out, a.ldo * size) == 16;
    switch (padded) {
        case 16: return launch_apply_rank<T, 16>(a, tiles, stream);
        case 32: return launch_apply_rank<T, 32>(a, tiles, stream);
        case 64: return launch_apply_rank<T, 64>(a, tiles, stream);
        default: return launch_apply_rank<T, 128>(a, tiles, stream);
    }
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
    INFMOE_CUDA_TRY(launch_chained(adapter_tiles_kernel, 1, PLAN_THREADS, 0, 1, (cudaStream_t)stream, T, adapter_count, offset,
                                   reinterpret_cast<int4*>(p + l.tiles), (int)max_tiles(T, adapter_count)));
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
    if (set->dtype == INFMOE_F32) return launch_apply<float>(a, tiles, (cudaStream_t)stream);
    if (set->dtype == INFMOE_F16) return launch_apply<__half>(a, tiles, (cudaStream_t)stream);
    return launch_apply<__nv_bfloat16>(a, tiles, (cudaStream_t)stream);
}

}  // extern "C"
