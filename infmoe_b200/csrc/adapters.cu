// Low-rank adapters of many requests at once, beside a shared projection: out[t] = y[t] + scale[a] B[a] (A[a] x[t]) with
// a the adapter of token t.  Tokens are grouped by adapter with the layer's own dispatch (an adapter takes the place of an
// expert); the plan that comes of it holds for every projection of the batch.
#include <climits>

#include "common.cuh"
#include "elem.cuh"
#include "kernels.h"

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
    int rank, d_in, d_out, adapters;
    const float* scale;       // [adapters] or NULL: 1
    const int* rank_of;       // [adapters] or NULL: all `rank`
    const int* pos;
    const int4* tiles;
};

// Simple form: one block per tile, row by row.
template <typename T>
__global__ void __launch_bounds__(APPLY_THREADS) adapter_apply_kernel(const ApplyArgs p) {
    extern __shared__ float s_v[];
    pdl_trigger();
    pdl_wait();
    const int4 tile = p.tiles[blockIdx.x];
    if (tile.z == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = tile.x < 0 ? 0 : p.rank_of ? max(0, min(p.rank, p.rank_of[tile.x])) : p.rank;
    if (tile.x < 0 && p.out == p.y) return;
    const float scale = tile.x >= 0 && p.scale ? p.scale[tile.x] : 1.f;
    const T* A = static_cast<const T*>(p.a) + (long long)max(tile.x, 0) * p.rank * p.d_in;
    const T* B = static_cast<const T*>(p.b) + (long long)max(tile.x, 0) * p.d_out * p.rank;
    for (int i = 0; i < tile.z; ++i) {
        const long long t = p.pos[tile.y + i];
        const T* x = static_cast<const T*>(p.x) + t * p.ldx;
        const T* y = static_cast<const T*>(p.y) + t * p.ldy;
        T* out = static_cast<T*>(p.out) + t * p.ldo;
        for (int r = warp; r < rank; r += APPLY_THREADS / 32) {
            float sum = 0.f;
            for (int d = lane; d < p.d_in; d += 32) sum = fmaf(to_float(x[d]), to_float(A[(long long)r * p.d_in + d]), sum);
            sum = warp_xor_sum(sum);
            if (lane == 0) s_v[r] = sum;
        }
        __syncthreads();
        for (int o = threadIdx.x; o < p.d_out; o += APPLY_THREADS) {
            float sum = 0.f;
            for (int r = 0; r < rank; ++r) sum = fmaf(s_v[r], to_float(B[(long long)o * p.rank + r]), sum);
            out[o] = from_float<T>(rank ? fmaf(scale, sum, to_float(y[o])) : to_float(y[o]));
        }
        __syncthreads();
    }
}

template <typename T>
int launch_apply(const ApplyArgs& a, long long tiles, cudaStream_t stream) {
    INFMOE_CUDA_TRY(launch_chained(adapter_apply_kernel<T>, (unsigned)tiles, APPLY_THREADS, sizeof(float) * (size_t)a.rank, 1,
                                   stream, a));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
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
    a.adapters = set->adapter_count;
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
