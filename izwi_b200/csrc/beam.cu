// Beam search on the device: the choice of the next beams from the logits, the reordering of the paged caches that
// follows it, and the walk back through the choices at the end.
#include <climits>
#include <type_traits>

#include "izb_common.cuh"

namespace {

// ---- selection -----------------------------------------------------------------------------------------------------
//   total(b, v) = score_b + logit_bv - lse_b,  lse_b = log sum over the finite logits of beam b of exp
// and the n_out largest totals of a group's beams, equal ones in the order of b * vocab + v.
//
// Inside a row the order is that of the logits, so one pass over them yields, for every tile of a row, the tile's
// maximum, its sum of exp(x - maximum) and its n_out largest (value, index) pairs; a second launch forms lse_b from
// the tiles, the totals of the few pairs that are left (in fp64: candidates of different beams are ranked by them),
// and their order.  32 x 8 rows of 151,936 bf16 logits: 26.1 us with the join (floor 11.9: reading them once), bound by
// the waits between a tile's three loops.

constexpr int BS_THREADS = 256;
constexpr int BS_WARPS = BS_THREADS / 32;
constexpr int BS_MAX_BEAMS = 32;
constexpr int BS_MAX_OUT = 64;
constexpr int BS_TILE_CAP = 512, BS_CAP = 1024;  // candidates of a tile, of a group kept in shared memory at a time

using u64 = unsigned long long;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// two multiply-adds, two additions in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// larger value <-> larger key, -0 as +0
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }
__device__ __forceinline__ u64 key_of(double v) {
    const u64 u = static_cast<u64>(__double_as_longlong(v + 0.0));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(u64 k) {
    return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k));
}

// The k-th largest of the 32 lanes' values (k <= 32): the lanes sorted by fifteen exchanges.
__device__ __forceinline__ uint32_t warp_kth(uint32_t x, int k) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int block = 2; block <= 32; block <<= 1)
#pragma unroll
        for (int step = block >> 1; step > 0; step >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, x, step);
            const bool larger = ((lane & block) == 0) == ((lane & step) == 0);
            x = larger ? max(x, other) : min(x, other);
        }
    return __shfl_sync(0xFFFFFFFFu, x, k - 1);
}

// A bound below which none of the k <= 64 largest candidates can lie, from the upper 32 bits of every thread's largest
// key.  The k-th largest of the maxima of 32 groups of threads is one (k groups hold a candidate that is no smaller), and a
// close one when k is well below 32 (22 candidates lie above the median of 32 maxima).
// So the block is cut into 32 groups, or for larger k into two or four sets of 32 smaller ones, and each set answers for its
// share of k.  Every thread returns the bound.
template <int THREADS>
__device__ __forceinline__ u64 block_bound(uint32_t mine, int k, uint32_t (*all)[32], uint32_t (&set)[4]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sets = k <= 20 ? 1 : k <= 40 ? 2 : 4, share = (k + sets - 1) / sets;
    all[warp][lane] = mine;  // group: the threads of a lane, of every (second, fourth) warp
    __syncthreads();
    if (warp < sets) {
        uint32_t v = 0;
        for (int w = warp; w < THREADS / 32; w += sets) v = max(v, all[w][lane]);
        v = warp_kth(v, share);
        if (lane == 0) set[warp] = v;
    }
    __syncthreads();
    uint32_t bound = set[0];
    for (int i = 1; i < sets; ++i) bound = min(bound, set[i]);
    return static_cast<u64>(bound) << 32;
}

// Candidates in shared memory: a key and, among equal keys, the lower index first.  PACKED: keys are different and say it all.
template <int N, bool PACKED>
struct Pool {
    static constexpr int CAP = N;
    u64 key[N];
    uint32_t idx[PACKED ? 1 : N];
    unsigned count;
    __device__ __forceinline__ static bool before(u64 ka, uint32_t ia, u64 kb, uint32_t ib) { return ka > kb || (!PACKED && ka == kb && ia < ib); }
    __device__ __forceinline__ uint32_t index(int i) const { return PACKED ? 0u : idx[PACKED ? 0 : i]; }
    __device__ __forceinline__ void put(int i, u64 k, uint32_t x) {
        key[i] = k;
        if (!PACKED) idx[PACKED ? 0 : i] = x;
    }
    __device__ __forceinline__ void add(u64 k, uint32_t x) {
        const unsigned at = atomicAdd(&count, 1u);
        if (at < N) put(at, k, x);
    }
};
// Descending order over the first n entries (n <= CAP).  Up to one entry per thread: each counts the entries in
// front of it (n broadcast reads, no barrier between them); more: bitonic exchange over the next power of two.
template <int THREADS, typename P>
__device__ void pool_sort(P& p, int n) {
    if (n <= THREADS) {
        const int i = threadIdx.x;
        const u64 key = i < n ? p.key[i] : 0;
        const uint32_t idx = i < n ? p.index(i) : 0;
        int rank = 0;
        if (i < n) {
#pragma unroll 4
            for (int j = 0; j < n; ++j) rank += P::before(p.key[j], p.index(j), key, idx);
        }
        __syncthreads();
        if (i < n) p.put(rank, key, idx);
        __syncthreads();
        return;
    }
    int size = 2 * THREADS;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += THREADS) p.put(i, 0, 0xFFFFFFFFu);
    __syncthreads();
    for (int block = 2; block <= size; block <<= 1)
        for (int step = block >> 1; step > 0; step >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += THREADS) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const bool down = (a & block) == 0;
                const u64 ka = p.key[a], kb = p.key[b];
                const uint32_t ia = p.index(a), ib = p.index(b);
                if (P::before(kb, ib, ka, ia) == down) {
                    p.put(a, kb, ib);
                    p.put(b, ka, ia);
                }
            }
            __syncthreads();
        }
}

// Fills the pool with every candidate not behind (bound_key, bound_idx); when they outgrow it, the k-th of those it
// caught is a tighter bound (any k candidates bound the k largest), and the scan is repeated: each repetition drops
// at least CAP - k candidates for good.  Then sorts.  Returns the number of sorted entries, at least the k
// largest if there are that many.  `scan(key, idx)` calls add for every candidate not behind the bound.  The pool's
// count is zero, and every thread knows it, on the first entry.
template <int THREADS, typename P, typename Scan>
__device__ int collect(P& p, u64 bound_key, int k, Scan scan) {
    uint32_t bound_idx = 0xFFFFFFFFu;
    for (;;) {
        scan(bound_key, bound_idx);
        __syncthreads();
        const unsigned n = p.count;
        pool_sort<THREADS>(p, n < P::CAP ? n : P::CAP);
        if (n <= P::CAP) return static_cast<int>(n);
        bound_key = p.key[k - 1];
        bound_idx = p.index(k - 1);
        if (threadIdx.x == 0) p.count = 0;
        __syncthreads();
    }
}

// A 16-byte vector of logits: its largest value (NaN ignored) and its elements.
template <typename T>
__device__ __forceinline__ float largest(const uint4& w) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else {
        uint32_t a, b;
        if constexpr (std::is_same<T, __half>::value) {
            asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
            asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
            asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
            return fmaxf(__half2float(__ushort_as_half(static_cast<unsigned short>(a))),
                         __half2float(__ushort_as_half(static_cast<unsigned short>(a >> 16))));
        } else {
            asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
            asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
            asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
            return fmaxf(izb::bf16_lo_to_f32(a), izb::bf16_hi_to_f32(a));
        }
    }
}
template <typename T>
__device__ __forceinline__ void elements(const uint4& w, float (&x)[16 / sizeof(T)]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(u[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            x[2 * i] = __half2float(__ushort_as_half(static_cast<unsigned short>(u[i])));
            x[2 * i + 1] = __half2float(__ushort_as_half(static_cast<unsigned short>(u[i] >> 16)));
        } else {
            x[2 * i] = izb::bf16_lo_to_f32(u[i]);
            x[2 * i + 1] = izb::bf16_hi_to_f32(u[i]);
        }
    }
}

struct SelectParams {
    const void* logits;
    const float* scores;
    const uint8_t* finished;
    float* scores_out;
    int* parents_out;
    int* tokens_out;
    uint8_t* finished_out;
    float2* tile_ml;  // [rows][tiles]: maximum and sum of exp(x - maximum)
    u64* tile_top;    // [rows][tiles][n_out]: key_of(value) << 32 | ~index, descending; 0: none
    long long ld;
    int vocab, beams, tiles, n_out, eos;
    int* status;
};

// A row whose beam is not alive or is finished is not read.
__device__ __forceinline__ bool row_counts(const SelectParams& p, int row) {
    return isfinite(p.scores[row]) && !(p.finished && p.finished[row]);
}

// One CTA per tile of THREADS * NV 16-byte vectors of a row, copied into shared memory, where three
// short loops look at it (maximum, sum, candidates); a thread works on every THREADS-th vector.  (Held in registers with
// everything unrolled, the tile made straight-line code that each CTA ran once, at the speed of instruction fetch: 144 us
// for 32 x 8 rows of 151936 bf16 logits.)  Rows may start anywhere: vectors are cut on 16-byte boundaries of memory; a tile
// inside its row is one bulk copy, and the ragged ends are read element by element.  Only finite logits count.
template <typename T, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, 8) beam_tile_kernel(const __grid_constant__ SelectParams p) {
    constexpr int V = 16 / sizeof(T), WARPS = THREADS / 32;
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __align__(128) uint4 tile_s[THREADS * NV];
    __shared__ Pool<BS_TILE_CAP, true> pool;  // key_of(value) << 32 | ~index
    __shared__ uint32_t sets[4];
    __shared__ float wm[WARPS], wl[WARPS];
    __shared__ unsigned long long landed;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        izb::mbar_init(izb::smem_u32(&landed), 1);
        izb::mbar_fence_init();
        pool.count = 0;
        abort_flag = 0;
    }
    __syncthreads();
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int row = blockIdx.x / p.tiles, tile = blockIdx.x - row * p.tiles;
    if (!row_counts(p, row)) return;
    const T* base = static_cast<const T*>(p.logits) + static_cast<long long>(row) * p.ld;
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
    const int first = tile * (THREADS * NV) + tid;
    uint4* mine = tile_s + tid;  // vector i at mine[i * THREADS]

    const long long tile0 = static_cast<long long>(tile) * (THREADS * NV * V) - skew;
    bool ok = true;
    if (tile0 >= 0 && tile0 + THREADS * NV * V <= p.vocab) {
        if (tid == 0) {
            izb::mbar_expect_tx(izb::smem_u32(&landed), sizeof(tile_s));
            izb::bulk_g2s(izb::smem_u32(tile_s), base + tile0, sizeof(tile_s), izb::smem_u32(&landed));
        }
        ok = izb::mbar_wait_bounded(izb::smem_u32(&landed), 0, &abort_flag);
    } else {
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
            const long long e0 = static_cast<long long>(first + i * THREADS) * V - skew;
            if (e0 >= 0 && e0 + V <= p.vocab) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(izb::smem_u32(mine + i * THREADS)), "l"(base + e0) : "memory");
            } else {
                T* w = reinterpret_cast<T*>(mine + i * THREADS);
                for (int k = 0; k < V; ++k) {
                    const long long e = e0 + k;
                    w[k] = e >= 0 && e < p.vocab ? base[e] : static_cast<T>(-INFINITY);
                }
            }
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    }

    float mx = -INFINITY, vm[NV];  // the largest of each vector
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        vm[i] = largest<T>(mine[i * THREADS]);
        mx = fmaxf(mx, vm[i]);
    }
    if (mx == INFINITY) {  // take the infinities out
        mx = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
            T* w = reinterpret_cast<T*>(mine + i * THREADS);
            for (int k = 0; k < V; ++k)
                if (static_cast<float>(w[k]) == INFINITY) w[k] = static_cast<T>(-INFINITY);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            vm[i] = largest<T>(mine[i * THREADS]);
            mx = fmaxf(mx, vm[i]);
        }
    }
    float top = mx;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (lane == 0) wm[warp] = top;
    if (!__syncthreads_and(ok)) {
        if (tid == 0) atomicExch(p.status, 1);
        if (!ok) {  // the copy under way lands in memory of this CTA
            abort_flag = 0;
            izb::mbar_wait_bounded(izb::smem_u32(&landed), 0, &abort_flag);
        }
        return;
    }
    // A bound of the tile's n_out largest; ties are left to collect().  With up to as many as there are warps, the n_out-th
    // largest of the warps' maxima (n_out warps have a value that is no smaller), else one from every thread's largest.
    u64 bound;
    if (p.n_out <= WARPS) {
        const float v = wm[lane % WARPS];
        int rank = 0;
#pragma unroll
        for (int j = 0; j < WARPS; ++j) rank += wm[j] > v || (wm[j] == v && j < lane % WARPS);
        const float b = __shfl_sync(0xFFFFFFFFu, v, __ffs(__ballot_sync(0xFFFFFFFFu, rank == p.n_out - 1)) - 1);
        bound = b > -INFINITY ? static_cast<u64>(key_of(b)) << 32 : 0ull;
    } else {
        bound = block_bound<THREADS>(mx > -INFINITY ? key_of(mx) : 0u, p.n_out, reinterpret_cast<uint32_t(*)[32]>(pool.key), sets);
    }

    float sum = 0.f;
    if (top > -INFINITY) {
        const float shift = top * LOG2E;
        float2 part = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < NV; ++i) {
            float x[V];
            elements<T>(mine[i * THREADS], x);
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                const float2 y = fma2(make_float2(x[k], x[k + 1]), make_float2(LOG2E, LOG2E), make_float2(-shift, -shift));
                part = add2(part, make_float2(ex2(y.x), ex2(y.y)));
            }
        }
        sum = part.x + part.y;
        if (sum != sum) {  // NaN among the logits: once more without them
            sum = 0.f;
#pragma unroll 1
            for (int i = 0; i < NV; ++i) {
                const T* w = reinterpret_cast<const T*>(mine + i * THREADS);
                for (int k = 0; k < V; ++k) {
                    const float x = static_cast<float>(w[k]);
                    if (x == x) sum += ex2(fmaf(x, LOG2E, -shift));
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) wl[warp] = sum;
    const int n = collect<THREADS>(pool, bound, p.n_out, [&](u64 bk, uint32_t) {
        const float floor_v = bk >> 32 ? value_of(static_cast<uint32_t>(bk >> 32)) : -INFINITY;
        // which vectors hold a candidate, then only those, element by element
        unsigned hits = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) hits |= vm[i] >= floor_v && vm[i] > -INFINITY ? 1u << i : 0u;
        while (hits) {
            const int i = __ffs(hits) - 1;
            hits &= hits - 1;
            float x[V];
            elements<T>(mine[i * THREADS], x);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (x[k] >= floor_v && x[k] > -INFINITY) {
                    const uint32_t e = static_cast<uint32_t>(first + i * THREADS) * V - skew + k;
                    const u64 key = static_cast<u64>(key_of(x[k])) << 32 | static_cast<uint32_t>(~e);
                    if (key >= bk) pool.add(key, 0);
                }
        }
    });
    if (tid == 0) {
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, wm[w]);
        for (int w = 0; w < WARPS; ++w) l += wm[w] > -INFINITY ? wl[w] * ex2((wm[w] - m) * LOG2E) : 0.f;
        p.tile_ml[blockIdx.x] = make_float2(m, l);
    }
    u64* out = p.tile_top + static_cast<long long>(blockIdx.x) * p.n_out;
    for (int i = tid; i < p.n_out; i += THREADS) out[i] = i < n ? pool.key[i] : 0ull;
}

// One CTA per group: log-sums of its beams, then the order of what the tiles kept.
__global__ void __launch_bounds__(BS_THREADS) beam_join_kernel(const __grid_constant__ SelectParams p) {
    using Candidates = Pool<BS_CAP, false>;
    __shared__ Candidates pool;
    __shared__ uint32_t sets[4];
    __shared__ double offset[BS_MAX_BEAMS];  // score - lse
    __shared__ uint8_t state[BS_MAX_BEAMS];  // 0: nothing, 1: its row, 2: finished
    __shared__ int open[BS_CAP];
    __shared__ unsigned n_open;
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = blockIdx.x, row0 = group * p.beams;
    if (tid == 0) pool.count = 0;
    // What the tiles left is read while the scores are on their way: the places exist, and those of rows that do not count
    // are not used.
    const int lists = p.beams * p.tiles;
    const u64* lists_from = p.tile_top + static_cast<long long>(row0) * p.tiles * p.n_out;
    const u64 first = tid < lists ? lists_from[static_cast<long long>(tid) * p.n_out] : 0ull;
    for (int b = warp; b < p.beams; b += BS_WARPS) {
        const float2* ml = p.tile_ml + static_cast<long long>(row0 + b) * p.tiles;
        float2 x0 = lane < p.tiles ? ml[lane] : make_float2(-INFINITY, 0.f);
        const float score = p.scores[row0 + b];
        const bool alive = isfinite(score), done = p.finished && p.finished[row0 + b];
        if (alive && !done) {
            float m = x0.x;
            for (int t = lane + 32; t < p.tiles; t += 32) m = fmaxf(m, ml[t].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            double s = 0.0;
            for (int t = lane; t < p.tiles; t += 32) {
                const float2 x = t == lane ? x0 : ml[t];
                if (x.x > -INFINITY) s += static_cast<double>(x.y) * static_cast<double>(expf(x.x - m));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (lane == 0) {
                offset[b] = static_cast<double>(score) - (static_cast<double>(m) + log(s));
                state[b] = m > -INFINITY ? 1 : 0;
            }
        } else if (lane == 0) {
            offset[b] = static_cast<double>(score);
            state[b] = alive && p.eos >= 0 ? 2 : 0;
        }
    }
    __syncthreads();
    // A list is a tile's sorted pairs; a finished beam is a list of its one candidate.  x: what the tile left in place i.
    auto pair_of = [&](int list, int i, u64 x, u64& key, uint32_t& idx) -> bool {
        const int b = list / p.tiles, t = list - b * p.tiles;
        if (state[b] == 2) {
            key = key_of(offset[b]);
            idx = static_cast<uint32_t>(b) * p.vocab + p.eos;
            return t == 0 && i == 0;
        }
        if (state[b] == 0 || x == 0) return false;
        key = key_of(static_cast<double>(value_of(static_cast<uint32_t>(x >> 32))) + offset[b]);
        idx = static_cast<uint32_t>(b) * p.vocab + static_cast<uint32_t>(~x);
        return true;
    };
    auto head_of = [&](int list) { return list == tid ? first : lists_from[static_cast<long long>(list) * p.n_out]; };
    uint32_t mine = 0;
    for (int l = tid; l < lists; l += BS_THREADS) {
        u64 key;
        uint32_t idx;
        if (pair_of(l, 0, head_of(l), key, idx)) mine = max(mine, static_cast<uint32_t>(key >> 32));
    }
    const u64 bound = block_bound<BS_THREADS>(mine, p.n_out, reinterpret_cast<uint32_t(*)[32]>(pool.key), sets);
    // the lists whose first pair is not behind the bound, BS_CAP at a time, then their pairs, all of them at once (one after
    // the other, list by list, every pair was a trip to memory: 190 us for 64 of 8 x 10 lists)
    const int n = collect<BS_THREADS>(pool, bound, p.n_out, [&](u64 bk, uint32_t bi) {
        for (int l0 = 0; l0 < lists; l0 += BS_CAP) {
            if (tid == 0) n_open = 0;
            __syncthreads();
            for (int l = l0 + tid; l < min(lists, l0 + BS_CAP); l += BS_THREADS) {
                u64 key;
                uint32_t idx;
                if (pair_of(l, 0, head_of(l), key, idx) && !Candidates::before(bk, bi, key, idx)) open[atomicAdd(&n_open, 1u)] = l;
            }
            __syncthreads();
            const int pairs = static_cast<int>(n_open) * p.n_out;
            for (int e = tid; e < pairs; e += BS_THREADS) {
                u64 key;
                uint32_t idx;
                const int o = e / p.n_out, i = e - o * p.n_out, l = open[o];
                if (pair_of(l, i, lists_from[static_cast<long long>(l) * p.n_out + i], key, idx) && !Candidates::before(bk, bi, key, idx)) pool.add(key, idx);
            }
            __syncthreads();
        }
    });
    for (int i = tid; i < p.n_out; i += BS_THREADS) {
        float score = -INFINITY;
        int parent = 0, token = p.eos >= 0 ? p.eos : 0;
        bool done = false;
        if (i < n) {
            const uint32_t idx = pool.idx[i];
            parent = static_cast<int>(idx / static_cast<uint32_t>(p.vocab));
            token = static_cast<int>(idx - static_cast<uint32_t>(parent) * p.vocab);
            score = static_cast<float>(value_of(pool.key[i]));
            done = state[parent] == 2 || token == p.eos;
        }
        const long long o = static_cast<long long>(group) * p.n_out + i;
        p.scores_out[o] = score;
        p.parents_out[o] = parent;
        p.tokens_out[o] = token;
        if (p.finished_out) p.finished_out[o] = done ? 1 : 0;
    }
}

int dtype_bytes(int dtype) { return dtype == IZB_F32 ? 4 : 2; }

// Tiles of 1,280 vectors of 16 bytes, ten for each of 128 threads: enough for a thread that what it does once a tile does not
// show, and eight tiles on an SM (32 x 8 rows of 151,936 bf16 logits: 26.1 us; sixteen vectors 27.4, eight 27.2, eight for each
// of 256 threads 28.9).  Tiles of 512 with 256 threads where the large ones would leave SMs without one, so that a few rows
// spread over the chip (4 x 4 rows of 51,865: 9.5 us against 10.1), unless a group's lists become many for the one CTA that
// joins them (8 rows of 151,936: 304 lists 13.5 us, 120 of the large tiles 9.2).
struct SelectPlan {
    bool large;
    int64_t tiles;
};
SelectPlan select_plan(const izb_ctx* ctx, int dtype, int64_t groups, int beams, int64_t vocab) {
    const int64_t v = 16 / dtype_bytes(dtype), vectors = (vocab + v - 1 + v - 1) / v;  // a row may start up to v - 1 elements into a vector
    const int64_t large = (vectors + 1279) / 1280, small = (vectors + 511) / 512;
    SelectPlan pl;
    pl.large = groups * beams * large >= (ctx && ctx->sm_count > 0 ? ctx->sm_count : 148) || beams * small > 128;
    pl.tiles = pl.large ? large : small;
    return pl;
}
size_t select_bytes(const SelectPlan& pl, int64_t rows, int n_out) {
    return static_cast<size_t>(rows) * pl.tiles * (static_cast<size_t>(n_out) * sizeof(u64) + sizeof(float2));
}

template <typename T>
cudaError_t launch_tiles(izb_ctx* ctx, cudaStream_t s, const SelectParams& p, bool large, unsigned grid) {
    if (large) return izb::launch_chained(ctx, beam_tile_kernel<T, 10, 128>, dim3(grid), dim3(128), 0, s, p);
    return izb::launch_chained(ctx, beam_tile_kernel<T, 2, 256>, dim3(grid), dim3(256), 0, s, p);
}

// ---- reordering of the paged caches --------------------------------------------------------------------------------
// Child k continues beam parents[k].  The pages a parent has filled are shared from now on: their table entries are
// copied.  Its last, partly filled page will be written by every child, so each child needs one of its own: the
// first child of a parent keeps the parent's page, and the others take the pages of beams without a child, in
// ascending order (there are exactly as many), and copy the rows held so far.  A page that is read is kept by
// somebody and a page that is written belonged to nobody any more, so copies of one call never meet.  Bound by DRAM:
// 16 x 8 beams, 36 layers of bf16 pages 98.2 us = 6.4 TB/s of reads and writes; 4 beams, 4 layers 3.0 us, one launch.

constexpr int RO_MAX_BEAMS = 32;
constexpr int RO_MAX_LAYERS = 64;
constexpr int RO_THREADS = 256;
constexpr int RO_WAVES = 8;  // of five CTAs an SM

struct LayerPtrs {
    uint8_t* k;
    uint8_t* v;
    float* k_scales;
    float* v_scales;
};
struct ReorderParams {
    LayerPtrs layer[RO_MAX_LAYERS];
    const int* table;
    int* table_out;
    const int* parents;
    const int* lens;
    int* status;
    long long max_pages;
    long long page_bytes, row_bytes;  // of the values
    int page_scales, row_scales;      // floats; Int8: one per page whatever it holds
    int beams, page_size, n_layers, splits;
};

// grid (CTAs of a child, groups * beams): CTA (0, child) also writes the child's table row
__global__ void __launch_bounds__(RO_THREADS) kv_pages_reorder_kernel(const __grid_constant__ ReorderParams p) {
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    __shared__ int sh_parent, sh_src, sh_dst, sh_full, sh_held;
    // units of 32 KB of a page of K or V of a layer, in turn among the CTAs of the child
    int unit = blockIdx.x, split, which, layer;
    auto where = [&]() {
        const int page = unit / p.splits;
        split = unit - page * p.splits;
        which = page & 1;
        layer = page >> 1;
    };
    where();
    const int child = blockIdx.y % p.beams, row0 = blockIdx.y - child;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const unsigned all = 0xFFFFFFFFu;
        const bool in = lane < p.beams;
        int par = in ? p.parents[row0 + lane] : -1 - lane;  // lanes past the beams match nobody
        const int len = p.lens[row0 + (in ? lane : 0)];
        const int len0 = __shfl_sync(all, len, 0);
        // beams of a group grow together, a parent is one of them and the pages they fill are in the table: else the
        // group's rows are left as they are
        const bool wrong = __any_sync(all, (in && (par < 0 || par >= p.beams)) || len != len0 || len0 < 0) ||
                           static_cast<long long>(len0) > p.max_pages * p.page_size;
        if (wrong) {
            if (lane == 0 && child == 0 && blockIdx.x == 0) atomicExch(p.status, 9);
            par = in ? lane : -1 - lane;
        }
        const int full = wrong ? 0 : len0 / p.page_size, held = wrong ? 0 : len0 - full * p.page_size;
        const unsigned same = __match_any_sync(all, par);
        const bool again = in && (same & ((1u << lane) - 1u)) != 0;  // not its parent's first child
        const unsigned again_mask = __ballot_sync(all, again);
        unsigned has_child = 0;
        for (int b = 0; b < p.beams; ++b)
            if (__any_sync(all, in && par == b)) has_child |= 1u << b;
        if (lane == child) {
            int from = par;
            if (again) {  // the page of the i-th beam without a child, i: further children before this one
                const unsigned left = ~has_child & (p.beams == 32 ? all : (1u << p.beams) - 1u);
                from = static_cast<int>(__fns(left, 0, __popc(again_mask & ((1u << lane) - 1u)) + 1));
            }
            sh_parent = par;
            sh_full = full;
            sh_held = held;
            sh_src = held ? p.table[(row0 + par) * p.max_pages + full] : 0;
            sh_dst = held ? p.table[(row0 + from) * p.max_pages + full] : 0;
        }
    }
    __syncthreads();
    const int held = sh_held, full = sh_full;
    if (blockIdx.x == 0) {
        const int* mine = p.table + static_cast<long long>(blockIdx.y) * p.max_pages;
        const int* theirs = p.table + (row0 + sh_parent) * p.max_pages;
        int* out = p.table_out + static_cast<long long>(blockIdx.y) * p.max_pages;
        for (long long c = threadIdx.x; c < p.max_pages; c += RO_THREADS)
            out[c] = c < full ? theirs[c] : (c == full && held) ? sh_dst : mine[c];
    }
    if (!held || sh_src == sh_dst) return;
    const int n = static_cast<int>(held * p.row_bytes / 16);
    constexpr int UN = 8;
    for (; unit < p.n_layers * 2 * p.splits; unit += gridDim.x, where()) {
        uint8_t* values = which ? p.layer[layer].v : p.layer[layer].k;
        float* scales = which ? p.layer[layer].v_scales : p.layer[layer].k_scales;
        const uint4* src = reinterpret_cast<const uint4*>(values + sh_src * p.page_bytes);
        uint4* dst = reinterpret_cast<uint4*>(values + sh_dst * p.page_bytes);
        const int i0 = split * RO_THREADS * UN + threadIdx.x;
        uint4 w[UN];
#pragma unroll
        for (int j = 0; j < UN; ++j)
            if (i0 + j * RO_THREADS < n) w[j] = __ldcs(src + i0 + j * RO_THREADS);
#pragma unroll
        for (int j = 0; j < UN; ++j)
            if (i0 + j * RO_THREADS < n) __stcs(dst + i0 + j * RO_THREADS, w[j]);
        if (scales && split == 0) {
            const int m = p.row_scales ? held * p.row_scales : p.page_scales;
            const float* from = scales + static_cast<long long>(sh_src) * p.page_scales;
            float* to = scales + static_cast<long long>(sh_dst) * p.page_scales;
            for (int i = threadIdx.x; i < m; i += RO_THREADS * UN) {
                float x[UN];
#pragma unroll
                for (int j = 0; j < UN; ++j)
                    if (i + j * RO_THREADS < m) x[j] = from[i + j * RO_THREADS];
#pragma unroll
                for (int j = 0; j < UN; ++j)
                    if (i + j * RO_THREADS < m) to[i + j * RO_THREADS] = x[j];
            }
        }
    }
}

// ---- walk back through the choices ---------------------------------------------------------------------------------
// out[j, s] = tokens[s, b_s],  b_{s-1} = parents[s, b_s],  b at the last step = last[j].
//
// A walk is a chain of dependent reads, one per step (0.25 us each from memory: 1,027 us for 4096 steps).  Up to 32
// beams, `beams` lanes hold a step's parents, so a step of the walk is a shuffle among them; and the steps are cut into
// chunks, 32 / beams of them side by side in a warp, one warp after the other: first every chunk maps all beams at its
// end to beams at its start and a warp's chunks are chained into one map, then the warps' maps are chained, and then
// every chunk is walked again from where the walks enter it, writing tokens.  Bound by that chain: 32 x 8 walks of 4,096
// steps 13.1 us, 14.1 with nothing in L2 (a group's warps in four CTAs of a cluster, 32 steps a lane in flight; 15.7 and 21.5
// with 16; one CTA 26.6), 5 of 37 steps 3.5 us, one launch.
constexpr int TR_WARPS = 32;
constexpr int TR_NONE = 0xFF;   // a walk that has left [0, beams)

// Rows s0 .. s0 + AHEAD - 1 of a lane's column (those below n), `ld` apart; whole: none is past n for any lane of the warp.
template <int AHEAD>
__device__ __forceinline__ void trace_rows(int (&r)[AHEAD], const int* from, long long ld, int s0, int n, bool whole) {
    const int* at = from + s0 * ld;
    if (whole) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j, at += ld) r[j] = __ldg(at);
    } else {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j, at += ld) r[j] = s0 + j < n ? __ldg(at) : 0;
    }
}

// AHEAD: steps whose rows a lane has in flight; more than 16 only where a CTA has a quarter of the warps.
template <int AHEAD>
__global__ void __launch_bounds__(AHEAD > 16 ? TR_WARPS * 8 : TR_WARPS * 32)
    beam_trace_chunks_kernel(const int* __restrict__ parents, const int* __restrict__ tokens, const int* __restrict__ last,
                             int* __restrict__ out, int steps, int beams, int picks, long long groups, long long ld_out, int chunk,
                             int ranks, int* status) {
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    // in the first CTA of a group: beam at the end of a warp's steps -> beam at the end of the warp's before
    __shared__ int map[TR_WARPS][32];
    // where each of `beams` walks enters a warp's steps
    __shared__ int enter[TR_WARPS][32];
    const int lane = threadIdx.x & 31, here = threadIdx.x >> 5, rank = static_cast<int>(blockIdx.x) % ranks;
    const int per_cta = static_cast<int>(blockDim.x >> 5), warp = rank * per_cta + here;
    const long long group = blockIdx.x / ranks, ld = groups * beams;
    auto sync_group = [&]() {
        if (ranks > 1) izb::cluster_sync_all();
        else __syncthreads();
    };
    const int chunks = (steps + chunk - 1) / chunk;
    const int side = 32 / beams, sub = lane / beams, me = lane - sub * beams, base = sub * beams;
    const int c = warp * side + sub;
    const long long lo = static_cast<long long>(c) * chunk;
    const int n = sub < side && c < chunks ? static_cast<int>(steps - lo < chunk ? steps - lo : chunk) : 0;  // steps of this lane's chunk
    const int warps = (chunks + side - 1) / side;                    // that have steps
    const int most = __reduce_max_sync(0xFFFFFFFFu, n);
    const bool even = __all_sync(0xFFFFFFFFu, n == most || sub >= side);
    const int* par = parents + (n ? lo : 0) * ld + group * beams + me;
    const int* tok = tokens + (n ? lo : 0) * ld + group * beams + me;
    // rows of out on 16-byte boundaries take four tokens a store: a lane writes a row of its own, so every store touches
    // as many sectors as it has lanes (4096 steps, 32 x 8 walks: 38.8 us with single stores, 26.6 us with these)
    const bool wide = ld_out % 4 == 0 && chunk % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    // `at` one step back; to: what the shuffle brought from the lane of beam `at`
    auto back = [&](int at, int to) { return at == TR_NONE || static_cast<unsigned>(to) >= static_cast<unsigned>(beams) ? TR_NONE : to; };

    // steps that fit one read are read once, tokens and the walks' ends with them: a short trace waits for memory once
    const bool once = most <= AHEAD;
    int r[AHEAD], t[AHEAD];
    if (once) {
        trace_rows(r, par, ld, 0, n, even && n == AHEAD);
        trace_rows(t, tok, ld, 0, n, even && n == AHEAD);
    }
    int end = warp == 0 && lane < beams && lane < picks ? last[group * picks + lane] : -1;

    int mine = me;  // beam `me` at the end of this lane's chunk -> beam at its start
    if (chunks > 1 && (side > 1 || warp > 0)) {  // nothing leads on from the first chunk of all
        for (int s0 = (most - 1) / AHEAD * AHEAD; s0 >= 0; s0 -= AHEAD) {
            if (!once) trace_rows(r, par, ld, s0, n, even && n && s0 + AHEAD <= most);
#pragma unroll
            for (int j = AHEAD - 1; j >= 0; --j) {
                const int to = __shfl_sync(0xFFFFFFFFu, r[j], (base + mine) & 31);
                if (s0 + j < n) mine = back(mine, to);
            }
        }
    }
    if (n == 0) mine = me;  // a chunk past the end leads nowhere else
    {
        int at = lane < beams ? lane : TR_NONE;
        for (int k = side - 1; k >= 0; --k) {
            const int to = __shfl_sync(0xFFFFFFFFu, mine, (k * beams + at) & 31);
            at = at == TR_NONE ? TR_NONE : to;
        }
        if (ranks > 1) izb::st_cluster_f32(izb::cluster_map_shared(izb::smem_u32(&map[warp][lane]), 0), __int_as_float(at));
        else map[warp][lane] = at;
    }
    for (int p0 = 0; p0 < picks; p0 += beams) {
        sync_group();
        if (warp == 0) {
            if (p0 > 0) end = lane < beams && p0 + lane < picks ? last[group * picks + p0 + lane] : -1;
            int at = end >= 0 && end < beams ? end : TR_NONE;
            for (int w = warps - 1; w >= 0; --w) {
                if (ranks > 1) izb::st_cluster_f32(izb::cluster_map_shared(izb::smem_u32(&enter[w][lane]), w / per_cta), __int_as_float(at));
                else enter[w][lane] = at;
                at = at == TR_NONE ? TR_NONE : map[w][at];
            }
        }
        sync_group();
        if (warp >= warps) continue;
        const bool walks = p0 + me < picks;
        int* dst = out + (group * picks + p0 + (walks ? me : 0)) * ld_out + (n ? lo : 0);
        // from the warp's end through the chunks behind this lane's own
        int at = enter[warp][me];
        for (int k = side - 1; k > 0; --k) {
            const int to = __shfl_sync(0xFFFFFFFFu, mine, (k * beams + at) & 31);
            if (k > sub && at != TR_NONE) at = to;
        }
        bool lost = false;
        for (int s0 = (most - 1) / AHEAD * AHEAD; s0 >= 0; s0 -= AHEAD) {
            const bool whole = even && n && s0 + AHEAD <= most;
            if (!once) trace_rows(r, par, ld, s0, n, whole);
            if (!once || p0 > 0) trace_rows(t, tok, ld, s0, n, whole);  // the tokens' registers become the results
#pragma unroll
            for (int j = AHEAD - 1; j >= 0; --j) {
                const int from = (base + at) & 31;
                const int token = __shfl_sync(0xFFFFFFFFu, t[j], from), to = __shfl_sync(0xFFFFFFFFu, r[j], from);
                t[j] = at == TR_NONE ? -1 : token;
                if (s0 + j < n) {
                    lost |= at == TR_NONE;
                    at = back(at, to);
                }
            }
            if (walks && wide && s0 + AHEAD <= n) {
#pragma unroll
                for (int j = 0; j < AHEAD; j += 4) *reinterpret_cast<int4*>(dst + s0 + j) = make_int4(t[j], t[j + 1], t[j + 2], t[j + 3]);
            } else if (walks) {
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (s0 + j < n) dst[s0 + j] = t[j];
            }
        }
        if (walks && lost) atomicExch(status, 9);
    }
}

// More beams than lanes: one thread per walk.
__global__ void __launch_bounds__(128)
    beam_trace_kernel(const int* __restrict__ parents, const int* __restrict__ tokens, const int* __restrict__ last,
                      int* __restrict__ out, int steps, int beams, int picks, long long groups, long long ld_out, int* status) {
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= groups * picks) return;
    const long long group = i / picks;
    int b = last[i];
    for (int s = steps - 1; s >= 0; --s) {
        if (b < 0 || b >= beams) {
            atomicExch(status, 9);
            for (; s >= 0; --s) out[i * ld_out + s] = -1;
            return;
        }
        const long long at = (s * groups + group) * beams + b;
        out[i * ld_out + s] = tokens[at];
        b = parents[at];
    }
}

}  // namespace

extern "C" {

size_t izb_beam_select_workspace_bytes(const izb_ctx* ctx, int32_t dtype, int64_t groups, int32_t beams, int64_t vocab, int32_t n_out) {
    if (groups <= 0 || beams <= 0 || beams > BS_MAX_BEAMS || vocab <= 0 || vocab > INT32_MAX / beams || n_out <= 0 || n_out > BS_MAX_OUT ||
        groups > INT32_MAX / beams)
        return 0;
    return select_bytes(select_plan(ctx, dtype, groups, beams, vocab), groups * beams, n_out);
}

int32_t izb_beam_select(izb_ctx* ctx, izb_stream stream, const void* logits, int32_t dtype, int64_t groups, int32_t beams, int64_t vocab,
                        int64_t ld, const float* scores, const uint8_t* finished, int32_t eos, int32_t n_out, float* scores_out,
                        int32_t* parents_out, int32_t* tokens_out, uint8_t* finished_out, void* workspace, size_t workspace_bytes) {
    if (!ctx || groups < 0 || beams <= 0 || vocab <= 0 || ld < vocab || n_out <= 0) return IZB_ERR_BAD_ARG;
    if (dtype != IZB_F32 && dtype != IZB_BF16 && dtype != IZB_F16) return IZB_ERR_BAD_ARG;
    if (eos >= vocab || (finished && eos < 0)) return IZB_ERR_BAD_ARG;  // a finished beam goes on with eos
    if (groups == 0) return IZB_OK;
    if (beams > BS_MAX_BEAMS || n_out > BS_MAX_OUT || vocab > INT32_MAX / beams || groups > INT32_MAX / beams) return IZB_ERR_UNSUPPORTED;
    if (!logits || !scores || !scores_out || !parents_out || !tokens_out) return IZB_ERR_BAD_ARG;
    if (!izb_aligned(logits, dtype_bytes(dtype)) || !izb_aligned(scores, 4) || !izb_aligned(scores_out, 4) || !izb_aligned(parents_out, 4) ||
        !izb_aligned(tokens_out, 4))
        return IZB_ERR_BAD_ARG;
    const int64_t rows = groups * beams, outs = groups * n_out;
    // a group's scores and marks are read before its results are written, so a call may update them in place: the whole
    // array or none of it
    const bool same_scores = scores == scores_out, same_marks = finished == finished_out;
    if (same_scores ? n_out != beams : (scores_out < scores + rows && scores < scores_out + outs)) return IZB_ERR_BAD_ARG;
    if (finished && finished_out && (same_marks ? n_out != beams : (finished_out < finished + rows && finished < finished_out + outs)))
        return IZB_ERR_BAD_ARG;
    const SelectPlan pl = select_plan(ctx, dtype, groups, beams, vocab);
    if (rows > INT32_MAX / pl.tiles) return IZB_ERR_UNSUPPORTED;
    const size_t need = select_bytes(pl, rows, n_out);
    if (!workspace || workspace_bytes < need || !izb_aligned(workspace, 8)) return IZB_ERR_BAD_ARG;
    SelectParams p = {};
    p.logits = logits;
    p.scores = scores;
    p.finished = finished;
    p.scores_out = scores_out;
    p.parents_out = parents_out;
    p.tokens_out = tokens_out;
    p.finished_out = finished_out;
    p.tile_ml = static_cast<float2*>(workspace);
    p.tile_top = reinterpret_cast<u64*>(p.tile_ml + rows * pl.tiles);
    p.ld = ld;
    p.vocab = static_cast<int>(vocab);
    p.beams = beams;
    p.tiles = static_cast<int>(pl.tiles);
    p.n_out = n_out;
    p.eos = eos;
    p.status = ctx->d_status;
    izb::DeviceGuard guard(ctx->device);
    if (!guard.ok) return IZB_ERR_LAUNCH;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(rows * pl.tiles);
    if (dtype == IZB_F32) IZB_CUDA_TRY(launch_tiles<float>(ctx, s, p, pl.large, grid));
    else if (dtype == IZB_F16) IZB_CUDA_TRY(launch_tiles<__half>(ctx, s, p, pl.large, grid));
    else IZB_CUDA_TRY(launch_tiles<__nv_bfloat16>(ctx, s, p, pl.large, grid));
    IZB_CUDA_TRY(izb::launch_chained(ctx, beam_join_kernel, dim3(static_cast<unsigned>(groups)), dim3(BS_THREADS), 0, s, p));
    ctx->launches.fetch_add(2, std::memory_order_relaxed);
    return IZB_OK;
}

int32_t izb_kv_pages_reorder(izb_ctx* ctx, izb_stream stream, const izb_kv_pages* layers, int32_t n_layers, const int32_t* parents,
                             int64_t groups, int32_t beams, const int32_t* seq_lens, int32_t* page_table_out) {
    if (!ctx || groups < 0 || beams <= 0 || n_layers <= 0 || !layers) return IZB_ERR_BAD_ARG;
    if (groups == 0) return IZB_OK;
    if (beams > RO_MAX_BEAMS || n_layers > RO_MAX_LAYERS || groups > 65535 / beams) return IZB_ERR_UNSUPPORTED;
    if (!parents || !seq_lens || !page_table_out) return IZB_ERR_BAD_ARG;
    if (!izb_aligned(parents, 4) || !izb_aligned(seq_lens, 4) || !izb_aligned(page_table_out, 4)) return IZB_ERR_BAD_ARG;
    const izb_kv_pages& a = layers[0];
    if (!a.page_table || !izb_aligned(a.page_table, 4)) return IZB_ERR_BAD_ARG;
    if (a.quantization < IZB_KV_NONE || a.quantization > IZB_KV_Q4_0 || a.page_size <= 0 || a.kv_heads <= 0 || a.max_pages_per_seq <= 0)
        return IZB_ERR_BAD_ARG;
    if (a.head_dim != 64 && a.head_dim != 128) return IZB_ERR_UNSUPPORTED;
    if (a.page_size > INT32_MAX / a.kv_heads / a.head_dim / 2) return IZB_ERR_UNSUPPORTED;
    // rows of the old table are read while rows of the new one are written
    const int64_t entries = groups * beams * a.max_pages_per_seq;
    if (page_table_out < a.page_table + entries && a.page_table < page_table_out + entries) return IZB_ERR_BAD_ARG;
    ReorderParams p = {};
    for (int i = 0; i < n_layers; ++i) {
        const izb_kv_pages& l = layers[i];
        if (l.page_table != a.page_table || l.quantization != a.quantization || l.page_size != a.page_size || l.kv_heads != a.kv_heads ||
            l.head_dim != a.head_dim || l.max_pages_per_seq != a.max_pages_per_seq)
            return IZB_ERR_BAD_ARG;
        if (!l.k_values || !l.v_values || !izb_aligned(l.k_values, 16) || !izb_aligned(l.v_values, 16)) return IZB_ERR_BAD_ARG;
        if (a.quantization != IZB_KV_NONE && (!l.k_scales || !l.v_scales || !izb_aligned(l.k_scales, 4) || !izb_aligned(l.v_scales, 4)))
            return IZB_ERR_BAD_ARG;
        p.layer[i] = {static_cast<uint8_t*>(l.k_values), static_cast<uint8_t*>(l.v_values),
                      a.quantization == IZB_KV_NONE ? nullptr : l.k_scales, a.quantization == IZB_KV_NONE ? nullptr : l.v_scales};
    }
    p.table = a.page_table;
    p.table_out = page_table_out;
    p.parents = parents;
    p.lens = seq_lens;
    p.status = ctx->d_status + 6;
    p.max_pages = a.max_pages_per_seq;
    p.page_bytes = static_cast<long long>(izb_kv_page_bytes(a.quantization, a.page_size, a.kv_heads, a.head_dim));
    p.row_bytes = p.page_bytes / a.page_size;
    p.page_scales = static_cast<int>(izb_kv_page_scales(a.quantization, a.page_size, a.kv_heads, a.head_dim));
    p.row_scales = a.quantization == IZB_KV_Q4_0 ? p.page_scales / a.page_size : 0;
    p.beams = beams;
    p.page_size = a.page_size;
    p.n_layers = n_layers;
    // 32 KB of a page per CTA and trip; a CTA finds out first what there is to copy, so a big batch gets no more of them than
    // keep the SMs busy eight times over (16 x 8 beams, 36 layers: bf16 98.2 us against 111.6 with a CTA for every 32 KB, Int8
    // 45.9 against 53.3, Q4_0 39.0 against 48.3; one group 10.8 against 10.0)
    p.splits = static_cast<int>((p.page_bytes + RO_THREADS * 128 - 1) / (RO_THREADS * 128));
    const int64_t units = static_cast<int64_t>(n_layers) * 2 * p.splits;
    const int64_t most = (static_cast<int64_t>(RO_WAVES) * 5 * ctx->sm_count + groups * beams - 1) / (groups * beams);
    const unsigned per_child = static_cast<unsigned>(units < most ? units : most);
    izb::DeviceGuard guard(ctx->device);
    if (!guard.ok) return IZB_ERR_LAUNCH;
    IZB_CUDA_TRY(izb::launch_chained(ctx, kv_pages_reorder_kernel, dim3(per_child, static_cast<unsigned>(groups * beams)),
                                     dim3(RO_THREADS), 0, static_cast<cudaStream_t>(stream), p));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

int32_t izb_beam_trace(izb_ctx* ctx, izb_stream stream, const int32_t* parents, const int32_t* tokens, int64_t steps, int64_t groups,
                       int32_t beams, const int32_t* last, int32_t picks, int32_t* out, int64_t ld_out) {
    if (!ctx || steps < 0 || groups < 0 || beams <= 0 || picks < 0 || ld_out < steps) return IZB_ERR_BAD_ARG;
    if (steps == 0 || groups == 0 || picks == 0) return IZB_OK;
    if (!parents || !tokens || !last || !out) return IZB_ERR_BAD_ARG;
    if (!izb_aligned(parents, 4) || !izb_aligned(tokens, 4) || !izb_aligned(last, 4) || !izb_aligned(out, 4)) return IZB_ERR_BAD_ARG;
    if (steps > INT32_MAX || groups > INT32_MAX / 128 || picks > INT32_MAX / groups) return IZB_ERR_UNSUPPORTED;
    izb::DeviceGuard guard(ctx->device);
    if (!guard.ok) return IZB_ERR_LAUNCH;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (beams <= 32) {
        // one chunk for every place of the CTA's warps, of whole reads ahead
        const int64_t places = TR_WARPS * (32 / beams), chunk = ((steps + places - 1) / places + 15) / 16 * 16;
        const int64_t warps = ((steps + chunk - 1) / chunk + 32 / beams - 1) / (32 / beams);  // a short trace is one warp's
        const int ranks = warps >= 8 && groups <= ctx->sm_count ? 4 : 1;
        // a lane's chunk of up to 32 steps is read once where the registers allow it
        auto kern = ranks == 4 && chunk > 16 ? beam_trace_chunks_kernel<32> : beam_trace_chunks_kernel<16>;
        IZB_CUDA_TRY(izb::launch_chained_cluster(ctx, ranks, kern, dim3(static_cast<unsigned>(groups * ranks)),
                                                 dim3(static_cast<unsigned>((warps + ranks - 1) / ranks * 32)), 0, st, parents, tokens, last, out, static_cast<int>(steps), beams, picks,
                                                 static_cast<long long>(groups), static_cast<long long>(ld_out), static_cast<int>(chunk), ranks,
                                                 ctx->d_status + 6));
    } else {
        const unsigned grid = static_cast<unsigned>((groups * picks + 127) / 128);
        IZB_CUDA_TRY(izb::launch_chained(ctx, beam_trace_kernel, dim3(grid), dim3(128), 0, st, parents, tokens, last, out,
                                         static_cast<int>(steps), beams, picks, static_cast<long long>(groups), static_cast<long long>(ld_out),
                                         ctx->d_status + 6));
    }
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

}  // extern "C"
