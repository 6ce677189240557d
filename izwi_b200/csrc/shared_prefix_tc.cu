// The prefix part of the shared-prefix attention on the 5th-generation tensor cores.
//
// One CTA per (group, KV head, block of query rows, chunk of prefix tokens).  Query rows are the 128 lanes of tensor
// memory; a tile is 128 tokens:
//   S = Q K^T   tcgen05.mma, both operands from shared memory            -> 128 fp32 columns
//   P = 2^(scale S - m), bf16, written over S by the threads that own the rows
//   O += P V    tcgen05.mma, P from tensor memory, V token-major           -> D fp32 columns
// Two accumulator sets keep the tensor cores busy while weights are computed: up to 128 rows both hold the same rows and
// take the tiles in turn (and are joined at the end); above, each holds 128 of 256 rows and
// every tile serves both, so that the prefix is read once for 256 rows.
//   warps 0..3, 4..7   weights of set 0, 1: a thread owns a row
//   bf16 pages:  warp 8 fetches tiles (TMA, four token rows of a paged pool at a time), warp 9 issues the products
//   codes:       warps 8..15 convert tiles through registers, once for all rows; warp 16 issues the products
// Rows of a tile are 128-byte swizzle rows, 64 channels each: K is the K-major operand, V the same bytes read MN-major.
#include <climits>

#include "shared_prefix.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace izb {
namespace shared_prefix {
namespace {

constexpr int TC_TILE = 128;                    // tokens
constexpr int TC_COPY = 256;                    // converting threads
constexpr int TC_CALLED = 3;                    // tiles ahead of the conversion that are called into L2
// Threads and, for codes, registers: 640 threads of 96 at launch become 256 x 128 + 256 x 88 + 128 x 48 = 640 x 96.  bf16:
// 384 threads of 168, enough for a row's 128 scores at once.
constexpr int TC_WEIGHT_REGS = 128, TC_COPY_REGS = 88, TC_ISSUE_REGS = 48, TC_LAUNCH_REGS = 96;
constexpr int tc_threads(int quant) { return quant == IZB_KV_NONE ? 384 : 256 + TC_COPY + 128; }
constexpr int TC_HALF = TC_TILE * 128;          // bytes of 64 channels of a tile

struct TcShared {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2];
    unsigned long long s_full[2], p_full[2][2], pv_done[2];  // p_full: per set and half of a tile's tokens
    uint32_t place[4][TC_TILE];  // per tile, four in turn: pool token of each tile token
    uint32_t page[4][TC_TILE];   // Int8: its page
    unsigned long long q_full;
    float2 ml[2][128];           // narrow blocks: maximum and sum of a row in either set
    uint32_t tmem;
    int copy_failed;  // the unit at which a wait gave up
    int failed;       // some wait gave up
};

// Waits for a phase of a barrier, at most IZB_WAIT_LIMIT_CLOCKS, suspended for up to 20 us at a time.
__device__ __forceinline__ bool wait_phase(unsigned long long* bar, int parity) {
    const uint32_t at = smem_u32(bar);
    auto try_wait = [&]() {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(at), "r"(parity), "r"(20000) : "memory");
        return ok != 0;
    };
    if (try_wait()) return true;
    const long long t0 = clock64();
    while (!try_wait())
        if (clock64() - t0 > IZB_WAIT_LIMIT_CLOCKS) return false;
    return true;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 lanes x 64 consecutive fp32 columns: thread i of the warp receives row (lane base + i).
__device__ __forceinline__ void tc_ld_32x64(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t* q = r + h * 32;
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]), "=r"(q[8]),
              "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]), "=r"(q[16]),
              "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]), "=r"(q[24]),
              "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
            : "r"(taddr + h * 32)
            : "memory");
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_st_32x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_st_32x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Rows of 128 bytes under the 128-byte swizzle with the row index the product's K: 64 consecutive elements of the other
// index per row, the next 64 `half` bytes on; groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_mn_major_sw128(uint32_t saddr, uint32_t half) {
    return umma_desc_k_major_sw128(saddr) | (static_cast<uint64_t>(half >> 4) << 16);
}

template <int D>
__device__ __forceinline__ uint32_t tile_place(int r, int c) {  // 16-byte chunk c of the row's D bf16 values
    return static_cast<uint32_t>((c >> 3) * TC_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Four rows of the pool, 64 channels from c, as four swizzled rows of 128 bytes; rows outside the tensor become zeros.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int c, int4 rows, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::
            "r"(dst), "l"(map), "r"(c), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(bar)
        : "memory");
}

// ---- tiles ---------------------------------------------------------------------------------------------------------
struct Maps {
    CUtensorMap box[2];   // K, V: 64 channels x box_rows consecutive pool tokens
    CUtensorMap row[2];   // 64 channels x 1 token, for the four-row form
    int box_rows;         // a power of two that divides the page, at most 64; 0: pages do not allow 8 or more
};

// bf16: one warp.  A full tile comes as boxes of consecutive tokens of a page; the last tile of a chunk, and every tile
// where pages are no multiple of eight tokens, four single rows at a time, rows past the end as zeros.  (Single rows move
// about 6 bytes a cycle, boxes several times as much.)
template <int D>
__device__ __forceinline__ void fetch_role(const Params& p, const Maps& maps, int src_row, int kh, int t0, int n_tok, uint32_t k_ring,
                                           uint32_t v_ring, TcShared& sh) {
    constexpr int TILE_BYTES = TC_TILE * D * 2;
    const Source& src = p.prefix;
    const int lane = threadIdx.x & 31;
    const int n_tiles = (n_tok + TC_TILE - 1) / TC_TILE;
    const int* table = src.table + static_cast<long long>(src_row) * src.max_pages;
    auto place = [&](int tok) -> int {  // pool token, or a row outside the tensor
        if (tok >= n_tok) return -1;
        const unsigned at = static_cast<unsigned>(t0 + tok), pg = at / static_cast<unsigned>(src.page_size);
        return table[pg] * src.page_size + static_cast<int>(at - pg * src.page_size);
    };
    const int boxes = maps.box_rows ? TC_TILE / maps.box_rows : 0;  // per 64 channels
    auto in_boxes = [&](int tile) { return boxes && (tile + 1) * TC_TILE <= n_tok; };
    const int my_half = boxes ? lane / boxes : 0, my_box = boxes ? lane - my_half * boxes : 0;
    auto places = [&](int tile) {
        if (in_boxes(tile)) return make_int4(place(tile * TC_TILE + my_box * maps.box_rows), 0, 0, 0);
        const int tok = tile * TC_TILE + 4 * lane;
        return make_int4(place(tok), place(tok + 1), place(tok + 2), place(tok + 3));
    };
    int4 rows = places(0);
    int units = 0;
    bool ok = true;
    for (int tile = 0; tile < n_tiles && ok; ++tile) {
        const int4 now = rows;
        if (tile + 1 < n_tiles) rows = places(tile + 1);
#pragma unroll
        for (int kv = 0; kv < 2 && ok; ++kv) {
            const int slot = tile & 1;
            ok = __all_sync(0xFFFFFFFFu, wait_phase(kv ? &sh.v_empty[slot] : &sh.k_empty[slot], ((tile >> 1) & 1) ^ 1));
            if (!ok) break;
            const uint32_t bar = smem_u32(kv ? &sh.v_full[slot] : &sh.k_full[slot]), dst = (kv ? v_ring : k_ring) + slot * TILE_BYTES;
            if (lane == 0) mbar_expect_tx(bar, TILE_BYTES);
            __syncwarp();
            if (in_boxes(tile)) {
                if (my_half < D / 64)
                    tma_load_2d(dst + my_half * TC_HALF + my_box * maps.box_rows * 128, &maps.box[kv], kh * D + my_half * 64, now.x, bar);
            } else {
#pragma unroll
                for (int h = 0; h < D / 64; ++h) tma_gather4(dst + h * TC_HALF + lane * 512, &maps.row[kv], kh * D + h * 64, now, bar);
            }
            ++units;
        }
    }
    if (!ok) {
        // shared memory is given back only after the copies under way have landed
        sh.failed = 1;
        for (int u = units > 4 ? units - 4 : 0; u < units; ++u) wait_phase((u & 1) ? &sh.v_full[(u >> 1) & 1] : &sh.k_full[(u >> 1) & 1], (u >> 2) & 1);
    }
}

// Codes.  Units of the stream: K of tile 0, V of tile 0, K of tile 1, ...  Slot (tile & 1) of either ring.
template <int D, int Q>
__device__ __forceinline__ void convert_role(const Params& p, int src_row, int kh, int t0, int n_tok, uint32_t k_ring, uint32_t v_ring, TcShared& sh) {
    constexpr int ROW = Q == IZB_KV_INT8 ? D : D / 2;
    constexpr int CHUNKS = ROW / 16, RSTEP = TC_COPY / CHUNKS, N = TC_TILE / RSTEP;  // chunks of a unit per thread
    constexpr int TILE_BYTES = TC_TILE * D * 2;
    const Source& src = p.prefix;
    const int t = threadIdx.x - 256, lane = t & 31, my_r = t / CHUNKS, my_c = t % CHUNKS;
    const int n_tiles = (n_tok + TC_TILE - 1) / TC_TILE;
    const uint32_t stride = static_cast<uint32_t>(p.kv_heads) * ROW;
    const uint8_t* from[2] = {src.k + kh * ROW + my_c * 16, src.v + kh * ROW + my_c * 16};
    const float* scales_from[2] = {src.k_scales, src.v_scales};
    const int* table = src.table + static_cast<long long>(src_row) * src.max_pages;
    int page = 0, in_page = 0;
    auto look_up = [&](int tok) {  // threads 0..127: the place of a tile's token, a tile ahead
        if (t < TC_TILE && tok < n_tok) {
            const unsigned at = static_cast<unsigned>(t0 + tok), pg = at / static_cast<unsigned>(src.page_size);
            in_page = static_cast<int>(at - pg * src.page_size);
            page = table[pg];
        }
    };
    auto publish = [&](int tile) {
        if (t < TC_TILE) {
            const bool in = tile * TC_TILE + t < n_tok;
            sh.place[tile & 3][t] = in ? static_cast<uint32_t>(page) * static_cast<uint32_t>(src.page_size) + static_cast<uint32_t>(in_page) : 0u;
            if (Q == IZB_KV_INT8) sh.page[tile & 3][t] = in ? static_cast<uint32_t>(page) : 0u;
        }
    };
    // One warp waits for a slot, the barrier behind it holds the others; then all see whether a wait has given up by now.
    auto slot_free = [&](unsigned long long* empty, int tile, int kv) {
        if (t < 32 && !wait_phase(&empty[tile & 1], ((tile >> 1) & 1) ^ 1)) {
            atomicMin(&sh.copy_failed, 2 * tile + kv);
            sh.failed = 1;
        }
    };
    auto given_up = [&](int tile, int kv) { return *static_cast<volatile int*>(&sh.copy_failed) <= 2 * tile + kv; };
    auto arrive = [&](unsigned long long* full, int tile) {
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full[tile & 1]));
    };
    look_up(t);

    const CodeBits<Q> bits;
    // the codes and scales of a unit, in registers; each buffer is filled again as soon as it has been converted, two units
    // ahead of its use
    uint4 raw[2][N];
    float sc[2][N];
    auto load = [&](int tile, int kv) {
        const int have = n_tok - tile * TC_TILE;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = j * RSTEP + my_r;
            const uint32_t place = sh.place[tile & 3][r];
            raw[kv][j] = make_uint4(0u, 0u, 0u, 0u);
            sc[kv][j] = 0.f;
            if (r < have) {
                raw[kv][j] = __ldcs(reinterpret_cast<const uint4*>(from[kv] + static_cast<uint64_t>(place) * stride));
                if constexpr (Q == IZB_KV_INT8) sc[kv][j] = scales_from[kv][sh.page[tile & 3][r]];
                else sc[kv][j] = scales_from[kv][static_cast<uint64_t>(place) * static_cast<uint32_t>(p.kv_heads * (D / 32)) + static_cast<uint32_t>(kh * (D / 32) + my_c)];
            }
        }
    };
    // Two units in registers are 32 KB on the way (Int8, D = 128), a third of what memory needs to run at its rate, so the
    // lines of tiles further ahead are called into L2.
    auto call = [&](int tile, int kv) {
        const int have = n_tok - tile * TC_TILE;
        if ((my_c * 16) % 128 != 0) return;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = j * RSTEP + my_r;
            if (r < have) asm volatile("prefetch.global.L2 [%0];" ::"l"(from[kv] + static_cast<uint64_t>(sh.place[tile & 3][r]) * stride));
        }
    };
#pragma unroll
    for (int i = 0; i < TC_CALLED; ++i) {
        publish(i);
        look_up((i + 1) * TC_TILE + t);
    }
    named_bar_sync(2, TC_COPY);
    load(0, 0);
    load(0, 1);
#pragma unroll
    for (int i = 1; i < TC_CALLED; ++i) {
        call(i, 0);
        call(i, 1);
    }
    for (int tile = 0; tile < n_tiles; ++tile) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            if (kv == 0) publish(tile + TC_CALLED);  // over a tile that nobody reads any more
            slot_free(kv ? sh.v_empty : sh.k_empty, tile, kv);
            named_bar_sync(2, TC_COPY);
            if (given_up(tile, kv)) return;
            if (kv == 0) look_up((tile + TC_CALLED + 1) * TC_TILE + t);
            const uint32_t base = (kv ? v_ring : k_ring) + (tile & 1) * TILE_BYTES;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int r = j * RSTEP + my_r;
                const uint32_t x[4] = {raw[kv][j].x, raw[kv][j].y, raw[kv][j].z, raw[kv][j].w};
                if constexpr (Q == IZB_KV_INT8) {
                    const uint32_t sc2 = pack_bf16x2(sc[kv][j], sc[kv][j]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t y[4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            y[2 * i] = hmul2(bits.pair(prmt(x[2 * h + i], 0u, 0x4140)), sc2);
                            y[2 * i + 1] = hmul2(bits.pair(prmt(x[2 * h + i], 0u, 0x4342)), sc2);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(base + tile_place<D>(r, my_c * 2 + h)), "r"(y[0]), "r"(y[1]),
                                     "r"(y[2]), "r"(y[3])
                                     : "memory");
                    }
                } else {
                    // a word's eight channels in the order 0, 4, 1, 5, 2, 6, 3, 7; so are the query rows, and the outputs are put back
                    uint32_t hi2, lo2;
                    split_scales(sc[kv][j], sc[kv][j], hi2, lo2);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = q4_value(bits.pair(x[w] >> (4 * e)), hi2, lo2);
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(base + tile_place<D>(r, my_c * 4 + w)), "r"(y[0]), "r"(y[1]),
                                     "r"(y[2]), "r"(y[3])
                                     : "memory");
                    }
                }
            }
            arrive(kv ? sh.v_full : sh.k_full, tile);
            if (tile + 1 < n_tiles) load(tile + 1, kv);
            call(tile + TC_CALLED, kv);
        }
    }
}

template <int D, int Q>
__global__ void __launch_bounds__(tc_threads(Q), 1)
    shared_prefix_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps, int wide) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ TcShared sh;
    constexpr int TILE_BYTES = TC_TILE * D * 2, Q_BYTES = 128 * D * 2;
    constexpr bool CODES = Q != IZB_KV_NONE;
    constexpr int ISSUE_WARP = CODES ? 16 : 9;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- the item ----
    int item = blockIdx.x;
    const int rb = item % p.row_blocks;
    item /= p.row_blocks;
    const int kh = item % p.kv_heads;
    item /= p.kv_heads;
    const int chunk = item % p.prefix.n_chunks, group = item / p.prefix.n_chunks;
    const int block_rows = wide ? 256 : 128;
    const int row0 = rb * block_rows, n_rows = min(block_rows, p.seqs * p.g - row0), seq0 = group * p.seqs;
    const int t0 = chunk * p.prefix.chunk;

    const uint32_t sq = smem_u32(smem), k_ring = sq + (wide ? 2 : 1) * Q_BYTES, v_ring = k_ring + 2 * TILE_BYTES;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), CODES ? TC_COPY / 32 : 1);
            mbar_init(smem_u32(&sh.v_full[i]), CODES ? TC_COPY / 32 : 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.p_full[i][0]), 4);
            mbar_init(smem_u32(&sh.p_full[i][1]), 4);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
        }
        mbar_init(smem_u32(&sh.q_full), 8);
        sh.copy_failed = INT_MAX;
        sh.failed = 0;
        mbar_fence_init();
    }
    __syncthreads();
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int n_tok = min(length_of(p.prefix, group) - t0, p.prefix.chunk);
    if (n_tok <= 0) return;  // the whole CTA, no tensor memory held
    const int n_tiles = (n_tok + TC_TILE - 1) / TC_TILE;
    // All 512 columns are this CTA's (the issuing warp takes them), so they begin at column 0.
    constexpr uint32_t tmem = 0;

    // Each role ends by itself: code shared behind it would have to fit the smallest of their register counts.
    if (CODES ? (warp >= 8 && warp < 16) : (warp >= 8 && warp != ISSUE_WARP)) {
        if constexpr (CODES) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_COPY_REGS));
            convert_role<D, Q>(p, group, kh, t0, n_tok, k_ring, v_ring, sh);
        } else if (warp == 8) {
            fetch_role<D>(p, maps, group, kh, t0, n_tok, k_ring, v_ring, sh);
        }
        __syncthreads();
    } else if (warp >= 8) {
        // ---------------- products ----------------
        if constexpr (CODES) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_ISSUE_REGS));
        if (warp == ISSUE_WARP) {
            tc_alloc(smem_u32(&sh.tmem), 512);
            // The whole warp walks the schedule, so that addresses and descriptors stay in uniform registers, and one lane
            // issues.  (With a single-lane loop each product's operands had to be moved there one by one between the other
            // warps' instructions: 110 to 280 cycles a product instead of 64.)
            const uint32_t s_idesc = umma_idesc_bf16(TC_TILE);
            const uint32_t o_idesc = umma_idesc_bf16(D) | (1u << 16);  // V is MN-major
            const uint64_t q_desc = umma_desc_k_major_sw128(sq), k_desc = umma_desc_k_major_sw128(k_ring);
            const uint64_t v_desc = desc_mn_major_sw128(v_ring, TC_HALF);
            bool ok = wait_phase(&sh.q_full, 0);
            auto scores = [&](int v, int tile, bool first_use, bool last_use) {
                if (first_use && ok) ok = wait_phase(&sh.k_full[tile & 1], (tile >> 1) & 1);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) return;
                tc_fence_after();
                const uint64_t a = q_desc + static_cast<uint64_t>((wide ? v : 0) * (Q_BYTES >> 4)), b = k_desc + static_cast<uint64_t>((tile & 1) * (TILE_BYTES >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t off = ((k >> 2) * TC_HALF + (k & 3) * 32) >> 4;
                        tc_mma_f16(v * 128, a + off, b + off, s_idesc, k != 0);
                    }
                    if (last_use) tc_commit(smem_u32(&sh.k_empty[tile & 1]));
                    tc_commit(smem_u32(&sh.s_full[v]));
                }
                __syncwarp();
            };
            auto values = [&](int v, int tile, int nth, bool first_use, bool last_use) {
                if (first_use && ok) ok = wait_phase(&sh.v_full[tile & 1], (tile >> 1) & 1);
                const uint64_t b = v_desc + static_cast<uint64_t>((tile & 1) * (TILE_BYTES >> 4));
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // the first 64 tokens while the weights of the others are computed
                    if (ok) ok = wait_phase(&sh.p_full[v][half], nth & 1);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) return;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = half * 4; k < half * 4 + 4; ++k)
                            mma_ts(256 + v * 128, v * 128 + k * 8, b + static_cast<uint64_t>(k * (2048 >> 4)), o_idesc, nth != 0 || k != 0);
                        if (half && last_use) tc_commit(smem_u32(&sh.v_empty[tile & 1]));
                        if (half) tc_commit(smem_u32(&sh.pv_done[v]));
                    }
                    __syncwarp();
                }
            };
            if (wide) {
                scores(0, 0, true, false);
                scores(1, 0, false, true);
                for (int t = 0; t < n_tiles && ok; ++t) {
                    values(0, t, t, true, false);
                    if (t + 1 < n_tiles) scores(0, t + 1, true, false);
                    values(1, t, t, false, true);
                    if (t + 1 < n_tiles) scores(1, t + 1, false, true);
                }
            } else {
                scores(0, 0, true, true);
                if (n_tiles > 1) scores(1, 1, true, true);
                for (int t = 0; t < n_tiles && ok; ++t) {
                    values(t & 1, t, t >> 1, true, true);
                    if (t + 2 < n_tiles) scores(t & 1, t + 2, true, true);
                }
            }
            if (!ok) sh.failed = 1;
        }
        __syncthreads();
        if (warp == ISSUE_WARP) {
            tc_fence_after();
            tc_dealloc(sh.tmem, 512);
            if (lane == 0 && sh.failed) atomicExch(p.status, 1);
        }
    } else {
        // ---------------- weights ----------------
        if constexpr (CODES) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_WEIGHT_REGS));
        // the query rows, K-major, all of a thread's 16-byte pieces under way at once
        {
            constexpr int C = D / 8, STEP = 256 / C, B = CODES ? 8 : 16;
            const int c = tid % C;
            for (int r0 = tid / C; r0 < block_rows; r0 += B * STEP) {
                uint4 x[B];
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int r = r0 + j * STEP, at = row0 + r;
                    x[j] = make_uint4(0u, 0u, 0u, 0u);
                    if (r < n_rows) {
                        const int s = at / p.g, h = at - s * p.g;
                        x[j] = *reinterpret_cast<const uint4*>(p.q + (seq0 + s) * p.ld_q + static_cast<long long>(kh * p.g + h) * D + c * 8);
                    }
                }
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int r = r0 + j * STEP;
                    uint4 y = make_uint4(x[j].x ^ p.q_sign, x[j].y ^ p.q_sign, x[j].z ^ p.q_sign, x[j].w ^ p.q_sign);
                    if (Q == IZB_KV_Q4_0) y = make_uint4(prmt(y.x, y.z, 0x5410), prmt(y.x, y.z, 0x7632), prmt(y.y, y.w, 0x5410), prmt(y.y, y.w, 0x7632));
                    if (r < block_rows)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(sq + (r >> 7) * Q_BYTES + tile_place<D>(r & 127, c)), "r"(y.x),
                                     "r"(y.y), "r"(y.z), "r"(y.w)
                                     : "memory");
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.q_full));
        }
        const int v = warp >> 2, row = (warp & 3) * 32 + lane;               // lane of tensor memory
        const int first = (wide ? v * 128 : 0) + (warp & 3) * 32;             // this warp's first row of the block
        const int mine = wide ? n_tiles : (n_tiles + 1 - v) / 2;              // tiles of this set
        const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + v * 128, t_o = t_lane + 256 + v * 128;
        const bool live = first < n_rows;                                      // else the warp only keeps the barriers going
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int n = 0; n < mine; ++n) {
            const int tile = wide ? n : 2 * n + v;
            if (!wait_phase(&sh.s_full[v], n & 1)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int left = n_tok - tile * TC_TILE;
            auto masked = [&](float(&s)[64], int c0) {
                if (left < c0 + 64) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (c0 + i >= left) s[i] = -INFINITY;
                }
            };
            auto largest = [&](const float(&s)[64]) {
                float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) t[k] = fmaxf(t[k], fmaxf(s[i + 2 * k], s[i + 2 * k + 1]));
                return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            };
            float s[2][64];  // codes: the halves one after the other, read twice
            if (live) {
                float top;
                tc_ld_32x64(t_s, s[0]);
                if constexpr (!CODES) tc_ld_32x64(t_s + 64, s[1]);
                masked(s[0], 0);
                top = largest(s[0]);
                if constexpr (CODES) tc_ld_32x64(t_s + 64, s[0]);
                masked(s[CODES ? 0 : 1], 64);
                top = fmaxf(top, largest(s[CODES ? 0 : 1]));
                // The reference point of a row follows its maximum only when that has grown by 2^8 in weight (not-less: also for
                // the first maximum): weights up to 2^8 are as exact as weights up to 1, and the output is seldom rescaled.
                if (__any_sync(0xFFFFFFFFu, !(top <= m + p.margin))) {
                    const float to = fmaxf(m, top), f = m == -INFINITY ? 0.f : ex2((m - to) * p.scale_log2);
                    m = to;
                    l *= f;
                    if (n > 0) {
                        if (!wait_phase(&sh.pv_done[v], (n - 1) & 1)) {  // the set's output so far is complete
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 8; ++c) {
                            uint32_t x[8];
                            tc_ld_32x8(t_o + c * 8, x);
#pragma unroll
                            for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                            tc_st_32x8(t_o + c * 8, x);
                        }
                    }
                }
            }
            const float u = m == -INFINITY ? 0.f : m * p.scale_log2;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (live) {
                    float(&x)[64] = s[CODES ? 0 : half];
                    if constexpr (CODES) {
                        tc_ld_32x64(t_s + half * 64, x);
                        masked(x, half * 64);
                    }
                    // weights over scores that have been read: 64 become 32 columns
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float a = ex2(fmaf(x[h * 32 + 2 * i], p.scale_log2, -u)), b = ex2(fmaf(x[h * 32 + 2 * i + 1], p.scale_log2, -u));
                            sum[i & 3] += a + b;
                            w[i] = pack_bf16x2(a, b);
                        }
                        tc_st_32x16(t_s + half * 32 + h * 16, w);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[v][half]));
            }
        }
        if (ok && mine > 0 && !wait_phase(&sh.pv_done[v], (mine - 1) & 1)) ok = false;
        if (!ok) sh.failed = 1;
        tc_fence_after();
        // Both sets are complete: the rows go through shared memory, where the tiles were, so that a row is written as one
        // run of memory.  Rows of D + 4 floats: consecutive ones start four banks apart.
        named_bar_sync(3, 256);
        constexpr int LD = D + 4;
        float* stage = reinterpret_cast<float*>(smem);
        if (live && mine > 0) {
            float* dst = stage + (v * 128 + row) * LD;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tc_ld_32x32(t_o + c * 32, o);
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float4 a = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]), b = make_float4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                    if (Q == IZB_KV_Q4_0) {
                        a = make_float4(o[i], o[i + 2], o[i + 4], o[i + 6]);
                        b = make_float4(o[i + 1], o[i + 3], o[i + 5], o[i + 7]);
                    }
                    *reinterpret_cast<float4*>(dst + c * 32 + i) = a;
                    *reinterpret_cast<float4*>(dst + c * 32 + i + 4) = b;
                }
            }
        }
        sh.ml[v][row] = make_float2(m, l);
        named_bar_sync(3, 256);
        const int chunks = p.prefix.n_chunks + p.own.n_chunks;
        constexpr int LANES = D / 4, RW = 32 / LANES;  // lanes of a row, rows of a warp at a time
        for (int r = warp * RW + lane / LANES; r < n_rows; r += 8 * RW) {
            const int d = (lane % LANES) * 4, at = row0 + r, s = at / p.g, h = at - s * p.g;
            const long long slot = (static_cast<long long>(seq0 + s) * p.heads + kh * p.g + h) * chunks + chunk;
            float4 x = *reinterpret_cast<const float4*>(stage + r * LD + d);  // row r & 127 of set r >> 7
            float2 a = sh.ml[r >> 7][r & 127];
            if (!wide && n_tiles > 1) {
                const float4 y = *reinterpret_cast<const float4*>(stage + (128 + r) * LD + d);
                const float2 b = sh.ml[1][r];
                const float top = fmaxf(a.x, b.x);
                const float f = a.x == -INFINITY ? 0.f : ex2((a.x - top) * p.scale_log2), g = b.x == -INFINITY ? 0.f : ex2((b.x - top) * p.scale_log2);
                x = make_float4(x.x * f + y.x * g, x.y * f + y.y * g, x.z * f + y.z * g, x.w * f + y.w * g);
                a = make_float2(top, a.y * f + b.y * g);
            }
            *reinterpret_cast<float4*>(p.acc + slot * D + d) = x;
            if (d == 0) p.ml[slot] = make_float2(a.x * p.scale_log2, a.y);
        }
        tc_fence_before();
        __syncthreads();
    }
}

template <int D, int Q>
int launch(izb_ctx* ctx, cudaStream_t s, const Params& p, int64_t items, bool wide) {
    auto kern = shared_prefix_tc_kernel<D, Q>;
    constexpr int RING = 4 * TC_TILE * D * 2, Q_BYTES = 128 * D * 2;
    static std::atomic<bool> ready[IZB_MAX_DEVICES];
    if (!ready[ctx->device].load(std::memory_order_relaxed)) {
        cudaFuncAttributes attr;
        IZB_CUDA_TRY(cudaFuncGetAttributes(&attr, kern));
        // the weight warps would wait for registers nobody has
        if (Q != IZB_KV_NONE && attr.numRegs < TC_LAUNCH_REGS) return IZB_ERR_LAUNCH;
        IZB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * Q_BYTES + RING));
        ready[ctx->device].store(true, std::memory_order_relaxed);
    }
    Maps maps = {};
    if (Q == IZB_KV_NONE) {
        int rows = 64;
        while (rows > 1 && p.prefix.page_size % rows) rows >>= 1;
        maps.box_rows = rows >= 8 ? rows : 0;
        // the pool as a matrix of tokens; how many it holds is not known here, and no row outside it is asked for
        const uint64_t dims[2] = {static_cast<uint64_t>(p.kv_heads) * D, 0x7FFFFFFFull}, strides[1] = {static_cast<uint64_t>(p.kv_heads) * D * 2};
        for (int i = 0; i < 4; ++i) {
            const uint32_t box[2] = {64, i < 2 && maps.box_rows ? static_cast<uint32_t>(maps.box_rows) : 1u};
            const int rc = tma_encode(i < 2 ? &maps.box[i] : &maps.row[i - 2], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, i & 1 ? p.prefix.v : p.prefix.k, dims,
                                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
            if (rc != IZB_OK) return rc;
        }
    }
    IZB_CUDA_TRY(launch_chained(ctx, kern, dim3(static_cast<unsigned>(items)), dim3(tc_threads(Q)), static_cast<size_t>((wide ? 2 : 1) * Q_BYTES + RING), s, p,
                                maps, wide ? 1 : 0));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

}  // namespace

int launch_prefix_tc(izb_ctx* ctx, cudaStream_t s, const Params& p, int head_dim, int64_t groups) {
    const bool wide = static_cast<int64_t>(p.seqs) * p.g > TC_ROWS;
    const int64_t items = groups * p.prefix.n_chunks * p.kv_heads * p.row_blocks;
    const int q = p.prefix.quant;
    if (head_dim == 128)
        return q == IZB_KV_NONE ? launch<128, IZB_KV_NONE>(ctx, s, p, items, wide) : q == IZB_KV_INT8 ? launch<128, IZB_KV_INT8>(ctx, s, p, items, wide)
                                                                                                       : launch<128, IZB_KV_Q4_0>(ctx, s, p, items, wide);
    return q == IZB_KV_NONE ? launch<64, IZB_KV_NONE>(ctx, s, p, items, wide) : q == IZB_KV_INT8 ? launch<64, IZB_KV_INT8>(ctx, s, p, items, wide)
                                                                                                  : launch<64, IZB_KV_Q4_0>(ctx, s, p, items, wide);
}

}  // namespace shared_prefix
}  // namespace izb
