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
//   codes:       four or eight warps convert K and as many V through registers, once for all rows; the next issues the products
// Measured: 64 sequences x 4 heads over 32,768 bf16 tokens, 8 KV heads of 128, 46.5 us with the join = 0.74 PFLOP/s; a tile
// under 256 rows takes 3,900 cycles of which the products need 2,048 and the exponentials 2,130: weights and products of a
// set wait for one another.  Codes, 32 rows: Int8 3,000 cycles a tile, Q4_0 2,000 (conversion and weights).
// Rows of a tile are 128-byte swizzle rows, 64 channels each: K is the K-major operand, V the same bytes read MN-major.
#include "shared_prefix.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace izb {
namespace shared_prefix {
namespace {

constexpr int TC_TILE = 128;                    // tokens
// Threads and registers.  bf16 pages: 384 threads of 168, enough for a row's 128 scores at once.  Codes: CONV threads convert
// K and as many V, and the launch's registers are shared out: 640 x 96 = 256 x 128 + 256 x 88 + 128 x 48 (CONV = 128),
// 896 x 72 = 256 x 112 + 512 x 64 + 128 x 24 (CONV = 256).
template <int Q, int CONV>
struct Roles {
    static constexpr bool CODES = Q != IZB_KV_NONE;
    static constexpr int THREADS = CODES ? 256 + 2 * CONV + 128 : 384;
    static constexpr int ISSUE_WARP = CODES ? 8 + 2 * CONV / 32 : 9;
    static constexpr int LAUNCH = !CODES ? 168 : CONV == 128 ? 96 : 72, WEIGHTS = CONV == 128 ? 128 : 112, COPY = CONV == 128 ? 88 : 64,
                         ISSUE = CONV == 128 ? 48 : 24;
    static_assert(!CODES || 256 * WEIGHTS + 2 * CONV * COPY + 128 * ISSUE <= THREADS * LAUNCH, "registers that nobody has");
};
constexpr int TC_HALF = TC_TILE * 128;          // bytes of 64 channels of a tile

struct TcShared {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2];
    unsigned long long s_full[2], p_full[2][2], pv_done[2][2];  // per set and half of a tile's tokens
    unsigned long long q_full;
    float2 ml[2][128];           // narrow blocks: maximum and sum of a row in either set
    uint32_t tmem;
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

// Codes.  CONV / 32 warps convert the K of every tile and as many others the V, each its share; no warp waits for another
// one, so that the copies, conversions and stores of some fill the pauses of others.  A lane copies (cp.async) exactly the
// pieces that it converts, `stages` tiles ahead, and so needs no barrier; in registers they would share the few counters
// on which a warp waits for loads, and waiting for a tile's would be waiting for the next one's.
// Slot (tile & 1) of either ring.
template <int D, int Q, int CONV>
struct Codes {
    static constexpr int ROW = Q == IZB_KV_INT8 ? D : D / 2;
    static constexpr int CHUNKS = ROW / 16, ROWS = 32 / CHUNKS, SHARE = TC_TILE / (CONV / 32), N = SHARE / ROWS;  // tokens copied at a time, a warp's share, copies of it
    static constexpr int SCALES = Q == IZB_KV_Q4_0 ? N * 32 * 4 : 0;
    static constexpr int STAGE = N * 32 * 16 + SCALES;                          // bytes of a warp's share of a tile
    static constexpr __host__ __device__ int bytes(int stages) { return Q == IZB_KV_NONE ? 0 : stages * 2 * (CONV / 32) * STAGE; }
    // tiles under way: what fits beside query rows and tiles of 16 bits
    static constexpr __host__ __device__ int stages(bool wide) { return D == 64 ? 3 : wide ? 1 : Q == IZB_KV_INT8 ? 2 : 3; }
};
template <int D, int Q, int CONV>
__device__ __forceinline__ void convert_role(const Params& p, int kv, int warp, int src_row, int kh, int t0, int n_tok, uint32_t ring, uint32_t staging,
                                             int stages, TcShared& sh) {
    using C = Codes<D, Q, CONV>;
    constexpr int LOW = C::CHUNKS / (D / 64);  // pieces of 16 bytes that hold 64 channels
    constexpr int TILE_BYTES = TC_TILE * D * 2;
    const Source& src = p.prefix;
    const int lane = threadIdx.x & 31, n_tiles = (n_tok + TC_TILE - 1) / TC_TILE;
    // The eight lanes of a store phase convert channels of the same 64 for several tokens, whose swizzles differ: eight
    // different 16-byte columns of the banks.
    const int my_c = (lane & (LOW - 1)) + (D == 128 ? ((lane >> 3) & 1) * LOW : 0);
    const int my_r = D == 128 ? (lane & 7) / LOW + (lane >> 4) * (8 / LOW) : lane / LOW;
    const uint32_t stride = static_cast<uint32_t>(p.kv_heads) * C::ROW;
    const uint8_t* from = (kv ? src.v : src.k) + kh * C::ROW + my_c * 16;
    const float* scales_from = (kv ? src.v_scales : src.k_scales) + (Q == IZB_KV_Q4_0 ? kh * (D / 32) + my_c : 0);
    const int* table = src.table + static_cast<long long>(src_row) * src.max_pages;
    unsigned long long *full = kv ? sh.v_full : sh.k_full, *empty = kv ? sh.v_empty : sh.k_empty;

    // This lane's token of the tiles to be copied: its page is asked for a tile ahead of that.
    const int my_tok = warp * C::SHARE + (lane & (C::SHARE - 1));
    int tok = my_tok, at_page = (t0 + my_tok) / src.page_size, rest = t0 + my_tok - at_page * src.page_size;
    int page = tok < n_tok ? table[at_page] : 0;
    float scale[3] = {0.f, 0.f, 0.f};  // Int8: of the page of the lane's token, in turn
    auto copy = [&](uint32_t to) {
        const bool in = tok < n_tok;  // what lies past the end becomes zeros with a zero scale
        const uint32_t my_place = in ? static_cast<uint32_t>(page) * static_cast<uint32_t>(src.page_size) + static_cast<uint32_t>(rest) : ~0u;
        if (Q == IZB_KV_INT8) {
            scale[0] = scale[1];
            scale[1] = scale[2];
            scale[2] = in ? scales_from[page] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < C::N; ++j) {
            uint32_t place = __shfl_sync(0xFFFFFFFFu, my_place, j * C::ROWS + my_r);
            const bool have = place != ~0u;
            place = have ? place : 0u;
            cp16(to + j * 512, from + static_cast<uint64_t>(place) * stride, have ? 16 : 0);
            if constexpr (Q == IZB_KV_Q4_0)
                cp4(to + C::N * 512 - lane * 12 + j * 128, scales_from + static_cast<uint64_t>(place) * static_cast<uint32_t>(p.kv_heads * (D / 32)), have ? 4 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        tok += TC_TILE;
        at_page += src.step_pages;
        rest += src.step_rest;
        if (rest >= src.page_size) { rest -= src.page_size; ++at_page; }
        page = tok < n_tok ? table[at_page] : 0;
    };
    const CodeBits<Q> bits;
    staging += ((kv * (CONV / 32) + warp) * stages) * C::STAGE + lane * 16;
    for (int i = 0; i < stages; ++i) copy(staging + i * C::STAGE);
    bool ok = true;
    uint32_t slot = staging;
    for (int tile = 0; tile < n_tiles; ++tile) {
        if (stages == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
        else if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 2;" ::: "memory");
        if (!wait_phase(&empty[tile & 1], ((tile >> 1) & 1) ^ 1)) {
            ok = false;
            break;
        }
        const uint32_t base = ring + (tile & 1) * TILE_BYTES;
        uint32_t my_scale = 0;
        if (Q == IZB_KV_INT8) {
            const float s = stages == 1 ? scale[2] : stages == 2 ? scale[1] : scale[0];
            my_scale = pack_bf16x2(s, s);
        }
#pragma unroll
        for (int j = 0; j < C::N; ++j) {
            const int r = warp * C::SHARE + j * C::ROWS + my_r;
            const uint4 raw = lds128(slot + j * 512);
            const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
            if constexpr (Q == IZB_KV_INT8) {
                const uint32_t sc2 = __shfl_sync(0xFFFFFFFFu, my_scale, j * C::ROWS + my_r);
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
                const float s = __uint_as_float(lds32(slot + C::N * 512 - lane * 12 + j * 128));
                uint32_t hi2, lo2;
                split_scales(s, s, hi2, lo2);
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
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full[tile & 1]));
        copy(slot);
        slot = slot == staging + (stages - 1) * C::STAGE ? staging : slot + C::STAGE;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) sh.failed = 1;
}

// The sequence of its group and the query head (of those of the KV head) a row of the block stands for, and a step of rows.
struct HeadStep {
    int s, h;
    __device__ __forceinline__ HeadStep(const Params& p, int rows) : s(rows / p.g), h(rows - s * p.g) {}
};
struct HeadRow {
    int s, h;
    __device__ __forceinline__ HeadRow(const Params& p, int row) : s(row / p.g), h(row - s * p.g) {}
    __device__ __forceinline__ void advance(const HeadStep& by, const Params& p) {
        s += by.s;
        h += by.h;
        if (h >= p.g) { h -= p.g; ++s; }
    }
};

template <int D, int Q, int CONV>
__global__ void __launch_bounds__(Roles<Q, CONV>::THREADS, 1)
    shared_prefix_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps, int wide) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ TcShared sh;
    constexpr int TILE_BYTES = TC_TILE * D * 2, Q_BYTES = 128 * D * 2;
    using R = Roles<Q, CONV>;
    constexpr bool CODES = R::CODES;
    constexpr int ISSUE_WARP = R::ISSUE_WARP;
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
            mbar_init(smem_u32(&sh.k_full[i]), CODES ? CONV / 32 : 1);
            mbar_init(smem_u32(&sh.v_full[i]), CODES ? CONV / 32 : 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.p_full[i][0]), 4);
            mbar_init(smem_u32(&sh.p_full[i][1]), 4);
            mbar_init(smem_u32(&sh.pv_done[i][0]), 1);
            mbar_init(smem_u32(&sh.pv_done[i][1]), 1);
        }
        mbar_init(smem_u32(&sh.q_full), 8);
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
    if (CODES ? (warp >= 8 && warp < ISSUE_WARP) : (warp >= 8 && warp != ISSUE_WARP)) {
        if constexpr (CODES) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::COPY));
            const int kv = (warp - 8) / (CONV / 32);
            convert_role<D, Q, CONV>(p, kv, (warp - 8) % (CONV / 32), group, kh, t0, n_tok, kv ? v_ring : k_ring, v_ring + 2 * TILE_BYTES,
                               Codes<D, Q, CONV>::stages(wide), sh);
        } else if (warp == 8) {
            fetch_role<D>(p, maps, group, kh, t0, n_tok, k_ring, v_ring, sh);
        }
        __syncthreads();
    } else if (warp >= 8) {
        // ---------------- products ----------------
        if constexpr (CODES) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::ISSUE));
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
                        tc_commit(smem_u32(&sh.pv_done[v][half]));
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
        if constexpr (CODES) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::WEIGHTS));
        // With at most 32 (64) rows the second set has them once more from lane 32 (64) on, so that the two sets' weights are
        // computed on different quarters of the SM.
        const int twin = wide || n_rows > 64 ? 128 : n_rows > 32 ? 64 : 32;
        // the query rows, K-major, all of a thread's 16-byte pieces under way at once
        {
            constexpr int C = D / 8, STEP = 256 / C, B = CODES ? 8 : 16;
            const int c = tid % C, start = tid / C;
            HeadRow at(p, row0 + start), again = at;
            const HeadStep by(p, STEP);
            for (int r0 = start; r0 < block_rows; r0 += B * STEP) {
                uint4 x[B];
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int r = r0 + j * STEP;
                    if (!wide && r == twin + start) at = again;
                    x[j] = make_uint4(0u, 0u, 0u, 0u);
                    if ((!wide && r >= twin ? r - twin : r) < n_rows)
                        x[j] = *reinterpret_cast<const uint4*>(p.q + (seq0 + at.s) * p.ld_q + static_cast<long long>(kh * p.g + at.h) * D + c * 8);
                    at.advance(by, p);
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
        const int v = warp >> 2;
        const int first = (wide ? v * 128 : -v * (twin & 127)) + (warp & 3) * 32;  // this warp's first row of the block
        const int mine = wide ? n_tiles : (n_tiles + 1 - v) / 2;              // tiles of this set
        const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + v * 128, t_o = t_lane + 256 + v * 128;
        const bool live = first >= 0 && first < n_rows;                        // else the warp only keeps the barriers going
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int n = 0; n < mine && ok; ++n) {
            const int tile = wide ? n : 2 * n + v;
            if (!wait_phase(&sh.s_full[v], n & 1)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int left = n_tok - tile * TC_TILE;
            auto largest = [&](float(&x)[64], int c0) {  // of 64 scores; those past the end become -inf
                if (left < c0 + 64) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (c0 + i >= left) x[i] = -INFINITY;
                }
                float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) t[k] = fmaxf(t[k], fmaxf(x[i + 2 * k], x[i + 2 * k + 1]));
                return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            };
            float s[2][64];  // bf16 pages: both halves are read at once; codes, with fewer registers: one after the other
            if (!CODES && live) {
                tc_ld_32x64(t_s, s[0]);
                tc_ld_32x64(t_s + 64, s[1]);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (live) {
                    float(&x)[64] = s[CODES ? 0 : half];
                    if constexpr (CODES) tc_ld_32x64(t_s + half * 64, x);
                    float top = -INFINITY;
                    if constexpr (CODES) top = largest(x, half * 64);
                    else if (half == 0) top = fmaxf(largest(s[0], 0), largest(s[1], 64));
                    // The reference point of a row follows its maximum only when that has grown by 2^8 in weight (not-less: also for
                    // the first maximum): weights up to 2^8 are as exact as weights up to 1, and the output is seldom rescaled.  With
                    // codes it may do so for either half of a tile: the scores are read once, and the first half's product does not wait
                    // for the second's maximum.
                    if ((CODES || half == 0) && __any_sync(0xFFFFFFFFu, !(top <= m + p.margin))) {
                        const float to = fmaxf(m, top), f = m == -INFINITY ? 0.f : ex2((m - to) * p.scale_log2);
                        m = to;
                        l *= f;
                        if (n > 0 || half > 0) {
                            if (!wait_phase(&sh.pv_done[v][half ^ 1], (n - 1 + half) & 1)) {  // the set's output so far is complete
                                ok = false;
                                break;
                            }
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 8; ++c) {
                                uint32_t y[8];
                                tc_ld_32x8(t_o + c * 8, y);
#pragma unroll
                                for (int i = 0; i < 8; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                                tc_st_32x8(t_o + c * 8, y);
                            }
                        }
                    }
                    const float u = m == -INFINITY ? 0.f : m * p.scale_log2;
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
        if (ok && mine > 0 && !wait_phase(&sh.pv_done[v][1], (mine - 1) & 1)) ok = false;
        if (!ok) sh.failed = 1;
        tc_fence_after();
        // Both sets are complete: the rows go through shared memory, where the tiles were, so that a row is written as one
        // run of memory.  Rows of D + 4 floats: consecutive ones start four banks apart.
        named_bar_sync(3, 256);
        constexpr int LD = D + 4;
        float* stage = reinterpret_cast<float*>(smem);
        if (live && mine > 0) {
            float* dst = stage + (wide ? first + lane : v * 128 + first + lane) * LD;
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
        if (live) sh.ml[v][(first & 127) + lane] = make_float2(m, l);
        named_bar_sync(3, 256);
        const int chunks = p.prefix.n_chunks + p.own.n_chunks;
        constexpr int LANES = D / 4, RW = 32 / LANES;  // lanes of a row, rows of a warp at a time
        HeadRow at(p, row0 + warp * RW + lane / LANES);
        const HeadStep by(p, 8 * RW);
#pragma unroll 4
        for (int r = warp * RW + lane / LANES; r < n_rows; r += 8 * RW) {
            const int d = (lane % LANES) * 4;
            const long long slot = (static_cast<long long>(seq0 + at.s) * p.heads + kh * p.g + at.h) * chunks + chunk;
            at.advance(by, p);
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

template <int D, int Q, int CONV>
int launch(izb_ctx* ctx, cudaStream_t s, const Params& p, int64_t items, bool wide) {
    auto kern = shared_prefix_tc_kernel<D, Q, CONV>;
    constexpr int RING = 4 * TC_TILE * D * 2, Q_BYTES = 128 * D * 2;
    auto smem = [](bool w) { return (w ? 2 : 1) * Q_BYTES + RING + Codes<D, Q, CONV>::bytes(Codes<D, Q, CONV>::stages(w)); };
    static std::atomic<bool> ready[IZB_MAX_DEVICES];
    if (!ready[ctx->device].load(std::memory_order_relaxed)) {
        cudaFuncAttributes attr;
        IZB_CUDA_TRY(cudaFuncGetAttributes(&attr, kern));
        // the weight warps would wait for registers nobody has
        if (Q != IZB_KV_NONE && attr.numRegs < Roles<Q, CONV>::LAUNCH) return IZB_ERR_LAUNCH;
        IZB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem(false) > smem(true) ? smem(false) : smem(true)));
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
    IZB_CUDA_TRY(launch_chained(ctx, kern, dim3(static_cast<unsigned>(items)), dim3(Roles<Q, CONV>::THREADS), static_cast<size_t>(smem(wide)), s, p,
                                maps, wide ? 1 : 0));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

// Converting warps: eight, and sixteen for Int8 under up to 128 rows.  Sixteen convert a tile faster and take issue slots
// from the weights.  D = 128, 32 rows per KV head: Int8 4,099 tokens x 32 groups 111 us with sixteen, 125 with
// eight; Q4_0 9,001 tokens x 32 groups 156 and 151; Int8 under 256 rows, 16,384 tokens x 8 groups, 195 and 184.
template <int D>
int launch_dim(izb_ctx* ctx, cudaStream_t s, const Params& p, int64_t items, bool wide) {
    if (p.prefix.quant == IZB_KV_NONE) return launch<D, IZB_KV_NONE, 128>(ctx, s, p, items, wide);
    if (p.prefix.quant == IZB_KV_Q4_0) return launch<D, IZB_KV_Q4_0, 128>(ctx, s, p, items, wide);
    return wide ? launch<D, IZB_KV_INT8, 128>(ctx, s, p, items, wide) : launch<D, IZB_KV_INT8, 256>(ctx, s, p, items, wide);
}

}  // namespace

int launch_prefix_tc(izb_ctx* ctx, cudaStream_t s, const Params& p, int head_dim, int64_t groups) {
    const bool wide = static_cast<int64_t>(p.seqs) * p.g > TC_ROWS;
    const int64_t items = groups * p.prefix.n_chunks * p.kv_heads * p.row_blocks;
    return head_dim == 128 ? launch_dim<128>(ctx, s, p, items, wide) : launch_dim<64>(ctx, s, p, items, wide);
}

}  // namespace shared_prefix
}  // namespace izb
