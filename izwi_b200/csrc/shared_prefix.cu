// Single-token attention for groups of sequences that share a prompt: the S sequences of group g attend to the
// prefix pages of the group, stored and read once for all of them, and then to pages of their own.
//
//   out[i, h] = sum_t p_t v_t,  p = softmax over t of (scale q[i, h] . k_t),  t over prefix(g) then own pages
//
// One decode step against n copies of the prompt reads its K and V n times; here the S * G query rows that meet a
// KV head of the prefix (G = heads / kv_heads) are the rows of one product, so the prefix crosses the memory bus
// once and its 16-bit fragments are used by S * G rows on the tensor cores.
//
// Work: an item is (group, KV head, block of query rows, chunk of prefix tokens) or (sequence, KV head, chunk of its
// own tokens); all items go out in one launch, one CTA each, or, with many rows or a long prefix, those of the prefix in
// a launch of their own on tensor memory (shared_prefix_tc.cu), behind which short own tokens join the last launch; a small
// call is one launch of clusters that join by themselves.  A CTA walks its chunk in tiles with a running maximum and sum
// per row and leaves (max, sum, weighted values) for a last launch that joins the chunks of every (sequence, head).  fp32
// for scores, maxima, sums and accumulators; p is rounded to bf16 for the product with v (half a step: 2^-8 relative at
// most, independent per token, which is what the bf16 output itself carries).
//
// Measured (device time of the whole call): 8 x 5 beams over 1,500 tokens, 20 heads of 64, bf16 15.5 us = 4.0 TB/s, bound by
// the ends of its items; 4 x 8 beams over 4,099 + 131 Int8 tokens, 32 / 8 heads of 128 27.1 us, bound by the instructions of
// two computing warps a scheduler; 4 beams over 100 + 5 tokens 6.2 us, a chain of trips to memory.
#include <climits>
#include <cmath>

#include "shared_prefix.cuh"

namespace {

using namespace izb::shared_prefix;

constexpr int SP_THREADS = 256;      // four computing warps, four that copy
constexpr int SP_TILE = 128;         // chunks are multiples of this, and so of every tile size
constexpr int SP_MAX_CHUNK = 768;    // tokens per item: with their table of places two CTAs still share an SM
constexpr int SP_MAX_G = 16;         // query heads per KV head: the rows of one own-pages item
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(izb::lds32(addr)); }
__device__ __forceinline__ void split_scale(float s, uint32_t& hi2, uint32_t& lo2) { split_scales(s, s, hi2, lo2); }

// How a tile of one item lies in shared memory.  Four computing warps share a tile, WT tokens each.
template <int D, int Q>
struct Layout {
    static constexpr int ROW = Q == IZB_KV_NONE ? 2 * D : Q == IZB_KV_INT8 ? D : D / 2;  // bytes of a token's K (or V)
    static constexpr int CHUNKS = ROW / 16;
    // tokens of a warp in a tile.  D = 128: the code of sixteen is what a warp runs without waiting for its instructions (Int8
    // 4 x 8 beams over 4,099 tokens 29.4 us against 30.0 with 32, Q4_0 2 x 8 over 9,001 19.5 against 20.7); D = 64, half as
    // much work a token: 88.6 us against 81.6 (Int8, 32 x 30 beams over 1,500 tokens).
    static constexpr int WT = D == 128 ? 16 : 32;
    static constexpr int TILE = 4 * WT;
    static constexpr int TILE_BYTES = TILE * ROW;
    static constexpr int SCALE_BYTES = Q == IZB_KV_Q4_0 ? TILE * (D / 32) * 4 : 0;
    static constexpr int STAGE = 2 * (TILE_BYTES + SCALE_BYTES);
    // what two CTAs (D = 64: three) of an SM can hold
    static constexpr int STAGES = D == 128 ? (STAGE > 24 * 1024 ? 3 : 4) : STAGE > 24 * 1024 ? 2 : STAGE > 12 * 1024 ? 3 : 4;
    // floats of a row of the final exchange between the warps: a store phase of bf16 tiles meets four rows of eight
    // consecutive banks, of codes two rows of four 16-byte columns
    static constexpr int EX_LD = Q == IZB_KV_NONE ? D + 8 : D + 4;
    // place of 16-byte chunk c of token row r: the chunk index is mixed with the row so that the eight lanes of a
    // shared-memory phase (ldmatrix: eight rows of one chunk; codes: two rows of four chunks) meet different banks
    static __device__ __forceinline__ int place(int r, int c) {
        if (CHUNKS >= 8) return r * ROW + ((c ^ (r & 7)) << 4);
        if (CHUNKS == 4) return r * ROW + ((c ^ ((r >> 1) & 3)) << 4);
        return r * ROW + ((c ^ ((r >> 2) & 1)) << 4);
    }
};

// shared memory of an item: query rows, table of token places, Int8 scales, then the tile ring, which the exchange reuses
template <int D, int MT, int Q>
constexpr int item_smem(int chunk) {
    const int ring = Layout<D, Q>::STAGE * Layout<D, Q>::STAGES;
    const int exchange = 4 * 16 * MT * Layout<D, Q>::EX_LD * 4;
    return 16 * MT * D * 2 + chunk * 4 + (Q == IZB_KV_INT8 ? chunk * 4 : 0) + (ring > exchange ? ring : exchange);
}

// Registers.  A launch of (256 threads, CTAS per SM) gets LAUNCH registers a thread; 128 copying threads keep COPY_REGS
// of them and 128 computing threads take the rest: COMPUTE + COPY_REGS = 2 LAUNCH.
constexpr int COPY_REGS = 24;
template <int D, int MT>
struct Regs {
    static constexpr int CTAS = D == 64 && MT == 1 ? 3 : 2;
    static constexpr int LAUNCH = CTAS == 3 ? 80 : 128;
    static constexpr int COMPUTE = 2 * LAUNCH - COPY_REGS;
};

struct Result {
    __nv_bfloat16* out;
    long long ld;
};

struct ItemShared {
    unsigned long long full[4], empty[4];
    long long slot[32];   // per row: its place among the partial results
    float2 wml[4][32];    // per warp and row: maximum and sum
    float factor[4][32];  // per warp and row: weight in the joined result
    float2 own[32];        // of an item that does not leave partial results: maximum (log2 scale) and sum of its rows
    int abort_flag;
};

// Chunks of the prefix a row of `group` has partial results of.
__device__ __forceinline__ int prefix_chunks_of(const Params& p, int group) {
    return p.prefix.n_chunks ? (length_of(p.prefix, group) + p.prefix.chunk - 1) / p.prefix.chunk : 0;
}

// Four channels of a row's result.  A row without any token gives zeros; NaN in a sum is not hidden.
template <int D>
__device__ __forceinline__ void leave(const Result& to, float4 a, float l, int seq, int head, int col) {
    const float4 y = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(a.x / l, a.y / l, a.z / l, a.w / l);
    __nv_bfloat16* out = to.out + seq * to.ld + static_cast<long long>(head) * D + col * 4;
    const uint32_t lo = izb::pack_bf16x2(y.x, y.y), hi = izb::pack_bf16x2(y.z, y.w);
    if ((reinterpret_cast<uintptr_t>(out) & 7) == 0) {
        *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
    } else {
        const __nv_bfloat162 b[2] = {*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi)};
        out[0] = b[0].x; out[1] = b[0].y; out[2] = b[1].x; out[3] = b[1].y;
    }
}

// `a`: weighted values of channels col * 4.. under maximum m (log2 scale) and sum l, joined with the row's partial results
// of the prefix from `slot` on; leaves the row's result.
template <int D>
__device__ __forceinline__ void finish(const Params& p, const Result& to, float4 a, float m, float l, long long slot, int np, int seq, int head,
                                       int col) {
#pragma unroll 6
    for (int c = 0; c < np; ++c) {
        const float2 x = p.ml[slot + c];
        const float4 v = *reinterpret_cast<const float4*>(p.acc + (slot + c) * D + col * 4);
        const float n = fmaxf(m, x.x), u = n == -INFINITY ? 0.f : n;
        const float f = ex2(m - u), g = ex2(x.x - u);
        l = l * f + x.y * g;
        m = n;
        a = make_float4(a.x * f + v.x * g, a.y * f + v.y * g, a.z * f + v.z * g, a.w * f + v.w * g);
    }
    leave<D>(to, a, l, seq, head, col);
}

// The items of a (group, KV head) lie in a cluster, prefix chunks first: each joins a share of the rows from all of them.
// 128 threads of every CTA.
template <int D>
__device__ __forceinline__ void join_cluster(const Params& p, const Result& to, ItemShared& sh, uint8_t* smem) {
    const int np = p.prefix.n_chunks, no = p.own.n_chunks, size = np + p.seqs * no;
    const int rank = static_cast<int>(blockIdx.x) % size, base = static_cast<int>(blockIdx.x) / size;
    const int group = base / p.kv_heads, kh = base - group * p.kv_heads;
    const uint32_t own = izb::smem_u32(&sh.own[0]), rows = izb::smem_u32(smem) + p.cluster_rows;
    izb::cluster_sync_all();
    for (int i = rank * 128 + static_cast<int>(threadIdx.x); i < p.seqs * p.g * (D / 4); i += size * 128) {
        const int row = i / (D / 4), col = i % (D / 4), s = row / p.g, h = row - s * p.g;
        float m = -INFINITY, l = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < np + no; ++c) {
            const int from = c < np ? c : np + s * no + c - np, r = c < np ? row : h;
            float2 x;
            float4 v;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(izb::cluster_map_shared(own + r * 8, from)) : "memory");
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(izb::cluster_map_shared(rows + (r * (D + 4) + col * 4) * 4, from))
                         : "memory");
            if (x.x == -INFINITY && x.y == 0.f) continue;  // no token: what lies there is nobody's
            const float n = fmaxf(m, x.x), u = n == -INFINITY ? 0.f : n;
            const float f = ex2(m - u), g = ex2(x.x - u);
            l = l * f + x.y * g;
            m = n;
            a = make_float4(a.x * f + v.x * g, a.y * f + v.y * g, a.z * f + v.z * g, a.w * f + v.w * g);
        }
        leave<D>(to, a, l, group * p.seqs + s, kh * p.g + h, col);
    }
    izb::cluster_sync_all();  // nobody leaves while its results are read
}

// One item: n_rows (at most 16 MT) query rows from row0 that meet KV head kh of `src` row `src_row`, a chunk of tokens from t0.
// Warps 0..3 compute, each on its share of every tile with a maximum, sum and accumulator of its own; warps 4..7
// copy tiles ahead of them through a ring of stages (cp.async onto an mbarrier), so that no warp waits for another one;
// registers the copying warps do not need go to the computing ones (setmaxnreg; their shares add up to the launch's).
//   Scores and outputs are mma.sync products of 16 rows: with at most 32 rows a 128-row tensor-memory tile would be idle
// for three quarters of its rows, while here a tile's fragments are read (or made from codes) exactly once.
//   PARTS: the chunk's result goes among the partial results.  FINISH: the item holds all own tokens of its rows and the prefix
// is done; it leaves the rows' results.  CLUSTER: so do together the items of a (group, KV head), which are a cluster.
enum Mode { PARTS, FINISHES, CLUSTER };
template <int D, int MT, int Q, int MT_LAUNCH, Mode MODE = PARTS>
__device__ __forceinline__ void attend(const Params& p, const Source& src, int src_row, int kh, int seq0, int row0, int n_rows, int t0,
                                       int chunk_slot, int chunks_total, uint8_t* smem, ItemShared& sh, const Result& to = Result{}) {
    using L = Layout<D, Q>;
    constexpr int ROWS = 16 * MT, WT = L::WT, NT = WT / 8, KS = D / 16, DT = D / 8;
    constexpr bool Q_IN_REGS = MT * D <= 128;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, tq = lane & 3;
    uint8_t* sq = smem;
    uint32_t* place = reinterpret_cast<uint32_t*>(sq + ROWS * D * 2);
    uint32_t* tok_scale = place + src.chunk;  // Int8: bf16 (k, v) scales of each token
    uint8_t* ring = reinterpret_cast<uint8_t*>(tok_scale + (Q == IZB_KV_INT8 ? src.chunk : 0));
    const uint32_t ring_u = izb::smem_u32(ring), sq_u = izb::smem_u32(sq);
    volatile int* abort_flag = &sh.abort_flag;

    // ---- where each token of the chunk lies, and the query rows ----
    // The loads of either half of the CTA are under way together: those of the table do not wait for the length (an entry
    // below max_len exists, what it holds is used only below the length), the copies not for scales and query rows.
    if (tid == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            izb::mbar_init(izb::smem_u32(&sh.full[s]), 128);
            izb::mbar_init(izb::smem_u32(&sh.empty[s]), 4);
        }
        sh.abort_flag = 0;
        izb::mbar_fence_init();
    }
    constexpr int U = SP_MAX_CHUNK / 128, QV = ROWS * (D / 8) / 128;
    const int t128 = tid & 127;
    const int first_page = (t0 + t128) / src.page_size, first_rest = t0 + t128 - first_page * src.page_size;
    int pages[U];
    if (warp >= 4 || Q == IZB_KV_INT8) {
        const int* table = src.table + static_cast<long long>(src_row) * src.max_pages;
        int pg = first_page, rest = first_rest;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * 128 + t128;
            pages[u] = 0;
            if (i < src.chunk && t0 + i < src.max_len) pages[u] = table[pg];
            pg += src.step_pages;
            rest += src.step_rest;
            if (rest >= src.page_size) { rest -= src.page_size; ++pg; }
        }
    }
    uint4 qv[QV];
    if (warp < 4) {
#pragma unroll
        for (int u = 0; u < QV; ++u) {
            const int i = u * 128 + tid, r = i / (D / 8), c = i % (D / 8), row = row0 + r;
            qv[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < n_rows) {
                const int s = row / p.g, h = row - s * p.g;
                qv[u] = *reinterpret_cast<const uint4*>(p.q + (seq0 + s) * p.ld_q + static_cast<long long>(kh * p.g + h) * D + c * 8);
            }
        }
    }
    const int n_tok = min(length_of(src, src_row) - t0, src.chunk);
    constexpr bool FINISH = MODE == FINISHES;
    const int np = FINISH ? prefix_chunks_of(p, seq0 / p.seqs) : 0;
    if (n_tok <= 0) {
        if (FINISH)
            for (int i = tid; i < n_rows * (D / 4); i += SP_THREADS) {
                const int r = i / (D / 4), head = kh * p.g + r;
                finish<D>(p, to, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f, (static_cast<long long>(seq0) * p.heads + head) * chunks_total, np, seq0, head,
                          i % (D / 4));
            }
        if (MODE == CLUSTER && tid < 128) {
            if (tid < n_rows) sh.own[tid] = make_float2(-INFINITY, 0.f);
            join_cluster<D>(p, to, sh, smem);
        }
        return;
    }
    const int n_tiles = (n_tok + L::TILE - 1) / L::TILE;
    __syncthreads();

    bool ok = true;
    if (warp >= 4) {
        // ---------------- copies ----------------
        int rest = first_rest;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * 128 + t128;  // tokens past the chunk: a place that can be addressed
            if (i < n_tiles * L::TILE)
                place[i] = i < n_tok ? static_cast<uint32_t>(pages[u]) * static_cast<uint32_t>(src.page_size) + static_cast<uint32_t>(rest) : 0u;
            rest += src.step_rest;
            if (rest >= src.page_size) rest -= src.page_size;
        }
        izb::named_bar_sync(2, 128);
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(COPY_REGS));
        const int t = t128;
        constexpr int RSTEP = 128 / L::CHUNKS;  // rows the 128 threads take at a time, a 16-byte chunk each
        const int my_r = t / L::CHUNKS, my_c = t % L::CHUNKS;
        const uint32_t stride = static_cast<uint32_t>(p.kv_heads) * L::ROW;
        const uint8_t* k_from = src.k + kh * L::ROW + my_c * 16;
        const uint8_t* v_from = src.v + kh * L::ROW + my_c * 16;
        for (int tile = 0; tile < n_tiles; ++tile) {
            const int stage = tile % L::STAGES;
            if (!izb::mbar_wait_bounded(izb::smem_u32(&sh.empty[stage]), ((tile / L::STAGES) & 1) ^ 1, abort_flag)) {
                ok = false;
                break;
            }
            const uint32_t base = ring_u + stage * L::STAGE;
            const int tok0 = tile * L::TILE;
            // rows past the chunk become zeros as far as a product step of 16 tokens reaches
            const int have = n_tok - tok0, need = min(L::TILE, (have + 15) & ~15);
#pragma unroll 4
            for (int j = 0; j < L::TILE / RSTEP; ++j) {
                const int r = j * RSTEP + my_r;
                if (r >= need) break;
                const uint64_t off = static_cast<uint64_t>(place[tok0 + r]) * stride;
                const int bytes = r < have ? 16 : 0;
                const uint32_t dst = base + L::place(r, my_c);
                cp16(dst, k_from + off, bytes);
                cp16(dst + L::TILE_BYTES, v_from + off, bytes);
            }
            if (Q == IZB_KV_Q4_0) {
                constexpr int B = D / 32;
#pragma unroll 4
                for (int j = 0; j < L::TILE * B / 128; ++j) {
                    const int i = j * 128 + t, r = i / B, c = i % B;
                    const int bytes = r < have ? 4 : 0;
                    const uint64_t off = static_cast<uint64_t>(place[tok0 + r]) * static_cast<uint32_t>(p.kv_heads * B) + static_cast<uint32_t>(kh * B + c);
                    cp4(base + 2 * L::TILE_BYTES + i * 4, src.k_scales + off, bytes);
                    cp4(base + 2 * L::TILE_BYTES + L::SCALE_BYTES + i * 4, src.v_scales + off, bytes);
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(izb::smem_u32(&sh.full[stage])) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok && lane == 0) atomicExch(p.status, 1);
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<D, MT_LAUNCH>::COMPUTE));
    if (Q == IZB_KV_INT8) {
        float ks[U], vs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ks[u] = vs[u] = 0.f;
            if (u * 128 + tid < n_tok) {
                ks[u] = src.k_scales[pages[u]];
                vs[u] = src.v_scales[pages[u]];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)  // zero past the chunk
            if (u * 128 + tid < n_tiles * L::TILE) tok_scale[u * 128 + tid] = izb::pack_bf16x2(ks[u], vs[u]);
    }
#pragma unroll
    for (int u = 0; u < QV; ++u) {
        const int i = u * 128 + tid, r = i / (D / 8), c = i % (D / 8);
        uint4 v = make_uint4(qv[u].x ^ p.q_sign, qv[u].y ^ p.q_sign, qv[u].z ^ p.q_sign, qv[u].w ^ p.q_sign);
        // Q4_0 codes leave their words as the channel pairs (0, 4), (1, 5), (2, 6), (3, 7) of eight
        if (Q == IZB_KV_Q4_0)
            v = make_uint4(izb::prmt(v.x, v.z, 0x5410), izb::prmt(v.x, v.z, 0x7632), izb::prmt(v.y, v.w, 0x5410), izb::prmt(v.y, v.w, 0x7632));
        *reinterpret_cast<uint4*>(sq + r * D * 2 + ((c ^ (r & 7)) << 4)) = v;
    }
    if (tid < n_rows) {
        const int row = row0 + tid, s = row / p.g, h = row - s * p.g;
        sh.slot[tid] = (static_cast<long long>(seq0 + s) * p.heads + kh * p.g + h) * chunks_total + chunk_slot;
    }
    izb::named_bar_sync(1, 128);
    float o[MT][DT][4], m[MT][2], l[MT][2];
    {
        const CodeBits<Q> bits;
        uint32_t qa[Q_IN_REGS ? MT : 1][Q_IN_REGS ? KS : 1][4];
        // fragment of query rows 16 mt.. for product step ks.  bf16: channels in order (ldmatrix); codes: the order of d
        // inside a product is free as long as both operands use it, lane tq takes the D / 4 channels from tq * D / 4, four
        // of them per step, so that it finds a token's codes for all steps in consecutive bytes
        auto q_frag = [&](uint32_t (&a)[4], int mt, int ks) {
            if constexpr (Q == IZB_KV_NONE) {
                const int r = mt * 16 + (lane & 15), c = ks * 2 + (lane >> 4);
                ldsm4(a, sq_u + r * D * 2 + ((c ^ (r & 7)) << 4));
            } else {
                const int r = mt * 16 + gq, e = tq * (D / 4) + ks * 4, c = e >> 3;
                const uint32_t at = sq_u + r * D * 2 + ((c ^ (r & 7)) << 4) + (e & 4) * 2;
                const uint2 lo = izb::lds64(at), hi = izb::lds64(at + 8 * D * 2);
                a[0] = lo.x; a[1] = hi.x; a[2] = lo.y; a[3] = hi.y;
            }
        };
        if constexpr (Q_IN_REGS) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) q_frag(qa[mt][ks], mt, ks);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < DT; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
        }
        const int wt = warp * WT;  // this warp's first token in a tile

        for (int tile = 0; tile < n_tiles; ++tile) {
            const int stage = tile % L::STAGES;
            if (!izb::mbar_wait_bounded(izb::smem_u32(&sh.full[stage]), (tile / L::STAGES) & 1, abort_flag)) {
                ok = false;
                break;
            }
            const uint32_t kt = ring_u + stage * L::STAGE, vt = kt + L::TILE_BYTES;
            const int left = n_tok - tile * L::TILE - wt;  // tokens of this warp's share that exist
            if (left > 0) {
                // ---- scores: S[rows, tokens] = Q K^T ----
                float s[MT][NT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int j = 0; j < NT; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    if (j * 8 >= left) break;
                    if constexpr (Q == IZB_KV_NONE) {
                        const int r = wt + j * 8 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            uint32_t b[4];
                            ldsm4(b, kt + L::place(r, ks * 2 + ((lane >> 3) & 1)));
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                uint32_t t[4];
                                if constexpr (!Q_IN_REGS) q_frag(t, mt, ks);
                                const uint32_t(&a)[4] = Q_IN_REGS ? qa[Q_IN_REGS ? mt : 0][Q_IN_REGS ? ks : 0] : t;
                                izb::mma_bf16_16816(s[mt][j], a[0], a[1], a[2], a[3], b[0], b[1]);
                                izb::mma_bf16_16816(s[mt][j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                            }
                        }
                    } else {
                        uint32_t b[2][KS * 2];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const int r = wt + (j + n) * 8 + gq;
                            if constexpr (Q == IZB_KV_INT8) {
                                const uint32_t sc = tok_scale[tile * L::TILE + r], sc2 = izb::prmt(sc, sc, 0x1010);
#pragma unroll
                                for (int h = 0; h < D / 64; ++h) {
                                    const uint4 w = izb::lds128(kt + L::place(r, tq * (D / 64) + h));
                                    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        b[n][h * 8 + i * 2] = hmul2(bits.pair(izb::prmt(x[i], 0u, 0x4140)), sc2);
                                        b[n][h * 8 + i * 2 + 1] = hmul2(bits.pair(izb::prmt(x[i], 0u, 0x4342)), sc2);
                                    }
                                }
                            } else {
                                uint32_t hi2, lo2;
                                split_scale(lds_f32(kt + 2 * L::TILE_BYTES + (r * (D / 32) + tq * (D / 4) / 32) * 4), hi2, lo2);
                                uint32_t x[D / 32];
                                if constexpr (D == 128) {
                                    const uint4 w = izb::lds128(kt + L::place(r, tq));
                                    x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
                                } else {
                                    const uint2 w = izb::lds64(kt + L::place(r, tq >> 1) + (tq & 1) * 8);
                                    x[0] = w.x; x[1] = w.y;
                                }
#pragma unroll
                                for (int i = 0; i < D / 32; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) b[n][i * 4 + e] = q4_value(bits.pair(x[i] >> (4 * e)), hi2, lo2);
                            }
                        }
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                uint32_t t[4];
                                if constexpr (!Q_IN_REGS) q_frag(t, mt, ks);
                                const uint32_t(&a)[4] = Q_IN_REGS ? qa[Q_IN_REGS ? mt : 0][Q_IN_REGS ? ks : 0] : t;
                                izb::mma_bf16_16816(s[mt][j], a[0], a[1], a[2], a[3], b[0][ks * 2], b[0][ks * 2 + 1]);
                                izb::mma_bf16_16816(s[mt][j + 1], a[0], a[1], a[2], a[3], b[1][ks * 2], b[1][ks * 2 + 1]);
                            }
                    }
                }

                // ---- running maximum and sum; s becomes the weights ----
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    if (left < WT) {
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (j * 8 + tq * 2 + (e & 1) >= left) s[mt][j][e] = -INFINITY;
                    }
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[mt][j][e]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 1));
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 2));
                    }
                    // The reference point of a row follows its maximum only when that has grown by 2^8: weights up to 2^8
                    // are as exact as weights up to 1, and the accumulators are seldom rescaled.  (Not-less: also for the
                    // first maximum.)
                    if (__any_sync(0xFFFFFFFFu, !(mx[0] <= m[mt][0] + p.margin) || !(mx[1] <= m[mt][1] + p.margin))) {
                        float f[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float n = fmaxf(m[mt][h], mx[h]);
                            f[h] = m[mt][h] == -INFINITY ? 0.f : ex2((m[mt][h] - n) * p.scale_log2);
                            m[mt][h] = n;
                            l[mt][h] *= f[h];
                        }
#pragma unroll
                        for (int j = 0; j < DT; ++j) {
                            o[mt][j][0] *= f[0]; o[mt][j][1] *= f[0];
                            o[mt][j][2] *= f[1]; o[mt][j][3] *= f[1];
                        }
                    }
                    // no token yet: nothing is subtracted, so that exp2(-inf) gives the zero weight
                    const float u0 = m[mt][0] == -INFINITY ? 0.f : m[mt][0] * p.scale_log2, u1 = m[mt][1] == -INFINITY ? 0.f : m[mt][1] * p.scale_log2;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        s[mt][j][0] = ex2(fmaf(s[mt][j][0], p.scale_log2, -u0));
                        s[mt][j][1] = ex2(fmaf(s[mt][j][1], p.scale_log2, -u0));
                        s[mt][j][2] = ex2(fmaf(s[mt][j][2], p.scale_log2, -u1));
                        s[mt][j][3] = ex2(fmaf(s[mt][j][3], p.scale_log2, -u1));
                        l[mt][0] += s[mt][j][0] + s[mt][j][1];
                        l[mt][1] += s[mt][j][2] + s[mt][j][3];
                    }
                }

                // ---- O += P V, sixteen tokens a step ----
#pragma unroll
                for (int k16 = 0; k16 < NT / 2; ++k16) {
                    if (k16 * 16 >= left) break;
                    uint32_t a[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        a[mt][0] = izb::pack_bf16x2(s[mt][2 * k16][0], s[mt][2 * k16][1]);
                        a[mt][1] = izb::pack_bf16x2(s[mt][2 * k16][2], s[mt][2 * k16][3]);
                        a[mt][2] = izb::pack_bf16x2(s[mt][2 * k16 + 1][0], s[mt][2 * k16 + 1][1]);
                        a[mt][3] = izb::pack_bf16x2(s[mt][2 * k16 + 1][2], s[mt][2 * k16 + 1][3]);
                    }
                    auto accumulate = [&](int j, uint32_t b0, uint32_t b1) {
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) izb::mma_bf16_16816(o[mt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
                    };
                    if constexpr (Q == IZB_KV_NONE) {
#pragma unroll
                        for (int j = 0; j < DT; j += 2) {
                            uint32_t b[4];
                            ldsm4t(b, vt + L::place(wt + k16 * 16 + (lane & 15), j + (lane >> 4)));
                            accumulate(j, b[0], b[1]);
                            accumulate(j + 1, b[2], b[3]);
                        }
                    } else {
                        // column n of output tile j stands for channel n * (D / 8) + j, so that a lane (n = gq) takes D / 8
                        // consecutive channels of its four tokens and pairs tokens 2 tq and 2 tq + 1 (and + 8) code by code
                        const int r0 = wt + k16 * 16 + tq * 2;
                        const int rows[4] = {r0, r0 + 1, r0 + 8, r0 + 9};
                        uint32_t x[4][4];  // the D / 8 codes of each token
                        if constexpr (Q == IZB_KV_INT8) {
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                if constexpr (D == 128) {
                                    const uint4 w = izb::lds128(vt + L::place(rows[t], gq));
                                    x[t][0] = w.x; x[t][1] = w.y; x[t][2] = w.z; x[t][3] = w.w;
                                } else {
                                    const uint2 w = izb::lds64(vt + L::place(rows[t], gq >> 1) + (gq & 1) * 8);
                                    x[t][0] = w.x; x[t][1] = w.y;
                                }
                            }
                            const uint32_t* ts = tok_scale + tile * L::TILE;
                            const uint32_t s01 = izb::prmt(ts[rows[0]], ts[rows[1]], 0x7632), s23 = izb::prmt(ts[rows[2]], ts[rows[3]], 0x7632);
#pragma unroll
                            for (int j = 0; j < DT; ++j) {
                                const int w = j >> 2, by = j & 3;
                                const uint32_t sel = by | ((4 + by) << 8);  // byte `by` of both words; the pair's mask drops the rest
                                accumulate(j, hmul2(bits.pair(izb::prmt(x[0][w], x[1][w], sel)), s01),
                                           hmul2(bits.pair(izb::prmt(x[2][w], x[3][w], sel)), s23));
                            }
                        } else {
                            const int blk = gq * (D / 8) / 32;
                            float sc[4];
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                sc[t] = lds_f32(kt + 2 * L::TILE_BYTES + L::SCALE_BYTES + (rows[t] * (D / 32) + blk) * 4);
                                if constexpr (D == 128) {
                                    const uint2 w = izb::lds64(vt + L::place(rows[t], gq >> 1) + (gq & 1) * 8);
                                    x[t][0] = w.x; x[t][1] = w.y;
                                } else {
                                    x[t][0] = izb::lds32(vt + L::place(rows[t], gq >> 2) + (gq & 3) * 4);
                                }
                            }
                            uint32_t ha, la, hb, lb;
                            split_scale(sc[0], ha, la);
                            split_scale(sc[1], hb, lb);
                            const uint32_t h01 = izb::prmt(ha, hb, 0x5410), l01 = izb::prmt(la, lb, 0x5410);
                            split_scale(sc[2], ha, la);
                            split_scale(sc[3], hb, lb);
                            const uint32_t h23 = izb::prmt(ha, hb, 0x5410), l23 = izb::prmt(la, lb, 0x5410);
#pragma unroll
                            for (int j = 0; j < DT; ++j) {
                                const uint32_t sel = (j & 4) ? 0x7632u : 0x5410u;  // four codes of both tokens side by side
                                const uint32_t w01 = izb::prmt(x[0][j >> 3], x[1][j >> 3], sel), w23 = izb::prmt(x[2][j >> 3], x[3][j >> 3], sel);
                                accumulate(j, q4_value(bits.pair(w01 >> (4 * (j & 3))), h01, l01), q4_value(bits.pair(w23 >> (4 * (j & 3))), h23, l23));
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) izb::mbar_arrive(izb::smem_u32(&sh.empty[stage]));
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 1);
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 2);
                if (tq == 0) sh.wml[warp][mt * 16 + h * 8 + gq] = make_float2(m[mt][h], l[mt][h]);
            }
    }
    if (!ok && lane == 0) atomicExch(p.status, 1);
    izb::named_bar_sync(1, 128);  // every tile of the ring has been read; from here on the four computing warps alone

    // ---- join the warps, leave the chunk's result ----
    // Codes leave a lane with runs of D / 8 channels; run n is turned by n 16-byte columns, so that the eight lanes of a
    // store phase (two rows, four runs) meet different banks.
    constexpr int LD = L::EX_LD;
    auto turned = [](int col) { return D == 128 ? col ^ (col >> 2) : col ^ ((col >> 3) << 1); };
    float* ex = reinterpret_cast<float*>(ring);  // [warp][16 MT][LD]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* row = ex + (warp * ROWS + mt * 16 + h * 8 + gq) * LD;
            if constexpr (Q == IZB_KV_NONE) {
#pragma unroll
                for (int j = 0; j < DT; ++j) *reinterpret_cast<float2*>(row + j * 8 + tq * 2) = make_float2(o[mt][j][h * 2], o[mt][j][h * 2 + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < DT; j += 4)
                        *reinterpret_cast<float4*>(row + turned(((tq * 2 + e) * DT + j) / 4) * 4) =
                            make_float4(o[mt][j][h * 2 + e], o[mt][j + 1][h * 2 + e], o[mt][j + 2][h * 2 + e], o[mt][j + 3][h * 2 + e]);
            }
        }
    if (tid < n_rows) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, sh.wml[w][tid].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 x = sh.wml[w][tid];
            const float f = x.x == -INFINITY ? 0.f : ex2((x.x - top) * p.scale_log2);
            sh.factor[w][tid] = f;
            sum += f * x.y;
        }
        if (MODE != PARTS) sh.own[tid] = make_float2(top * p.scale_log2, sum);
        else p.ml[sh.slot[tid]] = make_float2(top * p.scale_log2, sum);
    }
    izb::named_bar_sync(1, 128);
#pragma unroll 4
    for (int i = tid; i < n_rows * (D / 4); i += 128) {
        const int r = i / (D / 4), col = i % (D / 4), at = Q == IZB_KV_NONE ? col : turned(col);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = sh.factor[w][r];
            const float4 x = *reinterpret_cast<const float4*>(ex + (w * ROWS + r) * LD + at * 4);
            a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
        }
        if constexpr (FINISH) finish<D>(p, to, a, sh.own[r].x, sh.own[r].y, sh.slot[r] - chunk_slot, np, seq0, kh * p.g + r, col);
        else if constexpr (MODE == CLUSTER) *reinterpret_cast<float4*>(smem + p.cluster_rows + (r * (D + 4) + col * 4) * 4) = a;
        else *reinterpret_cast<float4*>(p.acc + sh.slot[r] * D + col * 4) = a;
    }
    if constexpr (MODE == CLUSTER) join_cluster<D>(p, to, sh, smem);
}

template <int D, int MT>
__global__ void __launch_bounds__(SP_THREADS, Regs<D, MT>::CTAS) shared_prefix_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ItemShared sh;
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int chunks = p.prefix.n_chunks + p.own.n_chunks;
    int item = blockIdx.x;
    if (item < p.prefix_items) {
        // row blocks of one (group, KV head, chunk) next to one another: they read the same tiles
        const int rb = item % p.row_blocks;
        item /= p.row_blocks;
        const int kh = item % p.kv_heads;
        item /= p.kv_heads;
        const int chunk = item % p.prefix.n_chunks, group = item / p.prefix.n_chunks;
        const int t0 = chunk * p.prefix.chunk, row0 = rb * 16 * MT, n = min(16 * MT, p.seqs * p.g - row0);
        if (p.prefix.quant == IZB_KV_NONE)
            attend<D, MT, IZB_KV_NONE, MT>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, chunk, chunks, smem, sh);
        else if (p.prefix.quant == IZB_KV_INT8)
            attend<D, MT, IZB_KV_INT8, MT>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, chunk, chunks, smem, sh);
        else
            attend<D, MT, IZB_KV_Q4_0, MT>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, chunk, chunks, smem, sh);
        return;
    }
    item -= p.prefix_items;
    const int kh = item % p.kv_heads;
    item /= p.kv_heads;
    const int chunk = item % p.own.n_chunks, seq = item / p.own.n_chunks;
    const int t0 = chunk * p.own.chunk, slot = p.prefix.n_chunks + chunk;
    if (p.own.quant == IZB_KV_NONE) attend<D, 1, IZB_KV_NONE, MT>(p, p.own, seq, kh, seq, 0, p.g, t0, slot, chunks, smem, sh);
    else if (p.own.quant == IZB_KV_INT8) attend<D, 1, IZB_KV_INT8, MT>(p, p.own, seq, kh, seq, 0, p.g, t0, slot, chunks, smem, sh);
    else attend<D, 1, IZB_KV_Q4_0, MT>(p, p.own, seq, kh, seq, 0, p.g, t0, slot, chunks, smem, sh);
}

// All items of a (group, KV head) in one cluster of up to eight CTAs, which joins their results through shared memory: a call
// of one launch.
template <int D, int MT>
__global__ void __launch_bounds__(SP_THREADS, Regs<D, MT>::CTAS) shared_prefix_cluster_kernel(const __grid_constant__ Params p, const __grid_constant__ Result to) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ItemShared sh;
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int np = p.prefix.n_chunks, no = p.own.n_chunks, size = np + p.seqs * no;
    const int rank = static_cast<int>(blockIdx.x) % size, base = static_cast<int>(blockIdx.x) / size;
    const int group = base / p.kv_heads, kh = base - group * p.kv_heads;
    if (rank < np) {
        const int t0 = rank * p.prefix.chunk, n = p.seqs * p.g;
        if (p.prefix.quant == IZB_KV_NONE) attend<D, MT, IZB_KV_NONE, MT, CLUSTER>(p, p.prefix, group, kh, group * p.seqs, 0, n, t0, 0, 0, smem, sh, to);
        else if (p.prefix.quant == IZB_KV_INT8) attend<D, MT, IZB_KV_INT8, MT, CLUSTER>(p, p.prefix, group, kh, group * p.seqs, 0, n, t0, 0, 0, smem, sh, to);
        else attend<D, MT, IZB_KV_Q4_0, MT, CLUSTER>(p, p.prefix, group, kh, group * p.seqs, 0, n, t0, 0, 0, smem, sh, to);
        return;
    }
    const int seq = group * p.seqs + (rank - np) / no, t0 = (rank - np) % no * p.own.chunk;
    if (p.own.quant == IZB_KV_NONE) attend<D, 1, IZB_KV_NONE, MT, CLUSTER>(p, p.own, seq, kh, seq, 0, p.g, t0, 0, 0, smem, sh, to);
    else if (p.own.quant == IZB_KV_INT8) attend<D, 1, IZB_KV_INT8, MT, CLUSTER>(p, p.own, seq, kh, seq, 0, p.g, t0, 0, 0, smem, sh, to);
    else attend<D, 1, IZB_KV_Q4_0, MT, CLUSTER>(p, p.own, seq, kh, seq, 0, p.g, t0, 0, 0, smem, sh, to);
}

// Behind the tensor-memory kernel: an item per (sequence, KV head) takes the sequence's own tokens, joins the chunks of the
// prefix and leaves the result, where there are few enough own tokens for one item.  (In a launch before it they cost that
// launch, and this one the reading of their partial results: 64 sequences of up to 256 own tokens 68.7 us against 64.2.)
template <int D>
__global__ void __launch_bounds__(SP_THREADS, Regs<D, 1>::CTAS) shared_prefix_finish_kernel(const __grid_constant__ Params p, const __grid_constant__ Result to) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ItemShared sh;
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    const int chunks = p.prefix.n_chunks + p.own.n_chunks;
    const int kh = blockIdx.x % p.kv_heads, seq = blockIdx.x / p.kv_heads;
    if (p.own.quant == IZB_KV_NONE) attend<D, 1, IZB_KV_NONE, 1, FINISHES>(p, p.own, seq, kh, seq, 0, p.g, 0, p.prefix.n_chunks, chunks, smem, sh, to);
    else if (p.own.quant == IZB_KV_INT8) attend<D, 1, IZB_KV_INT8, 1, FINISHES>(p, p.own, seq, kh, seq, 0, p.g, 0, p.prefix.n_chunks, chunks, smem, sh, to);
    else attend<D, 1, IZB_KV_Q4_0, 1, FINISHES>(p, p.own, seq, kh, seq, 0, p.g, 0, p.prefix.n_chunks, chunks, smem, sh, to);
}

// One CTA per (sequence, head): four warps take every fourth chunk, a lane D / 32 channels.
template <int D>
__global__ void __launch_bounds__(128)
    shared_prefix_join_kernel(const __grid_constant__ Params p, __nv_bfloat16* __restrict__ out, long long ld_out) {
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    constexpr int E = D / 32, AHEAD = 4;
    __shared__ float sm_acc[4][D], sm_m[4], sm_l[4];
    const int row = blockIdx.x, seq = row / p.heads, head = row - seq * p.heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = p.prefix.n_chunks + p.own.n_chunks;
    const int len_p = p.prefix.n_chunks ? length_of(p.prefix, seq / p.seqs) : 0, len_o = p.own.n_chunks ? length_of(p.own, seq) : 0;
    const long long base = static_cast<long long>(row) * chunks;
    auto used = [&](int c) { return c < p.prefix.n_chunks ? c * p.prefix.chunk < len_p : c < chunks && (c - p.prefix.n_chunks) * p.own.chunk < len_o; };
    float m = -INFINITY, l = 0.f, a[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = 0.f;
    for (int c0 = warp; c0 < chunks; c0 += 4 * AHEAD) {
        // The first results are read while the lengths are on their way: their places exist, and what is not in use is not used.
        float2 x[AHEAD];
        float v[AHEAD][E];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int c = c0 + 4 * i;
            if (c0 == warp ? c < chunks : used(c)) {
                x[i] = p.ml[base + c];
                const float* from = p.acc + (base + c) * D + lane * E;
                if constexpr (E == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(from);
                    v[i][0] = y.x; v[i][1] = y.y; v[i][2] = y.z; v[i][3] = y.w;
                } else {
                    const float2 y = *reinterpret_cast<const float2*>(from);
                    v[i][0] = y.x; v[i][1] = y.y;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (!used(c0 + 4 * i)) continue;
            const float n = fmaxf(m, x[i].x);
            const float u = n == -INFINITY ? 0.f : n;
            const float f = ex2(m - u), g = ex2(x[i].x - u);
            l = l * f + x[i].y * g;
            m = n;
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = a[e] * f + v[i][e] * g;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_acc[warp][lane * E + e] = a[e];
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += 128) {
        const float top = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
        float sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = sm_m[w] == -INFINITY ? 0.f : ex2(sm_m[w] - top);
            sum += f * sm_l[w];
            v += f * sm_acc[w][d];
        }
        // a row without any token gives zeros; NaN in a sum is not hidden
        out[seq * ld_out + static_cast<long long>(head) * D + d] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
struct Plan {
    bool tc;         // the prefix goes to the tensor-memory kernel
    bool cluster;    // one launch: the items of a (group, KV head) are a cluster
    bool own_finishes;  // the own tokens are taken behind it, by the launch that joins
    int rows;        // query rows of a prefix item
    int row_blocks;
    int prefix_chunk, prefix_chunks, own_chunk, own_chunks;
};

// Tokens per item.  `base` items per chunk of the sequence meet `slots` resident CTAs in waves; an item costs its
// tiles plus `extra` for the query rows, the first loads and the result.  The split counts from the fewest whose chunks
// are allowed are tried.
int choose_chunk(int64_t base, int64_t tokens, int64_t slots, int tile, int extra, int most_tiles) {
    const int64_t tiles = (tokens + tile - 1) / tile;
    const int64_t fewest = (tiles + most_tiles - 1) / most_tiles, most = fewest + 63;
    int64_t best = 0, best_cost = INT64_MAX;
    for (int64_t n = fewest; n <= tiles && n <= most; ++n) {
        const int64_t per = (tiles + n - 1) / n, items = base * ((tiles + per - 1) / per);
        const int64_t cost = ((items + slots - 1) / slots) * (per + extra);
        if (cost < best_cost) {
            best_cost = cost;
            best = per;
        }
        if (per == 1) break;
    }
    return static_cast<int>(best * tile);
}

Plan make_plan(const izb_ctx* ctx, int64_t groups, int64_t seqs, int kv_heads, int g, int head_dim, int quant, int64_t max_prefix, int64_t max_own) {
    Plan pl = {};
    const int64_t rows = seqs * g, sms = ctx && ctx->sm_count > 0 ? ctx->sm_count : 148;
    // Which kernel takes the prefix.  Above 32 rows a second block of 32 would read the tiles again, and the tensor-memory
    // kernel holds 128 or 256.  Up to 32 its rows are mostly idle, but a tile of 128 tokens of 128 channels takes it less time
    // (bf16 1,900 cycles against 3,300 to 4,900 here); against that stand some 5 us for an item's first loads, tensor memory
    // and result, and another 5 to 9 where own tokens follow it, which here fill the same launch.  So its items have to be
    // long, longer with own tokens.  Microseconds there against here, tiles an item in brackets:
    //   17 to 32 rows  bf16 20.6/19.6 (9) 31.0/35.5 (16) 51.6/60.4 (32), own tokens 39.6/39.7 (16) 58.8/62.0 (28);
    //                  Int8 21.4/22.4 (8) 22.2/21.8 (9) 32.2/39.5 (16), own 29.5/26.9 (8) 42.4/42.7 (16);
    //                  Q4_0, whose conversion takes most, 14.4/15.1 (4) 20.5/22.1 (9), own 22.6/22.4 (4) 27.6/28.4 (8)
    //   up to 16       bf16 30.5/31.0 (16) 50.9/52.5 (28) 89.2/105.9 (57), own 62.5/53.6 (28) 100.6/107.9 (57);
    //                  Int8 52.5/48.3 (32), Q4_0 50.1/46.3 (32)
    // D = 64: 54 against 31 (bf16), 64 against 48 (Int8, 30 rows) at 12 tiles an item.
    const int tc_rows = rows <= TC_ROWS ? TC_ROWS : 2 * TC_ROWS;
    const int64_t tc_items = groups * kv_heads * ((rows + tc_rows - 1) / tc_rows);
    const int tc_chunk = max_prefix > 0 ? choose_chunk(tc_items, max_prefix, sms, 128, 4, 1 << 20) : 0;
    const bool own = max_own > 0;
    const int least = rows > 16 ? (quant == IZB_KV_NONE ? (own ? 24 : 12) : quant == IZB_KV_INT8 ? (own ? 16 : 10) : own ? 8 : 4) : own ? 48 : 24;
    pl.tc = rows > 32 || (head_dim == 128 && (rows > 16 || quant == IZB_KV_NONE) && tc_chunk >= least * 128);
    pl.rows = pl.tc ? tc_rows : rows <= 16 ? 16 : 32;
    pl.row_blocks = static_cast<int>((rows + pl.rows - 1) / pl.rows);
    const int64_t slots = (head_dim == 64 && (rows <= 16 || pl.tc) ? 3 : 2) * sms;  // of the other kernel
    if (max_prefix > 0) {
        const int64_t base = groups * kv_heads * pl.row_blocks;
        pl.prefix_chunk = pl.tc ? tc_chunk : choose_chunk(base, max_prefix, slots, SP_TILE, 1, SP_MAX_CHUNK / SP_TILE);
        pl.prefix_chunks = static_cast<int>((max_prefix + pl.prefix_chunk - 1) / pl.prefix_chunk);
    }
    if (max_own > 0) {
        pl.own_chunk = choose_chunk(groups * seqs * kv_heads, max_own, slots, SP_TILE, 1, SP_MAX_CHUNK / SP_TILE);
        pl.own_chunks = static_cast<int>((max_own + pl.own_chunk - 1) / pl.own_chunk);
    }
    pl.own_finishes = pl.tc && pl.own_chunks == 1;
    // One launch instead of two saves its issue on the host and up to 1 us on the device, as long as all items are resident at
    // once; clusters of more than two need more room than there is, since they do not fill every place (two launches against
    // one, us: 160 clusters of two 16.5 / 15.5, 8 of five 6.2 / 6.2 and 13.3 / 11.1 issued by the host, 64 of four 12.2 / 17.0,
    // 240 of four 16.0 / 23.6).
    const int64_t size = pl.prefix_chunks + seqs * pl.own_chunks;
    pl.cluster = !pl.tc && pl.row_blocks == 1 && size > 0 && size <= 8 && groups * kv_heads * size <= (size <= 2 ? slots : sms);
    return pl;
}

size_t plan_bytes(const Plan& pl, int64_t batch, int heads, int head_dim) {
    return static_cast<size_t>(batch) * heads * (pl.prefix_chunks + pl.own_chunks) * (head_dim + 2) * sizeof(float);
}

int source_from(const izb_kv_pages* a, const int32_t* lens, int64_t max_len, Source* s) {
    if (!a->k_values || !a->v_values || !a->page_table || !lens) return IZB_ERR_BAD_ARG;
    if (a->quantization < IZB_KV_NONE || a->quantization > IZB_KV_Q4_0) return IZB_ERR_BAD_ARG;
    if (a->page_size <= 0 || a->kv_heads <= 0 || a->max_pages_per_seq <= 0) return IZB_ERR_BAD_ARG;
    if (a->head_dim != 64 && a->head_dim != 128) return IZB_ERR_UNSUPPORTED;
    if (a->quantization != IZB_KV_NONE && (!a->k_scales || !a->v_scales)) return IZB_ERR_BAD_ARG;
    if (!izb_aligned(a->k_values, 16) || !izb_aligned(a->v_values, 16) || !izb_aligned(a->page_table, 4) || !izb_aligned(lens, 4) ||
        !izb_aligned(a->k_scales, 4) || !izb_aligned(a->v_scales, 4))
        return IZB_ERR_BAD_ARG;
    // a length never leads past the row's table entries
    if (max_len < 0 || max_len > INT32_MAX - SP_MAX_CHUNK || (max_len + a->page_size - 1) / a->page_size > a->max_pages_per_seq)
        return IZB_ERR_BAD_ARG;
    s->k = static_cast<const uint8_t*>(a->k_values);
    s->v = static_cast<const uint8_t*>(a->v_values);
    s->k_scales = a->k_scales;
    s->v_scales = a->v_scales;
    s->table = a->page_table;
    s->lens = lens;
    s->max_pages = a->max_pages_per_seq;
    s->quant = a->quantization;
    s->page_size = a->page_size;
    s->step_pages = 128 / a->page_size;
    s->step_rest = 128 % a->page_size;
    s->max_len = static_cast<int>(max_len);
    return IZB_OK;
}

template <int D, int MT>
size_t smem_for(const Source& s) {
    if (s.n_chunks == 0) return 0;
    return s.quant == IZB_KV_NONE ? item_smem<D, MT, IZB_KV_NONE>(s.chunk)
           : s.quant == IZB_KV_INT8 ? item_smem<D, MT, IZB_KV_INT8>(s.chunk) : item_smem<D, MT, IZB_KV_Q4_0>(s.chunk);
}

template <int D, int MT, typename... Args>
int launch_items(izb_ctx* ctx, cudaStream_t s, void (*kern)(Params, Args...), std::atomic<bool>* ready, size_t smem, int cluster, int64_t items,
                 const Params& p, const Args&... args) {
    if (!ready[ctx->device].load(std::memory_order_relaxed)) {
        cudaFuncAttributes attr;
        IZB_CUDA_TRY(cudaFuncGetAttributes(&attr, kern));
        if (attr.numRegs < Regs<D, MT>::LAUNCH) return IZB_ERR_LAUNCH;  // the computing warps would wait for registers nobody has
        IZB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->max_smem_optin - static_cast<int>(attr.sharedSizeBytes)));
        ready[ctx->device].store(true, std::memory_order_relaxed);
    }
    IZB_CUDA_TRY(izb::launch_chained_cluster(ctx, cluster, kern, dim3(static_cast<unsigned>(items)), dim3(SP_THREADS), smem, s, p, args...));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

template <int D, int MT>
int launch_all_items(izb_ctx* ctx, cudaStream_t s, const Params& p, int64_t items) {
    static std::atomic<bool> ready[IZB_MAX_DEVICES];
    const size_t prefix = p.prefix_items > 0 ? smem_for<D, MT>(p.prefix) : 0, own = smem_for<D, 1>(p.own);
    return launch_items<D, MT>(ctx, s, shared_prefix_kernel<D, MT>, ready, prefix > own ? prefix : own, 1, items, p);
}

// Where an item's exchange between its warps ends.
template <int D, int MT>
size_t exchange_end(const Source& s) {
    if (s.n_chunks == 0) return 0;
    const int q = s.quant, ld = q == IZB_KV_NONE ? Layout<D, IZB_KV_NONE>::EX_LD : Layout<D, IZB_KV_INT8>::EX_LD;
    return 16 * MT * D * 2 + s.chunk * 4 + (q == IZB_KV_INT8 ? s.chunk * 4 : 0) + 4 * 16 * MT * ld * 4;
}

template <int D, int MT>
int launch_cluster(izb_ctx* ctx, cudaStream_t s, Params p, int64_t groups, __nv_bfloat16* out, long long ld_out) {
    static std::atomic<bool> ready[IZB_MAX_DEVICES];
    // the rows' results lie at the end, where the tiles have been and no exchange reaches
    const size_t rows = 16 * MT * (D + 4) * 4;
    const size_t sizes[4] = {smem_for<D, MT>(p.prefix), smem_for<D, 1>(p.own), exchange_end<D, MT>(p.prefix) + rows, exchange_end<D, 1>(p.own) + rows};
    size_t smem = 0;
    for (size_t x : sizes) smem = x > smem ? x : smem;
    smem = (smem + 15) / 16 * 16;
    p.cluster_rows = static_cast<int>(smem - rows);
    const int size = p.prefix.n_chunks + p.seqs * p.own.n_chunks;
    return launch_items<D, MT>(ctx, s, shared_prefix_cluster_kernel<D, MT>, ready, smem, size, groups * p.kv_heads * size, p, Result{out, ld_out});
}

template <int D>
int launch_dim(izb_ctx* ctx, cudaStream_t s, const Params& p, const Plan& pl, int64_t items, int64_t batch, __nv_bfloat16* out,
               long long ld_out) {
    if (pl.cluster) return pl.rows == 16 ? launch_cluster<D, 1>(ctx, s, p, batch / p.seqs, out, ld_out) : launch_cluster<D, 2>(ctx, s, p, batch / p.seqs, out, ld_out);
    if (items > 0) {
        const int rc = pl.tc || pl.rows == 16 ? launch_all_items<D, 1>(ctx, s, p, items) : launch_all_items<D, 2>(ctx, s, p, items);
        if (rc != IZB_OK) return rc;
    }
    if (pl.tc && p.prefix.n_chunks > 0) {
        const int rc = launch_prefix_tc(ctx, s, p, D, batch / p.seqs);
        if (rc != IZB_OK) return rc;
    }
    if (pl.own_finishes) {
        static std::atomic<bool> ready[IZB_MAX_DEVICES];
        return launch_items<D, 1>(ctx, s, shared_prefix_finish_kernel<D>, ready, smem_for<D, 1>(p.own), 1, batch * p.kv_heads, p, Result{out, ld_out});
    }
    IZB_CUDA_TRY(izb::launch_chained(ctx, shared_prefix_join_kernel<D>, dim3(static_cast<unsigned>(batch * p.heads)), dim3(128), 0, s, p, out,
                                     ld_out));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

}  // namespace

extern "C" {

size_t izb_shared_prefix_decode_gqa_attention_workspace_bytes(const izb_ctx* ctx, int64_t groups, int64_t seqs_per_group, int32_t heads,
                                                              int32_t kv_heads, int32_t head_dim, int64_t max_prefix_len,
                                                              int64_t max_seq_len) {
    if (groups <= 0 || seqs_per_group <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 ||
        max_prefix_len < 0 || max_seq_len < 0 || groups > INT32_MAX / seqs_per_group || max_prefix_len > INT32_MAX || max_seq_len > INT32_MAX)
        return 0;
    // the query does not know how the pages are stored: enough for every plan
    size_t most = 0;
    for (int quant = IZB_KV_NONE; quant <= IZB_KV_Q4_0; ++quant) {
        const Plan pl = make_plan(ctx, groups, seqs_per_group, kv_heads, heads / kv_heads, head_dim, quant, max_prefix_len, max_seq_len);
        const size_t need = plan_bytes(pl, groups * seqs_per_group, heads, head_dim);
        most = need > most ? need : most;
    }
    return most;
}

int32_t izb_shared_prefix_decode_gqa_attention(izb_ctx* ctx, izb_stream stream, const void* q, const izb_kv_pages* prefix,
                                               const int32_t* prefix_lens, const izb_kv_pages* pages, const int32_t* seq_lens, void* out,
                                               int64_t groups, int64_t seqs_per_group, int32_t heads, int64_t max_prefix_len,
                                               int64_t max_seq_len, int64_t ld_q, int64_t ld_out, float scale, void* workspace,
                                               size_t workspace_bytes) {
    if (!ctx || !prefix || groups < 0 || seqs_per_group < 0 || heads <= 0) return IZB_ERR_BAD_ARG;
    if (groups == 0 || seqs_per_group == 0) return IZB_OK;
    Params p = {};
    int rc = source_from(prefix, prefix_lens, max_prefix_len, &p.prefix);
    if (rc != IZB_OK) return rc;
    const int kv_heads = prefix->kv_heads, d = prefix->head_dim;
    if (pages) {
        rc = source_from(pages, seq_lens, max_seq_len, &p.own);
        if (rc != IZB_OK) return rc;
        if (pages->kv_heads != kv_heads || pages->head_dim != d) return IZB_ERR_BAD_ARG;
    } else if (max_seq_len != 0) {
        return IZB_ERR_BAD_ARG;
    }
    if (!q || !out || !izb_aligned(q, 16) || ld_q % 8 != 0 || !izb_aligned(out, 2)) return IZB_ERR_BAD_ARG;
    if (heads % kv_heads != 0 || heads / kv_heads > SP_MAX_G) return IZB_ERR_UNSUPPORTED;
    if (ld_q < static_cast<int64_t>(heads) * d || ld_out < static_cast<int64_t>(heads) * d) return IZB_ERR_BAD_ARG;
    if (groups > INT32_MAX / seqs_per_group || groups * seqs_per_group > INT32_MAX / heads) return IZB_ERR_UNSUPPORTED;
    const int64_t batch = groups * seqs_per_group;
    const Plan pl = make_plan(ctx, groups, seqs_per_group, kv_heads, heads / kv_heads, d, p.prefix.quant, max_prefix_len, max_seq_len);
    const size_t need = plan_bytes(pl, batch, heads, d);
    if (need && (!workspace || workspace_bytes < need || !izb_aligned(workspace, 16))) return IZB_ERR_BAD_ARG;
    p.prefix.chunk = pl.prefix_chunk;
    p.prefix.n_chunks = pl.prefix_chunks;
    p.own.chunk = pl.own_chunk;
    p.own.n_chunks = pl.own_chunks;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.acc = static_cast<float*>(workspace);
    p.ml = reinterpret_cast<float2*>(p.acc + static_cast<size_t>(batch) * heads * (pl.prefix_chunks + pl.own_chunks) * d);
    p.ld_q = ld_q;
    p.seqs = static_cast<int>(seqs_per_group);
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.g = heads / kv_heads;
    p.row_blocks = pl.row_blocks;
    p.status = ctx->d_status;
    p.q_sign = scale < 0.f ? 0x80008000u : 0u;
    p.scale_log2 = fmaxf(fabsf(scale) * LOG2E, 1e-30f);  // not 0: a masked product is -inf and must stay it
    p.margin = 8.f / p.scale_log2;
    const int64_t prefix_items = pl.tc ? 0 : groups * pl.prefix_chunks * kv_heads * pl.row_blocks, items = prefix_items + (pl.own_finishes ? 0 : batch * kv_heads * pl.own_chunks);
    if (items > INT32_MAX || batch * kv_heads > INT32_MAX || groups * pl.prefix_chunks > INT32_MAX / kv_heads / pl.row_blocks) return IZB_ERR_UNSUPPORTED;
    p.prefix_items = static_cast<int>(prefix_items);
    izb::DeviceGuard guard(ctx->device);
    if (!guard.ok) return IZB_ERR_LAUNCH;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto* op = static_cast<__nv_bfloat16*>(out);
    return d == 128 ? launch_dim<128>(ctx, s, p, pl, items, batch, op, ld_out) : launch_dim<64>(ctx, s, p, pl, items, batch, op, ld_out);
}

}  // extern "C"
