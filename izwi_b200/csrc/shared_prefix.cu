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
// own tokens); all items go out in one launch, one CTA each.  A CTA walks its chunk in tiles of 64 tokens with a
// running maximum and sum per row and leaves (max, sum, weighted values) for a second launch that joins the chunks
// of every (sequence, head).  fp32 for scores, maxima, sums and accumulators; p is rounded to bf16 for the product
// with v (half a step: 2^-9 relative, independent per token, which is what the bf16 output itself carries).
#include <climits>

#include "izb_common.cuh"

namespace {

constexpr int SP_THREADS = 128;
constexpr int SP_TILE = 64;          // tokens per tile
constexpr int SP_MAX_CHUNK = 2048;   // tokens per item: bounds the shared table of token places
constexpr int SP_MAX_G = 16;         // query heads per KV head: the rows of one own-pages item
constexpr float LOG2E = 1.4426950408889634f;

struct Source {
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scales;
    const float* v_scales;
    const int* table;
    const int* lens;
    long long max_pages;
    int quant, page_size;
    int max_len;     // lengths on the device are cut to this
    int chunk;       // tokens per item
    int n_chunks;
};

struct Params {
    Source prefix, own;
    const __nv_bfloat16* q;
    float* acc;       // [rows][chunks][D], rows = batch * heads
    float2* ml;       // [rows][chunks]: maximum (log2 scale) and sum
    long long ld_q;
    int seqs, heads, kv_heads, g;  // sequences per group, query heads per KV head
    int row_blocks, prefix_items;
    float scale_log2;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool fill) {
    const int n = fill ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool fill) {
    const int n = fill ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(izb::lds32(addr)); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two Int8 codes in the low bytes of the halves of x (code = byte - 128) -> bf16x2.  128 + (byte & 127) is the bf16
// 0x4300 | low bits; what is left is -256 for bytes below 128 and -128 above: every step is exact.
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) {
    return hsub2((x & 0x007F007Fu) | 0x43004300u, (~x & 0x00800080u) | 0x43004300u);
}
// Two 4-bit codes in the low nibbles of the halves (code = nibble - 8) -> bf16x2, exact.
__device__ __forceinline__ uint32_t q4_pair(uint32_t x) { return hsub2((x & 0x000F000Fu) | 0x43004300u, 0x43084308u); }
// code * scale rounded to bf16 as the stored value is defined.  The fp32 scale enters as two bf16 parts; the product
// with the small part is rounded to 8 bits at 2^-8 of the value, so the sum's one rounding sees the product to 2^-17.
__device__ __forceinline__ uint32_t q4_value(uint32_t code2, uint32_t hi2, uint32_t lo2) { return hfma2(code2, hi2, hmul2(code2, lo2)); }
__device__ __forceinline__ void split_scale(float s, uint32_t& hi2, uint32_t& lo2) {
    const __nv_bfloat16 h = __float2bfloat16_rn(s);
    const __nv_bfloat16 l = __float2bfloat16_rn(s - __bfloat162float(h));
    const uint32_t hu = __bfloat16_as_ushort(h), lu = __bfloat16_as_ushort(l);
    hi2 = hu | (hu << 16);
    lo2 = lu | (lu << 16);
}

template <int D, int Q, int ROWS>
struct Layout {
    static constexpr int ROW = Q == IZB_KV_NONE ? 2 * D : Q == IZB_KV_INT8 ? D : D / 2;  // bytes of a token's K (or V)
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int TILE_BYTES = SP_TILE * ROW;
    static constexpr int SCALE_BYTES = Q == IZB_KV_Q4_0 ? SP_TILE * (D / 32) * 4 : 0;
    static constexpr int STAGE = 2 * (TILE_BYTES + SCALE_BYTES);
    // two CTAs share an SM (113 KB each): the ring takes what the query rows leave
    static constexpr int STAGES = Q == IZB_KV_NONE ? (ROWS <= 32 ? 3 : 2) : Q == IZB_KV_INT8 ? (ROWS <= 64 ? 5 : 4) : 6;
    // place of 16-byte chunk c of token row r: the chunk index is mixed with the row so that the eight lanes of a
    // shared-memory phase (ldmatrix: eight rows of one chunk; codes: two rows of four chunks) meet different banks
    static __device__ __forceinline__ int place(int r, int c) {
        if (CHUNKS >= 8) return r * ROW + ((c ^ (r & 7)) << 4);
        if (CHUNKS == 4) return r * ROW + ((c ^ ((r >> 1) & 3)) << 4);
        return r * ROW + ((c ^ ((r >> 2) & 1)) << 4);
    }
};

// shared memory of an item: query rows, table of token places, Int8 scales, cross-warp scratch, then the tile ring
// (which the final exchange between warps reuses)
template <int D, int ROWS, int Q>
constexpr int item_smem(int chunk) {
    const int ring = Layout<D, Q, ROWS>::STAGE * Layout<D, Q, ROWS>::STAGES;
    const int exchange = 4 * 32 * D * 4;  // at most 32 rows from each of four warps
    return ROWS * D * 2 + chunk * 4 + (Q == IZB_KV_INT8 ? chunk * 4 : 0) + 4 * 32 * 8 + (ring > exchange ? ring : exchange);
}

// One item: rows [row0, row0 + n_rows) of the query rows that meet KV head kh of `src` row `src_row`, tokens
// [t0, t1).  WM warps side by side over the rows (16 * MT rows each), 4 / WM over the tokens of a tile.
template <int D, int WM, int MT, int Q>
__device__ __forceinline__ void attend(const Params& p, const Source& src, int src_row, int kh, int seq0, int row0, int n_rows, int t0,
                                       int t1, int chunk_slot, int chunks_total, uint8_t* smem) {
    constexpr int WN = 4 / WM, ROWS = 16 * MT * WM, TOK = SP_TILE / WN, NT = TOK / 8, KS = D / 16, DT = D / 8;
    using L = Layout<D, Q, ROWS>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wn = warp / WM;
    const int gq = lane >> 2, tq = lane & 3;
    const int n_tok = t1 - t0, n_tiles = (n_tok + SP_TILE - 1) / SP_TILE;

    uint8_t* sq = smem;
    uint32_t* place = reinterpret_cast<uint32_t*>(sq + ROWS * D * 2);
    uint32_t* tok_scale = place + src.chunk;                                     // Int8: bf16 (k, v) scales of each token
    float2* wml = reinterpret_cast<float2*>(tok_scale + (Q == IZB_KV_INT8 ? src.chunk : 0));
    uint8_t* ring = reinterpret_cast<uint8_t*>(wml + 4 * 32);
    const uint32_t ring_u = izb::smem_u32(ring), sq_u = izb::smem_u32(sq);

    // ---- where each token of the chunk lies, and the query rows ----
    for (int i = tid; i < n_tiles * SP_TILE; i += SP_THREADS) {
        uint32_t at = 0, sc = 0;
        if (i < n_tok) {
            const int t = t0 + i, pg = t / src.page_size;
            const int page = src.table[static_cast<long long>(src_row) * src.max_pages + pg];
            at = static_cast<uint32_t>(page) * static_cast<uint32_t>(src.page_size) + static_cast<uint32_t>(t - pg * src.page_size);
            if (Q == IZB_KV_INT8) sc = izb::pack_bf16x2(src.k_scales[page], src.v_scales[page]);
        }
        place[i] = at;
        if (Q == IZB_KV_INT8) tok_scale[i] = sc;
    }
    for (int i = tid; i < ROWS * (D / 8); i += SP_THREADS) {
        const int r = i / (D / 8), c = i % (D / 8), row = row0 + r;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < n_rows) {
            const int s = row / p.g, h = row - s * p.g;
            v = *reinterpret_cast<const uint4*>(p.q + (seq0 + s) * p.ld_q + static_cast<long long>(kh * p.g + h) * D + c * 8);
        }
        *reinterpret_cast<uint4*>(sq + r * D * 2 + ((c ^ (r & 7)) << 4)) = v;
    }
    __syncthreads();

    auto issue = [&](int tile) {
        if (tile < n_tiles) {
            const uint32_t base = ring_u + (tile % L::STAGES) * L::STAGE;
            const int tok0 = tile * SP_TILE;
#pragma unroll
            for (int j = 0; j < SP_TILE * L::CHUNKS / SP_THREADS; ++j) {
                const int i = j * SP_THREADS + tid, r = i / L::CHUNKS, c = i % L::CHUNKS;
                const bool ok = tok0 + r < n_tok;
                const long long off =
                    (static_cast<long long>(ok ? place[tok0 + r] : 0u) * p.kv_heads + kh) * L::ROW + c * 16;
                cp16(base + L::place(r, c), src.k + (ok ? off : 0), ok);
                cp16(base + L::TILE_BYTES + L::place(r, c), src.v + (ok ? off : 0), ok);
            }
            if (Q == IZB_KV_Q4_0) {
                constexpr int B = D / 32;
#pragma unroll
                for (int j = 0; j < SP_TILE * B / SP_THREADS; ++j) {
                    const int i = j * SP_THREADS + tid, r = i / B, c = i % B;
                    const bool ok = tok0 + r < n_tok;
                    const long long off = (static_cast<long long>(ok ? place[tok0 + r] : 0u) * p.kv_heads + kh) * B + c;
                    cp4(base + 2 * L::TILE_BYTES + i * 4, src.k_scales + (ok ? off : 0), ok);
                    cp4(base + 2 * L::TILE_BYTES + L::SCALE_BYTES + i * 4, src.v_scales + (ok ? off : 0), ok);
                }
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < L::STAGES - 1; ++s) issue(s);

    float o[MT][DT][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt][0] = m[mt][1] = -INFINITY;
        l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < DT; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
    }

    for (int tile = 0; tile < n_tiles; ++tile) {
        cp_wait<L::STAGES - 2>();
        __syncthreads();
        issue(tile + L::STAGES - 1);
        const uint32_t kt = ring_u + (tile % L::STAGES) * L::STAGE, vt = kt + L::TILE_BYTES;
        const int wt = wn * TOK;  // this warp's first token in the tile

        // ---- scores: S[rows, tokens] = Q K^T ----
        float s[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < NT; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
        if constexpr (Q == IZB_KV_NONE) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int r = (wm * MT + mt) * 16 + (lane & 15), c = ks * 2 + (lane >> 4);
                    ldsm4(a[mt], sq_u + r * D * 2 + ((c ^ (r & 7)) << 4));
                }
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t b[4];
                    const int r = wt + j * 8 + (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
                    ldsm4(b, kt + L::place(r, c));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        izb::mma_bf16_16816(s[mt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[0], b[1]);
                        izb::mma_bf16_16816(s[mt][j + 1], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[2], b[3]);
                    }
                }
            }
        } else {
            // Codes become fragments in registers.  The order of d inside a product is free as long as both operands
            // use it: lane tq takes the D / 4 consecutive channels from tq * D / 4, four of them per mma step.
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int r = wt + j * 8 + gq;
                uint32_t b[KS * 2];
                if constexpr (Q == IZB_KV_INT8) {
                    const uint32_t sc = tok_scale[tile * SP_TILE + r];
                    const uint32_t sc2 = izb::prmt(sc, sc, 0x1010);
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) {
                        const uint4 w = izb::lds128(kt + L::place(r, tq * (D / 64) + h));
                        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            b[h * 8 + i * 2] = hmul2(int8_pair(izb::prmt(x[i], 0u, 0x4140)), sc2);
                            b[h * 8 + i * 2 + 1] = hmul2(int8_pair(izb::prmt(x[i], 0u, 0x4342)), sc2);
                        }
                    }
                } else {
                    const int blk = tq * (D / 4) / 32;
                    uint32_t hi2, lo2;
                    split_scale(lds_f32(kt + 2 * L::TILE_BYTES + (r * (D / 32) + blk) * 4), hi2, lo2);
                    uint32_t x[D / 32];
                    if constexpr (D == 128) {
                        const uint4 w = izb::lds128(kt + L::place(r, tq));
                        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
                    } else {
                        const uint2 w = izb::lds64(kt + L::place(r, tq >> 1) + (tq & 1) * 8);
                        x[0] = w.x; x[1] = w.y;
                    }
                    // eight codes of a word, low nibble first: byte i holds channels 2 i and 2 i + 1
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t by = (x[i] >> (8 * e)) & 0xFFu;
                            b[i * 4 + e] = q4_value(q4_pair(by | (by << 12)), hi2, lo2);
                        }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int r0 = (wm * MT + mt) * 16 + gq;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const int e = tq * (D / 4) + ks * 4, c = e >> 3, half = (e & 4) * 2;
                        const uint2 a0 = izb::lds64(sq_u + r0 * D * 2 + ((c ^ (r0 & 7)) << 4) + half);
                        const uint2 a1 = izb::lds64(sq_u + (r0 + 8) * D * 2 + ((c ^ (r0 & 7)) << 4) + half);
                        izb::mma_bf16_16816(s[mt][j], a0.x, a1.x, a0.y, a1.y, b[ks * 2], b[ks * 2 + 1]);
                    }
                }
            }
        }

        // ---- running maximum and sum; s becomes the weights ----
        const int left = n_tok - tile * SP_TILE - wt;  // tokens of this warp's share that exist
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = j * 8 + tq * 2 + (e & 1) < left;
                    s[mt][j][e] = in ? s[mt][j][e] * p.scale_log2 : -INFINITY;
                    if (e < 2) mx0 = fmaxf(mx0, s[mt][j][e]);
                    else mx1 = fmaxf(mx1, s[mt][j][e]);
                }
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xFFFFFFFFu, mx0, 1));
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xFFFFFFFFu, mx0, 2));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xFFFFFFFFu, mx1, 1));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xFFFFFFFFu, mx1, 2));
            const float n0 = fmaxf(m[mt][0], mx0), n1 = fmaxf(m[mt][1], mx1);
            // no token yet: subtract 0 so that exp2(-inf) gives the zero weight
            const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
            if (__any_sync(0xFFFFFFFFu, n0 != m[mt][0] || n1 != m[mt][1])) {
                const float f0 = ex2(m[mt][0] - u0), f1 = ex2(m[mt][1] - u1);
                l[mt][0] *= f0;
                l[mt][1] *= f1;
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    o[mt][j][0] *= f0; o[mt][j][1] *= f0;
                    o[mt][j][2] *= f1; o[mt][j][3] *= f1;
                }
                m[mt][0] = n0;
                m[mt][1] = n1;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                s[mt][j][0] = ex2(s[mt][j][0] - u0);
                s[mt][j][1] = ex2(s[mt][j][1] - u0);
                s[mt][j][2] = ex2(s[mt][j][2] - u1);
                s[mt][j][3] = ex2(s[mt][j][3] - u1);
                l[mt][0] += s[mt][j][0] + s[mt][j][1];
                l[mt][1] += s[mt][j][2] + s[mt][j][3];
            }
        }

        // ---- O += P V, sixteen tokens a step ----
#pragma unroll
        for (int kt16 = 0; kt16 < NT / 2; ++kt16) {
            uint32_t a[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                a[mt][0] = izb::pack_bf16x2(s[mt][2 * kt16][0], s[mt][2 * kt16][1]);
                a[mt][1] = izb::pack_bf16x2(s[mt][2 * kt16][2], s[mt][2 * kt16][3]);
                a[mt][2] = izb::pack_bf16x2(s[mt][2 * kt16 + 1][0], s[mt][2 * kt16 + 1][1]);
                a[mt][3] = izb::pack_bf16x2(s[mt][2 * kt16 + 1][2], s[mt][2 * kt16 + 1][3]);
            }
            if constexpr (Q == IZB_KV_NONE) {
#pragma unroll
                for (int j = 0; j < DT; j += 2) {
                    uint32_t b[4];
                    const int r = wt + kt16 * 16 + (lane & 15), c = j + (lane >> 4);
                    ldsm4t(b, vt + L::place(r, c));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        izb::mma_bf16_16816(o[mt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[0], b[1]);
                        izb::mma_bf16_16816(o[mt][j + 1], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[2], b[3]);
                    }
                }
            } else {
                // column n of output tile j stands for channel n * (D / 8) + j, so that a lane (n = gq) takes D / 8
                // consecutive channels of its four tokens and pairs tokens 2 tq and 2 tq + 1 (and + 8) byte by byte
                const int r0 = wt + kt16 * 16 + tq * 2;
                const int rows[4] = {r0, r0 + 1, r0 + 8, r0 + 9};
                uint32_t x[4][4];  // the D / 8 codes of each token
                uint32_t h01, l01, h23, l23;
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
                    const uint32_t* ts = tok_scale + tile * SP_TILE;
                    h01 = izb::prmt(ts[rows[0]], ts[rows[1]], 0x7632);
                    h23 = izb::prmt(ts[rows[2]], ts[rows[3]], 0x7632);
                    l01 = l23 = 0u;
#pragma unroll
                    for (int j = 0; j < DT; ++j) {
                        const int w = j >> 2, by = j & 3;
                        const uint32_t sel = by | ((4 + by) << 8);  // byte `by` of both words; int8_pair masks the rest
                        const uint32_t b0 = hmul2(int8_pair(izb::prmt(x[0][w], x[1][w], sel)), h01);
                        const uint32_t b1 = hmul2(int8_pair(izb::prmt(x[2][w], x[3][w], sel)), h23);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            izb::mma_bf16_16816(o[mt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
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
                    split_scale(sc[0], ha, la); split_scale(sc[1], hb, lb);
                    h01 = izb::prmt(ha, hb, 0x5410); l01 = izb::prmt(la, lb, 0x5410);
                    split_scale(sc[2], ha, la); split_scale(sc[3], hb, lb);
                    h23 = izb::prmt(ha, hb, 0x5410); l23 = izb::prmt(la, lb, 0x5410);
#pragma unroll
                    for (int j = 0; j < DT; ++j) {
                        const int w = j >> 3, sh = 4 * (j & 7);
                        const uint32_t b0 = q4_value(q4_pair(((x[0][w] >> sh) & 0xFu) | (((x[1][w] >> sh) & 0xFu) << 16)), h01, l01);
                        const uint32_t b1 = q4_value(q4_pair(((x[2][w] >> sh) & 0xFu) | (((x[3][w] >> sh) & 0xFu) << 16)), h23, l23);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            izb::mma_bf16_16816(o[mt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
                    }
                }
            }
        }
    }
    cp_wait<0>();

    // ---- join the warps that shared the rows, leave the chunk's result ----
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 1);
            l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 2);
            if (tq == 0) wml[warp * 32 + mt * 16 + h * 8 + gq] = make_float2(m[mt][h], l[mt][h]);
        }
    __syncthreads();  // also: every tile of the ring has been read
    float* ex = reinterpret_cast<float*>(ring);  // [warp][16 MT][D]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = mt * 16 + gq + (e >> 1) * 8;
                const int n = tq * 2 + (e & 1);
                const int d = Q == IZB_KV_NONE ? j * 8 + n : n * DT + j;
                ex[(warp * 16 * MT + r) * D + d] = o[mt][j][e];
            }
    __syncthreads();
    for (int i = tid; i < n_rows * D; i += SP_THREADS) {
        const int r = i / D, d = i - r * D;
        const int w = r / (16 * MT), rr = r - w * 16 * MT;
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < WN; ++n) top = fmaxf(top, wml[(n * WM + w) * 32 + rr].x);
        float sum = 0.f, a = 0.f;
#pragma unroll
        for (int n = 0; n < WN; ++n) {
            const float2 x = wml[(n * WM + w) * 32 + rr];
            const float f = x.x == -INFINITY ? 0.f : ex2(x.x - top);
            sum += f * x.y;
            a += f * ex[((n * WM + w) * 16 * MT + rr) * D + d];
        }
        const int row = row0 + r, sq_i = row / p.g, h = row - sq_i * p.g;
        const long long slot = (static_cast<long long>(seq0 + sq_i) * p.heads + kh * p.g + h) * chunks_total + chunk_slot;
        p.acc[slot * D + d] = a;
        if (d == 0) p.ml[slot] = make_float2(top, sum);
    }
}

__device__ __forceinline__ int length_of(const Source& s, int row) { return min(max(s.lens[row], 0), s.max_len); }

template <int D, int WM, int MT>
__global__ void __launch_bounds__(SP_THREADS) shared_prefix_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
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
        const int len = length_of(p.prefix, group), t0 = chunk * p.prefix.chunk, t1 = min(len, t0 + p.prefix.chunk);
        if (t0 >= t1) return;
        constexpr int ROWS = 16 * MT * WM;
        const int row0 = rb * ROWS, n = min(ROWS, p.seqs * p.g - row0);
        if (p.prefix.quant == IZB_KV_NONE)
            attend<D, WM, MT, IZB_KV_NONE>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, t1, chunk, chunks, smem);
        else if (p.prefix.quant == IZB_KV_INT8)
            attend<D, WM, MT, IZB_KV_INT8>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, t1, chunk, chunks, smem);
        else
            attend<D, WM, MT, IZB_KV_Q4_0>(p, p.prefix, group, kh, group * p.seqs, row0, n, t0, t1, chunk, chunks, smem);
        return;
    }
    item -= p.prefix_items;
    const int kh = item % p.kv_heads;
    item /= p.kv_heads;
    const int chunk = item % p.own.n_chunks, seq = item / p.own.n_chunks;
    const int len = length_of(p.own, seq), t0 = chunk * p.own.chunk, t1 = min(len, t0 + p.own.chunk);
    if (t0 >= t1) return;
    const int slot = p.prefix.n_chunks + chunk;
    if (p.own.quant == IZB_KV_NONE) attend<D, 1, 1, IZB_KV_NONE>(p, p.own, seq, kh, seq, 0, p.g, t0, t1, slot, chunks, smem);
    else if (p.own.quant == IZB_KV_INT8) attend<D, 1, 1, IZB_KV_INT8>(p, p.own, seq, kh, seq, 0, p.g, t0, t1, slot, chunks, smem);
    else attend<D, 1, 1, IZB_KV_Q4_0>(p, p.own, seq, kh, seq, 0, p.g, t0, t1, slot, chunks, smem);
}

// One CTA per (sequence, head): four warps take every fourth chunk, a lane D / 32 channels.
template <int D>
__global__ void __launch_bounds__(128)
    shared_prefix_join_kernel(const __grid_constant__ Params p, __nv_bfloat16* __restrict__ out, long long ld_out) {
    izb::pdl_launch_dependents();
    izb::pdl_wait();
    constexpr int E = D / 32;
    __shared__ float sm_acc[4][D], sm_m[4], sm_l[4];
    const int row = blockIdx.x, seq = row / p.heads, head = row - seq * p.heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = p.prefix.n_chunks + p.own.n_chunks;
    const int np = p.prefix.n_chunks ? (length_of(p.prefix, seq / p.seqs) + p.prefix.chunk - 1) / p.prefix.chunk : 0;
    const int no = p.own.n_chunks ? (length_of(p.own, seq) + p.own.chunk - 1) / p.own.chunk : 0;
    const long long base = static_cast<long long>(row) * chunks;
    float m = -INFINITY, l = 0.f, a[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = 0.f;
#pragma unroll 4
    for (int c = warp; c < np + no; c += 4) {
        const long long slot = base + (c < np ? c : p.prefix.n_chunks + c - np);
        const float2 x = p.ml[slot];
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = p.acc[slot * D + lane * E + e];
        const float n = fmaxf(m, x.x);
        const float u = n == -INFINITY ? 0.f : n;
        const float f = ex2(m - u), g = ex2(x.x - u);
        l = l * f + x.y * g;
        m = n;
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] = a[e] * f + v[e] * g;
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
    int rows;        // query rows of a prefix item: 16, 32, 64 or 128
    int row_blocks;
    int prefix_chunk, prefix_chunks, own_chunk, own_chunks;
};

// Tokens per item.  `base` items per chunk of the sequence meet `slots` resident CTAs in waves; an item costs its
// tiles plus about one tile for the query rows, the table of places and the result.  The split counts from the
// fewest whose chunks fit the table of places are tried.
int choose_chunk(int64_t base, int64_t tokens, int64_t slots) {
    const int64_t tiles = (tokens + SP_TILE - 1) / SP_TILE;
    const int64_t fewest = (tiles + SP_MAX_CHUNK / SP_TILE - 1) / (SP_MAX_CHUNK / SP_TILE), most = fewest + 48;
    int64_t best = 0, best_cost = INT64_MAX;
    for (int64_t n = fewest; n <= tiles && n <= most; ++n) {
        const int64_t per = (tiles + n - 1) / n, items = base * ((tiles + per - 1) / per);
        const int64_t cost = ((items + slots - 1) / slots) * (per + 1);
        if (cost < best_cost) {
            best_cost = cost;
            best = per;
        }
        if (per == 1) break;
    }
    return static_cast<int>(best * SP_TILE);
}

Plan make_plan(const izb_ctx* ctx, int64_t groups, int64_t seqs, int kv_heads, int g, int64_t max_prefix, int64_t max_own) {
    Plan pl = {};
    const int64_t rows = seqs * g, slots = 2 * static_cast<int64_t>(ctx && ctx->sm_count > 0 ? ctx->sm_count : 148);
    // the smallest block that holds the rows: a tile's fragments serve all rows of a block, idle rows cost mma steps
    pl.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    pl.row_blocks = static_cast<int>((rows + pl.rows - 1) / pl.rows);
    if (max_prefix > 0) {
        pl.prefix_chunk = choose_chunk(groups * kv_heads * pl.row_blocks, max_prefix, slots);
        pl.prefix_chunks = static_cast<int>((max_prefix + pl.prefix_chunk - 1) / pl.prefix_chunk);
    }
    if (max_own > 0) {
        pl.own_chunk = choose_chunk(groups * seqs * kv_heads, max_own, slots);
        pl.own_chunks = static_cast<int>((max_own + pl.own_chunk - 1) / pl.own_chunk);
    }
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
    s->max_len = static_cast<int>(max_len);
    return IZB_OK;
}

template <int D, int ROWS>
size_t smem_for(const Source& s) {
    if (s.n_chunks == 0) return 0;
    return s.quant == IZB_KV_NONE ? item_smem<D, ROWS, IZB_KV_NONE>(s.chunk)
           : s.quant == IZB_KV_INT8 ? item_smem<D, ROWS, IZB_KV_INT8>(s.chunk) : item_smem<D, ROWS, IZB_KV_Q4_0>(s.chunk);
}

template <int D, int WM, int MT>
int launch_items(izb_ctx* ctx, cudaStream_t s, const Params& p, int64_t items) {
    size_t smem = smem_for<D, 16 * MT * WM>(p.prefix);
    const size_t own = smem_for<D, 16>(p.own);
    if (own > smem) smem = own;
    auto kern = shared_prefix_kernel<D, WM, MT>;
    static std::atomic<int> smem_set[IZB_MAX_DEVICES];
    if (smem_set[ctx->device].load(std::memory_order_relaxed) < static_cast<int>(smem)) {
        IZB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->max_smem_optin));
        smem_set[ctx->device].store(ctx->max_smem_optin, std::memory_order_relaxed);
    }
    IZB_CUDA_TRY(izb::launch_chained(ctx, kern, dim3(static_cast<unsigned>(items)), dim3(SP_THREADS), smem, s, p));
    ctx->launches.fetch_add(1, std::memory_order_relaxed);
    return IZB_OK;
}

template <int D>
int launch_dim(izb_ctx* ctx, cudaStream_t s, const Params& p, const Plan& pl, int64_t items, int64_t batch, __nv_bfloat16* out,
               long long ld_out) {
    if (items > 0) {
        const int rc = pl.rows == 16   ? launch_items<D, 1, 1>(ctx, s, p, items)
                       : pl.rows == 32 ? launch_items<D, 1, 2>(ctx, s, p, items)
                       : pl.rows == 64 ? launch_items<D, 2, 2>(ctx, s, p, items)
                                       : launch_items<D, 4, 2>(ctx, s, p, items);
        if (rc != IZB_OK) return rc;
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
    const Plan pl = make_plan(ctx, groups, seqs_per_group, kv_heads, heads / kv_heads, max_prefix_len, max_seq_len);
    return plan_bytes(pl, groups * seqs_per_group, heads, head_dim);
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
    const Plan pl = make_plan(ctx, groups, seqs_per_group, kv_heads, heads / kv_heads, max_prefix_len, max_seq_len);
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
    p.scale_log2 = scale * LOG2E;
    const int64_t prefix_items = groups * pl.prefix_chunks * kv_heads * pl.row_blocks, items = prefix_items + batch * kv_heads * pl.own_chunks;
    if (items > INT32_MAX) return IZB_ERR_UNSUPPORTED;
    p.prefix_items = static_cast<int>(prefix_items);
    izb::DeviceGuard guard(ctx->device);
    if (!guard.ok) return IZB_ERR_LAUNCH;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto* op = static_cast<__nv_bfloat16*>(out);
    return d == 128 ? launch_dim<128>(ctx, s, p, pl, items, batch, op, ld_out) : launch_dim<64>(ctx, s, p, pl, items, batch, op, ld_out);
}

}  // extern "C"
