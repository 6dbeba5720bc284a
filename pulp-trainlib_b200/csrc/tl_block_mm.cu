// The products of the feed-forward block and of the 8-bit linear layer on the tensor cores (tcgen05, operands by TMA, accumulators in tensor memory).
// Persistent CTAs walk tiles of 128 rows (256 for a CTA pair) x BN accumulator columns: a producer warp fills a ring of shared-memory
// stages of 128 bytes of K per row, a thread of another warp multiplies them, eight warps take finished accumulators out and apply the epilogue.
//   gate:      the B operand of a tile is BN / 2 rows of Wg and the same rows of Wu (in a pair: one CTA's shared memory holds Wg's, the
//              other's Wu's), so that gate and up of a result lie BN / 2 columns apart in the same lane: H, and if wanted G and U, leave from
//              registers and the pre-activations are never read back.
//   gate, bw:  dH stays in the accumulator; the epilogue reads G and U and writes H, dG and dU.
//   8 bits:    kind::i8, 32-bit integer accumulators (exact); scales and bias in the epilogue.
//   fp32:      3xTF32 on packed (hi, lo) pairs: D0 = A_hi [B_hi | B_lo]^T, D1 = A_lo B_hi^T.  The accumulator truncates: each step takes up to 2^-23 of it
//              off towards zero, which over a chain of n steps is 0.24 n 2^-23 of the result (4e-6 at K = 1024).  So every 128 of K
//              the accumulators are added to sums in registers, rounded to nearest, and started anew: 5e-7 at any K.
// Few tiles: `splits` CTAs share a tile's K and leave partial tiles, which bm_reduce_kernel adds in order (with the same epilogue).
// Measured with 4096 tokens, 2048 x 8192 x 2048, half precision (1627 TFLOP/s in short runs): gate and up with all results kept 180 us (1523 TFLOP/s, tensor pipe
// active 93% of the cycles), the product behind them 100 (1374), dH with its epilogue 138 (996: shared memory carries five tensors beside the operands),
// the four gradients in one launch 475 (1446, 97%).  8 bits, 4096 x 8192 -> 4096: 95 us (2890).  In a stream of passes the power limit sets the clock.
// No multicast loads.  Every wait is bounded and reports through the status word.
#include "tl_tma_mm.cuh"
#include "tl_gate.cuh"
#include <algorithm>

namespace tl {

enum { MM_F16 = 0, MM_TF32 = 1, MM_I8 = 2 };
static constexpr int BM_ROWS = 128, BM_EPI = 8, BM_THREADS = 32 * (BM_EPI + 2), BM_MAX_STAGES = 8;
static constexpr uint32_t BM_RING = 192 * 1024;
static constexpr int BM_CHUNK = 4;                     // fp32: K steps of 32 between two drains of the accumulators

template <int KIND> struct BmCfg { static constexpr int BK = KIND == MM_F16 ? 64 : KIND == MM_TF32 ? 32 : 128, PARTS = KIND == MM_TF32 ? 2 : 1; };

// A product of a launch.  Its units (tiles x splits) follow those of the product before; a CTA (or pair) takes every step-th unit of the launch.
template <class T> struct BmJob {
    T *C, *g, *u, *dg, *du;
    const T *bias; const float *xs, *ws;
    uint32_t *part;
    int N, M, ld, tiles_m, tiles_n, kps, ksteps, splits, first, reduce_first, a_mn, b_mn;  // ld: elements between the rows of C, dg and du (g and u: M); kps: K steps of a term
    int c_align, g_align;                                                                  // ALIGN_* of C, dg, du and of g, u
};
// What all rows of a tensor start on: 16 bytes (and are whole groups of 16 long, or padded so), 4 bytes, or their elements' size
enum { ALIGN_ELEMENT = 0, ALIGN_WORD = 1, ALIGN_16 = 2 };
static constexpr int BM_JOBS = 4;
constexpr int bm_jobs(int epi) { return epi == FFN_PLAIN ? BM_JOBS : 1; }
template <class T, int JOBS> struct BmParams {
    BmJob<T> job[JOBS];
    int jobs, units, stages, reduce_blocks;
    uint32_t stage_bytes;
    int *status;
};
struct BmMaps { CUtensorMap a[2], b[2]; };
template <int JOBS> struct BmMapList { BmMaps of[JOBS]; };

// The four MMAs of a stage, 32 bytes (or 16 rows) of K each; a, b: lower words of the first one's descriptors, SA, SB: 16-byte units to the next one's.  What the
// issuing thread does per stage decides where tiles are small: with 64-bit descriptors added up, steps in registers and the barrier asked only when its stage
// was wanted a stage took 490 cycles (128 x 64 of 8 bits: 128 on the tensor cores).
constexpr uint32_t BM_DESC_UPPER = 1024u >> 4 | 1u << 14 | LAYOUT_SW128 << 29;
#define TL_BM_MMA(GROUP, TYPE, ACC) \
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t" ACC "add.u32 la, %1, %4;\n\tadd.u32 lb, %2, %5;\n\t" \
                 "mov.b64 da, {la, %6};\n\tmov.b64 db, {lb, %6};\n\ttcgen05.mma.cta_group::" GROUP ".kind::" TYPE " [%0], da, db, %3, p;\n\t}" \
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(kk * SA), "n"(kk * SB), "n"(BM_DESC_UPPER), "r"(acc) : "memory")
#define TL_BM_MMA_KIND(ACC)                                                                                   \
    do {                                                                                                      \
        if constexpr (KIND == MM_F16) { if constexpr (PAIR) TL_BM_MMA("2", "f16", ACC); else TL_BM_MMA("1", "f16", ACC); }         \
        else if constexpr (KIND == MM_TF32) { if constexpr (PAIR) TL_BM_MMA("2", "tf32", ACC); else TL_BM_MMA("1", "tf32", ACC); } \
        else { if constexpr (PAIR) TL_BM_MMA("2", "i8", ACC); else TL_BM_MMA("1", "i8", ACC); }               \
    } while (0)
template <int KIND, bool PAIR, int SA, int SB, int kk> __device__ __forceinline__ void bm_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    if constexpr (kk == 0) TL_BM_MMA_KIND("setp.ne.b32 p, %7, 0;\n\t");
    else TL_BM_MMA_KIND("setp.eq.b32 p, 0, 0;\n\t");
}
#undef TL_BM_MMA_KIND
#undef TL_BM_MMA
template <int KIND, bool PAIR, int SA, int SB> __device__ __forceinline__ void bm_step(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    bm_mma<KIND, PAIR, SA, SB, 0>(d, a, b, idesc, acc);
    bm_mma<KIND, PAIR, SA, SB, 1>(d, a, b, idesc, acc);
    bm_mma<KIND, PAIR, SA, SB, 2>(d, a, b, idesc, acc);
    bm_mma<KIND, PAIR, SA, SB, 3>(d, a, b, idesc, acc);
}
// has the phase completed? (asked without waiting: mbarrier.try_wait may suspend the thread, for a stage that is not coming too)
__device__ __forceinline__ bool bm_peek(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// accumulators of 32-bit integers (2), operands of signed 8 bits (1), both K-major
__host__ __device__ constexpr uint32_t i8_idesc(uint32_t M, uint32_t N) { return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24); }

// ---------------------------------------------------------------- epilogue of W neighbouring results of a row
template <int W> __device__ __forceinline__ void bm_st(float *p, const float (&v)[W], int live, bool vec)
{
    if (vec && live >= W) {
#pragma unroll
        for (int j = 0; j < W; j += 4) *reinterpret_cast<float4 *>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) if (j < live) p[j] = v[j];
    }
}
__device__ __forceinline__ uint32_t bm_half2(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int W> __device__ __forceinline__ void bm_st(__half *p, const float (&v)[W], int live, bool vec)
{
    if (vec && live >= W) {
        if constexpr (W % 8 == 0) {
#pragma unroll
            for (int j = 0; j < W; j += 8)
                *reinterpret_cast<uint4 *>(p + j) = make_uint4(bm_half2(v[j], v[j + 1]), bm_half2(v[j + 2], v[j + 3]), bm_half2(v[j + 4], v[j + 5]), bm_half2(v[j + 6], v[j + 7]));
        } else *reinterpret_cast<uint2 *>(p) = make_uint2(bm_half2(v[0], v[1]), bm_half2(v[2], v[3]));
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) if (j < live) st(p + j, v[j]);
    }
}
template <int W> __device__ __forceinline__ void bm_ld(const float *p, float (&v)[W], int live, bool vec)
{
    if (vec && live >= W) {
#pragma unroll
        for (int j = 0; j < W; j += 4) { const float4 x = *reinterpret_cast<const float4 *>(p + j); v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w; }
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = ld0(j < live, p + j);
    }
}
__device__ __forceinline__ void bm_unpack(uint32_t w, float &a, float &b)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    a = f.x; b = f.y;
}
template <int W> __device__ __forceinline__ void bm_ld(const __half *p, float (&v)[W], int live, bool vec)
{
    if (vec && live >= W) {
        if constexpr (W % 8 == 0) {
#pragma unroll
            for (int j = 0; j < W; j += 8) {
                const uint4 x = *reinterpret_cast<const uint4 *>(p + j);
                bm_unpack(x.x, v[j], v[j + 1]); bm_unpack(x.y, v[j + 2], v[j + 3]); bm_unpack(x.z, v[j + 4], v[j + 5]); bm_unpack(x.w, v[j + 6], v[j + 7]);
            }
        } else { const uint2 x = *reinterpret_cast<const uint2 *>(p); bm_unpack(x.x, v[0], v[1]); bm_unpack(x.y, v[2], v[3]); }
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = ld0(j < live, p + j);
    }
}
// ---------------------------------------------------------------- tiles of 32 rows x W columns between a warp's registers and memory
// In registers a lane has a row (as tensor memory gives it), in memory neighbouring lanes should have neighbouring columns: the tile turns in 2 KB of shared
// memory per warp, 16-byte chunks XOR-swizzled with the row so that neither side has bank conflicts.  A lane storing its own row's 16 bytes
// touches 32 lines per instruction; so the gradient's epilogue (two tensors in, three out) took 50000 cycles per tile, three times its products.
template <class T, int W> struct BmTile {
    static constexpr int CHUNKS = W * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T);        // of a row; elements of a chunk
    static __device__ __forceinline__ int at(int row, int chunk) { return (row * CHUNKS + (chunk ^ (row / (8 / CHUNKS) & (CHUNKS - 1)))) * 16; }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        if constexpr (sizeof(T) == 2) return make_uint4(bm_half2(v[0], v[1]), bm_half2(v[2], v[3]), bm_half2(v[4], v[5]), bm_half2(v[6], v[7]));
        else return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    // Rows that do not start on 16 bytes move in 32-bit words, neighbouring lanes neighbouring words of a row: in memory as a word where rows start on four bytes,
    // as two halves otherwise.  (Element by element, each load waited for the one before: with 1650 columns the gradient's epilogue took 38 us, now 10.)
    static constexpr int WORDS = CHUNKS * 4, ROW_WORDS = W * (int)sizeof(T) / 4;           // of a lane; of a row
    static __device__ __forceinline__ uint32_t &word(uint4 (&q)[CHUNKS], int i) { return reinterpret_cast<uint32_t *>(&q[i / 4])[i % 4]; }
    // registers -> memory; base: the tensor's element (first row of the warp, first column of the tile); rows, cols: how many of them exist
    static __device__ __forceinline__ void store(T *base, int ld, int rows, int cols, int align, const float (&v)[W], unsigned char *stage, int lane)
    {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) *reinterpret_cast<uint4 *>(stage + at(lane, c)) = pack(v + c * E);
        __syncwarp();
        if (align == ALIGN_16) {
#pragma unroll
            for (int i = 0; i < CHUNKS; i++) {
                const int r = i * (32 / CHUNKS) + lane / CHUNKS, c = lane % CHUNKS;
                const uint4 x = *reinterpret_cast<const uint4 *>(stage + at(r, c));
                if (r < rows && c * E < cols) *reinterpret_cast<uint4 *>(base + (size_t)r * ld + c * E) = x;
            }
        } else if (sizeof(T) == 4 || align == ALIGN_WORD) {
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                const int r = (i * 32 + lane) / ROW_WORDS, k = (i * 32 + lane) % ROW_WORDS, c = k * 4 / (int)sizeof(T);
                const uint32_t x = *reinterpret_cast<const uint32_t *>(stage + at(r, k / 4) + k % 4 * 4);
                if (r < rows && c < cols) *reinterpret_cast<uint32_t *>(base + (size_t)r * ld + c) = x;
            }
        } else {                                             // (neighbouring elements from neighbouring lanes: halves of words alternating would be two writes of every sector)
#pragma unroll 8
            for (int i = 0; i < W; i++) {
                const int r = (i * 32 + lane) / W, c = (i * 32 + lane) % W;
                const T x = *reinterpret_cast<const T *>(stage + at(r, c / E) + c % E * (int)sizeof(T));
                if (r < rows && c < cols) base[(size_t)r * ld + c] = x;
            }
        }
        __syncwarp();
    }
    // memory -> registers in two steps, so that the loads can be under way long before the tile is needed
    static __device__ __forceinline__ void fetch(const T *base, int ld, int rows, int cols, int align, uint4 (&q)[CHUNKS], int lane)
    {
#pragma unroll
        for (int i = 0; i < CHUNKS; i++) q[i] = make_uint4(0, 0, 0, 0);
        if (align == ALIGN_16) {
#pragma unroll
            for (int i = 0; i < CHUNKS; i++) {
                const int r = i * (32 / CHUNKS) + lane / CHUNKS, c = lane % CHUNKS;
                if (r < rows && c * E < cols) q[i] = *reinterpret_cast<const uint4 *>(base + (size_t)r * ld + c * E);
            }
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                const int r = (i * 32 + lane) / ROW_WORDS, c = (i * 32 + lane) % ROW_WORDS * 4 / (int)sizeof(T);
                const T *from = base + (size_t)r * ld + c;
                if (r >= rows || c >= cols) continue;
                if (sizeof(T) == 4 || align == ALIGN_WORD) word(q, i) = *reinterpret_cast<const uint32_t *>(from);
                else {
                    const unsigned short *h = reinterpret_cast<const unsigned short *>(from);
                    word(q, i) = h[0] | (c + 1 < cols ? (uint32_t)h[1] << 16 : 0u);
                }
            }
        }
    }
    static __device__ __forceinline__ void turn(int align, uint4 (&q)[CHUNKS], float (&v)[W], unsigned char *stage, int lane)
    {
        if (align == ALIGN_16) {
#pragma unroll
            for (int i = 0; i < CHUNKS; i++) *reinterpret_cast<uint4 *>(stage + at(i * (32 / CHUNKS) + lane / CHUNKS, lane % CHUNKS)) = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                const int r = (i * 32 + lane) / ROW_WORDS, k = (i * 32 + lane) % ROW_WORDS;
                *reinterpret_cast<uint32_t *>(stage + at(r, k / 4) + k % 4 * 4) = word(q, i);
            }
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            const uint4 x = *reinterpret_cast<const uint4 *>(stage + at(lane, c));
            if constexpr (sizeof(T) == 2) {
                bm_unpack(x.x, v[c * E], v[c * E + 1]); bm_unpack(x.y, v[c * E + 2], v[c * E + 3]); bm_unpack(x.z, v[c * E + 4], v[c * E + 5]); bm_unpack(x.w, v[c * E + 6], v[c * E + 7]);
            } else { v[c * E] = __uint_as_float(x.x); v[c * E + 1] = __uint_as_float(x.y); v[c * E + 2] = __uint_as_float(x.z); v[c * E + 3] = __uint_as_float(x.w); }
        }
        __syncwarp();
    }
};
// The results of W columns from col on of the 32 rows from row0 on.  v: the accumulators (gate), w: the second ones (up); gq, uq: G and U as BmTile::fetch left them.
template <class T, int EPI, int W>
__device__ __forceinline__ void bm_tile_results(const BmJob<T> &p, int row0, int col, float (&v)[W], float (&w)[W], uint4 (&gq)[BmTile<T, W>::CHUNKS],
                                                uint4 (&uq)[BmTile<T, W>::CHUNKS], unsigned char *stage, int lane)
{
    typedef BmTile<T, W> Tile;
    constexpr bool FAST = sizeof(T) == 2;
    const size_t at = (size_t)row0 * p.ld + col;
    const int rows = p.N - row0, cols = p.M - col;
    if constexpr (EPI == FFN_GATE) {
        if (p.g) {
            const size_t of = (size_t)row0 * p.M + col;
            Tile::store(p.g + of, p.M, rows, cols, p.g_align, v, stage, lane);
            Tile::store(p.u + of, p.M, rows, cols, p.g_align, w, stage, lane);
        }
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = gate_fw<FAST>(v[j], w[j]);
    } else if constexpr (EPI == FFN_GATE_BW) {
        float g[W], u[W];
        Tile::turn(p.g_align, gq, g, stage, lane);
        Tile::turn(p.g_align, uq, u, stage, lane);
#pragma unroll
        for (int j = 0; j < W; j++) { const float dh = v[j]; gate_bw<FAST>(g[j], u[j], dh, v[j], g[j], u[j]); }
        Tile::store(p.dg + at, p.ld, rows, cols, p.c_align, g, stage, lane);
        Tile::store(p.du + at, p.ld, rows, cols, p.c_align, u, stage, lane);
    } else if constexpr (EPI == FFN_INT8) {
        const float xs = ld0(lane < rows, p.xs + row0 + lane);
        const bool even = cols >= W && ((uintptr_t)p.ws & 15) == 0;
        float s[W];
        bm_ld<W>(p.ws + col, s, cols, even);
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = v[j] * xs * s[j];
        if (p.bias) {
            bm_ld<W>(p.bias + col, s, cols, cols >= W && ((uintptr_t)p.bias & 15) == 0);
#pragma unroll
            for (int j = 0; j < W; j++) v[j] += s[j];
        }
    }
    Tile::store(p.C + at, p.ld, rows, cols, p.c_align, v, stage, lane);
}
// The same for four columns of a row (from partial tiles)
template <class T, int EPI> __device__ __forceinline__ void bm_results(const BmJob<T> &p, int row, int col, float (&v)[4], float (&w)[4])
{
    constexpr bool FAST = sizeof(T) == 2;
    const size_t at = (size_t)row * p.ld + col, of = (size_t)row * p.M + col;
    const int live = p.M - col;
    const bool c_vec = p.c_align == ALIGN_16, g_vec = p.g_align == ALIGN_16;
    if constexpr (EPI == FFN_GATE) {
        if (p.g) { bm_st<4>(p.g + of, v, live, g_vec); bm_st<4>(p.u + of, w, live, g_vec); }
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = gate_fw<FAST>(v[j], w[j]);
    } else if constexpr (EPI == FFN_GATE_BW) {
        float g[4], u[4];
        bm_ld<4>(p.g + of, g, live, g_vec); bm_ld<4>(p.u + of, u, live, g_vec);
#pragma unroll
        for (int j = 0; j < 4; j++) { const float dh = v[j]; gate_bw<FAST>(g[j], u[j], dh, v[j], g[j], u[j]); }
        bm_st<4>(p.dg + at, g, live, c_vec); bm_st<4>(p.du + at, u, live, c_vec);
    } else if constexpr (EPI == FFN_INT8) {
        const float xs = p.xs[row];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = v[j] * xs * ld0(j < live, p.ws + col + j) + ld0(p.bias && j < live, p.bias + col + j);
    }
    bm_st<4>(p.C + at, v, live, c_vec);
}

// tile -> row block, column block: eight row blocks share a sweep over the columns
template <class T> __device__ __forceinline__ void bm_locate(const BmJob<T> &p, int tile, int &rb, int &cb)
{
    const int g = tile / (8 * p.tiles_m), in = tile - g * 8 * p.tiles_m, rows = min(8, p.tiles_n - 8 * g);
    rb = 8 * g + in % rows; cb = in / rows;
}

// unit of a launch -> product, tile, part of its K
struct BmUnit { int job, tile, rank, ks0, ks1; };
template <class T, int JOBS> __device__ __forceinline__ BmUnit bm_unit(const BmParams<T, JOBS> &p, int unit)
{
    BmUnit u;
    u.job = 0;
#pragma unroll
    for (int i = 1; i < JOBS; i++) if (i < p.jobs && unit >= p.job[i].first) u.job = i;
    const BmJob<T> &j = p.job[u.job];
    unit -= j.first;
    u.tile = unit / j.splits; u.rank = unit - u.tile * j.splits;
    u.ks0 = j.ksteps * u.rank / j.splits; u.ks1 = j.ksteps * (u.rank + 1) / j.splits;
    return u;
}

template <int KIND, class T, int EPI, int BN, bool PAIR>
__global__ void __launch_bounds__(BM_THREADS) block_mm_kernel(const __grid_constant__ BmMapList<bm_jobs(EPI)> maps, const __grid_constant__ BmParams<T, bm_jobs(EPI)> p)
{
    constexpr int BK = BmCfg<KIND>::BK, PARTS = BmCfg<KIND>::PARTS;
    constexpr int BNL = PAIR ? BN / 2 : BN;                                         // rows of B in this CTA's shared memory
    constexpr int BNC = EPI == FFN_GATE ? BN / 2 : BN;                              // result columns of a tile
    constexpr int CW = BNC / 2;                                                     // of a warp
    constexpr int ROWS = PAIR ? 2 * BM_ROWS : BM_ROWS;
    constexpr uint32_t A_BYTES = BM_ROWS * 128u, B_BYTES = BNL * 128u;
    constexpr int NBUF = KIND == MM_TF32 && BN > 64 ? 1 : 2;
    constexpr uint32_t BUF_COLS = 256;
    constexpr int W = CW < 64 / (int)sizeof(T) ? CW : 64 / (int)sizeof(T);                // columns that a warp's epilogue takes at a time
    extern __shared__ unsigned char bsm_raw[];
    const uint32_t sbase = (smem_u32(bsm_raw) + 1023u) & ~1023u;                    // swizzle atoms want 1024-byte alignment
    __shared__ uint64_t full[BM_MAX_STAGES], empty[BM_MAX_STAGES], acc_full[2], acc_empty[2], last_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed_s;
    __shared__ __align__(16) unsigned char stages_out[BM_EPI][2048];
    volatile int *failed = &failed_s;

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int ST = p.stages;
    const int rank = PAIR ? (int)blockIdx.x % 2 : 0, first = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x, step = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
    const int row_of_tile = PAIR ? rank * BM_ROWS : 0;

    if (tid == 0) {
        for (int s = 0; s < ST; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; b++) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], PAIR ? 2 * BM_EPI : BM_EPI); }
        mbar_init(&last_bar, 1);
        failed_s = 0;
        fence_barrier_init();
        tma_prefetch_desc(&maps.of[0].a[0]); tma_prefetch_desc(&maps.of[0].b[0]);
    }
    if (warp == 0) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
    }
    tc_fence_before();
    if constexpr (PAIR) tm_cluster_sync();                                          // the other CTA's barriers are initialised too
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    if (warp == BM_EPI) {
        // producer (whole warp; a thread is elected around the instructions)
        const uint32_t full0 = PAIR ? tm_mapa(smem_u32(&full[0]), 0) : 0u;          // the pair's leader counts both CTAs' bytes
        int s = 0;
        uint32_t phase = 1, issued = 0;                                             // the first pass over the ring finds it empty
        bool ok = true;
        for (int unit = first; unit < p.units && ok; unit += step) {
            const BmUnit un = bm_unit(p, unit);
            const BmJob<T> &j = p.job[un.job];
            const BmMaps &map = maps.of[un.job];
            int rb, cb;
            bm_locate(j, un.tile, rb, cb);
            const int row0 = rb * ROWS + row_of_tile, col0 = cb * BNC;
            int term = un.ks0 / j.kps, kt = un.ks0 - term * j.kps;
            for (int k = un.ks0; k < un.ks1; k++) {
                if (!tm_wait(&empty[s], phase, failed)) { ok = false; break; }
                if (elect_one()) {
                    const uint32_t st = sbase + s * p.stage_bytes, sb = st + PARTS * A_BYTES;
                    const uint32_t bar = full0 + 8u * s;
                    auto load = [&](uint32_t dst, const CUtensorMap *m, int x, int y, int z) {
                        if constexpr (PAIR) tma_load_3d_pair(dst, m, bar, x, y, z);
                        else tma_load_3d(dst, m, &full[s], x, y, z);
                    };
                    if (!PAIR || rank == 0) mbar_arrive_expect_tx(&full[s], PAIR ? 2 * p.stage_bytes : p.stage_bytes);
                    const CUtensorMap *ma = &map.a[term], *mb = &map.b[EPI == FFN_GATE ? 0 : term];
#pragma unroll
                    for (int z = 0; z < PARTS; z++) {
                        if (KIND == MM_F16 && j.a_mn) { for (int q = 0; q < 2; q++) load(st + q * 8192u, ma, row0 + 64 * q, kt * BK, 0); }
                        else load(st + z * A_BYTES, ma, kt * BK, row0, z);
                        if constexpr (EPI == FFN_GATE) {
                            if constexpr (PAIR) load(sb, &map.b[rank], kt * BK, col0, 0);
                            else {
                                load(sb + z * B_BYTES, &map.b[0], kt * BK, col0, z);
                                load(sb + z * B_BYTES + B_BYTES / 2, &map.b[1], kt * BK, col0, z);
                            }
                        } else {
                            const int c = col0 + (PAIR ? rank * BNL : 0);
                            if (KIND == MM_F16 && j.b_mn) { for (int q = 0; q < BNL / 64; q++) load(sb + q * 8192u, mb, c + 64 * q, kt * BK, 0); }
                            else load(sb + z * B_BYTES, mb, kt * BK, c, z);
                        }
                    }
                }
                __syncwarp();
                issued++;
                if (++kt == j.kps) { kt = 0; term++; }
                if (++s == ST) { s = 0; phase ^= 1u; }
            }
        }
        // given up: the copies still under way land before the shared memory is left (the pair's leader sees both CTAs')
        if (!ok && (!PAIR || rank == 0))
            for (int j = 0; j < ST; j++) {
                if ((uint32_t)j >= issued && issued < (uint32_t)ST) break;
                const uint32_t parity = j < s ? phase ^ 1u : phase;
                for (int i = 0; i < 100000 && !mbar_try_wait(&full[j], parity); i++) __nanosleep(100);
            }
    } else if (warp == BM_EPI + 1) {
        if ((!PAIR || rank == 0) && elect_one()) {                                // one thread walks the loop
            const uint32_t stage_step = p.stage_bytes >> 4;
            bool ready = false;                                                     // the next stage was seen full
            const uint32_t idesc_lo = mma_idesc(FMT_TF32, ROWS, BN);
            int s = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = first; unit < p.units && ok; unit += step) {
                const BmUnit un = bm_unit(p, unit);
                const bool a_mn = KIND == MM_F16 && p.job[un.job].a_mn, b_mn = KIND == MM_F16 && p.job[un.job].b_mn;
                const uint32_t majors = (a_mn ? IDESC_A_MN_MAJOR : 0u) | (b_mn ? IDESC_B_MN_MAJOR : 0u);
                const uint32_t idesc = KIND == MM_F16 ? (mma_idesc(FMT_F16, ROWS, BN) | majors) : KIND == MM_I8 ? i8_idesc(ROWS, BN) : mma_idesc(FMT_TF32, ROWS, 2 * BN);
                // lower descriptor words of stage 0 (the upper one is the same in every layout used)
                const uint32_t low_a = (uint32_t)(a_mn ? smem_desc_swizzled(sbase, 8192u, 1024u, LAYOUT_SW128) : smem_desc_kmajor_sw128(sbase, 1024));
                const uint32_t low_b = (uint32_t)(b_mn ? smem_desc_swizzled(sbase + PARTS * A_BYTES, 8192u, 1024u, LAYOUT_SW128) : smem_desc_kmajor_sw128(sbase + PARTS * A_BYTES, 1024));
                for (int kc = un.ks0; kc < un.ks1 && ok; it++) {
                    const int kend = KIND == MM_TF32 ? min(un.ks1, kc + BM_CHUNK) : un.ks1, buf = it % NBUF, use = it / NBUF;
                    if (use > 0 && !tm_wait(&acc_empty[buf], (uint32_t)(use - 1) & 1u, failed)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t d = tmem + buf * BUF_COLS;
                    uint32_t acc = 0;
                    for (; kc < kend; kc++) {
                        if (!ready && !tm_wait(&full[s], phase, failed)) { ok = false; break; }
                        const int now = s;
                        if (++s == ST) { s = 0; phase ^= 1u; }
                        ready = bm_peek(&full[s], phase);                       // of the next step: its answer comes while this one's MMAs are issued
                        tc_fence_after();
                        const uint32_t a = low_a + now * stage_step, b = low_b + now * stage_step;
                        if (KIND != MM_F16 || !(a_mn || b_mn)) bm_step<KIND, PAIR, 2, 2>(d, a, b, idesc, acc);
                        else if (a_mn && b_mn) bm_step<KIND, PAIR, 128, 128>(d, a, b, idesc, acc);
                        else if (b_mn) bm_step<KIND, PAIR, 2, 128>(d, a, b, idesc, acc);
                        else bm_step<KIND, PAIR, 128, 2>(d, a, b, idesc, acc);
                        if constexpr (KIND == MM_TF32) bm_step<KIND, PAIR, 2, 2>(d + 2 * BN, a + (A_BYTES >> 4), b, idesc_lo, acc);
                        tm_commit<PAIR>(&empty[now]);
                        acc = 1u;
                    }
                    if (ok) tm_commit<PAIR>(&acc_full[buf]);
                }
            }
            if (!ok) {                                                              // given up: what was issued ends first
                tm_commit<PAIR>(&last_bar);
                for (int i = 0; i < 100000 && !mbar_try_wait(&last_bar, 0); i++) __nanosleep(100);
            }
        }
        __syncwarp();
    } else {
        // epilogue: warp w owns TMEM lanes 32 (w % 4) .. + 31, one row each, and one half of the tile's result columns
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const int row_in = quarter * 32 + lane;
        unsigned char *stage = stages_out[warp];
        typedef BmTile<T, W> Tile;
        int it = 0;
        bool ok = true;
        for (int unit = first; unit < p.units && ok; unit += step) {
            const BmUnit un = bm_unit(p, unit);
            const BmJob<T> &j = p.job[un.job];
            const int ks0 = un.ks0, ks1 = un.ks1;
            int rb, cb;
            bm_locate(j, un.tile, rb, cb);
            const int row0 = rb * ROWS + row_of_tile + quarter * 32, col0 = cb * BNC + half * CW;
            constexpr int NS = KIND == MM_TF32 ? CW : 1, NS2 = KIND == MM_TF32 && EPI == FFN_GATE ? CW : 1;
            float sum[NS], sum2[NS2];
            const bool whole = PAIR || j.splits == 1;                               // results leave from here, not partial tiles
            auto take = [&](uint32_t d, int c, float (&v)[W]) {                     // W accumulators of this lane's row
                uint32_t a[W];
                if constexpr (W == 32) tmem_ld32w(d + c, a); else tmem_ld16w(d + c, a);
                if constexpr (KIND == MM_TF32) {
                    uint32_t b[W], x[W];
                    if constexpr (W == 32) { tmem_ld32w(d + BN + c, b); tmem_ld32w(d + 2 * BN + c, x); } else { tmem_ld16w(d + BN + c, b); tmem_ld16w(d + 2 * BN + c, x); }
                    tmem_wait_ld();
#pragma unroll
                    for (int q = 0; q < W; q++) v[q] = __uint_as_float(a[q]) + (__uint_as_float(b[q]) + __uint_as_float(x[q]));
                } else {
                    tmem_wait_ld();
#pragma unroll
                    for (int q = 0; q < W; q++) v[q] = KIND == MM_I8 && whole ? (float)(int)a[q] : __uint_as_float(a[q]);
                }
            };
            auto release = [&](int buf) {                                           // the accumulators are in registers: they may be overwritten
                tc_fence_before();
                __syncwarp();
                if (lane == 0) { if constexpr (PAIR) tm_arrive_at(tm_mapa(smem_u32(&acc_empty[buf]), 0)); else mbar_arrive(&acc_empty[buf]); }
            };
            auto arrived = [&](int buf, int use) {
                bool there = true;
                if (lane == 0) there = tm_wait(&acc_full[buf], (uint32_t)use & 1u, failed, 32);
                there = __shfl_sync(0xffffffffu, there ? 1 : 0, 0) != 0;
                tc_fence_after();
                return there;
            };
            uint4 gq[Tile::CHUNKS], uq[Tile::CHUNKS], g1[Tile::CHUNKS], u1[Tile::CHUNKS];       // G and U of this piece and the next
            auto fetch = [&](int c) {
                if constexpr (EPI == FFN_GATE_BW) {
                    if (!whole || row0 >= j.N || c >= CW || col0 + c >= j.M) return;
                    const size_t at = (size_t)row0 * j.M + col0 + c;
                    Tile::fetch(j.g + at, j.M, j.N - row0, j.M - col0 - c, j.g_align, g1, lane);
                    Tile::fetch(j.u + at, j.M, j.N - row0, j.M - col0 - c, j.g_align, u1, lane);
                }
            };
            uint32_t *mine = j.part + ((size_t)(un.tile * j.splits + un.rank) * BM_ROWS + row_in) * BN;        // row of the partial tile (splits > 1)
            auto leave = [&](int c, float (&v)[W], float (&w)[W]) {
                if (!whole) {
#pragma unroll
                    for (int q = 0; q < W; q += 4) {
                        *reinterpret_cast<float4 *>(mine + half * CW + c + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
                        if constexpr (EPI == FFN_GATE) *reinterpret_cast<float4 *>(mine + BNC + half * CW + c + q) = make_float4(w[q], w[q + 1], w[q + 2], w[q + 3]);
                    }
                } else if (row0 < j.N && col0 + c < j.M) bm_tile_results<T, EPI, W>(j, row0, col0 + c, v, w, gq, uq, stage, lane);
            };
            auto turn_over = [&]() {
#pragma unroll
                for (int i = 0; i < Tile::CHUNKS; i++) { gq[i] = g1[i]; uq[i] = u1[i]; }
            };
            fetch(0);
            if constexpr (KIND == MM_TF32) {
#pragma unroll
                for (int q = 0; q < NS; q++) sum[q] = 0.f;
#pragma unroll
                for (int q = 0; q < NS2; q++) sum2[q] = 0.f;
                for (int kc = ks0; kc < ks1; kc += BM_CHUNK, it++) {
                    const int buf = it % NBUF, use = it / NBUF;
                    if (!arrived(buf, use)) { ok = false; break; }
                    const uint32_t d = tmem + lane_addr + buf * BUF_COLS;
#pragma unroll
                    for (int c = 0; c < CW; c += W) {
                        float v[W];
                        take(d, half * CW + c, v);
#pragma unroll
                        for (int q = 0; q < W; q++) sum[c + q] += v[q];
                        if constexpr (EPI == FFN_GATE) {
                            take(d, BNC + half * CW + c, v);
#pragma unroll
                            for (int q = 0; q < W; q++) sum2[c + q] += v[q];
                        }
                    }
                    release(buf);
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < CW; c += W) {
                    float v[W], w[W];
#pragma unroll
                    for (int q = 0; q < W; q++) { v[q] = sum[c + q]; w[q] = EPI == FFN_GATE ? sum2[EPI == FFN_GATE ? c + q : 0] : 0.f; }
                    turn_over();
                    fetch(c + W);
                    leave(c, v, w);
                }
            } else {
                const int buf = it % NBUF, use = it / NBUF;
                it++;
                if (!arrived(buf, use)) { ok = false; break; }
                const uint32_t d = tmem + lane_addr + buf * BUF_COLS;
#pragma unroll 1
                for (int c = 0; c < CW; c += W) {
                    float v[W], w[W];
                    turn_over();
                    fetch(c + W);
                    take(d, half * CW + c, v);
                    if constexpr (EPI == FFN_GATE) take(d, BNC + half * CW + c, w);
                    if (c + W >= CW) release(buf);
                    leave(c, v, w);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*failed && tid == 0) atomicCAS(p.status, 0, 9);
    if constexpr (PAIR) {
        tm_cluster_sync();                                                          // both CTAs are done with each other's memory
        if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        tm_cluster_sync();
    } else if (warp == 0) tmem_dealloc(tmem, 512);
}

// four neighbouring sums over the partial tiles: whole numbers as such
template <int KIND, int BN> __device__ __forceinline__ void bm_add_parts(const uint32_t *from, int splits, float (&t)[4])
{
    if constexpr (KIND == MM_I8) {
        int n[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int k = 0; k < splits; k++) { const int4 x = *reinterpret_cast<const int4 *>(from + (size_t)k * BM_ROWS * BN); n[0] += x.x; n[1] += x.y; n[2] += x.z; n[3] += x.w; }
#pragma unroll
        for (int j = 0; j < 4; j++) t[j] = (float)n[j];
    } else {
        t[0] = t[1] = t[2] = t[3] = 0.f;
#pragma unroll 4
        for (int k = 0; k < splits; k++) { const float4 x = *reinterpret_cast<const float4 *>(from + (size_t)k * BM_ROWS * BN); t[0] += x.x; t[1] += x.y; t[2] += x.z; t[3] += x.w; }
    }
}
// The results from the partial tiles of the launch's split contractions: a thread per four neighbouring results, partial tiles added in order.
template <int KIND, class T, int EPI, int BN> __global__ void __launch_bounds__(256) bm_reduce_kernel(const __grid_constant__ BmParams<T, bm_jobs(EPI)> all)
{
    pdl_wait();
    int job = 0;
#pragma unroll
    for (int k = 1; k < bm_jobs(EPI); k++) if (k < all.jobs && (int)blockIdx.x >= all.job[k].reduce_first) job = k;        // (one that is not split has no blocks: the next one starts there too)
    const BmJob<T> &p = all.job[job];
    constexpr int BNC = EPI == FFN_GATE ? BN / 2 : BN, QUADS = BNC / 4, PER = BM_ROWS * QUADS;       // (PER is a multiple of 256: a block stays inside one tile)
    const int block = (int)blockIdx.x - p.reduce_first, tile = block / (PER / 256), e = (block % (PER / 256) + tile * (PER / 256)) * 256 + threadIdx.x, in = e - tile * PER, r = in / QUADS, c = (in - r * QUADS) * 4;
    int rb, cb;
    bm_locate(p, tile, rb, cb);
    const int row = rb * BM_ROWS + r, col = cb * BNC + c;
    if (row >= p.N || col >= p.M) return;
    const uint32_t *src = p.part + ((size_t)tile * p.splits * BM_ROWS + r) * BN + c;
    float v[4], w[4];
    bm_add_parts<KIND, BN>(src, p.splits, v);
    if constexpr (EPI == FFN_GATE) bm_add_parts<KIND, BN>(src + BNC, p.splits, w);
    bm_results<T, EPI>(p, row, col, v, w);
}

// ---------------------------------------------------------------- launch
static bool bm_map(CUtensorMap *m, CUtensorMapDataType type, int esize, const void *base, int inner, int outer, int parts, long long os, long long ps, int box_inner, int box_outer)
{
    EncodeTiledFn enc = (EncodeTiledFn)tc_encode_tiled_fn();
    cuuint64_t gdim[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)parts};
    cuuint64_t gstr[2] = {(cuuint64_t)(os * esize), (cuuint64_t)((parts > 1 ? ps : (long long)outer * os) * esize)};
    cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1u}, estr[3] = {1, 1, 1};
    return enc && enc(m, type, 3, (void *)base, gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tile and CTAs per tile with the fewest cycles by a model: a K step costs its tensor time or what its bytes take into an SM (58 per cycle with several tiles for
// every SM, 100 with one at most: its shared memory feeds the tensor cores no faster), a pair's a third more than its tensor time; a tile 1000 cycles beside its K
// steps, a launch 2000 (pairs 8000), partial tiles 2000 and their bytes.  On 38 products of 64 to 4096 rows, timed with every tile and up to 16 parts, what it takes is 0.8% slower than the fastest on average.
struct BmPlan { int BN, pair; };
// Several products in one launch: the sum of their units' cycles over the CTAs and the longest unit, for which a product's K is split while CTAs are idle.
template <class T, int JOBS> static BmPlan bm_plan(int kind, int epi, BmParams<T, JOBS> &p)
{
    BmPlan plan = {64, 0};
    double best = 1e30;
    const int bns[4] = {256, 128, 64, 256};
    for (int i = kind == MM_TF32 ? 1 : 0; i < (kind == MM_TF32 ? 3 : 4); i++) {
        const bool two = i == 3;
        const int bn = bns[i], bnc = epi == FFN_GATE ? bn / 2 : bn, places = two ? sm_count() / 2 : sm_count();
        int splits[JOBS] = {}, tiles[JOBS] = {}, units = 0;
        for (int k = 0; k < p.jobs; k++) { splits[k] = 1; units += tiles[k] = ceil_div(p.job[k].N, two ? 256 : 128) * ceil_div(p.job[k].M, bnc); }
        const double tensor = (kind == MM_TF32 ? 6.0 : 2.0) * bn * (two ? 4.0 / 3.0 : 1.0);
        for (;;) {
            const double fill = (kind == MM_TF32 ? 2 : 1) * 128.0 * (128 + (two ? bn / 2 : bn)) / (units <= places ? 100.0 : 58.0), step = std::max(tensor, fill);
            double sum = 0, longest = 0, reduce = 0;
            int at = 0;
            for (int k = 0; k < p.jobs; k++) {
                const double unit = step * ceil_div(p.job[k].ksteps, splits[k]) + 1000.0;
                sum += unit * tiles[k] * splits[k];
                if (unit > longest) { longest = unit; at = k; }
                if (splits[k] > 1) reduce += 2000.0 + 512.0 * bn * tiles[k] * splits[k] / 2000.0;
            }
            const double work = p.jobs == 1 ? ceil_div(units, places) * longest : std::max(sum / places + 0.3 * longest, longest);
            const double cost = (two ? 8000.0 : 2000.0) + work + reduce;
            if (cost < 0.97 * best) { best = cost; plan = {bn, two ? 1 : 0}; for (int k = 0; k < p.jobs; k++) p.job[k].splits = splits[k]; }
            // alone, a product's parts have to fit the CTAs once; among others, parts shorten the unit that the launch would wait for
            const bool more = p.jobs == 1 ? units + tiles[at] <= places : longest > 0.5 * sum / places && (long long)tiles[at] * (splits[at] + 1) * BM_ROWS * bn <= (16ll << 20);
            if (two || splits[at] >= 32 || !more || p.job[at].ksteps < 2 * (splits[at] + 1)) break;
            splits[at]++;
            units += tiles[at];
        }
    }
    return plan;
}

template <int KIND, class T, int EPI, int BN, bool PAIR> static void bm_launch(const BmMapList<bm_jobs(EPI)> &maps, const BmParams<T, bm_jobs(EPI)> &p)
{
    const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
    static bool attr_set = false;
    if (!attr_set) {
        cudaFuncSetAttribute(block_mm_kernel<KIND, T, EPI, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(BM_RING + 1024));
        attr_set = true;
    }
    if constexpr (PAIR) TL_LAUNCH_CLUSTER((block_mm_kernel<KIND, T, EPI, BN, PAIR>), (unsigned)(2 * std::min(p.units, sm_count() / 2)), BM_THREADS, smem, 2, maps, p);
    else {
        TL_LAUNCH((block_mm_kernel<KIND, T, EPI, BN, PAIR>), (unsigned)std::min(p.units, sm_count()), BM_THREADS, smem, maps, p);
        if (p.reduce_blocks) TL_LAUNCH((bm_reduce_kernel<KIND, T, EPI, BN>), (unsigned)p.reduce_blocks, 256, 0, p);
    }
}
template <int KIND, class T, int EPI> static void bm_dispatch(const BmPlan &plan, const BmMapList<bm_jobs(EPI)> &maps, const BmParams<T, bm_jobs(EPI)> &p)
{
    if constexpr (KIND != MM_TF32) {
        if (plan.pair) return bm_launch<KIND, T, EPI, 256, true>(maps, p);
        if (plan.BN == 256) return bm_launch<KIND, T, EPI, 256, false>(maps, p);
    }
    if (plan.BN == 128) bm_launch<KIND, T, EPI, 128, false>(maps, p);
    else bm_launch<KIND, T, EPI, 64, false>(maps, p);
}
// what does not depend on the operands' layout; false: no memory for the partial tiles
template <int KIND, class T, int EPI> static bool bm_setup(Scope &sc, const BmPlan &plan, BmParams<T, bm_jobs(EPI)> &p)
{
    const int bnc = EPI == FFN_GATE ? plan.BN / 2 : plan.BN;
    p.status = tc_status_word();
    p.stage_bytes = BmCfg<KIND>::PARTS * (BM_ROWS * 128u + (uint32_t)(plan.pair ? plan.BN / 2 : plan.BN) * 128u);
    p.stages = std::min<int>(BM_MAX_STAGES, BM_RING / p.stage_bytes);
    p.units = p.reduce_blocks = 0;
    for (int k = 0; k < p.jobs; k++) {
        BmJob<T> &j = p.job[k];
        j.reduce_first = p.reduce_blocks;
        j.tiles_m = ceil_div(j.M, bnc); j.tiles_n = ceil_div(j.N, plan.pair ? 2 * BM_ROWS : BM_ROWS);
        j.first = p.units;
        p.units += j.tiles_m * j.tiles_n * j.splits;
        if (j.splits > 1) p.reduce_blocks += j.tiles_m * j.tiles_n * (BM_ROWS * bnc / 4 / 256);
        if (j.splits > 1 && !(j.part = sc.scratch<uint32_t>((size_t)j.tiles_m * j.tiles_n * j.splits * BM_ROWS * plan.BN))) return false;
    }
    return true;
}

template <class T> static int bm_align(int ld, const void *a, const void *b, const void *c)
{
    const uintptr_t at = (uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)((size_t)ld * sizeof(T));
    return at % 16 == 0 ? ALIGN_16 : at % 4 == 0 ? ALIGN_WORD : ALIGN_ELEMENT;
}
static bool bm_ready()
{
    if (!tc_encode_tiled_fn()) set_error(TL_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    else if (!tc_status_word()) set_error(TL_ERR_NO_MEMORY, "no memory for the word in which a kernel's waits report");
    else return true;
    return false;
}
static bool bm_no_map()
{
    set_error(TL_ERR_CUDA, "cuTensorMapEncodeTiled refused an operand");
    return false;
}
// copies of up to twelve operands in one launch
template <class T> struct BmPacks { PackOp<T> op[12]; int count, blocks; };
template <class T> __global__ void __launch_bounds__(256) bm_pack_kernel(const __grid_constant__ BmPacks<T> ops)
{
    pdl_wait();
    int k = 0;
    while (k + 1 < ops.count && (int)blockIdx.x >= ops.op[k + 1].first) k++;
    pack_kmajor_block<T>(ops.op[k]);
}
template <class T, int EPI> bool block_mm(Scope &sc, const FfnProduct<T> *list, int count)
{
    constexpr int KIND = sizeof(T) == 2 ? MM_F16 : MM_TF32, BK = BmCfg<KIND>::BK, JOBS = bm_jobs(EPI);
    constexpr long long EB = 16 / (long long)sizeof(T);
    if (!bm_ready()) return false;
    // what takes longest goes first
    const FfnProduct<T> *order[JOBS] = {};
    for (int k = 0; k < count; k++) order[k] = list + k;
    auto length = [](const FfnProduct<T> *f) { return (long long)f->K * f->terms; };
    for (int k = 1; k < count; k++)
        for (int i = k; i > 0 && length(order[i]) > length(order[i - 1]); i--) std::swap(order[i], order[i - 1]);
    struct Op { const T *at; long long os, ps; int mn; };
    struct Done { const T *src; long long rs, cs; int rows, K; Op op; } done[12];
    BmPacks<T> pack;
    pack.count = pack.blocks = 0;
    // one layout for all operands of a side: they share strides, and all are read in place or none.  An operand of two products is copied once.
    auto side = [&](const T *const *src, int n, long long rs, long long cs, int rows, int K, Op *o) -> bool {
        const int Kp = (int)(((long long)K + 8 * EB - 1) / (8 * EB) * (8 * EB));           // (whole lines: a box's 128 bytes over two of them are fetched as two)
        int where = tm_in_place<T>(src[0], rs, cs, 0, rows, K, 1);
        if (n > 1 && tm_in_place<T>(src[1], rs, cs, 0, rows, K, 1) != where) where = 0;
        for (int i = 0; i < n; i++) {
            if (where) { o[i] = {src[i], where == 1 ? rs : cs, 0, where - 1}; continue; }
            int k = 0;
            while (k < pack.count && !(done[k].src == src[i] && done[k].rs == rs && done[k].cs == cs && done[k].rows == rows && done[k].K == K)) k++;
            if (k < pack.count) { o[i] = done[k].op; continue; }
            const size_t size = ((size_t)rows * Kp + 63) & ~(size_t)63;
            T *hi = sc.scratch<T>(BmCfg<KIND>::PARTS * size);
            if (!hi) return false;
            const bool straight = cs == 1;
            PackOp<T> &op = pack.op[pack.count];
            op = {src[i], hi, sizeof(T) == 4 ? hi + size : nullptr, rs, cs, 0, rows, K, Kp, ceil_div(Kp, straight ? 64 : 32), ceil_div(rows, straight ? 32 : 64), pack.blocks, straight,
                  (straight ? rs : rs == 1 ? cs : 1) % EB == 0 && ((uintptr_t)src[i] & 15) == 0};
            pack.blocks += op.nk * op.nr;
            o[i] = {hi, Kp, (long long)size, 0};
            done[pack.count++] = {src[i], rs, cs, rows, K, o[i]};
        }
        return true;
    };
    Op a[JOBS][2], b[JOBS][2];
    BmParams<T, JOBS> p = {};
    p.jobs = count;
    for (int k = 0; k < count; k++) {
        const FfnProduct<T> &f = *order[k];
        BmJob<T> &j = p.job[k];
        if (!side(f.A, f.terms, f.a_rs, f.a_cs, f.N, f.K, a[k]) || !side(f.B, EPI == FFN_GATE ? 2 : f.terms, f.b_cs, f.b_rs, f.M, f.K, b[k])) return false;
        j.C = f.C; j.g = f.g; j.u = f.u; j.dg = f.dg; j.du = f.du; j.N = f.N; j.M = f.M; j.ld = f.ld;
        j.kps = ceil_div(f.K, BK); j.ksteps = j.kps * f.terms;
        j.a_mn = a[k][0].mn; j.b_mn = b[k][0].mn;
        j.c_align = bm_align<T>(f.ld, f.C, f.dg, f.du); j.g_align = bm_align<T>(f.M, f.g, f.u, nullptr);
    }
    const BmPlan plan = bm_plan<T, JOBS>(KIND, EPI, p);
    if (!bm_setup<KIND, T, EPI>(sc, plan, p)) return false;
    const CUtensorMapDataType type = sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    BmMapList<JOBS> maps;
    const int b_rows = EPI == FFN_GATE || plan.pair ? plan.BN / 2 : plan.BN;
    for (int k = 0; k < count; k++) {
        const FfnProduct<T> &f = *order[k];
        auto map_of = [&](CUtensorMap *m, const Op &o, int rows, int box_rows) -> bool {
            return o.mn ? bm_map(m, type, (int)sizeof(T), o.at, rows, f.K, 1, o.os, 0, 64, 64) : bm_map(m, type, (int)sizeof(T), o.at, f.K, rows, BmCfg<KIND>::PARTS, o.os, o.ps, BK, box_rows);
        };
        for (int i = 0; i < f.terms; i++) if (!map_of(&maps.of[k].a[i], a[k][i], f.N, BM_ROWS)) return bm_no_map();
        for (int i = 0; i < (EPI == FFN_GATE ? 2 : f.terms); i++) if (!map_of(&maps.of[k].b[i], b[k][i], f.M, b_rows)) return bm_no_map();
    }
    if (pack.count) TL_LAUNCH((bm_pack_kernel<T>), pack.blocks, 256, 0, pack);
    bm_dispatch<KIND, T, EPI>(plan, maps, p);
    return true;
}
#define INST(T)                                                             \
    template bool block_mm<T, FFN_PLAIN>(Scope &, const FfnProduct<T> *, int);   \
    template bool block_mm<T, FFN_GATE>(Scope &, const FfnProduct<T> *, int);    \
    template bool block_mm<T, FFN_GATE_BW>(Scope &, const FfnProduct<T> *, int);
INST(float)
INST(__half)

// Rows of `size` bytes that do not lie on 16-byte boundaries -> rows of `quads` 16-byte groups (behind the end: never read), of both operands; a thread per group,
// from the five words around its bytes (2338 rows of 7772 bytes and 192: 14.8 us byte by byte).
struct BmRows { const unsigned char *src[2], *end[2]; uint4 *dst[2]; long long groups[2]; };
__global__ void __launch_bounds__(256) pack_rows_int8_kernel(const __grid_constant__ BmRows p, int size, int quads)
{
    pdl_wait();
    long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const int which = e >= p.groups[0];
    if (which) e -= p.groups[0];
    if (e >= p.groups[which]) return;
    const long long r = e / quads;
    const int k = (int)(e - r * quads) * 16;
    if (k >= size) return;
    const unsigned char *s = p.src[which] + (size_t)r * size + k, *begin = p.src[which], *end = p.end[which];
    const int off = (int)((uintptr_t)s & 3);
    uint32_t v[5], w[4];
#pragma unroll
    for (int i = 0; i < 5; i++) {
        const unsigned char *a = s - off + 4 * i;
        v[i] = 0;
        if (a >= begin && a + 4 <= end) v[i] = *reinterpret_cast<const uint32_t *>(a);
        else {
#pragma unroll
            for (int b = 0; b < 4; b++) if (a + b >= begin && a + b < end) v[i] |= (uint32_t)a[b] << (8 * b);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * off);
    p.dst[which][e] = make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T> void linear_int8(Scope &sc, const signed char *x, const float *xs, const signed char *w, const float *ws, const T *bias, T *y, int rows, int in, int out)
{
    if (rows <= FEW_ROWS) return few_rows_int8<T>(sc, x, xs, w, ws, bias, y, rows, in, out);
    if (!bm_ready()) return;
    const int quads = in < 128 ? ceil_div(in, 16) : ceil_div(in, 128) * 8;         // (whole lines, as above, where a row has one)
    const signed char *at[2] = {x, w};
    signed char *copy[2] = {nullptr, nullptr};
    const int count[2] = {rows, out};
    for (int i = 0; i < 2; i++)
        if (in % 16 || ((uintptr_t)at[i] & 15)) {
            if (!(copy[i] = sc.scratch<signed char>((size_t)count[i] * quads * 16))) return;
        }
    BmParams<T, 1> p = {};
    BmJob<T> &j = p.job[0];
    p.jobs = 1;
    j.C = y; j.bias = bias; j.xs = xs; j.ws = ws; j.N = rows; j.M = j.ld = out;
    j.kps = j.ksteps = ceil_div(in, BmCfg<MM_I8>::BK);
    j.c_align = bm_align<T>(out, y, nullptr, nullptr);
    const BmPlan plan = bm_plan<T, 1>(MM_I8, FFN_INT8, p);
    if (!bm_setup<MM_I8, T, FFN_INT8>(sc, plan, p)) return;
    BmMapList<1> maps;
    for (int i = 0; i < 2; i++)
        if (!bm_map(i ? &maps.of[0].b[0] : &maps.of[0].a[0], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, copy[i] ? copy[i] : at[i], in, count[i], 1, copy[i] ? (long long)quads * 16 : in, 0, BmCfg<MM_I8>::BK,
                    i ? (plan.pair ? plan.BN / 2 : plan.BN) : BM_ROWS)) { bm_no_map(); return; }
    if (copy[0] || copy[1]) {
        BmRows q;
        for (int i = 0; i < 2; i++) { q.src[i] = (const unsigned char *)at[i]; q.end[i] = q.src[i] + (size_t)count[i] * in; q.dst[i] = (uint4 *)copy[i]; q.groups[i] = copy[i] ? (long long)count[i] * quads : 0; }
        TL_LAUNCH(pack_rows_int8_kernel, ceil_div(q.groups[0] + q.groups[1], 256), 256, 0, q, in, quads);
    }
    bm_dispatch<MM_I8, T, FFN_INT8>(plan, maps, p);
}
template void linear_int8<float>(Scope &, const signed char *, const float *, const signed char *, const float *, const float *, float *, int, int, int);
template void linear_int8<__half>(Scope &, const signed char *, const float *, const signed char *, const float *, const __half *, __half *, int, int, int);

} // namespace tl
