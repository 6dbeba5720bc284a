// What the TMA-fed tcgen05 products share: loads and MMAs of single CTAs and of pairs, bounded waits, tensor maps, and the packing of operands
// that cannot be read in place.
#pragma once
#include "tl_kernels.h"
#include "tl_tc.cuh"

namespace tl {

using namespace tc;

int *tc_status_word();          // tl_conv_tc.cu
void *tc_encode_tiled_fn();     // tl_conv_tc.cu: cuTensorMapEncodeTiled through the runtime's driver entry point query

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *m, uint64_t *bar, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
// The same for a CTA pair: the barrier (a cluster address) may be the other CTA's.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *m, uint32_t bar, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// One MMA; PAIR: 256 rows, 128 in each CTA of the pair, and half of B's rows from each CTA's shared memory.
template <bool HALF, bool PAIR> __device__ __forceinline__ void tm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    if constexpr (!PAIR) { if constexpr (HALF) mma_f16_ss(d, a, b, idesc, acc); else mma_tf32_ss(d, a, b, idesc, acc); }
    else if constexpr (HALF)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// An arrival on the barrier (PAIR: of both CTAs) when the MMAs issued so far have completed.
template <bool PAIR> __device__ __forceinline__ void tm_commit(uint64_t *bar)
{
    if constexpr (!PAIR) mma_commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ uint32_t tm_mapa(uint32_t addr, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void tm_arrive_at(uint32_t bar)           // a cluster address
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait (about a second): polls back to back, or `nap` ns apart.
__device__ __forceinline__ bool tm_wait(uint64_t *bar, uint32_t parity, volatile int *failed, uint32_t nap = 0)
{
    for (uint32_t i = 0; i < 20000000u; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (nap) __nanosleep(nap);
        if ((i & 63u) == 63u && *failed) return false;
    }
    *failed = 1;
    return false;
}
__device__ __forceinline__ void tm_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// ---------------------------------------------------------------- operand packing
// dst[(b * rows + r) * Kp + k] = src[b*bs + r*rs + k*cs] for k < K (columns K..Kp-1 are never read: the tensor map ends at K).
// fp32: hi part to dst, lo part to lo.  One launch for both operands of a product.  K-contiguous sources go straight through
// registers, 32 rows x 64 k per block and eight k per thread; the others through a shared-memory tile of 32 k x 64 rows, read
// as vectors along the rows where they are contiguous and aligned, written as whole 128-byte rows of 32 k (64 x [64 x 784]
// transposed and split: 15.5 us with scalar reads of 32 rows, 9.2 us so).
template <class T> struct PackOp { const T *src; T *dst, *lo; long long rs, cs, bs; int rows, K, Kp, nk, nr, first, straight, vec; };
template <class T> struct PackOps { PackOp<T> op[2]; int count; };

template <class T> __device__ __forceinline__ void pack_kmajor_block(const PackOp<T> &o)
{
    __shared__ float tile[32][65];
    const int t = (int)blockIdx.x - o.first, tr = t / o.nk, b = tr / o.nr;
    if (!o.straight) {
        const int k0 = (t - tr * o.nk) * 32, r0 = (tr - b * o.nr) * 64, left = o.rows - r0;
        const T *s = o.src + (long long)b * o.bs + (long long)r0 * o.rs;
        if (sizeof(T) == 4 && o.vec) {
            const int rq = (threadIdx.x & 15) * 4, kk = threadIdx.x >> 4;
            float4 v[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const T *p = s + rq + (long long)(k0 + kk + 16 * q) * o.cs;
                v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + kk + 16 * q < o.K) {
                    if (rq + 4 <= left) v[q] = *reinterpret_cast<const float4 *>(p);
                    else { if (rq < left) v[q].x = ld(p); if (rq + 1 < left) v[q].y = ld(p + 1); if (rq + 2 < left) v[q].z = ld(p + 2); }
                }
            }
#pragma unroll
            for (int q = 0; q < 2; q++) { float *d = &tile[kk + 16 * q][rq]; d[0] = v[q].x; d[1] = v[q].y; d[2] = v[q].z; d[3] = v[q].w; }
        } else {
            const int rr = threadIdx.x & 63, kk = threadIdx.x >> 6;
            const T *p = s + (long long)rr * o.rs + (long long)(k0 + kk) * o.cs;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; q++, p += 4 * o.cs) v[q] = ld0(rr < left && k0 + kk + 4 * q < o.K, p);
#pragma unroll
            for (int q = 0; q < 8; q++) tile[kk + 4 * q][rr] = v[q];
        }
        __syncthreads();
        const int kq = (threadIdx.x & 7) * 4;
        if (k0 + kq >= o.Kp) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = (threadIdx.x >> 3) + 32 * h;
            if (row >= left) return;
            const long long at = ((long long)b * o.rows + r0 + row) * o.Kp + k0 + kq;
            if constexpr (sizeof(T) == 4) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int q = 0; q < 4; q++) split_tf32(tile[kq + q][row], hi[q], lo[q]);
                *reinterpret_cast<uint4 *>(o.dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(o.lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            } else {
                const __half2 x = __floats2half2_rn(tile[kq][row], tile[kq + 1][row]), y = __floats2half2_rn(tile[kq + 2][row], tile[kq + 3][row]);
                *reinterpret_cast<uint2 *>(o.dst + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
            }
        }
        return;
    }
    const int k0 = (t - tr * o.nk) * 64, r0 = (tr - b * o.nr) * 32;
    const T *s = o.src + (long long)b * o.bs;
    const int r = threadIdx.x >> 3, kq = (threadIdx.x & 7) * 8;
    float v[8];
    {
        const T *p = s + (long long)(r0 + r) * o.rs + k0 + kq;
        if (o.vec && r0 + r < o.rows && k0 + kq + 8 <= o.K) {
            if constexpr (sizeof(T) == 4) {
                const float4 x = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(p + 4);
                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
            } else {
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = ld(p + q);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = ld0(r0 + r < o.rows && k0 + kq + q < o.K, p + q);
        }
    }
    if (r0 + r >= o.rows || k0 + kq >= o.Kp) return;
    const long long at = ((long long)b * o.rows + r0 + r) * o.Kp + k0 + kq;          // Kp is a multiple of 16 bytes
    if constexpr (sizeof(T) == 4) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int q = 0; q < 8; q++) split_tf32(v[q], hi[q], lo[q]);
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (k0 + kq + 4 * h < o.Kp) {
                *reinterpret_cast<uint4 *>(o.dst + at + 4 * h) = make_uint4(hi[4 * h], hi[4 * h + 1], hi[4 * h + 2], hi[4 * h + 3]);
                *reinterpret_cast<uint4 *>(o.lo + at + 4 * h) = make_uint4(lo[4 * h], lo[4 * h + 1], lo[4 * h + 2], lo[4 * h + 3]);
            }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; q++) { const __half2 h = __floats2half2_rn(v[2 * q], v[2 * q + 1]); w[q] = *reinterpret_cast<const uint32_t *>(&h); }
        *reinterpret_cast<uint4 *>(o.dst + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <class T>
__global__ void __launch_bounds__(256) pack_kmajor_kernel(const __grid_constant__ PackOps<T> ops)
{
    pdl_wait();
    pack_kmajor_block<T>(ops.op[ops.count > 1 && (int)blockIdx.x >= ops.op[1].first ? 1 : 0]);
}

// inner: extent of the contiguous index, outer: of the other one, `os` elements apart
template <class T> static bool make_map(EncodeTiledFn enc, CUtensorMap *m, const T *base, int inner, int outer, int batch, long long os, long long bs, int box_inner, int box_outer)
{
    cuuint64_t gdim[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)batch};
    cuuint64_t gstr[2] = {(cuuint64_t)os * sizeof(T), (cuuint64_t)(batch > 1 ? bs : (long long)outer * os) * sizeof(T)};
    cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1u};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, (void *)base, gdim, gstr, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// fp16 operands stay where they are when one index is contiguous (returns 1: the contracted one, 2: the rows) and the other steps in
// multiples of 16 bytes; 0 = the operand is packed
template <class T> static int tm_in_place(const T *src, long long rs, long long cs, long long bs, int rows, int K, int batch)
{
    constexpr long long EB = 16 / (long long)sizeof(T);
    if (sizeof(T) != 2 || ((uintptr_t)src & 15) || (batch > 1 && bs % EB)) return 0;
    return cs == 1 && rs % EB == 0 && rs >= K ? 1 : rs == 1 && cs % EB == 0 && cs >= rows ? 2 : 0;
}

} // namespace tl
