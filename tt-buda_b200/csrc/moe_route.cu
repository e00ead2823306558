// K10: the router of a mixture of experts for a few tokens, one launch.
//
//   l[t, e] = sum_h x[t, h] w[e, h],  p = softmax(l[t, :]),  the `top` largest l of a token in descending order (of equal
//   ones the lowest index first),  weight = p, or p over the sum of the chosen ones
//
// Bound: for a few tokens the latency of one pass over w (E * H values that every cluster reads once, from L2 after the
// first).  A cluster of 8 CTAs takes a block of tokens; its CTAs share the experts, the warps of a CTA share an expert's
// row when there are fewer experts than warps, so that all of w is asked for at once.  The scores meet in distributed
// shared memory; the warp of token i chooses in CTA i % 8.  Most of a call is waiting for w, so a warp asks for a row's piece in one
// go (8 octets a lane).  w may be what the launch in front has written, as x may: before that one is complete its addresses are
// only named to L2, which brings no value into the kernel.
// Scores decide which experts run: a lane adds 8 products in binary32 (off by at most 7 * 2^-24 of their magnitudes), everything
// behind that is binary64 up to the choice, and the softmax takes binary64 differences.  Sums and choice in binary32 take 0.8 us less
// for the 16 tokens below, but experts closer than 2^-24 of their scores come in the wrong order and the weights are off by
// 1.4e-7 instead of 6e-8.  Keeping what every addition rounds off leaves 5.9e-8 and takes 4 us more.
// Measured (B200): one token, 8 experts of 1024 binary32 weights 3.5 us; 16 tokens, 128 experts of 4096 bfloat16 weights 11.6 us
// (16 clusters read and widen the same 1 MB).
#include <cuda_bf16.h>

#include "few_rows.cuh"

namespace buda {
namespace route {

constexpr int kCluster = 8;
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kPerCta = kMaxExperts / kCluster;

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double ld_cluster_f64(const double *p, uint32_t rank)
{
    uint32_t a;
    double v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
    return v;
}

// Eight consecutive values of a row, fetched (16-byte loads where `vec`, zero past H) and turned into binary32 later, so that
// many rows' loads are under way before the first is used.
template <typename T>
struct Octet;
template <>
struct Octet<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *row, int h, int H, bool vec)
    {
        if (vec && h + 8 <= H) {
            r = *reinterpret_cast<const uint4 *>(row + h);
            return;
        }
        const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = h + i < H ? p[h + i] : 0u;
        r = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};
template <>
struct Octet<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *row, int h, int H, bool vec)
    {
        if (vec && h + 8 <= H) {
            a = *reinterpret_cast<const float4 *>(row + h);
            b = *reinterpret_cast<const float4 *>(row + h + 4);
            return;
        }
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = h + i < H ? row[h + i] : 0.0f;
        a = make_float4(v[0], v[1], v[2], v[3]);
        b = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

// Binary64 in an order that unsigned integers have: NaN below every number, 0 for "already chosen".
__device__ __forceinline__ uint64_t order_of(double l)
{
    if (isnan(l)) return 1u;
    const uint64_t b = (uint64_t)__double_as_longlong(l + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}

constexpr int kStaged = 28 * 1024;       // activations of a block of tokens up to this size are kept in shared memory

template <typename TW, int TB>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 2)
    route_kernel(const __nv_bfloat16 *x, int64_t ldx, int T, int H, const TW *w, int64_t ldw, int E, int top, int renorm, int split,
                 float *weights, int *ids)
{
    __shared__ double part[kPerCta * TB * kWarps];      // [expert of this CTA][token][piece of the row]
    __shared__ double score[kPerCta * TB];
    extern __shared__ __align__(16) __nv_bfloat16 xs[]; // [TB][8 * octets], zero past H
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int t0 = (blockIdx.x / kCluster) * TB, nt = min(T - t0, TB);
    const int mine = E > (int)rank ? (E - (int)rank + kCluster - 1) / kCluster : 0;   // experts rank, rank + 8, ...
    const bool xvec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * 2)) & 15) == 0;
    const bool wvec = ((reinterpret_cast<uintptr_t>(w) | (uintptr_t)(ldw * sizeof(TW))) & 15) == 0;
    const int octets = (H + 7) / 8;
    const bool staged = TB * octets * 16 <= kStaged;

    // A warp's work: batches of kBatch octets (of every lane) of its tasks, a task being a piece of an expert's row.
    constexpr int kBatch = (TB == 1 ? 8 : 4) * 2 / (int)sizeof(TW);
    const int batches = (octets + split * 32 * kBatch - 1) / (split * 32 * kBatch);   // of a piece; the last ones may be empty
    const int tasks = mine * split > warp ? (mine * split - warp + kWarps - 1) / kWarps : 0;
    Octet<TW> a[kBatch];
    int el, piece, o0, o1;
    const TW *row;
    auto place = [&](int it) {
        const int task = warp + it / batches * kWarps;
        el = task / split;
        piece = task % split;
        o0 = (int)((int64_t)octets * piece / split) + it % batches * 32 * kBatch + lane;
        o1 = (int)((int64_t)octets * (piece + 1) / split);
        row = w + (int64_t)(rank + el * kCluster) * ldw;
    };
    auto load = [&](int it) {
        place(it);
#pragma unroll
        for (int u = 0; u < kBatch; u++) a[u].load(row, o0 + 32 * u < o1 ? (o0 + 32 * u) * 8 : H, H, wvec);
    };
    if (tasks) {
        place(0);
#pragma unroll
        for (int u = 0; u < kBatch; u++)
            if (o0 + 32 * u < o1) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + (o0 + 32 * u) * 8));
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");                // the launch in front may write x and w
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tasks) load(0);
    if (staged) {
        for (int i = tid; i < nt * octets; i += kThreads) {
            Octet<__nv_bfloat16> b;
            const int t = i / octets, o = i - t * octets;
            b.load(x + (int64_t)(t0 + t) * ldx, o * 8, H, xvec);
            *reinterpret_cast<uint4 *>(xs + (int64_t)i * 8) = b.r;
        }
        __syncthreads();
    }
    double s[TB];
    for (int it = 0; it < tasks * batches; it++) {
        if (it) load(it);
        if (it % batches == 0)
#pragma unroll
            for (int i = 0; i < TB; i++) s[i] = 0.0;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            if (o0 + 32 * u >= o1) break;
            float av[8];
            a[u].get(av);
#pragma unroll
            for (int i = 0; i < TB; i++) {
                const int t = min(i, nt - 1);
                Octet<__nv_bfloat16> b;
                if (staged) b.r = *reinterpret_cast<const uint4 *>(xs + (t * octets + o0 + 32 * u) * 8);
                else b.load(x + (int64_t)(t0 + t) * ldx, (o0 + 32 * u) * 8, H, xvec);
                float bv[8], p = 0.0f;
                b.get(bv);
#pragma unroll
                for (int v = 0; v < 8; v++) p = fmaf(av[v], bv[v], p);
                s[i] += p;
            }
        }
        if (it % batches == batches - 1) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < TB; i++) {
                double all = s[i];
#pragma unroll
                for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
                if (lane == 0) part[(el * TB + i) * split + piece] = all;
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < mine * TB; i += kThreads) {
        double v = 0.0;
        for (int p = 0; p < split; p++) v += part[i * split + p];
        score[i] = v;
    }
    cluster_sync();
    // warp `warp` of CTA `rank` chooses for token 8 * warp + rank of the block
    const int i = warp * kCluster + (int)rank;
    if (i < nt) {
        constexpr int kPer = kMaxExperts / 32;
        const int per = (E + 31) / 32;
        double l[kPer];
        uint64_t key[kPer];
#pragma unroll
        for (int q = 0; q < kPer; q++) {
            l[q] = 0.0;
            key[q] = 0u;
            if (q < per) {
                const int e = q * 32 + lane;
                if (e < E) {
                    l[q] = ld_cluster_f64(&score[(e / kCluster) * TB + i], e % kCluster);
                    key[q] = order_of(l[q]);
                }
            }
        }
        int my_id = 0;              // lane s keeps the s-th choice
        double my_l = 0.0, most = 0.0;
        for (int s = 0; s < top; s++) {
            uint64_t best = 0;
            int at = 0;
            double bl = 0.0;
#pragma unroll
            for (int q = 0; q < kPer; q++)
                if (q < per && key[q] > best) {
                    best = key[q];
                    at = q * 32 + lane;
                    bl = l[q];
                }
            const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
            const uint32_t among = __ballot_sync(0xffffffffu, (uint32_t)(best >> 32) == high);
            int id;
            if (__popc(among) == 1) {
                id = __shfl_sync(0xffffffffu, at, __ffs(among) - 1);
            } else {            // the same in the upper 32 bits
                const uint32_t low = __reduce_max_sync(0xffffffffu, among >> lane & 1 ? (uint32_t)best : 0u);
                id = (int)__reduce_min_sync(0xffffffffu, (among >> lane & 1) && (uint32_t)best == low ? (uint32_t)at : 0xffffffffu);
            }
            const double v = __shfl_sync(0xffffffffu, bl, id & 31);
#pragma unroll
            for (int q = 0; q < kPer; q++)
                if (q * 32 + lane == id) key[q] = 0;
            if (s == 0) most = v;
            if (lane == s) {
                my_id = id;
                my_l = v;
            }
        }
        float sum = 0.0f;
        if (renorm) {
            sum = lane < top ? expf((float)(my_l - most)) : 0.0f;
        } else {
#pragma unroll
            for (int q = 0; q < kPer; q++)
                if (q * 32 + lane < E) sum += expf((float)(l[q] - most));
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane < top) {
            const int64_t o = (int64_t)(t0 + i) * top + lane;
            ids[o] = my_id;
            weights[o] = expf((float)(my_l - most)) / sum;
        }
    }
    cluster_sync();      // no CTA leaves while another reads its scores
}

template <typename TW>
cudaError_t launch_tw(const void *x, int64_t ldx, int T, int H, const void *w, int64_t ldw, int E, int top, int renorm, float *weights,
                      int *ids, int sm_count, cudaStream_t stream)
{
    // enough tokens to a cluster that all clusters are resident at once
    const int clusters = sm_count / kCluster > 0 ? sm_count / kCluster : 1;
    const int tb = T <= clusters ? 1 : T <= 2 * clusters ? 2 : 4;
    const int most = (E + kCluster - 1) / kCluster;
    int split = 1;                                  // pieces of a row: as many warps as there are, but 32 octets for each
    while (split * 2 * most <= kWarps && H >= split * 2 * 256) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((T + tb - 1) / tb * kCluster));
    cfg.blockDim = dim3(kThreads);
    const int64_t x_bytes = (int64_t)tb * ((H + 7) / 8) * 16;
    cfg.dynamicSmemBytes = x_bytes <= kStaged ? x_bytes : 0;
    cfg.stream = stream;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;     // begins while the launch in front of it ends, if that one lets it
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    auto kernel = tb == 1 ? route_kernel<TW, 1> : tb == 2 ? route_kernel<TW, 2> : route_kernel<TW, 4>;
    return cudaLaunchKernelEx(&cfg, kernel, (const __nv_bfloat16 *)x, ldx, T, H, (const TW *)w, ldw, E, top, renorm, split, weights, ids);
}

}  // namespace route

cudaError_t launch_moe_route(const void *x, int64_t ldx, int T, int H, const void *w, int w_f32, int64_t ldw, int E, int top, int renorm,
                             float *weights, int *ids, int sm_count, cudaStream_t stream)
{
    return w_f32 ? route::launch_tw<float>(x, ldx, T, H, w, ldw, E, top, renorm, weights, ids, sm_count, stream)
                 : route::launch_tw<__nv_bfloat16>(x, ldx, T, H, w, ldw, E, top, renorm, weights, ids, sm_count, stream);
}

}  // namespace buda
