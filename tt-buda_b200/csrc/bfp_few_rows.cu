// K9: products of a few rows (tokens) with block-float weights, for serving.
//
//   matvec      Y[m, n]  = sum_k A[m, k] W[k, n]
//   experts     h[s, i]  = w_s act((x_t G_e)[i]) (x_t U_e)[i]            ("in")
//               y[t, n]  = sum over the slots s of token t of sum_i h[s, i] D_e[i, n]
// The second product of the experts has two forms.  Up to 3 tokens ("out"): a column group runs through all reached experts
// as if their rows were one long sum, with zeros where a token has not chosen an expert; nothing is left to add up.  More
// tokens ("each"): every expert's products on their own with only its own tokens, into binary32 rows of the workspace that a third
// launch adds up -- otherwise most columns of the tensor product would be zeros (16 experts, 32 tokens, two each: 4 of 32).
//
// W, G, U, D are queue images in the default byte layout: tile records of 64 shared exponents and four 16x16 faces, a
// stored datum of m magnitude bits standing for (-1)^s q 2^(E - 126 - m).
//
// Bound: bytes of the images (1.0625 / 0.5625 / 0.3125 a weight) -- every weight meets only a few rows.  What decides is
// how few instructions a weight costs on its way and how much of the images is on its way at once:
//   * A warp owns 128 output columns (4 tile columns) and walks tile rows.  Each lane loads its own pieces of the records
//     straight into registers, one tile row ahead: four whole rows (4t .. 4t+3) of a face, the four exponents beside them and
//     the four activations they meet, each consecutive bytes; the four lanes of a face read its 128 bytes (Bfp4) in one
//     access.  With 16 warps an SM that is 37 KB under way.  (The same through bulk copies into a ring of shared memory took
//     half as many instructions again: barrier, copy issue, second load; 11.0 us against 9.8 for 1x4096x16384 Bfp4_b.)
//   * Decode: a datum's sign and magnitude bits are moved to bit 15 and to the top of the 7 mantissa bits of a
//     bfloat16, which makes the subnormal number (-1)^s q 2^(-126 - m); a packed multiply by 2^E finishes it, exactly.
//     One byte permute puts the same byte of two weight rows into both halves of a register in both places, so a pair
//     costs one AND (plus a shift for all but one datum of a byte) and the multiply.
//   * The products go through mma.sync m16n8k16 with the WEIGHTS as the 16-row operand and the tokens as the 8 columns:
//     a lane's fragment is two weight columns at four weight rows (which four of the sum's rows a lane takes is free, as long as
//     the activations follow), so decoded weights never leave the registers.  (tcgen05 reads its operands from shared or
//     tensor memory: the decoded weights would be written and read once more there for a product whose tensor work is small.)
//   * The tile rows are split over the warps of a CTA and, where there are few columns, over a cluster of up to 8 CTAs;
//     sums are joined through shared and distributed shared memory in a fixed order: no workspace, no atomics, the same bits
//     every time.
// Measured (B200, images in turn that exceed L2 four times): 1x4096x16384 Bfp4_b 9.0 us, 4.2 TB/s of its 37.8 MB, integer pipe 50 %
// active; 32x4096x16384 Bfp8_b 24.7 us, 2.9 TB/s; the products of 16 tokens' 4 of 32 experts, 4096 x 2048 gated Bfp4_b, 123 us,
// 3.3 TB/s.
// Sums are held in binary32 throughout, and so is h between the two launches: a lane cuts the values it loads into three bfloat16
// pieces (8 bits of the significand each, exactly all 24), for three times the tensor work of the second product and a fifth more
// instructions (the layer of those 32 experts takes 128 us; with two pieces, within 2^-16 of h, it took 119).
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "few_rows.cuh"

namespace buda {
namespace few {

constexpr int kUnitWarps = 8;           // a CTA has once or twice as many warps
constexpr int kGroupTiles = 4;          // tile columns of one warp
constexpr int kPitch = 132;             // floats per token of a warp's sums: 8-byte stores of 4 x 4 lanes meet no bank twice
constexpr int kDown = 24;               // single-token sums are held times 2^-24 (see single_step)

enum { kMatvec = 0, kExpertsIn = 1, kExpertsOut = 2, kExpertsEach = 3 };
enum { kUsual = 0, kPlain = 1, kWide = 2 };   // forms of a sweep (see products)
__host__ __device__ constexpr bool from_h(int mode) { return mode == kExpertsOut || mode == kExpertsEach; }

// How many units of 8 warps an SM holds, by registers: 128 a thread for up to 16 tokens in a pass.  Of 9 to 16 tokens that is too few
// (Bfp8_b spills 256 bytes a thread in the product, 372 and 672 in the experts' launches), and twice the warps are the faster all the same (12x4096x16384 Bfp8_b 19.2 us against 20.7; 64 tokens, 4 of 32 experts of
// 1024 x 2048 Bfp4_b 68-74 against 86-90).
__host__ __device__ constexpr int units_per_sm(int nt) { return nt <= 2 ? 2 : 1; }

template <int MB>
struct Fmt {
    static constexpr int kRow = 2 * (MB + 1);               // bytes of one face row
    static constexpr int kFace = 16 * kRow;
    static constexpr int kRec = 64 + 4 * kFace;
};

struct Args {
    const __nv_bfloat16 *x;      // [rows, K], row stride ldx (matvec, experts-in; the others read h)
    int64_t ldx;
    int rows, K, Kt, N, Nt;
    const uint8_t *w0, *w1;      // w1: the up matrix of gated experts
    void *out;
    int64_t ldo;
    int out_f32;
    const int *ids;
    const float *wts;
    int top, E, act;
    float *h;                    // [rows * top][32 * tile rows of the down matrix]
    int hpad;
    float *partial;              // experts-each: [rows * top][32 * tile columns of the down matrix]
    uint32_t m4, m16, m64;       // 4, 16, 64: multiplying by a parameter keeps a shift off the integer pipe (see pair_of)
    int cluster;
};

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// The raw data of one lane for one 16-row step: four face rows, as pairs p = 0 and 1, and their exponents.
template <int MB>
struct Raw {
    uint32_t w[2][2][(MB + 1) / 2];   // [p][row][32-bit word]
    uint32_t e;
};

// 32 bytes that nothing reads again: a whole sector for every lane
struct Words8 {
    uint32_t v[8];
};
__device__ __forceinline__ Words8 load_sector(const uint8_t *p)
{
    Words8 r;
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7])
                 : "l"(p));
    return r;
}

// A lane's four rows, at `data`
template <int MB>
__device__ __forceinline__ void load_rows(Raw<MB> &r, const uint8_t *data)
{
    if constexpr (MB == 7) {
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const Words8 a = load_sector(data + p * 32);
#pragma unroll
            for (int i = 0; i < 8; i++) r.w[p][i >> 2][i & 3] = a.v[i];
        }
    } else if constexpr (MB == 3) {
        const Words8 a = load_sector(data);
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i >> 2][(i >> 1) & 1][i & 1] = a.v[i];
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(data));
        r.w[0][0][0] = a.x; r.w[0][1][0] = a.y;
        r.w[1][0][0] = a.z; r.w[1][1][0] = a.w;
    }
}

// Weight columns 2j and 2j+1 of the pair of rows p as subnormal bfloat16 pairs (low half: the even row).  The integer pipe, which
// permutes and masks, is what these kernels run into; the shifts go to the multiply-add pipe, as products with 4, 16 and 64 that the
// compiler does not know.
template <int MB>
__device__ __forceinline__ void pair_of(const Raw<MB> &r, int p, int j, const Args &A, uint32_t &even, uint32_t &odd)
{
    constexpr uint32_t keep = 0x80008000u | (((0x7fu << (7 - MB)) & 0x7fu) * 0x00010001u);
    if constexpr (MB == 7) {
        const int w = j >> 1, b = (j & 1) * 2;
        even = __byte_perm(r.w[p][0][w], r.w[p][1][w], 0x4400u + 0x1111u * b) & keep;
        odd = __byte_perm(r.w[p][0][w], r.w[p][1][w], 0x4400u + 0x1111u * (b + 1)) & keep;
    } else if constexpr (MB == 3) {
        const uint32_t d = __byte_perm(r.w[p][0][j >> 2], r.w[p][1][j >> 2], 0x4400u + 0x1111u * (j & 3));
        even = (d * A.m16) & keep;
        odd = d & keep;
    } else {
        const uint32_t d = __byte_perm(r.w[p][0][0], r.w[p][1][0], 0x4400u + 0x1111u * (j >> 1));
        even = (j & 1) ? (d * A.m4) & keep : (d * A.m64) & keep;
        odd = (j & 1) ? d & keep : (d * A.m16) & keep;
    }
}

// 2^a and 2^b (-127 < a, b <= 127) as a bfloat16 pair
__device__ __forceinline__ uint32_t pow2_pair(int a, int b) { return ((uint32_t)(a + 127) << 7) | ((uint32_t)(b + 127) << 23); }

// the shared exponents of row pair p, moved by `by`, as a pair of powers of two (0 < exponent + by + 127 < 255)
__device__ __forceinline__ uint32_t scale_pair(uint32_t e, int p, int by)
{
    return (__byte_perm(e, 0u, p ? 0x4342u : 0x4140u) + (uint32_t)(by + 127) * 0x00010001u) << 7;
}

// A pair of weights for the pieces of h behind the first: 0 in the place of an infinity.  The first piece alone meets it, for the
// sum of the pieces times an infinity is what the first one gives, and another one of zero would make it a NaN.
__device__ __forceinline__ uint32_t finite_pair(uint32_t v)
{
    return v & ~__vcmpeq2(v & 0x7fff7fffu, 0x7f807f80u);
}

// One 16-row step for up to 8 * NT tokens: the weights are scaled.  BIG where a shared exponent is above 127 (2^E is no
// bfloat16 then: up to three factors).
template <int MB, int NT, int PIECES, bool BIG>
__device__ __forceinline__ void step(float (&acc)[8][NT][4], const Raw<MB> &raw, const Args &A, const uint2 (&x)[PIECES][NT])
{
    uint32_t s[2], s2[2], s3[2];
#pragma unroll
    for (int p = 0; p < 2; p++) {
        if constexpr (BIG) {
            const int a = (raw.e >> (16 * p)) & 0xff, b = (raw.e >> (16 * p + 8)) & 0xff;
            s[p] = pow2_pair(min(a, 127), min(b, 127));
            s2[p] = pow2_pair(min(max(a - 127, 0), 127), min(max(b - 127, 0), 127));
            s3[p] = pow2_pair(max(a - 254, 0), max(b - 254, 0));
        } else {
            s[p] = scale_pair(raw.e, p, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        uint32_t a[4];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            pair_of<MB>(raw, p, j, A, a[2 * p], a[2 * p + 1]);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t v = mul_bf16x2(a[2 * p + c], s[p]);
                if constexpr (BIG) v = mul_bf16x2(mul_bf16x2(v, s2[p]), s3[p]);
                a[2 * p + c] = v;
            }
        }
#pragma unroll
        for (int q = 0; q < PIECES; q++) {
            if (BIG && q == 1)         // and for those behind
#pragma unroll
                for (int c = 0; c < 4; c++) a[c] = finite_pair(a[c]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma16816(acc[j][nt], a, x[q][nt].x, x[q][nt].y);
        }
    }
}

// The same for ONE token: the 8 columns of the product are free, so column g carries the token's values scaled by the
// shared exponents of lane group g's own face, and the weights stay the unscaled subnormals -- 2 multiplies instead of 32.
// Only the diagonal (row group g, column g) counts.  The columns are held times 2^-24, which keeps x 2^E inside bfloat16
// up to |x| max|w| = 2^24 (a product below 2^-102 is then rounded at 2^-125).
template <int MB, int PIECES>
__device__ __forceinline__ void single_step(float (&acc)[8][1][4], const Raw<MB> &raw, const Args &A, const uint32_t (&b)[PIECES][2])
{
#pragma unroll
    for (int j = 0; j < 8; j++) {
        uint32_t a[4];
        pair_of<MB>(raw, 0, j, A, a[0], a[1]);
        pair_of<MB>(raw, 1, j, A, a[2], a[3]);
#pragma unroll
        for (int q = 0; q < PIECES; q++) mma16816(acc[j][0], a, b[q][0], b[q][1]);
    }
}

// One token where some x 2^(E - 24) is no finite bfloat16: what is too much for the column goes to the weights.  Of E = 255 all of it
// does: such a weight is taken to its own size first, where 2^128 and above becomes an infinity, and the 2^-24 comes behind that
// (the activations would lose their last bits to it below 2^-102, and such a product may still be as large as 2^26).
template <int MB, int PIECES>
__device__ __forceinline__ void single_step_wide(float (&acc)[8][1][4], const Raw<MB> &raw, const Args &A, const uint2 (&x)[PIECES][1])
{
#pragma unroll
    for (int q = 0; q < PIECES; q++) {
        uint32_t b[2], s1[2], s2[2], s3[2], s4[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            int d[2], v[2], last[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int E = (raw.e >> (16 * p + 8 * h)) & 0xff, ex = ((p ? x[q][0].y : x[q][0].x) >> (7 + 16 * h)) & 0xff;
                d[h] = E == 255 ? 255 : max(ex + E - kDown - 254, 0);
                v[h] = E == 255 ? 0 : E - kDown - d[h];
                last[h] = E == 255 ? -kDown : 0;
            }
            b[p] = mul_bf16x2(mul_bf16x2(p ? x[q][0].y : x[q][0].x, pow2_pair(min(v[0], 127), min(v[1], 127))), pow2_pair(max(v[0] - 127, 0), max(v[1] - 127, 0)));
            s1[p] = pow2_pair(min(d[0], 127), min(d[1], 127));
            s2[p] = pow2_pair(min(max(d[0] - 127, 0), 127), min(max(d[1] - 127, 0), 127));
            s3[p] = pow2_pair(max(d[0] - 254, 0), max(d[1] - 254, 0));
            s4[p] = pow2_pair(last[0], last[1]);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t a[4];
            pair_of<MB>(raw, 0, j, A, a[0], a[1]);
            pair_of<MB>(raw, 1, j, A, a[2], a[3]);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                a[c] = mul_bf16x2(mul_bf16x2(mul_bf16x2(mul_bf16x2(a[c], s1[c >> 1]), s2[c >> 1]), s3[c >> 1]), s4[c >> 1]);
                if (q > 0) a[c] = finite_pair(a[c]);
            }
            mma16816(acc[j][0], a, b[0], b[1]);
        }
    }
}

// Activations as the tensor operand takes them: pairs of bfloat16, of a binary32 value (h) in three pieces that add up to it.  Each
// piece is the upper half of what is left, so the sign stays and nothing overflows.  What is not finite leaves a rest that is no
// number, which shows in the sums; the wide form (EXACT) then takes the rest as zero.
template <bool EXACT, int PIECES, int NT, int WORDS>
__device__ __forceinline__ void pieces_of(uint2 (&b)[PIECES][NT], const uint32_t (&x)[NT][WORDS])
{
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        if constexpr (WORDS == 2) {
            b[0][nt] = make_uint2(x[nt][0], x[nt][1]);
        } else {
            uint32_t v[4] = {x[nt][0], x[nt][1], x[nt][2], x[nt][3]};
#pragma unroll
            for (int q = 0; q < PIECES; q++) {
                b[q][nt] = make_uint2(__byte_perm(v[0], v[1], 0x7632u), __byte_perm(v[2], v[3], 0x7632u));
                if (q + 1 < PIECES)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float rest = __uint_as_float(v[i]) - __uint_as_float(v[i] & 0xffff0000u);
                        v[i] = EXACT && !isfinite(rest) ? 0u : __float_as_uint(rest);
                    }
            }
        }
    }
}

// Elements k .. k+3 of a row (k a multiple of 4), zero past K; `pairs`: 4-byte loads are allowed.
__device__ __forceinline__ uint2 load_four(const __nv_bfloat16 *row, int k, int K, bool pairs)
{
    if (pairs && k + 4 <= K) {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(row + k);
        return make_uint2(p[0], p[1]);
    }
    const uint16_t *p = reinterpret_cast<const uint16_t *>(row) + k;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = k + i < K ? p[i] : 0u;
    return make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
}

__device__ __forceinline__ float activate(float v, int act)
{
    if (act == BUDA_ACT_SILU) return v / (1.0f + expf(-v));
    return 0.5f * v * erfcf(v * -0.70710678118654752f);      // 1 + erf(z) = erfc(-z), which keeps its digits where erf is near -1
}

// Shared memory: [the warps' sums][the CTA's sums][tables]
template <int MB, int NT>
struct Lay {
    static constexpr int kTok = NT ? 8 * NT : 1;
    static constexpr int kSums = kTok * kPitch * 4;                       // of one warp
    // behind the warps' sums:
    static constexpr int kPart = 0;                                       // [kTok][128] floats
    static constexpr int kMap = kPart + kTok * 128 * 4;                   // 8 words: bit e set where expert e has a token
    static constexpr int kCount = kMap + kMaxExperts / 8;
    static constexpr int kList = kCount + 16;                             // in, each: (slot, weight) of the expert's tokens; out: experts
    static constexpr int kRows = kList + 4 * kMaxExperts;                 // out: the slot of (expert, token)
    __host__ __device__ static constexpr int ids(int mode) { return mode == kExpertsOut ? kRows + 2 * kMaxExperts * kTok : kRows; }
    static constexpr int bytes(int mode, int warps)
    {
        return warps * kSums + (mode == kMatvec ? kMap : ids(mode) + (NT ? 4 * kMaxFewRows * kMaxTop : 0));
    }
};

// What a CTA works on: `units` tile rows, in the out form of (expert, tile row) pairs.
struct Work {
    int n_tok, tok0;             // tokens of this pass; the first one
    bool begin;                  // the first pass of this CTA
    int units;
    int64_t w_off;               // experts-in: where this expert's images begin
    const int *list;
    const int16_t *rows;
};

// The sums of this warp's share of the tile rows, left in sums[warp][token][j][g][2].  SINGLE: one token (NT = 1 then).
template <int MB, int NT, int MODE, bool SINGLE>
__device__ __forceinline__ void products(const Args &A, const Work &W, uint8_t *smem, int group, int me, int workers, int tok_pitch)
{
    using F = Fmt<MB>;
    constexpr int PIECES = from_h(MODE) ? 3 : 1, WORDS = from_h(MODE) ? 4 : 2;      // of four activations: in products, as loaded
    using X = std::conditional_t<from_h(MODE), float, __nv_bfloat16>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t image = (int64_t)A.Kt * A.Nt * F::kRec, row_bytes = (int64_t)A.Nt * F::kRec;
    const uint32_t each = (uint32_t)W.units / (uint32_t)workers, extra = (uint32_t)W.units - each * workers;
    const int u0 = (int)(me * each + min((uint32_t)me, extra)), n = (int)(each + ((uint32_t)me < extra));
    const int s0 = MODE == kExpertsOut ? (int)((uint32_t)u0 / (uint32_t)A.Kt) : 0, kt0 = u0 - s0 * A.Kt;

    // Lane group g reads face column (g >> 1) & 1 of tile (g & 1) + 2 * (g >> 2) of the column group; of gated experts the
    // last two tiles are the up matrix's.  Tiles past the last column are read as the first one and dropped.
    const bool gated = MODE == kExpertsIn && A.w1 != nullptr;
    const int span = gated ? kGroupTiles / 2 : kGroupTiles;
    int tile = (g & 1) | ((g >> 2) << 1);
    const uint8_t *matrix = A.w0;
    if (gated && tile >= span) {
        tile -= span;
        matrix = A.w1;
    }
    const int col = group * span + tile, fc = (g >> 1) & 1;
    matrix += (int64_t)(col < A.Nt ? col : group * span) * F::kRec;

    const bool vec = from_h(MODE) || ((reinterpret_cast<uintptr_t>(A.x) | (A.rows > 1 ? (uintptr_t)(A.ldx * 2) : 0)) & 7) == 0;
    const bool pairs = ((reinterpret_cast<uintptr_t>(A.x) | (A.rows > 1 ? (uintptr_t)(A.ldx * 2) : 0)) & 3) == 0;
    const int whole = from_h(MODE) ? A.Kt : vec ? A.K / 32 : 0;    // tile rows whose activations are loaded four at a time

    // What a lane loads ahead: its rows of one face or of the upper and the lower one, and token g's activations beside them.
    // Lanes past the last token read the first one's row: their columns of the product are dropped.
    constexpr int HALVES = MB == 7 || NT == 2 || (NT == 4 && MODE != kMatvec) ? 1 : 2;      // by registers
    struct Part {
        Raw<MB> raw[HALVES];
        uint32_t x[HALVES][NT][WORDS];
    };
    float acc[8][NT][4];
    uint32_t seen = 0;                // all shared exponents met, ORed

    // One sweep over the share.  The first one takes every step as it usually is and looks afterwards whether one was not (an
    // exponent of 128 or more, a sum that is no finite number): then all of the warp's share is done again with the exact wide steps,
    // which load nothing ahead.  One such block makes 1x4096x16384 Bfp4_b take 14.9 us instead of 8.9, 32x4096x16384 Bfp8_b 40 instead
    // of 25; blocks in every share 24 and 50, and 16 tokens' 4 of 32 experts 292 instead of 122.  The plain
    // form is for activations that are not aligned.  The usual form's loop has no test in it, so that the compiler schedules
    // two tile rows as one; the last rows, where activations may end inside a tile row, come behind it (1x4096x16384 Bfp4_b 9.8
    // -> 8.7 us).
    auto sweep = [&](auto kind_tag) {
        constexpr bool WIDE = decltype(kind_tag)::value == kWide, PLAIN = decltype(kind_tag)::value == kPlain;
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int v = 0; v < 4; v++) acc[j][nt][v] = 0.0f;
        int w_s = s0, w_kt = kt0, x_s = s0, x_kt = kt0;     // the tile rows that weights and activations are asked for
        const int64_t first = kt0 * row_bytes + (MODE == kExpertsOut ? (n > 0 ? W.list[s0] * image : 0) : W.w_off);
        const uint8_t *at = matrix + first;
        // lane t of a quad takes rows 4t .. 4t+3 of the upper (f = 0), then of the lower face
        auto load_w = [&](Raw<MB> &raw, int f) {
            const int face = 2 * f + fc;
            load_rows<MB>(raw, at + 64 + face * F::kFace + 4 * t * F::kRow);
            raw.e = __ldg(reinterpret_cast<const uint32_t *>(at + face * 16 + 4 * t));
        };
        auto ask_l2 = [&]() {             // a tile row's pieces, by address alone
#pragma unroll
            for (int f = 0; f < 2; f++) {
                const int face = 2 * f + fc;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 64 + face * F::kFace + 4 * t * F::kRow));
                if (MB == 7) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 64 + face * F::kFace + 4 * t * F::kRow + 32));
                if (t == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + face * 16));
            }
        };
        auto next_w = [&]() {
            at += row_bytes;
            if (MODE == kExpertsOut && ++w_kt == A.Kt) {
                w_kt = 0;
                if (++w_s * A.Kt < W.units) at = matrix + W.list[w_s] * image;
            }
        };
        const X *xp[NT];
        uint32_t present[NT];             // experts-out: all ones where the token has this expert
        auto rows_of = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                int tk = SINGLE ? 0 : nt * 8 + g;
                if (tk >= W.n_tok) tk = 0;
                present[nt] = ~0u;
                if constexpr (MODE == kMatvec) {
                    xp[nt] = A.x + (int64_t)(W.tok0 + tk) * A.ldx;
                } else if constexpr (MODE == kExpertsIn) {
                    xp[nt] = A.x + (int64_t)(W.list[2 * (W.tok0 + tk)] / A.top) * A.ldx;
                } else if constexpr (MODE == kExpertsEach) {
                    xp[nt] = A.h + (int64_t)W.list[2 * (W.tok0 + tk)] * A.hpad;
                } else {
                    const int r = W.rows[x_s * tok_pitch + tk];
                    if (r < 0) present[nt] = 0u;
                    xp[nt] = A.h + (int64_t)max(r, 0) * A.hpad;
                }
                xp[nt] += x_kt * 32 + 4 * t;
            }
        };
        auto load_x = [&](uint32_t (&x)[NT][WORDS], int f, bool inside) {    // inside: the tile row is known to lie inside the rows
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if constexpr (from_h(MODE)) {
                    const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(xp[nt] + f * 16));
                    x[nt][0] = v.x; x[nt][1] = v.y; x[nt][2] = v.z; x[nt][3] = v.w;
                    if (MODE == kExpertsOut && !SINGLE)
#pragma unroll
                        for (int i = 0; i < 4; i++) x[nt][i] &= present[nt];
                } else {
                    const uint2 v = inside || x_kt < whole ? *reinterpret_cast<const uint2 *>(xp[nt] + f * 16)
                                                           : load_four(xp[nt] - x_kt * 32 - 4 * t, x_kt * 32 + f * 16 + 4 * t, A.K, pairs);
                    x[nt][0] = v.x; x[nt][1] = v.y;
                }
            }
        };
        auto next_x = [&]() {
            x_kt++;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) xp[nt] += 32;
            if (MODE == kExpertsOut && x_kt == A.Kt) {
                x_kt = 0;
                if (++x_s * A.Kt < W.units) rows_of();
            }
        };
        auto compute = [&](const Raw<MB> &raw, const uint32_t (&loaded)[NT][WORDS]) {
            if (!WIDE) seen |= raw.e;
            uint2 x[PIECES][NT];
            pieces_of<WIDE>(x, loaded);
            if constexpr (WIDE && MODE == kExpertsOut && !SINGLE) {
                // a stored infinity times the zero that stands for "not this token's expert" is no zero: such columns are left out
                float part[8][NT][4] = {};
                step<MB, NT, PIECES, true>(part, raw, A, x);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int v = 0; v < 2; v++) {
                        const uint32_t here = __shfl_sync(0xffffffffu, present[nt], 4 * (2 * t + v));   // column 2t + v is lane group 2t + v's token
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            acc[j][nt][v] += here ? part[j][nt][v] : 0.0f;
                            acc[j][nt][2 + v] += here ? part[j][nt][2 + v] : 0.0f;
                        }
                    }
            } else if constexpr (!SINGLE) {
                step<MB, NT, PIECES, WIDE>(acc, raw, A, x);
            } else if constexpr (WIDE) {
                single_step_wide<MB, PIECES>(acc, raw, A, x);
            } else {
                uint32_t b[PIECES][2];
#pragma unroll
                for (int q = 0; q < PIECES; q++) {
                    b[q][0] = mul_bf16x2(x[q][0].x, scale_pair(raw.e, 0, -kDown));
                    b[q][1] = mul_bf16x2(x[q][0].y, scale_pair(raw.e, 1, -kDown));
                }
                single_step<MB, PIECES>(acc, raw, A, b);
            }
        };
        if constexpr (WIDE || (PLAIN && MODE != kMatvec)) {   // rare: nothing ahead, which leaves the registers to the usual form
            Part P;
            if (n > 0) rows_of();
#pragma unroll 1
            for (int i = 0; i < n; i++) {
#pragma unroll
                for (int f = 0; f < 2; f++) {
                    load_w(P.raw[0], f);
                    load_x(P.x[0], f, false);
                    compute(P.raw[0], P.x[0]);
                }
                next_w();
                next_x();
            }
        } else {
            Part P0, P1;
            // What the launch in front of this one computes is waited for before anything it may have written is read.  Of the
            // experts' second launch that is the first one, which writes h and no image and waited itself for all that came before: the
            // images may be read at once.  The product's launch stands behind any other launch, which may have written the image:
            // it only names its first rows to L2 before the wait.
            auto first_w = [&]() {
                if (n > 0) {
#pragma unroll
                    for (int f = 0; f < HALVES; f++) load_w(P0.raw[f], f);
                    if (HALVES == 2) next_w();
                }
            };
            if (W.begin && MODE != kExpertsIn) {
                if (MODE == kMatvec) {
                    if (n > 0) ask_l2();
                } else {
                    first_w();
                }
                griddep_wait();
                griddep_launch();
                if (MODE == kMatvec) first_w();
            } else {
                first_w();
            }
            if (n > 0) {
                rows_of();
#pragma unroll
                for (int f = 0; f < HALVES; f++) load_x(P0.x[f], f, false);
                if (HALVES == 2) next_x();
            }
            int i = 0;
            if constexpr (HALVES == 2) {
                auto both = [&](Part &P, bool inside) {
                    load_w(P.raw[0], 0);
                    load_w(P.raw[1], 1);
                    next_w();
                    load_x(P.x[0], 0, inside);
                    load_x(P.x[1], 1, inside);
                    next_x();
                };
                auto compute2 = [&](const Part &P) {
                    compute(P.raw[0], P.x[0]);
                    compute(P.raw[1], P.x[1]);
                };
#pragma unroll 1
                for (; i + 3 < n; i += 2) {
                    both(P1, !PLAIN);
                    compute2(P0);
                    both(P0, !PLAIN);
                    compute2(P1);
                }
                const int left = n - i;      // up to 3, the first one in P0
                if (left > 0) {
                    if (left > 1) both(P1, false);
                    compute2(P0);
                    if (left > 1) {
                        if (left > 2) both(P0, false);
                        compute2(P1);
                        if (left > 2) compute2(P0);
                    }
                }
            } else {
                auto lower = [&](bool inside) {
                    load_w(P1.raw[0], 1);
                    load_x(P1.x[0], 1, inside);
                    next_w();
                    next_x();
                };
                auto upper = [&](bool inside) {
                    load_w(P0.raw[0], 0);
                    load_x(P0.x[0], 0, inside);
                };
#pragma unroll 1
                for (; i + 2 < n; i++) {
                    lower(!PLAIN);
                    compute(P0.raw[0], P0.x[0]);
                    upper(!PLAIN);
                    compute(P1.raw[0], P1.x[0]);
                }
#pragma unroll 1
                for (; i < n; i++) {
                    lower(false);
                    compute(P0.raw[0], P0.x[0]);
                    if (i + 1 < n) upper(false);
                    compute(P1.raw[0], P1.x[0]);
                }
            }
        }
    };
    using Usual = std::integral_constant<int, kUsual>;
    if (from_h(MODE) || vec) sweep(Usual());
    else if constexpr (!from_h(MODE)) sweep(std::integral_constant<int, kPlain>());
    bool again = (seen & 0x80808080u) != 0;
    if constexpr (SINGLE || from_h(MODE)) {
        float z = 0.0f;                   // a sum of zeros, unless something is not finite
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int v = 0; v < 4; v++) z = fmaf(acc[j][nt][v], 0.0f, z);
        again |= z != 0.0f;
    }
    if (__any_sync(0xffffffffu, again)) sweep(std::integral_constant<int, kWide>());

    float *sums = reinterpret_cast<float *>(smem);
    if constexpr (SINGLE) {
        if (t == (g >> 1))
#pragma unroll
            for (int j = 0; j < 8; j++)
                *reinterpret_cast<float2 *>(sums + warp * tok_pitch * kPitch + j * 16 + g * 2) =
                    make_float2(((g & 1) ? acc[j][0][1] : acc[j][0][0]) * (float)(1 << kDown),
                                ((g & 1) ? acc[j][0][3] : acc[j][0][2]) * (float)(1 << kDown));
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int v = 0; v < 2; v++)
                if (nt * 8 + 2 * t + v < W.n_tok)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        *reinterpret_cast<float2 *>(sums + (warp * tok_pitch + nt * 8 + 2 * t + v) * kPitch + j * 16 + g * 2) =
                            make_float2(acc[j][nt][v], acc[j][nt][2 + v]);
    }
    __syncthreads();
}

// NT: groups of 8 tokens in one pass; 0: one token.
template <int MB, int NT, int MODE>
__global__ void __launch_bounds__(32 * kUnitWarps * units_per_sm(NT), 1) few_rows_kernel(const __grid_constant__ Args A)
{
    using F = Fmt<MB>;
    using L = Lay<MB, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = A.cluster, threads = blockDim.x, warps = threads >> 5;
    const int rank = c > 1 ? (int)cluster_rank() : 0;
    const int group = blockIdx.x / c;
    uint8_t *base = smem + warps * L::kSums;
    uint32_t *map = reinterpret_cast<uint32_t *>(base + L::kMap);
    volatile int *found_at = reinterpret_cast<volatile int *>(base + L::kCount);
    int *list = reinterpret_cast<int *>(base + L::kList);
    int16_t *rows = reinterpret_cast<int16_t *>(base + L::kRows);
    int *ids = reinterpret_cast<int *>(base + L::ids(MODE));

    // ---- which tokens and which matrices
    Work W;
    W.list = list;
    W.rows = rows;
    W.units = A.Kt;
    W.w_off = 0;
    W.tok0 = blockIdx.y * L::kTok;
    W.begin = true;
    int found = 0;                                     // in, each: the tokens of this CTA's expert
    const int64_t image = (int64_t)A.Kt * A.Nt * F::kRec;
    if (MODE == kMatvec) {
        W.n_tok = min(A.rows - W.tok0, L::kTok);
    } else {
        if (MODE == kExpertsIn) {
            griddep_wait();
            griddep_launch();
        }
        if constexpr (NT == 0) {
            // One token: lane s looks at slot s.  A slot counts where its expert exists and is not named before.
            const int e = lane < A.top ? __ldcg(A.ids + lane) : -1;
            const float w = lane < A.top ? __ldcg(A.wts + lane) : 0.0f;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const bool counts = e >= 0 && e < A.E && __ffs(same) - 1 == lane;
            const uint32_t m = __ballot_sync(0xffffffffu, counts);
            const int count = __popc(m);
            W.n_tok = 1;
            W.tok0 = 0;
            if (MODE == kExpertsIn) {
                if ((int)blockIdx.y >= count) return;  // the whole cluster: it shares blockIdx.y
                const int s = (int)__fns(m, 0, blockIdx.y + 1);
                W.w_off = __shfl_sync(0xffffffffu, e, s) * image;
                float sum = 0.0f;                      // in the order of the slots
                for (int i = 0; i < A.top; i++) {
                    const float wi = __shfl_sync(0xffffffffu, w, i);
                    if (__shfl_sync(0xffffffffu, e, i) == __shfl_sync(0xffffffffu, e, s)) sum += wi;
                }
                if (lane == 0) {                       // every warp writes the same
                    list[0] = s;
                    list[1] = __float_as_int(sum);
                }
            } else {
                if (counts) {
                    list[__popc(m & ((1u << lane) - 1u))] = e;
                    rows[__popc(m & ((1u << lane) - 1u))] = (int16_t)lane;
                }
                W.units = count * A.Kt;
            }
            __syncwarp();
        } else {
            if (MODE != kExpertsOut) W.tok0 = 0;
            const int t_end = MODE == kExpertsOut ? min(A.rows, W.tok0 + L::kTok) : A.rows, first = W.tok0 * A.top, slots = t_end * A.top - first;
            if (tid < kMaxExperts / 32) map[tid] = 0;
            __syncthreads();
            for (int i = tid; i < slots; i += threads) {
                int e = __ldcg(A.ids + first + i);
                if (e < 0 || e >= A.E) e = -1;
                ids[i] = e;
                if (e >= 0) atomicOr(&map[e >> 5], 1u << (e & 31));
            }
            __syncthreads();
            int count = 0;
            for (int w = 0; w < kMaxExperts / 32; w++) count += __popc(map[w]);
            if (MODE == kExpertsOut) {
                W.n_tok = t_end - W.tok0;
                if (tid < kMaxExperts && (map[tid >> 5] >> (tid & 31) & 1u)) {     // expert e is number (set bits below e)
                    int at = __popc(map[tid >> 5] & ((1u << (tid & 31)) - 1u));
                    for (int w = 0; w < (tid >> 5); w++) at += __popc(map[w]);
                    list[at] = tid;
                }
                for (int i = tid; i < count * L::kTok; i += threads) rows[i] = -1;
                __syncthreads();
                if (tid < W.n_tok)
                    for (int s = A.top - 1; s >= 0; s--) {                         // of a repeated expert the first slot stays
                        const int e = ids[tid * A.top + s];
                        if (e < 0) continue;
                        int at = __popc(map[e >> 5] & ((1u << (e & 31)) - 1u));
                        for (int w = 0; w < (e >> 5); w++) at += __popc(map[w]);
                        rows[at * L::kTok + tid] = (int16_t)((W.tok0 + tid) * A.top + s);
                    }
                __syncthreads();
                W.units = count * A.Kt;
            } else {
                if ((int)blockIdx.y >= count) {                                    // the whole cluster: it shares blockIdx.y
                    // where no slot counts at all, some block still has to stand behind the launch in front
                    if (MODE == kExpertsEach && blockIdx.y == 0) griddep_wait();
                    return;
                }
                int e = 0, left = blockIdx.y;
                for (int w = 0; w < kMaxExperts / 32; w++) {
                    const int here = __popc(map[w]);
                    if (left >= 0 && left < here) e = 32 * w + (int)__fns(map[w], 0, left + 1);
                    left -= here;
                }
                W.w_off = e * image;
                if (warp == 0) {                       // the tokens of this expert, in order; a repeated slot adds its weight
                    int n = 0;
                    for (int b = 0; b < A.rows; b += 32) {
                        const int tk = b + lane;
                        int slot = -1;
                        float w = 0.0f;
                        if (tk < A.rows)
                            for (int s = 0; s < A.top; s++)
                                if (ids[tk * A.top + s] == e) {
                                    if (MODE == kExpertsIn) w += __ldcg(A.wts + tk * A.top + s);
                                    if (slot < 0) slot = s;
                                }
                        const uint32_t m = __ballot_sync(0xffffffffu, slot >= 0);
                        if (slot >= 0) {
                            const int at = n + __popc(m & ((1u << lane) - 1u));
                            list[2 * at] = tk * A.top + slot;
                            list[2 * at + 1] = __float_as_int(w);
                        }
                        n += __popc(m);
                    }
                    if (lane == 0) *found_at = n;
                }
                __syncthreads();
                found = *found_at;
            }
        }
    }

    const int workers = c * warps, me = rank * warps + warp;
    const float *sums = reinterpret_cast<const float *>(smem);
    float *part = reinterpret_cast<float *>(base + L::kPart);
    const bool gated = MODE == kExpertsIn && A.w1 != nullptr;
    const int col0 = group * (gated ? kGroupTiles / 2 : kGroupTiles) * 32;
    auto of_cta = [&](int tk, int q) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 8
        for (int w = 0; w < warps; w++) {
            const float2 v = *reinterpret_cast<const float2 *>(sums + (w * L::kTok + tk) * kPitch + 2 * q);
            s.x += v.x;
            s.y += v.y;
        }
        return s;
    };
    auto total = [&](int tk, int q) {
        if (c == 1) return of_cta(tk, q);
        float2 s = make_float2(0.0f, 0.0f);
        const uint32_t at = smem_u32(part + tk * 128 + 2 * q);
        for (int r = 0; r < c; r++) {
            const float2 v = ld_cluster_f2(map_rank(at, r));
            s.x += v.x;
            s.y += v.y;
        }
        return s;
    };

    // ---- one pass, or (in, each) as many as the expert has groups of kTok tokens
    while (true) {
        if (NT != 0 && (MODE == kExpertsIn || MODE == kExpertsEach)) W.n_tok = min(found - W.tok0, L::kTok);
        if constexpr (NT == 0) {
            products<MB, 1, MODE, true>(A, W, smem, group, me, workers, 1);
        } else {
            products<MB, NT, MODE, false>(A, W, smem, group, me, workers, L::kTok);
        }

        // join the warps, and the CTAs of a cluster (each finishes its share of the outputs)
        if (c > 1) {
            for (int i = tid; i < W.n_tok * 64; i += threads)
                *reinterpret_cast<float2 *>(part + (i >> 6) * 128 + 2 * (i & 63)) = of_cta(i >> 6, i & 63);
            cluster_sync();
        }
        const int per_tok = gated ? 32 : 64, items = W.n_tok * per_tok;
        for (int i = rank * threads + tid; i < items; i += c * threads) {
            const int tk = gated ? i >> 5 : i >> 6, r = i & (per_tok - 1);
            const int j = gated ? r >> 2 : r >> 3, gg = gated ? r & 3 : r & 7, q = j * 8 + gg;
            const int col = col0 + ((gg & 1) | ((gg >> 2) << 1)) * 32 + ((gg >> 1) & 1) * 16 + 2 * j;
            float2 v = total(tk, q);
            if (MODE == kExpertsIn) {
                float2 up = make_float2(1.0f, 1.0f);
                if (gated) up = total(tk, q + 4);
                const float w = __int_as_float(list[2 * (W.tok0 + tk) + 1]);
                float r2[2] = {activate(v.x, A.act) * up.x * w, activate(v.y, A.act) * up.y * w};
                if (col < A.hpad)                  // tile padding is zero: its weights are
                    *reinterpret_cast<float2 *>(A.h + (int64_t)list[2 * (W.tok0 + tk)] * A.hpad + col) =
                        make_float2(col < A.N ? r2[0] : 0.0f, col + 1 < A.N ? r2[1] : 0.0f);
            } else if (MODE == kExpertsEach) {
                if (col < 32 * A.Nt)
                    *reinterpret_cast<float2 *>(A.partial + (int64_t)list[2 * (W.tok0 + tk)] * 32 * A.Nt + col) = v;
            } else {
                const int64_t at = (int64_t)(W.tok0 + tk) * A.ldo + col;
#pragma unroll
                for (int b = 0; b < 2; b++)
                    if (col + b < A.N) {
                        const float f = b ? v.y : v.x;
                        if (A.out_f32) reinterpret_cast<float *>(A.out)[at + b] = f;
                        else reinterpret_cast<__nv_bfloat16 *>(A.out)[at + b] = __float2bfloat16_rn(f);
                    }
            }
        }
        if (c > 1) cluster_sync();                     // no CTA goes on while another reads its sums
        if (NT == 0 || MODE == kMatvec || MODE == kExpertsOut || W.tok0 + L::kTok >= found) break;
        W.tok0 += L::kTok;
        W.begin = false;
        __syncthreads();                               // the sums are read: they may be written again
    }
}

// y[t] = the sum of the rows of token t's slots, each expert once: a block for 1024 columns of a token.
__global__ void __launch_bounds__(256) sum_slots_kernel(const float *partial, int64_t pitch, const int *ids, int top, int E, int H,
                                                        __nv_bfloat16 *y, int64_t ldy)
{
    griddep_wait();
    griddep_launch();
    const int t = blockIdx.y, lane = threadIdx.x & 31, col = blockIdx.x * 1024 + threadIdx.x * 4;
    const int e = lane < top ? __ldcg(ids + t * top + lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    uint32_t m = __ballot_sync(0xffffffffu, e >= 0 && e < E && __ffs(same) - 1 == lane);
    if (col >= H) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (; m; m &= m - 1) {
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(partial + (int64_t)(t * top + __ffs(m) - 1) * pitch + col));
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int b = 0; b < 4; b++)
        if (col + b < H) y[(int64_t)t * ldy + col + b] = __float2bfloat16_rn(f[b]);
}

// Every launch may begin before the one in front of it is done.  It waits for that one before it reads or writes anything that any
// launch in front may have written or may read; the exception (images, in the experts' second launch) is explained in `products`.
// Only launches that say so let it: those of this file and of the router, each after its own wait.
template <int MB, int NT, int MODE>
cudaError_t launch_one(const Args &a, dim3 grid, int warps, cudaStream_t stream)
{
    constexpr int most = Lay<MB, NT>::bytes(MODE, kUnitWarps * units_per_sm(NT));
    static_assert(most <= 227 * 1024, "shared memory of the largest CTA");
    static std::atomic<uint64_t> ready{0};      // devices whose kernel may take this much shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(few_rows_kernel<MB, NT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = Lay<MB, NT>::bytes(MODE, warps);
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = a.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, few_rows_kernel<MB, NT, MODE>, a);
}

int groups_of_8(int rows) { return rows == 1 ? 0 : rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// How the tile rows of a column group are shared out: over the warps of a CTA and over a cluster.
struct Split {
    int units, cluster;       // units of 8 warps in a CTA; CTAs
};
// CTAs of a cluster first, one to an SM, while each warp of 8 keeps a tile row, and as many as fit while it keeps two; then more
// warps in a CTA, while each keeps 4.
// Measured, us, as CTAs x warps (B200): 1x1024x1024 Bfp4_b, 8 column groups: 4x8 2.46, 8x8 2.91, 1x16 3.19.  8x4096x1024 Bfp8_b, 8
// groups: 8x8 4.81, 8x16 4.99, 1x16 10.3.  12x4096x4096 Bfp4_b, 32 groups: 8x8 6.70, 4x8 7.91, 4x16 7.06.  1x4096x16384 Bfp4_b,
// 128 groups: 1x16 9.75, 2x8 10.5, 1x8 12.4.
Split split_of(int64_t groups, int64_t tile_rows, int sm_count, int per_sm)
{
    int64_t c = std::min<int64_t>(sm_count / groups, (tile_rows + kUnitWarps - 1) / kUnitWarps);
    if (2 * groups <= sm_count) c = std::max(c, std::min<int64_t>((int64_t)per_sm * sm_count / groups, tile_rows / (2 * kUnitWarps)));
    c = std::max<int64_t>(1, std::min<int64_t>(c, 8));
    int64_t u = tile_rows / (c * kUnitWarps * 4);
    u = std::min<int64_t>(u, (int64_t)sm_count * per_sm / (groups * c));
    u = std::max<int64_t>(1, std::min<int64_t>(u, per_sm));
    return {(int)u, (int)c};
}

template <int MODE, int MB>
cudaError_t launch_nt(int nt, const Args &a, dim3 grid, int warps, cudaStream_t stream)
{
    // one sum over all experts serves up to kOneSum tokens, sums of their own more than that
    if constexpr (MODE != kExpertsEach)
        if (nt == 0) return launch_one<MB, 0, MODE>(a, grid, warps, stream);
    if constexpr (MODE != kExpertsOut) {
        if (nt == 2) return launch_one<MB, 2, MODE>(a, grid, warps, stream);
        if (nt == 4) return launch_one<MB, 4, MODE>(a, grid, warps, stream);
    }
    return launch_one<MB, 1, MODE>(a, grid, warps, stream);
}

// groups: column groups; copies: how many times each, for other experts or rows; y: grid rows
template <int MODE>
cudaError_t dispatch(int mant_bits, int nt, Args &a, int groups, double copies, int64_t tile_rows, int y, int sm_count, cudaStream_t stream)
{
    const Split s = split_of((int64_t)(groups * copies + 0.5), tile_rows, sm_count, units_per_sm(nt));
    const dim3 grid((unsigned)(groups * s.cluster), y);
    const int warps = s.units * kUnitWarps;
    a.cluster = s.cluster;
    a.m4 = 4;
    a.m16 = 16;
    a.m64 = 64;
    switch (mant_bits) {
        case 7: return launch_nt<MODE, 7>(nt, a, grid, warps, stream);
        case 3: return launch_nt<MODE, 3>(nt, a, grid, warps, stream);
        default: return launch_nt<MODE, 1>(nt, a, grid, warps, stream);
    }
}

}  // namespace few

using namespace few;

cudaError_t launch_bfp_matvec(const void *A, int64_t M, int64_t K, int64_t lda, const void *W, int64_t N, int mant_bits, void *Y, int64_t ldy,
                              int out_f32, int sm_count, cudaStream_t stream)
{
    Args a = {};
    a.x = (const __nv_bfloat16 *)A; a.ldx = lda;
    a.rows = (int)M; a.K = (int)K; a.Kt = (int)((K + 31) / 32); a.N = (int)N; a.Nt = (int)((N + 31) / 32);
    a.w0 = (const uint8_t *)W;
    a.out = Y; a.ldo = ldy; a.out_f32 = out_f32;
    const int nt = groups_of_8(a.rows), groups = (a.Nt + kGroupTiles - 1) / kGroupTiles, passes = (a.rows + 31) / 32;
    return dispatch<kMatvec>(mant_bits, nt, a, groups, passes, a.Kt, passes, sm_count, stream);
}

cudaError_t launch_moe_experts(const MoeArgs &m, int sm_count, cudaStream_t stream)
{
    const int Ht = (m.H + 31) / 32, It = (m.I + 31) / 32;
    const int slots = m.T * m.top, most = m.E < slots ? m.E : slots;
    // The experts that independent choices reach on average, and the tokens of one.  A pass over an expert's weights takes 8, 16 or
    // 32 tokens.  Measured, us, passes of 8 / 16 / 32, gated, 4 of 16 experts (B200):
    //   tokens an expert       5                   6                   8                   10                  12                  16
    //   1024 x 1024 Bfp4_b     22.5 / 27.5 / 31.9  28.5 / 28.2 / 32.4  31.6 / 28.4 / 32.7  32.8 / 29.6 / 34.5  39.5 / 38.0 / 35.1  45.2 / 46.8 / 36.2
    //   2048 x 1024 Bfp2_b     25.7 / 32.5 / 51.2  32.8 / 33.1 / 52.0  36.7 / 33.5 / 52.6  37.8 / 34.6 / 54.6  44.4 / 45.3 / 55.8  53.1 / 56.7 / 57.1
    //   1024 x 2048 Bfp8_b     35.4 / 45.6 / 66.4  42.8 / 46.3 / 67.2  47.1 / 47.1 / 68.1  50.8 / 49.2 / 71.1  58.6 / 63.3 / 72.3  67.4 / 74.5 / 74.3
    // and 2 of 4 experts, 16 tokens an expert: 29.7 / 26.0 / 19.5, 33.0 / 32.2 / 23.2, 34.8 / 38.4 / 23.7.
    // One sum over all experts (up to kOneSum tokens) against sums of their own for 2, 3, 4 and 8 tokens:
    //   4 of 32 of 1024 x 1024 Bfp4_b  14.3, 16.8, 22.6, 30.0 against 14.4, 17.4, 18.6, 27.2
    //   2 of 16 of 2048 x 1024 Bfp2_b  13.6, 15.3, 17.2, 22.9 against 14.7, 16.8, 17.8, 20.2
    //   2 of 16 of 4096 x 1024 Bfp8_b  20.7, 30.0, 34.3, 43.8 against 22.8, 26.7, 28.3, 41.9
    //   8 of 64 of 2048 x 1024 Bfp4_b  31.0, 51.4, 57.7, 79.4 against 26.5, 42.2, 44.3, 58.6
    //   2 of 8 of 4096 x 2048 Bfp4_b   30.4, 38.9, 38.6, 41.2 against 26.1, 44.5, 37.6, 39.1
    const double miss = m.top < m.E ? 1.0 - (double)m.top / m.E : 0.0, reached = m.E * (1.0 - pow(miss, m.T));
    const double share = (double)slots / m.E;
    const int nt = m.T == 1 ? 0 : m.T <= 8 || share <= 6.0 ? 1 : share <= 10.0 ? 2 : 4;
    Args a = {};
    a.x = (const __nv_bfloat16 *)m.x; a.ldx = m.ldx;
    a.rows = m.T; a.K = m.H; a.Kt = Ht; a.N = m.I; a.Nt = It;
    a.w0 = (const uint8_t *)m.gate; a.w1 = (const uint8_t *)m.up;
    a.ids = m.ids; a.wts = m.weights; a.top = m.top; a.E = m.E; a.act = m.act;
    a.h = (float *)m.h; a.hpad = 32 * It;
    const int span = m.up ? kGroupTiles / 2 : kGroupTiles;
    cudaError_t e = dispatch<kExpertsIn>(m.mant_bits, nt, a, (It + span - 1) / span, reached, Ht, most, sm_count, stream);
    if (e != cudaSuccess) return e;
    a.K = m.I; a.Kt = It; a.N = m.H; a.Nt = Ht;
    a.w0 = (const uint8_t *)m.down; a.w1 = nullptr;
    a.out = m.y; a.ldo = m.ldy; a.out_f32 = 0;
    const int groups = (Ht + kGroupTiles - 1) / kGroupTiles;
    if (m.T <= kOneSum) return dispatch<kExpertsOut>(m.mant_bits, nt, a, groups, 1.0, (int64_t)(It * reached + 0.5), 1, sm_count, stream);
    a.partial = reinterpret_cast<float *>((uint8_t *)m.h + moe_h_bytes(m.T, m.top, m.I));
    e = dispatch<kExpertsEach>(m.mant_bits, nt, a, groups, reached, It, most, sm_count, stream);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((m.H + 1023) / 1024, m.T);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, sum_slots_kernel, (const float *)a.partial, (int64_t)32 * Ht, m.ids, m.top, m.E, m.H, (__nv_bfloat16 *)m.y,
                              m.ldy);
}

}  // namespace buda
