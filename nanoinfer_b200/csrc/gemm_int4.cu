// Products with 4-bit weights: out[tokens, N] = X[tokens, K] . W[N, K]^T, W[n, k] = (code[n, k] - 8) * scale[n, k / group], bfloat16
// activations and scales, 32-bit sums, for up to 64 tokens. A weight's bytes are needed once, which is what a product cannot do without (2 x 18,944 x
// 3,584: 11 us); up to 16 tokens it takes some 1.7 times that (8: 18.8 us, bfloat16 weights 49), with more its time is the instructions, which grow
// with the tokens (32: 41 us, 64: 80, bfloat16 weights 46 and 48).
//
// Layout (made once, when a model is loaded). A tile is 16 rows x 64 k, 512 bytes: 16 bytes for each lane of a warp, which are the
// lane's share of the weight operand of four tensor-core instructions (mma.sync m16n8k16, weights as the 16 rows, tokens as the 8
// columns), so a tile is one load of 512 contiguous bytes and goes from memory to the tensor core through registers alone. Lane (g, t)
// holds of every 32 k the columns 8t .. 8t + 7 of the rows g and g + 8: word 2b + j of its four has the k 32b + 8t + 4j + e, e = 0..3, in
// the order of nibbles (row g, e 0) (row g + 8, e 0) (g, 2) (g + 8, 2) (g, 1) (g + 8, 1) (g, 3) (g + 8, 3). A code in the low bits of
// 128.0 is the bfloat16 number 128 + code; minus 136 it is the weight without its scale, exactly. Tiles lie [row tile][k tile]; scales
// [row tile][group][8] pairs of the rows g and g + 8.
//
// The scale multiplies a group's 32-bit sum, not its weights: the products are exact, and a group costs one multiply-add for each
// result instead of one multiplication for each weight.
//
// What bounds a product of many weights is the instructions that make a code a number: 11 for eight codes as above, 65 for a tile and
// its row tile, where memory delivers a tile to an SM every 22 cycles. So there (F16) a code is fed as it lies in its word: in the low
// bits of a 16-bit float it is code * 2^-24 (a number below the normal ones, which the tensor core multiplies exactly), four bits
// further up 16 times that, and one shift reaches the word's other half: 5 instructions. The activations are 16-bit floats too,
// scaled by a power of two for each token so that the largest lies in 2^13 .. 2^14 (every element that counts is exact), and the 8 of
// (code - 8) leaves a group's sum as 8 times the sum of the group's activations, where the sum begins. A small kernel before makes
// the scaled activations, those sums and the factors, which small products cannot wait for.
#include "pipeline.cuh"
#include <cuda_fp16.h>
#include <cmath>

using namespace nibp;

namespace {

constexpr int WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16_once(unsigned dst, const void* src) {          // (past L1: weights are read once)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_or_zero(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned lds4(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float2 lds8f(unsigned at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

// The four fragments of a word as they lie there: 16-bit floats code * 2^-24, the rows g + 8 (fragments 1 and 3) 16 times that.
__device__ __forceinline__ void codes_of(unsigned w, unsigned (&a)[4]) {
    const unsigned u = w >> 8;
    a[0] = w & 0x000f000fu; a[1] = w & 0x00f000f0u; a[2] = u & 0x000f000fu; a[3] = u & 0x00f000f0u;
}
// The four fragments of a word: nibble pairs as bfloat16 numbers code - 8.
__device__ __forceinline__ void weights_of(unsigned w, unsigned (&a)[4]) {
    const __nv_bfloat162 off = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));       // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
        a[i] = *reinterpret_cast<const unsigned*>(&v);
    }
}

struct Args {
    const __nv_bfloat16* x; const uint4* w; const unsigned* scales; const float* bias; void* out;
    const float* sums; const float* factors;        // F16: -8 * 2^-24 * the sums of the activations [k / 64 or 32][64 tokens], a factor for each token
    int tokens, n_out, k, ldx, ldo, epi, row_tiles, k_tiles, group_shift, groups, ksplit, csize;      // group_shift: log2(group)
    NibGlu glu;
};

// The activations of F16: a CTA a token. x16 [tokens][k] = x * 2^e, sums as Args has them, factors = 2^24 / 2^e. step: 64 or 32.
constexpr int PREP_THREADS = 512;
__global__ void __launch_bounds__(PREP_THREADS)
prepare_f16_kernel(const __nv_bfloat16* x, int ldx, __half* __restrict__ x16, float* __restrict__ sums, float* __restrict__ factors, int k, int step) {
    __shared__ unsigned s_top[PREP_THREADS / 32];
    const int token = blockIdx.x, lane = threadIdx.x & 31;
    const uint4* row = reinterpret_cast<const uint4*>(x + (size_t)token * ldx);
    pdl_launch_dependents();        // (the product sends for its weights meanwhile)
    pdl_wait();
    unsigned top = 0;
    for (int i = threadIdx.x; i < k / 8; i += PREP_THREADS) {
        const uint4 u = row[i];
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PREP_THREADS / 32; ++i) top = max(top, s_top[i]);
    // the exponent field e of the largest element: 2^(140 - e) takes it to 2^13 (in two factors: the power may leave the range)
    const int e = (int)(top >> 7), up = (e == 0 || e == 255) ? 0 : 140 - e;
    const float f1 = __uint_as_float((unsigned)(127 + up / 2) << 23), f2 = __uint_as_float((unsigned)(127 + up - up / 2) << 23);
    if (threadIdx.x == 0)
        factors[token] = 0x1p24f * __uint_as_float((unsigned)(127 - up / 2) << 23) * __uint_as_float((unsigned)(127 - (up - up / 2)) << 23);
    const int lanes = step / 8;                     // that hold a step between them
    for (int i0 = 0; i0 < k / 8; i0 += PREP_THREADS) {
        const int i = i0 + threadIdx.x;
        float sum = 0.f;
        if (i < k / 8) {
            const uint4 u = row[i];
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
            unsigned r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * f1 * f2, __uint_as_float(w[j] & 0xffff0000u) * f1 * f2);
                const float2 v = __half22float2(h);
                sum += v.x + v.y;
                r[j] = *reinterpret_cast<const unsigned*>(&h);
            }
            reinterpret_cast<uint4*>(x16 + (size_t)token * k)[i] = make_uint4(r[0], r[1], r[2], r[3]);
        }
        for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (i < k / 8 && (i & (lanes - 1)) == 0) sums[(size_t)(i / lanes) * 64 + token] = sum * (-8.f * 0x1p-24f);
    }
}

// A stage of a warp's ring in shared memory: R tiles of weights and the activations of 64 k of NT * 8 tokens, every lane's own 16-byte
// pieces (what a lane uses it has copied itself), and the scales and sums of G groups.
template <int NT, int R, bool G32, bool F16> struct Ring {
    static constexpr int G = G32 ? 2 : 1;
    static constexpr int X_AT = R * 512, S_AT = X_AT + NT * 1024, C_AT = S_AT + R * G * 32;
    static constexpr int STAGE = C_AT + (F16 ? G * NT * 32 : 0);
    static constexpr int SPLIT = NT <= 2 ? 4 : 1;           // CTAs that may share K
    static constexpr int SENT = SPLIT > 1 ? SPLIT * R * NT * 512 : 0;       // what they send to the first of them
    static constexpr int FIT = (108 * 1024 - SENT) / WARPS / STAGE, D = FIT < 2 ? 2 : FIT > 8 ? 8 : FIT;      // two CTAs an SM
    static constexpr int RING = WARPS * D * STAGE, PART = WARPS * R * NT * 4 * 32 * 4;
    static constexpr int OWN = RING > PART ? RING : PART, BYTES = OWN + SENT;
    static_assert(OWN % 16 == 0, "results are sent 16 bytes at a time");
};

__device__ __forceinline__ void st_peer_f32x4(unsigned addr, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// R row tiles a warp, which share the activations they multiply with (with DUAL half of them a gate's and half an up's); NT tiles of 8
// tokens. ``ksplit`` warps of a CTA share a row unit's K and are summed in order; where all eight do, up to four CTAs of a cluster may
// share it further, and the first of them sums what the others send it, in order.
template <int NT, int R, bool DUAL, bool G32, bool F16>
__global__ void __launch_bounds__(WARPS * 32)
gemm_int4_kernel(const Args a) {
    using C = Ring<NT, R, G32, F16>;
    constexpr int D = C::D, G = C::G, OUT = DUAL ? R / 2 : R;              // row tiles of the result
    extern __shared__ __align__(16) float part[];             // the rings; then [WARPS][R][NT][4][32] where K is split
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = a.csize > 1 ? (int)cluster_rank() : 0;
    if (a.csize > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");       // this CTA is there: its peers may send
    const int unit = (blockIdx.x / a.csize) * (WARPS / a.ksplit) + warp / a.ksplit, kpart = warp % a.ksplit;
    const int out_tiles = (a.n_out + 15) / 16;
    const int rt0 = unit * OUT;                                             // first row tile of the unit's results
    const bool live = rt0 < out_tiles;
    const int per = (a.k_tiles + a.ksplit * a.csize - 1) / (a.ksplit * a.csize);
    const int begin = live ? min(a.k_tiles, (rank * a.ksplit + kpart) * per) : 0, end = live ? min(a.k_tiles, begin + per) : 0;
    const uint4* wp[R];
    size_t scale_row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        // (a tile behind the last is computed and not stored)
        const int rt = min(DUAL ? min(rt0 + r / 2, out_tiles - 1) + (r & 1) * out_tiles : rt0 + r, a.row_tiles - 1);
        wp[r] = a.w + (size_t)rt * a.k_tiles * 32 + lane;
        scale_row[r] = (size_t)rt * a.groups;
    }
    const unsigned ring = (unsigned)__cvta_generic_to_shared(part) + warp * D * C::STAGE;
    const int groups = a.groups;
    auto send_weights = [&](int kt, unsigned dst) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            copy16_once(dst + r * 512 + lane * 16, wp[r] + (size_t)kt * 32);
#pragma unroll
            for (int b = 0; b < G; ++b) {
                const int at = G32 ? 2 * kt + b : (kt << 6) >> a.group_shift;
                if (lane < 8) copy4_or_zero(dst + C::S_AT + (r * G + b) * 32 + lane * 4, a.scales + (scale_row[r] + min(at, groups - 1)) * 8 + lane, at < groups);
            }
        }
    };
    const __nv_bfloat16* xp[NT];            // (16 bits either way)
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = a.x + (size_t)min(n * 8 + g, a.tokens - 1) * a.ldx + 8 * t;
    auto send_activations = [&](int kt, unsigned dst) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool valid = n * 8 + g < a.tokens && kt * 64 + b * 32 < a.k;
                copy16_or_zero(dst + C::X_AT + (n * 2 + b) * 512 + lane * 16, xp[n] + (valid ? kt * 64 + b * 32 : 0), valid);
            }
        if (F16) {
#pragma unroll
            for (int b = 0; b < G; ++b) {
                const int at = G32 ? 2 * kt + b : kt;
                for (int i = lane; i < NT * 8; i += 32) copy4_or_zero(dst + C::C_AT + (b * NT * 8 + i) * 4, a.sums + (size_t)at * 64 + i, i < a.tokens && at * (G32 ? 32 : 64) < a.k);
            }
        }
    };
    pdl_launch_dependents();
    // weights are nobody's output: the first stages' are sent for before the wait, the activations behind it
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (begin + d < end) send_weights(begin + d, ring + d * C::STAGE);
    pdl_wait();
#pragma unroll
    for (int d = 0; d < D - 1; ++d) {
        if (begin + d < end) send_activations(begin + d, ring + d * C::STAGE);
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    }

    float acc[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
    auto add = [&](float (&to)[4], const float (&s)[4], unsigned scale) {
        const float s0 = __uint_as_float(scale << 16), s1 = __uint_as_float(scale & 0xffff0000u);
        to[0] = fmaf(s[0], s0, to[0]); to[1] = fmaf(s[1], s0, to[1]);
        to[2] = fmaf(s[2], s1, to[2]); to[3] = fmaf(s[3], s1, to[3]);
    };
    unsigned src = ring, dst = ring + (D - 1) * C::STAGE;
    const unsigned ring_end = ring + D * C::STAGE;
#pragma unroll 1
    for (int kt = begin; kt < end; ++kt) {
        if (kt + D - 1 < end) { send_weights(kt + D - 1, dst); send_activations(kt + D - 1, dst); }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group %0;\n" ::"n"(D - 1) : "memory");
        __syncwarp();               // (scales and sums are other lanes' copies)
        float s[R][NT][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (G32 || b == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 c = F16 ? lds8f(src + C::C_AT + (G32 ? b * NT * 32 : 0) + n * 32 + t * 8) : make_float2(0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < R; ++r) { s[r][n][0] = c.x; s[r][n][1] = c.y; s[r][n][2] = 16.f * c.x; s[r][n][3] = 16.f * c.y; }
                }
            }
            uint4 x[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n] = lds16(src + C::X_AT + (n * 2 + b) * 512 + lane * 16);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned at = src + r * 512 + lane * 16 + b * 8;
                const float2 words = lds8f(at);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned f[4];
                    const unsigned word = __float_as_uint(h == 0 ? words.x : words.y);
                    if (F16) codes_of(word, f); else weights_of(word, f);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const unsigned b0 = h == 0 ? x[n].x : x[n].z, b1 = h == 0 ? x[n].y : x[n].w;
                        if (F16) mma_f16(s[r][n], f, b0, b1); else mma_bf16(s[r][n], f, b0, b1);
                    }
                }
            }
            if (G32 || b == 1) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const unsigned scale = lds4(src + C::S_AT + (r * G + (G32 ? b : 0)) * 32 + g * 4);
#pragma unroll
                    for (int n = 0; n < NT; ++n) add(acc[r][n], s[r][n], scale);
                }
            }
        }
        __syncwarp();               // the shared places are free
        src = src + C::STAGE == ring_end ? ring : src + C::STAGE;
        dst = dst + C::STAGE == ring_end ? ring : dst + C::STAGE;
    }

    // ---- the results of token tile n: element e is row g + 8 * (e / 2), token n * 8 + 2t + (e & 1)
    auto emit = [&](float (&v)[R][4], int n) {
        if (F16) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int tok = n * 8 + 2 * t + j;
                const float f = tok < a.tokens ? __ldcg(a.factors + tok) : 0.f;        // (the kernel before this one writes them)
#pragma unroll
                for (int r = 0; r < R; ++r) { v[r][j] *= f; v[r][2 + j] *= f * 0.0625f; }
            }
        }
#pragma unroll
        for (int r = 0; r < OUT; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = (rt0 + r) * 16 + g + 8 * (e >> 1), tok = n * 8 + 2 * t + (e & 1);
                if (f >= a.n_out || tok >= a.tokens) continue;
                const size_t at = (size_t)tok * a.ldo + f;
                if (DUAL) {
                    const float gate = v[DUAL ? 2 * r : 0][e], up = v[DUAL ? 2 * r + 1 : 0][e];
                    const float y = a.epi == EPI_GEGLU ? nib_geglu_fast(gate, up)
                                  : a.epi == EPI_GLU ? nib_glu_fast(a.glu, gate, up) : __fdividef(gate, 1.0f + __expf(-gate)) * up;
                    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
                } else {
                    const float y = v[r][e] + (a.bias ? __ldg(a.bias + f) : 0.f);
                    if (a.epi == EPI_STORE) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
                    else if (a.epi == EPI_ADD) static_cast<float*>(a.out)[at] += y;
                    else static_cast<float*>(a.out)[at] = y;
                }
            }
    };
    if (a.ksplit == 1) {
        if (!live) return;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float v[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[r][e] = acc[r][n][e];
            emit(v, n);
        }
        return;
    }
    __syncthreads();                // every warp is through with its ring
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(((warp * R + r) * NT + n) * 4 + e) * 32 + lane] = acc[r][n][e];
    __syncthreads();
    const int first = warp - kpart;             // the unit's first warp
    auto sum_of = [&](int r, int n) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < a.ksplit; ++p) {
            const float* at = part + (((first + p) * R + r) * NT + n) * 128 + lane;
            v.x += at[0]; v.y += at[32]; v.z += at[64]; v.w += at[96];
        }
        return v;
    };
    if constexpr (C::SPLIT > 1) {
        if (a.csize > 1) {          // (all eight warps share one unit)
            float4* sent = reinterpret_cast<float4*>(reinterpret_cast<unsigned char*>(part) + C::OWN);         // [csize][R * NT][32]
            asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");           // every CTA is there
            for (int i = warp; i < R * NT; i += WARPS) st_peer_f32x4(peer_smem(sent + (rank * R * NT + i) * 32 + lane, 0), sum_of(i / NT, i % NT));
            cluster_sync();
            if (rank != 0) return;
            for (int n = warp; n < NT; n += WARPS) {
                float v[R][4];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int p = 0; p < a.csize; ++p) {
                        const float4 x = sent[(p * R * NT + r * NT + n) * 32 + lane];
                        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
                    }
                    v[r][0] = sum.x; v[r][1] = sum.y; v[r][2] = sum.z; v[r][3] = sum.w;
                }
                emit(v, n);
            }
            return;
        }
    }
    if (!live) return;
    for (int n = kpart; n < NT; n += a.ksplit) {
        float v[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float4 sum = sum_of(r, n);
            v[r][0] = sum.x; v[r][1] = sum.y; v[r][2] = sum.z; v[r][3] = sum.w;
        }
        emit(v, n);
    }
}

// The weights as numbers: rows of K in bfloat16 or 32 bits, a lane's share of a tile a thread. part 0: the weight (rounded, in
// bfloat16); part 1: what that rounding leaves, which bfloat16 holds exactly (a code has 3 significant bits and a scale 8).
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&f)[8]) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const unsigned*>(&v);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename T>
__global__ void __launch_bounds__(256)
unpack_int4_kernel(const uint4* __restrict__ w, const unsigned* __restrict__ scales, T* __restrict__ out, int n, int k, int k_tiles, int group_shift,
                   int groups, long long items, int part) {
    pdl_wait();
    pdl_launch_dependents();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int lane = (int)(i & 31), g = lane >> 2, t = lane & 3;
    const long long tile = i >> 5;
    const int rt = (int)(tile / k_tiles), kt = (int)(tile - (long long)rt * k_tiles);
    const uint4 u = w[i];
    const unsigned words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int k0 = kt * 64 + b * 32 + 8 * t;
        if (k0 >= k) continue;
        const unsigned pair = __ldg(scales + ((size_t)rt * groups + (k0 >> group_shift)) * 8 + g);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = rt * 16 + half * 8 + g;
            if (row >= n) continue;
            const float s = __uint_as_float(half ? pair & 0xffff0000u : pair << 16);
            float f[8];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int shift = 4 * half + 8 * (e >> 1) + 16 * (e & 1);
                    float v = (float)((int)((words[2 * b + j] >> shift) & 15u) - 8) * s;
                    if (part == 1) v -= __bfloat162float(__float2bfloat16_rn(v));
                    f[4 * j + e] = v;
                }
            store8<T>(out + (size_t)row * k + k0, f);
        }
    }
}

template <int NT, int R, bool DUAL, bool G32, bool F16>
int launch(const Args& a, int blocks, cudaStream_t stream) {
    constexpr int bytes = Ring<NT, R, G32, F16>::BYTES;
    NIB_CUDA((allow_smem_once<gemm_int4_kernel<NT, R, DUAL, G32, F16>>(bytes)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.csize > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.csize;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (nib_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    NIB_CUDA(cudaLaunchKernelEx(&cfg, gemm_int4_kernel<NT, R, DUAL, G32, F16>, a));
    return 0;
}

template <int R, bool DUAL, bool G32, bool F16>
int by_tokens(const Args& a, int blocks, cudaStream_t stream) {
    if (a.tokens <= 8) return launch<1, R, DUAL, G32, F16>(a, blocks, stream);
    if (a.tokens <= 16) return launch<2, R, DUAL, G32, F16>(a, blocks, stream);
    if constexpr (R <= 2 && !F16) {
        if (a.tokens <= 32) return launch<4, R, DUAL, G32, F16>(a, blocks, stream);
        return launch<8, R, DUAL, G32, F16>(a, blocks, stream);
    }
    nib_set_error("gemm_int4: four row tiles a warp and prepared activations are for up to 16 tokens");
    return 1;
}

bool fits(int n, int k, int group) { return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0; }

}  // namespace

// The arguments of a product, one block of memory.
struct NibGemmInt4 {
    const void* x; const void* w; const void* scales; const float* bias; void* out;
    void* scratch;              // nib_gemm_int4_scratch bytes, 16-byte aligned; without, the codes meet the activations as they are
    int tokens, n, k, group, ldx, ldo, epi, sms;        // sms: SMs of the device
    float alpha, limit, shift;                          // the constants of EPI_GLU
    int pad;
};

// Bytes of scratch with which a product prepares its activations as 16-bit floats.
NIB_API long long nib_gemm_int4_scratch(int tokens, int k) { return (long long)tokens * k * 2 + (long long)ceil_div(k, 32) * 64 * 4 + 256; }

// out[tokens, n] from the packed weights of n rows (of 2 n rows, gate then up, for the gated epilogues). -1, and nothing done, where
// another product has to take these operands: more than 64 tokens, rows that do not begin on 16 bytes, a gated product whose halves
// are not whole row tiles.
NIB_API int nib_gemm_int4(const void* args, cudaStream_t stream) {
    NibGemmInt4 c;
    memcpy(&c, args, sizeof c);
    const int tokens = c.tokens, n = c.n, k = c.k, group = c.group, epi = c.epi, sms = c.sms;
    const bool dual = epi_dual(epi);
    NIB_REQUIRE(tokens >= 0 && sms > 0 && fits(n, k, group), "gemm_int4: %d tokens, %d x %d weights in groups of %d are not supported", tokens, n, k, group);
    NIB_REQUIRE(epi == EPI_STORE || epi == EPI_ADD || epi == EPI_F32 || dual, "gemm_int4: unknown epilogue %d", epi);
    NIB_REQUIRE((((uintptr_t)c.w) & 15) == 0 && (((uintptr_t)c.scales) & 3) == 0, "gemm_int4: weights must be 16-byte aligned, scales 4-byte");
    NIB_REQUIRE(((uintptr_t)c.scratch & 15) == 0, "gemm_int4: scratch must be 16-byte aligned");
    if (tokens > 64 || c.ldx % 8 != 0 || ((uintptr_t)c.x & 15) != 0 || (dual && n % 16 != 0)) return -1;
    if (tokens == 0) return 0;
    const int out_tiles = ceil_div(n, 16);
    const bool g32 = group == 32, f16 = c.scratch != nullptr;
    Args a{(const __nv_bfloat16*)c.x, (const uint4*)c.w, (const unsigned*)c.scales, c.bias, c.out, nullptr, nullptr, tokens, n, k, c.ldx, c.ldo, epi,
           dual ? 2 * out_tiles : out_tiles, ceil_div(k, 64), group == 32 ? 5 : group == 64 ? 6 : 7, k / group, 1, 1, NibGlu{c.alpha, c.limit, c.shift}};
    if (f16) {
        float* sums = (float*)c.scratch;
        float* factors = sums + (size_t)ceil_div(k, 32) * 64;
        __half* x16 = (__half*)(factors + 64);
        NIB_CUDA(launch_pdl(prepare_f16_kernel, dim3(tokens), dim3(PREP_THREADS), (size_t)0, stream, (const __nv_bfloat16*)c.x, c.ldx, x16, sums, factors, k, g32 ? 32 : 64));
        a.x = (const __nv_bfloat16*)x16;
        a.ldx = k;
        a.sums = sums;
        a.factors = factors;
    }
    // How the work is cut: row tiles a warp (they share the activations' copies), warps of a CTA and CTAs that share K. A tile costs about
    // 60 instructions and a step of a warp 40 besides; an SM issues some 2.2 a cycle, a warp alone one in four.
    int rows = dual ? 2 : 1, best_rows = rows;
    double best = 1e30;
    for (; rows <= (tokens <= 16 ? 4 : 2); rows *= 2)
        for (int ks = 1; ks <= WARPS; ks *= 2)
            for (int cs = 1; cs <= (ks == WARPS && tokens <= 16 ? 4 : 1); ++cs) {
                if (ks * cs > a.k_tiles) continue;
                const int per_token_tile = (tokens + 7) / 8 - 1;             // (more tokens: more copies and products)
                const double step = ceil_div(a.k_tiles, ks * cs) * (rows * (60.0 + 8.0 * per_token_tile) + 40.0 + 12.0 * per_token_tile);
                const double ctas = (double)ceil_div((long long)ceil_div(a.row_tiles, rows) * ks, WARPS) * cs;
                const double busy = ceil(ctas / sms) * WARPS * step / 2.2, alone = 4.0 * step;
                const double cost = (busy > alone ? busy : alone) + (ks > 1 ? 300.0 : 0.0) + (cs > 1 ? 1500.0 : 0.0);
                if (cost < best) { best = cost; best_rows = rows; a.ksplit = ks; a.csize = cs; }
            }
    rows = best_rows;
    const int blocks = ceil_div((long long)ceil_div(a.row_tiles, rows) * a.ksplit, WARPS) * a.csize;
#define CALL(R, DUAL)                                                                                                                                  \
    (f16 ? (g32 ? by_tokens<R, DUAL, true, true>(a, blocks, stream) : by_tokens<R, DUAL, false, true>(a, blocks, stream))                               \
         : (g32 ? by_tokens<R, DUAL, true, false>(a, blocks, stream) : by_tokens<R, DUAL, false, false>(a, blocks, stream)))
    if (dual) return rows == 4 ? CALL(4, true) : CALL(2, true);
    return rows == 4 ? CALL(4, false) : rows == 2 ? CALL(2, false) : CALL(1, false);
#undef CALL
}

// The weights of n rows as bfloat16 or 32-bit numbers [n, k]; part 1: what the rounding to bfloat16 leaves.
NIB_API int nib_unpack_int4(const void* w, const void* scales, void* out, int n, int k, int group, int part, int dtype, cudaStream_t stream) {
    NIB_REQUIRE(fits(n, k, group), "unpack_int4: %d x %d weights in groups of %d are not supported", n, k, group);
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "unpack_int4: unknown dtype %d", dtype);
    NIB_REQUIRE((((uintptr_t)w | (uintptr_t)out) & 15) == 0 && ((uintptr_t)scales & 3) == 0, "unpack_int4: weights and result must be 16-byte aligned, scales 4-byte");
    const int k_tiles = ceil_div(k, 64), shift = group == 32 ? 5 : group == 64 ? 6 : 7;
    const long long items = (long long)ceil_div(n, 16) * k_tiles * 32, grid = (items + 255) / 256;
    NIB_REQUIRE(grid < (1LL << 31) - 1, "unpack_int4: too many weights for one launch");
#define CALL(T) NIB_CUDA(launch_pdl(unpack_int4_kernel<T>, dim3((unsigned)grid), dim3(256), (size_t)0, stream, (const uint4*)w, (const unsigned*)scales, \
                                    (T*)out, n, k, k_tiles, shift, k / group, items, part))
    if (dtype == NIB_F32) CALL(float); else CALL(__nv_bfloat16);
#undef CALL
    return 0;
}
