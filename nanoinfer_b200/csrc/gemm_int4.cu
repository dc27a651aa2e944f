// Products with 4-bit weights: out[tokens, N] = X[tokens, K] . W[N, K]^T, W[n, k] = (code[n, k] - 8) * scale[n, k / group], bfloat16
// activations and scales, 32-bit sums. For up to 64 tokens the weights' bytes are what a product costs, and each is needed once.
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
#include "common.cuh"
#include <cuda_fp16.h>

namespace {

constexpr int WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Weights are read once: they are not to push the activations out of L1.
__device__ __forceinline__ uint4 ldg16_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
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
    int tokens, n_out, k, ldx, ldo, epi, row_tiles, k_tiles, group_shift, groups, ksplit;      // group_shift: log2(group)
    NibGlu glu;
};

// The activations of F16: a CTA a token. x16 [tokens][k] = x * 2^e, sums as Args has them, factors = 2^24 / 2^e. step: 64 or 32.
constexpr int PREP_THREADS = 512;
__global__ void __launch_bounds__(PREP_THREADS)
prepare_f16_kernel(const __nv_bfloat16* __restrict__ x, int ldx, __half* __restrict__ x16, float* __restrict__ sums, float* __restrict__ factors, int k, int step) {
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

// R row tiles a warp, which share the activations they multiply with (two of one matrix, or with DUAL a gate's and an up's); NT tiles
// of 8 tokens; D tiles of weights on their way at any time. ``ksplit`` warps of a CTA share a row unit's K and are summed in order.
template <int NT, int R, bool DUAL, bool G32, bool F16, int D>
__global__ void __launch_bounds__(WARPS * 32)
gemm_int4_kernel(const Args a) {
    extern __shared__ float part[];             // [WARPS][R][NT][4][32] where K is split
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int unit = blockIdx.x * (WARPS / a.ksplit) + warp / a.ksplit, kpart = warp % a.ksplit;
    const int out_tiles = (a.n_out + 15) / 16;
    const int rt0 = DUAL ? unit : unit * R;                                 // first row tile of the unit
    const bool live = rt0 < out_tiles;
    const int per = (a.k_tiles + a.ksplit - 1) / a.ksplit;
    const int begin = live ? min(a.k_tiles, kpart * per) : 0, end = live ? min(a.k_tiles, begin + per) : 0;
    const uint4* wp[R];
    const unsigned* sp[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int rt = min(DUAL ? rt0 + r * out_tiles : rt0 + r, a.row_tiles - 1);      // (a tile behind the last is computed and not stored)
        wp[r] = a.w + (size_t)rt * a.k_tiles * 32 + lane;
        sp[r] = a.scales + (size_t)rt * a.groups * 8 + g;
    }
    pdl_launch_dependents();
    uint4 w[D][R];
    unsigned sc[D][R][G32 ? 2 : 1];
    auto load = [&](int d, int kt) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            w[d][r] = ldg16_stream(wp[r] + (size_t)kt * 32);
            if (G32) {
                sc[d][r][0] = __ldg(sp[r] + (size_t)(2 * kt) * 8);
                sc[d][r][G32 ? 1 : 0] = 2 * kt + 1 < a.groups ? __ldg(sp[r] + (size_t)(2 * kt + 1) * 8) : 0u;
            } else {
                sc[d][r][0] = __ldg(sp[r] + (size_t)((kt << 6) >> a.group_shift) * 8);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (begin + d < end) load(d, begin + d);
    pdl_wait();                                 // weights are nobody's output; the activations are
    const __nv_bfloat16* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = n * 8 + g < a.tokens ? a.x + (size_t)(n * 8 + g) * a.ldx + 8 * t : nullptr;        // (16 bits either way)

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
    for (int base = begin; base < end; base += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int kt = base + d;
            if (kt >= end) break;
            uint4 x[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    x[n][b] = make_uint4(0u, 0u, 0u, 0u);
                    if (xp[n] != nullptr && kt * 64 + b * 32 < a.k) x[n][b] = *reinterpret_cast<const uint4*>(xp[n] + kt * 64 + b * 32);
                }
            float s[R][NT][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (G32 || b == 0) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float2 c = make_float2(0.f, 0.f);
                        if (F16) c = __ldg(reinterpret_cast<const float2*>(a.sums + (size_t)min(G32 ? 2 * kt + b : kt, a.k / (G32 ? 32 : 64) - 1) * 64 + n * 8 + 2 * t));
#pragma unroll
                        for (int r = 0; r < R; ++r) { s[r][n][0] = c.x; s[r][n][1] = c.y; s[r][n][2] = 16.f * c.x; s[r][n][3] = 16.f * c.y; }
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    unsigned f[4];
                    auto multiply = [&](unsigned word, bool second) {
                        if (F16) codes_of(word, f); else weights_of(word, f);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const unsigned b0 = second ? x[n][b].z : x[n][b].x, b1 = second ? x[n][b].w : x[n][b].y;
                            if (F16) mma_f16(s[r][n], f, b0, b1); else mma_bf16(s[r][n], f, b0, b1);
                        }
                    };
                    multiply(b == 0 ? w[d][r].x : w[d][r].z, false);
                    multiply(b == 0 ? w[d][r].y : w[d][r].w, true);
                }
                if (G32 || b == 1) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int n = 0; n < NT; ++n) add(acc[r][n], s[r][n], sc[d][r][G32 ? b : 0]);
                }
            }
            if (kt + D < end) load(d, kt + D);
        }
    }

    // ---- the results of token tile n: element e is row g + 8 * (e / 2), token n * 8 + 2t + (e & 1)
    auto emit = [&](float (&v)[R][4], int n) {
        if (F16) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int tok = n * 8 + 2 * t + j;
                const float f = tok < a.tokens ? __ldg(a.factors + tok) : 0.f;
#pragma unroll
                for (int r = 0; r < R; ++r) { v[r][j] *= f; v[r][2 + j] *= f * 0.0625f; }
            }
        }
#pragma unroll
        for (int r = 0; r < (DUAL ? 1 : R); ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = (rt0 + r) * 16 + g + 8 * (e >> 1), tok = n * 8 + 2 * t + (e & 1);
                if (f >= a.n_out || tok >= a.tokens) continue;
                const size_t at = (size_t)tok * a.ldo + f;
                if (DUAL) {
                    const float gate = v[0][e], up = v[R - 1][e];
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
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(((warp * R + r) * NT + n) * 4 + e) * 32 + lane] = acc[r][n][e];
    __syncthreads();
    if (!live) return;
    const int first = warp - kpart;             // the unit's first warp
    for (int n = kpart; n < NT; n += a.ksplit) {
        float v[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float sum = 0.f;
                for (int p = 0; p < a.ksplit; ++p) sum += part[((((first + p) * R + r) * NT + n) * 4 + e) * 32 + lane];
                v[r][e] = sum;
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
    constexpr int D = NT <= 2 ? 4 : 2;
    const size_t smem = a.ksplit > 1 ? (size_t)WARPS * R * NT * 4 * 32 * 4 : 0;
    static const cudaError_t set = cudaFuncSetAttribute(gemm_int4_kernel<NT, R, DUAL, G32, F16, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        WARPS * R * NT * 4 * 32 * 4);
    NIB_CUDA(set);
    NIB_CUDA(launch_pdl(gemm_int4_kernel<NT, R, DUAL, G32, F16, D>, dim3(blocks), dim3(WARPS * 32), smem, stream, a));
    return 0;
}

template <int R, bool DUAL, bool G32, bool F16>
int by_tokens(const Args& a, int blocks, cudaStream_t stream) {
    if (a.tokens <= 8) return launch<1, R, DUAL, G32, F16>(a, blocks, stream);
    if (a.tokens <= 16) return launch<2, R, DUAL, G32, F16>(a, blocks, stream);
    if (a.tokens <= 32) return launch<4, R, DUAL, G32, F16>(a, blocks, stream);
    return launch<8, R, DUAL, G32, F16>(a, blocks, stream);
}

bool fits(int n, int k, int group) { return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0; }

}  // namespace

// The arguments of a product, one block of memory.
struct NibGemmInt4 {
    const void* x; const void* w; const void* scales; const float* bias; void* out;
    void* scratch;                                      // nib_gemm_int4_scratch bytes, 16-byte aligned
    int tokens, n, k, group, ldx, ldo, epi, sms;        // sms: SMs of the device
    float alpha, limit, shift;                          // the constants of EPI_GLU
    int pad;
};

// Whether a product's activations are prepared as 16-bit floats, and the scratch bytes that takes (0: not).
static long long f16_scratch(int tokens, int n, int k, bool dual) {
    return (long long)(dual ? 2 : 1) * n * k / 2 >= (4 << 20) ? (long long)tokens * k * 2 + (long long)ceil_div(k, 32) * 64 * 4 + 256 : 0;
}
NIB_API long long nib_gemm_int4_scratch(int tokens, int n, int k, int dual) { return tokens > 64 ? 0 : f16_scratch(tokens, n, k, dual != 0); }

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
    NIB_REQUIRE((((uintptr_t)c.w) & 15) == 0 && (((uintptr_t)c.scales) & 3) == 0, "gemm_int4: weights must be 16-byte aligned");
    if (tokens > 64 || c.ldx % 8 != 0 || ((uintptr_t)c.x & 15) != 0 || (dual && n % 16 != 0)) return -1;
    if (tokens == 0) return 0;
    const int out_tiles = ceil_div(n, 16);
    const bool g32 = group == 32, f16 = c.scratch != nullptr && f16_scratch(tokens, n, k, dual) > 0;
    Args a{(const __nv_bfloat16*)c.x, (const uint4*)c.w, (const unsigned*)c.scales, c.bias, c.out, nullptr, nullptr, tokens, n, k, c.ldx, c.ldo, epi,
           dual ? 2 * out_tiles : out_tiles, ceil_div(k, 64), group == 32 ? 5 : group == 64 ? 6 : 7, k / group, 1, NibGlu{c.alpha, c.limit, c.shift}};
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
    // Two row tiles a warp share the activations' loads; one where two would leave SMs without work.
    const bool two = dual || (tokens <= 32 && out_tiles >= 2 * WARPS * sms);
    const int units = dual || !two ? out_tiles : ceil_div(out_tiles, 2);
    // As many warps share a unit's K as it takes to have 16 warps an SM, while each has a tile.
    while (a.ksplit < WARPS && (long long)units * a.ksplit < 16LL * sms && a.k_tiles >= 2 * a.ksplit) a.ksplit *= 2;
    const int blocks = ceil_div((long long)units * a.ksplit, WARPS);
#define CALL(R, DUAL)                                                                                                                                  \
    (f16 ? (g32 ? by_tokens<R, DUAL, true, true>(a, blocks, stream) : by_tokens<R, DUAL, false, true>(a, blocks, stream))                               \
         : (g32 ? by_tokens<R, DUAL, true, false>(a, blocks, stream) : by_tokens<R, DUAL, false, false>(a, blocks, stream)))
    if (dual) return CALL(2, true);
    return two ? CALL(2, false) : CALL(1, false);
#undef CALL
}

// The weights of n rows as bfloat16 or 32-bit numbers [n, k]; part 1: what the rounding to bfloat16 leaves.
NIB_API int nib_unpack_int4(const void* w, const void* scales, void* out, int n, int k, int group, int part, int dtype, cudaStream_t stream) {
    NIB_REQUIRE(fits(n, k, group), "unpack_int4: %d x %d weights in groups of %d are not supported", n, k, group);
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "unpack_int4: unknown dtype %d", dtype);
    NIB_REQUIRE((((uintptr_t)w | (uintptr_t)out) & 15) == 0, "unpack_int4: weights and result must be 16-byte aligned");
    const int k_tiles = ceil_div(k, 64), shift = group == 32 ? 5 : group == 64 ? 6 : 7;
    const long long items = (long long)ceil_div(n, 16) * k_tiles * 32, grid = (items + 255) / 256;
    NIB_REQUIRE(grid < (1LL << 31) - 1, "unpack_int4: too many weights for one launch");
#define CALL(T) NIB_CUDA(launch_pdl(unpack_int4_kernel<T>, dim3((unsigned)grid), dim3(256), (size_t)0, stream, (const uint4*)w, (const unsigned*)scales, \
                                    (T*)out, n, k, k_tiles, shift, k / group, items, part))
    if (dtype == NIB_F32) CALL(float); else CALL(__nv_bfloat16);
#undef CALL
    return 0;
}
