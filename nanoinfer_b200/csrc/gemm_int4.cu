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
#include "common.cuh"

namespace {

constexpr int WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Weights are read once: they are not to push the activations out of L1.
__device__ __forceinline__ uint4 ldg16_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
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
    int tokens, n_out, k, ldx, ldo, epi, row_tiles, k_tiles, group_shift, groups, ksplit;      // group_shift: log2(group)
    NibGlu glu;
};

// R row tiles a warp, which share the activations they multiply with (two of one matrix, or with DUAL a gate's and an up's); NT tiles
// of 8 tokens; D tiles of weights on their way at any time. ``ksplit`` warps of a CTA share a row unit's K and are summed in order.
template <int NT, int R, bool DUAL, bool G32, int D>
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
    for (int n = 0; n < NT; ++n) xp[n] = n * 8 + g < a.tokens ? a.x + (size_t)(n * 8 + g) * a.ldx + 8 * t : nullptr;

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
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int n = 0; n < NT; ++n) s[r][n][0] = s[r][n][1] = s[r][n][2] = s[r][n][3] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    unsigned f[4];
                    weights_of(b == 0 ? w[d][r].x : w[d][r].z, f);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(s[r][n], f, x[n][b].x, x[n][b].y);
                    weights_of(b == 0 ? w[d][r].y : w[d][r].w, f);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(s[r][n], f, x[n][b].z, x[n][b].w);
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
    auto emit = [&](const float (&v)[R][4], int n) {
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

template <int NT, int R, bool DUAL, bool G32>
int launch(const Args& a, int blocks, cudaStream_t stream) {
    constexpr int D = NT <= 2 ? 4 : 2;
    const size_t smem = a.ksplit > 1 ? (size_t)WARPS * R * NT * 4 * 32 * 4 : 0;
    static const cudaError_t set = cudaFuncSetAttribute(gemm_int4_kernel<NT, R, DUAL, G32, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        WARPS * R * NT * 4 * 32 * 4);
    NIB_CUDA(set);
    NIB_CUDA(launch_pdl(gemm_int4_kernel<NT, R, DUAL, G32, D>, dim3(blocks), dim3(WARPS * 32), smem, stream, a));
    return 0;
}

template <int R, bool DUAL, bool G32>
int by_tokens(const Args& a, int blocks, cudaStream_t stream) {
    if (a.tokens <= 8) return launch<1, R, DUAL, G32>(a, blocks, stream);
    if (a.tokens <= 16) return launch<2, R, DUAL, G32>(a, blocks, stream);
    if (a.tokens <= 32) return launch<4, R, DUAL, G32>(a, blocks, stream);
    return launch<8, R, DUAL, G32>(a, blocks, stream);
}

bool fits(int n, int k, int group) { return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0; }

}  // namespace

// The arguments of a product, one block of memory.
struct NibGemmInt4 {
    const void* x; const void* w; const void* scales; const float* bias; void* out;
    int tokens, n, k, group, ldx, ldo, epi, sms;        // sms: SMs of the device
    float alpha, limit, shift;                          // the constants of EPI_GLU
    int pad;
};

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
    Args a{(const __nv_bfloat16*)c.x, (const uint4*)c.w, (const unsigned*)c.scales, c.bias, c.out, tokens, n, k, c.ldx, c.ldo, epi,
           dual ? 2 * out_tiles : out_tiles, ceil_div(k, 64), group == 32 ? 5 : group == 64 ? 6 : 7, k / group, 1, NibGlu{c.alpha, c.limit, c.shift}};
    // Two row tiles a warp share the activations' loads; one where two would leave SMs without work.
    const bool two = dual || (tokens <= 32 && out_tiles >= 2 * WARPS * sms);
    const int units = dual || !two ? out_tiles : ceil_div(out_tiles, 2);
    // As many warps share a unit's K as it takes to have 16 warps an SM, while each has a tile.
    while (a.ksplit < WARPS && (long long)units * a.ksplit < 16LL * sms && a.k_tiles >= 2 * a.ksplit) a.ksplit *= 2;
    const int blocks = ceil_div((long long)units * a.ksplit, WARPS);
    const bool g32 = group == 32;
    if (dual) return g32 ? by_tokens<2, true, true>(a, blocks, stream) : by_tokens<2, true, false>(a, blocks, stream);
    if (two) return g32 ? by_tokens<2, false, true>(a, blocks, stream) : by_tokens<2, false, false>(a, blocks, stream);
    return g32 ? by_tokens<1, false, true>(a, blocks, stream) : by_tokens<1, false, false>(a, blocks, stream);
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
