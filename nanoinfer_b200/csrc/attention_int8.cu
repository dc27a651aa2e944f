// Attention of single decoded tokens over the 8-bit cache (cache_int8.cu): codes of 8 bits, a scale for each page and kv head.
//
//     s_j = scale * q . (ck_j * sk_j),  w = softmax(s),  o = sum_j w_j cv_j sv_j        (keys at positions lo..p)
//
// The key scale multiplies a score. The value scale would multiply a row of V before a tensor core sums it; it goes into the
// softmax instead: with t_j = s_j log2(e) + log2(sv_j) and a running reference M of max t,
//     w_j = 2^(s_j log2(e) - M + 20),  p_j = w_j sv_j 2^-20  (about 1 at most),  l = sum_j w_j,  o = 2^20 sum_j p_j cv_j / l,
// so the tensor core multiplies p_j, in 16 bits, with whole numbers that 16 bits hold exactly, and a row is right to its own
// size however much the scales of its blocks differ. l and o are summed in 32 bits; with scales of 2^-80 .. 2^121 the terms of l that
// count lie between 2^-125 and 2^106 (the 20 is what centres them).
//
// Two kernels. The one on the tensor cores takes heads of 64 and 128, at most 16 query heads a kv head and pages of a multiple of
// 8 tokens; the general one takes any shape and 32-bit rows. The keys of a (token, kv head) are cut in one of two ways. Few rows: among
// the CTAs of a cluster, which merge their partial (max, sum, output) through distributed shared memory and store the row. Many, or
// long ones: into spans of equal length, a CTA each, whatever the contexts' lengths, merged in order by a second kernel (clusters of
// eight find room on 15 places of the GPU at a time, and contexts of different lengths would keep SMs waiting).
#include "attention_common.cuh"
#include "pipeline.cuh"
#include <cuda_fp16.h>

using namespace nibp;

namespace {

constexpr int WARPS = 4;
constexpr float LIFT = 20.f, UNLIFT = 0x1p-20f, RELIFT = 0x1p20f;

struct Args {
    const int* ctx_lens; const int* block_table; const signed char* k_pages; const signed char* v_pages;
    const float* k_scales; const float* v_scales; float* part_o; float* part_ml;
    int q_stride, bt_stride, bt_width, page_size, shift, num_pages, heads, kv_heads, n_rep, head_dim, window;
    int csize, span, parts;         // CTAs of a cluster and span 0; or 1, the keys of a span and the most spans a row has
    float scale;
};

__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// The keys lo..p of a token, and of those the steps of ``step`` keys (aligned to absolute multiples) that are this CTA's.
struct Range { int lo, p, begin, end; };
__device__ __forceinline__ Range range_of(const Args& a, int token, int step) {
    Range r;
    r.p = a.ctx_lens[token] - 1;                            // the token's own position; -1: a padding row
    r.lo = a.window > 0 ? max(0, r.p - a.window + 1) : 0;
    const int first = r.lo / step, n = r.p >= 0 ? r.p / step - first + 1 : 0;
    const int per = a.span ? a.span / step : (n + a.csize - 1) / a.csize;
    r.begin = first + blockIdx.x * per;
    r.end = min(first + n, r.begin + per);
    return r;
}

// What a CTA leaves: its output, relative to its own maximum, in cta_o [n_rep][hd], its (max, sum) in cta_ml. With spans it is stored
// for the kernel behind; in a cluster this CTA finishes its slice of the outputs. All threads take part.
template <typename T>
__device__ __forceinline__ void finish(const float* cta_o, const float* cta_ml, const Args& a, int hd, T* __restrict__ out, int threads) {
    const size_t th0 = (size_t)blockIdx.y * a.heads + (size_t)blockIdx.z * a.n_rep;
    const int total = a.n_rep * hd;
    if (a.span) {
        for (int i = threadIdx.x; i < total; i += threads) {
            const int row = i / hd, d = i - row * hd;
            a.part_o[((th0 + row) * a.parts + blockIdx.x) * hd + d] = cta_o[i];
        }
        for (int i = threadIdx.x; i < 2 * a.n_rep; i += threads) a.part_ml[((th0 + (i >> 1)) * a.parts + blockIdx.x) * 2 + (i & 1)] = cta_ml[i];
        return;
    }
    if (a.csize > 1) cluster_sync(); else __syncthreads();
    const int rank = a.csize > 1 ? (int)cluster_rank() : 0;
    const int slice = (total + a.csize - 1) / a.csize, end = min(total, (rank + 1) * slice);
    for (int i = rank * slice + threadIdx.x; i < end; i += threads) {
        const int row = i / hd, d = i - row * hd;
        float m_all = -INFINITY, l_all = 0.f, acc = 0.f;
        if (a.csize > 1) {
            float mr[8], lr[8], orr[8];        // asked for together: one round trip
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                mr[r] = -INFINITY; lr[r] = 0.f; orr[r] = 0.f;
                if (r < a.csize) {
                    mr[r] = ld_peer_f32(peer_smem(cta_ml + row * 2, r));
                    lr[r] = ld_peer_f32(peer_smem(cta_ml + row * 2 + 1, r));
                    orr[r] = ld_peer_f32(peer_smem(cta_o + i, r));
                }
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) m_all = fmaxf(m_all, mr[r]);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float f = (mr[r] == -INFINITY) ? 0.f : exp2_ftz(mr[r] - m_all);
                l_all += lr[r] * f;
                acc += orr[r] * f;
            }
        } else {
            l_all = cta_ml[row * 2 + 1];
            acc = cta_o[i];
        }
        Elem<T>::store(out + (th0 + row) * hd + d, l_all == 0.f ? 0.f : acc / l_all * RELIFT);      // a row that sees nothing is zero, an undefined one NaN
    }
    if (a.csize > 1) cluster_sync();        // nobody leaves while a peer may still read its shared memory
}

// Merges the spans of one (token, head), in order. grid: (heads, tokens). step: as the kernel before cut the keys.
template <typename T>
__global__ void __launch_bounds__(128)
merge_int8_kernel(T* __restrict__ out, const Args a, int step) {
    pdl_wait();
    pdl_launch_dependents();
    const int p = a.ctx_lens[blockIdx.y] - 1, lo = a.window > 0 ? max(0, p - a.window + 1) : 0, hd = a.head_dim;
    const int steps = p >= 0 ? p / step - lo / step + 1 : 0, per = a.span / step;
    const int parts = min(a.parts, (steps + per - 1) / per);
    const size_t th = (size_t)blockIdx.y * a.heads + blockIdx.x;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + th * a.parts;
    const float* po = a.part_o + th * a.parts * hd;
    float m = -INFINITY;
    for (int s = 0; s < parts; ++s) m = fmaxf(m, ml[s].x);
    for (int d = threadIdx.x; d < hd; d += 128) {
        float l = 0.f, acc = 0.f;
        for (int s0 = 0; s0 < parts; s0 += 8) {
            float v[8];
            float2 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = min(s0 + u, parts - 1);
                v[u] = po[(size_t)s * hd + d];
                x[u] = ml[s];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = s0 + u >= parts || x[u].x == -INFINITY ? 0.f : exp2_ftz(x[u].x - m);
                if (s0 + u < parts) { l += x[u].y * f; acc += v[u] * f; }
            }
        }
        Elem<T>::store(out + th * hd + d, l == 0.f ? 0.f : acc / l * RELIFT);
    }
}

// log2 of a value scale, for the reference M alone (any value near it serves). Of a scale of 0 or one below the cache's: what a score
// may be above M without the sum leaving the range of 32 bits.
__device__ __forceinline__ float reference_log2(float scale) { return fmaxf(__log2f(scale), -80.f); }

__device__ __forceinline__ int page_at(const Args& a, const int* __restrict__ bt, int key, int& slot) {
    const int lp = a.shift >= 0 ? key >> a.shift : key / a.page_size;
    slot = key - lp * a.page_size;
    if (lp >= a.bt_width) return -1;
    const int page = __ldg(bt + lp);
    return page < a.num_pages ? page : -1;
}

// ------------------------------------------------------------------------------------------ on the tensor cores
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two value codes (bytes sel of ``biased``, codes plus 128) as 16-bit floats: in the low bits of 1024.0 they are 1152 + code, exactly.
__device__ __forceinline__ unsigned two_codes(unsigned biased, unsigned sel) {
    const unsigned u = __byte_perm(biased, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}

// The codes of KU * 16 keys as a warp holds them: thread (g, t) has 16-byte pieces t, t + 4 of the key rows g and g + 8, and the
// dims g * HD/8 .. of the value rows 2t, 2t + 1, 2t + 8, 2t + 9: every row of 64 or 128 bytes is read whole, by one instruction,
// straight into the registers that the tensor core is fed from.
template <int HD, int KU> struct Codes {
    uint4 k[KU][2][HD / 64];
    unsigned v[KU][4][HD / 32];
    float ks[KU][2], vs[KU][2];         // of the rows 0..7 and 8..15
};

// A key code enters the tensor core as the 16-bit number (code + 128) 2^-24, which is the code's byte, its first bit turned over, with
// zeros before it; what the 128 adds to a score, 128 2^-24 sum of the head's elements, is what the accumulator begins at.
// WHOLE: pages of a multiple of 16 tokens, so that 16 keys lie in one.
template <int HD, int NH, int KU, bool WHOLE>
__global__ void __launch_bounds__(WARPS * 32)
attention_int8_mma_kernel(const __nv_bfloat16* __restrict__ q_rows, __nv_bfloat16* __restrict__ out, const Args a) {
    constexpr int STEP = KU * 16, MS = HD + 4, ROWS = NH * 8;
    extern __shared__ __align__(16) float smem[];
    const int token = blockIdx.y, kvh = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();
    const Range range = range_of(a, token, STEP);
    const int p = range.p, lo = range.lo, end = range.end;
    if (a.span && range.begin >= end) return;               // (a shorter context than the longest one)
    const int* bt = a.block_table + (size_t)token * a.bt_stride;
    const long long page_bytes = (long long)a.kv_heads * a.page_size * HD;
    const signed char* k_lane = a.k_pages + (size_t)kvh * a.page_size * HD + g * HD + t * 16;
    const signed char* v_lane = a.v_pages + (size_t)kvh * a.page_size * HD + 2 * t * HD + g * (HD / 8);

    // A page that the request does not hold is read as the pool's first with scales of 0: nothing leaves the pool.
    auto load = [&](Codes<HD, KU>& c, int step) {
#pragma unroll
        for (int ku = 0; ku < KU; ++ku) {
            int slot = 0, page = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = step * STEP + ku * 16 + h * 8;
                if (!WHOLE || h == 0) page = (key <= p && key + (WHOLE ? 16 : 8) > lo) ? page_at(a, bt, key, slot) : -1;
                const bool held = page >= 0;
                const int at_page = held ? page : 0, at_slot = (held ? slot : 0) + (WHOLE ? h * 8 : 0);
                const long long at = at_page * page_bytes + at_slot * HD;
                if (!WHOLE || h == 0) {
                    const size_t block = (size_t)at_page * a.kv_heads + kvh;
                    c.ks[ku][h] = __ldg(a.k_scales + block);
                    c.vs[ku][h] = __ldg(a.v_scales + block);
                    if (!held) c.ks[ku][h] = c.vs[ku][h] = 0.f;
                } else {
                    c.ks[ku][h] = c.ks[ku][0];
                    c.vs[ku][h] = c.vs[ku][0];
                }
#pragma unroll
                for (int i = 0; i < HD / 64; ++i) c.k[ku][h][i] = __ldg(reinterpret_cast<const uint4*>(k_lane + at + i * 64));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (HD == 64) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(v_lane + at + j * HD));
                        c.v[ku][2 * h + j][0] = x.x; c.v[ku][2 * h + j][1] = x.y;
                    } else {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(v_lane + at + j * HD));
                        c.v[ku][2 * h + j][0] = x.x; c.v[ku][2 * h + j][1] = x.y;
                        c.v[ku][2 * h + j][2] = x.z; c.v[ku][2 * h + j][3] = x.w;
                    }
                }
            }
        }
    };
    Codes<HD, KU> c[2];
    int step = range.begin + warp;
    if (step < end) load(c[0], step);

    // Q^T as the column operand, its dims in the order in which the key rows' pieces hold them. A head is scaled by a power of two so
    // that its largest element lies in 2^12 .. 2^13: 16-bit floats then hold every element that counts exactly.
    unsigned qb[HD / 16][NH][2];
    float factor[NH][2], bias[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
        const int head = nh * 8 + g;
        const __nv_bfloat16* qp = q_rows + (size_t)token * a.q_stride + (size_t)(kvh * a.n_rep + head) * HD + t * 16;
        unsigned raw[HD / 16][2], top = 0;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                raw[kk][j] = head < a.n_rep ? *reinterpret_cast<const unsigned*>(qp + (kk >> 2) * 64 + (kk & 3) * 4 + 2 * j) : 0u;
                top = max(top, max(raw[kk][j] & 0x7fffu, (raw[kk][j] >> 16) & 0x7fffu));
            }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the exponent field of the largest element: 2^(139 - e) takes it to 2^12 (in two factors: the power may leave the range)
        const int e = (int)(top >> 7), up = (e == 0 || e == 255) ? 0 : 139 - e;
        const float f1 = __uint_as_float((unsigned)(127 + up / 2) << 23), f2 = __uint_as_float((unsigned)(127 + up - up / 2) << 23);
        float sum = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                qb[kk][nh][j] = pack_f16(__uint_as_float(raw[kk][j] << 16) * f1 * f2, __uint_as_float(raw[kk][j] & 0xffff0000u) * f1 * f2);
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&qb[kk][nh][j]));
                sum += x.x + x.y;
            }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // 2^24 / 2^up, in factors that stay in range
        const float mine = a.scale * LOG2E * __uint_as_float((unsigned)(127 - up / 2) << 23) * __uint_as_float((unsigned)(127 - (up - up / 2)) << 23) * 0x1p24f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {           // of the heads 2t, 2t + 1
            factor[nh][q] = __shfl_sync(0xffffffffu, mine, 8 * t + 4 * q);
            bias[nh][q] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * q) * (-128.f * 0x1p-24f);
        }
    }

    float o[HD / 16][NH][4], m_ref[NH][2], l_part[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
        m_ref[nh][0] = m_ref[nh][1] = -INFINITY;
        l_part[nh][0] = l_part[nh][1] = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[d][nh][0] = o[d][nh][1] = o[d][nh][2] = o[d][nh][3] = 0.f;
    }

    auto compute = [&](const Codes<HD, KU>& c, int step) {
        float s[KU][NH][4];
        // S^T = K Q^T
#pragma unroll
        for (int ku = 0; ku < KU; ++ku) {
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) { s[ku][nh][0] = s[ku][nh][2] = bias[nh][0]; s[ku][nh][1] = s[ku][nh][3] = bias[nh][1]; }
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const unsigned w0[4] = {c.k[ku][0][i].x, c.k[ku][0][i].y, c.k[ku][0][i].z, c.k[ku][0][i].w};
                const unsigned w1[4] = {c.k[ku][1][i].x, c.k[ku][1][i].y, c.k[ku][1][i].z, c.k[ku][1][i].w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const unsigned u0 = w0[b] ^ 0x80808080u, u1 = w1[b] ^ 0x80808080u;
                    const unsigned a0 = __byte_perm(u0, 0, 0x4140), a1 = __byte_perm(u1, 0, 0x4140), a2 = __byte_perm(u0, 0, 0x4342), a3 = __byte_perm(u1, 0, 0x4342);
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh) mma_f16(s[ku][nh], a0, a1, a2, a3, qb[i * 4 + b][nh][0], qb[i * 4 + b][nh][1]);
                }
            }
        }
        // element e of a tile: key g + 8 * (e / 2), head 2t + (e & 1)
        const int key0 = step * STEP + g;
        const bool edge = step * STEP < lo || step * STEP + STEP - 1 > p;
        float lv[KU][2], vs[KU][2];
#pragma unroll
        for (int ku = 0; ku < KU; ++ku)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                lv[ku][h] = WHOLE && h == 1 ? lv[ku][0] : reference_log2(c.vs[ku][h]);
                vs[ku][h] = WHOLE && h == 1 ? vs[ku][0] : c.vs[ku][h] * UNLIFT;
            }
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int ku = 0; ku < KU; ++ku)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = s[ku][nh][e] * (factor[nh][e & 1] * c.ks[ku][e >> 1]);
                    if (edge) {
                        const int key = key0 + ku * 16 + 8 * (e >> 1);
                        if (key < lo || key > p) v = -INFINITY;
                    }
                    s[ku][nh][e] = v;
                    top[e & 1] = fmaxf(top[e & 1], v + lv[ku][e >> 1]);
                }
            // the reference moves only where a key is 2^6 above it: p stays far inside 16 bits meanwhile
            if (__any_sync(0xffffffffu, top[0] > m_ref[nh][0] + 6.f || top[1] > m_ref[nh][1] + 6.f)) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 4));
                    top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 8));
                    top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 16));
                    const float m_new = fmaxf(m_ref[nh][q], top[q]);
                    const float corr = (m_ref[nh][q] == -INFINITY) ? 0.f : exp2_ftz(m_ref[nh][q] - m_new);
                    m_ref[nh][q] = m_new;
                    l_part[nh][q] *= corr;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) { o[d][nh][q] *= corr; o[d][nh][2 + q] *= corr; }
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float m_use = (m_ref[nh][q] == -INFINITY) ? 0.f : m_ref[nh][q] - LIFT;       // nothing visible yet: 2^(-inf - 0) = 0
#pragma unroll
                for (int ku = 0; ku < KU; ++ku)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float w = exp2_ftz(s[ku][nh][2 * h + q] - m_use);
                        l_part[nh][q] += w;
                        float pv = w * vs[ku][h];
                        if (edge && w == 0.f) pv = 0.f;             // (a hidden key's block may be undefined)
                        s[ku][nh][2 * h + q] = pv;
                    }
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int ku = 0; ku < KU; ++ku) {
            unsigned pb[NH][2];
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
                pb[nh][0] = movmatrix_trans(pack_f16(s[ku][nh][0], s[ku][nh][1]));
                pb[nh][1] = movmatrix_trans(pack_f16(s[ku][nh][2], s[ku][nh][3]));
            }
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {             // four dims: two row tiles of V^T
                const unsigned x0 = c.v[ku][0][w] ^ 0x80808080u, x1 = c.v[ku][1][w] ^ 0x80808080u;
                const unsigned x2 = c.v[ku][2][w] ^ 0x80808080u, x3 = c.v[ku][3][w] ^ 0x80808080u;
                const unsigned lo01 = __byte_perm(x0, x1, 0x5140), hi01 = __byte_perm(x0, x1, 0x7362);      // dims 0, 1 and 2, 3 of two keys
                const unsigned lo23 = __byte_perm(x2, x3, 0x5140), hi23 = __byte_perm(x2, x3, 0x7362);
                const unsigned d0a = two_codes(lo01, 0x4140), d1a = two_codes(lo01, 0x4342), d0b = two_codes(lo23, 0x4140), d1b = two_codes(lo23, 0x4342);
                const unsigned d2a = two_codes(hi01, 0x4140), d3a = two_codes(hi01, 0x4342), d2b = two_codes(hi23, 0x4140), d3b = two_codes(hi23, 0x4342);
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    mma_f16(o[2 * w][nh], d0a, d1a, d0b, d1b, pb[nh][0], pb[nh][1]);
                    mma_f16(o[2 * w + 1][nh], d2a, d3a, d2b, d3b, pb[nh][0], pb[nh][1]);
                }
            }
        }
    };

    while (step < end) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (step < end) {
                if (step + WARPS < end) load(c[b ^ 1], step + WARPS);
                compute(c[b], step);
                step += WARPS;
            }
        }
    }

    // ---- merge the warps through shared memory
    float* sm_o = smem;                                     // [WARPS][ROWS][MS]
    float* sm_ml = sm_o + WARPS * ROWS * MS;                // [WARPS][ROWS][2]
    float* cta_o = sm_ml + WARPS * ROWS * 2;                // [ROWS][HD]
    float* cta_ml = cta_o + ROWS * HD;                      // [ROWS][2]
#pragma unroll
    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int row = warp * ROWS + nh * 8 + 2 * t + q;
            float l = l_part[nh][q];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)           // row g of tile d is the dim g * HD/8 + 2d, row g + 8 the one behind it
                *reinterpret_cast<float2*>(sm_o + row * MS + g * (HD / 8) + 2 * d) = make_float2(o[d][nh][q], o[d][nh][2 + q]);
            if (g == 0) { sm_ml[row * 2] = m_ref[nh][q]; sm_ml[row * 2 + 1] = l; }
        }
    __syncthreads();
    for (int i = tid; i < a.n_rep * HD; i += WARPS * 32) {
        const int row = i / HD, d = i - row * HD;
        float mw[WARPS], m_row = -INFINITY, acc = 0.f, l_row = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { mw[w] = sm_ml[(w * ROWS + row) * 2]; m_row = fmaxf(m_row, mw[w]); }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = (mw[w] == -INFINITY) ? 0.f : exp2_ftz(mw[w] - m_row);
            acc += sm_o[(w * ROWS + row) * MS + d] * f;
            l_row += sm_ml[(w * ROWS + row) * 2 + 1] * f;
        }
        cta_o[i] = acc;
        if (d == 0) { cta_ml[row * 2] = m_row; cta_ml[row * 2 + 1] = l_row; }
    }
    if (a.span) __syncthreads();
    finish(cta_o, cta_ml, a, HD, out, WARPS * 32);
}

template <int HD, int NH> constexpr int mma_smem() { return (WARPS * NH * 8 * (HD + 4 + 2) + NH * 8 * (HD + 2)) * 4; }

// ------------------------------------------------------------------------------------------ any shape
// Tiles of 32 keys, as 32-bit values in shared memory: a thread has one (query head, key) of the scores at a time, then one
// (query head, dim) of the sums. VEC: heads of a multiple of 16, whose rows are read 16 bytes at a time.
constexpr int GT = 32, GEN_THREADS = 128;

template <typename T, bool VEC>
__global__ void __launch_bounds__(GEN_THREADS)
attention_int8_any_kernel(const T* __restrict__ q_rows, T* __restrict__ out, const Args a) {
    extern __shared__ __align__(16) float smem[];
    const int hd = a.head_dim, n_rep = a.n_rep, token = blockIdx.y, kvh = blockIdx.z, tid = threadIdx.x;
    const int ks_stride = VEC ? hd + 4 : hd | 1;        // (a warp's threads read 32 rows at the same column)
    float* kt = smem;                           // [GT][ks_stride]
    float* vt = kt + GT * ks_stride;            // [GT][hd]
    float* q = vt + GT * hd;                    // [n_rep][hd]
    float* cta_o = q + n_rep * hd;              // [n_rep][hd]
    float* w = cta_o + n_rep * hd;              // [n_rep][GT]
    float* corr = w + n_rep * GT;               // [n_rep]
    float* cta_ml = corr + n_rep;               // [n_rep][2]
    __shared__ float ks[GT], vs[GT];
    __shared__ long long from[GT];              // where a key's codes are; -1: nowhere
    pdl_wait();
    pdl_launch_dependents();
    const Range range = range_of(a, token, GT);
    const int p = range.p, lo = range.lo;
    if (a.span && range.begin >= range.end) return;
    const int* bt = a.block_table + (size_t)token * a.bt_stride;
    for (int i = tid; i < n_rep * hd; i += GEN_THREADS) {
        q[i] = Elem<T>::load(q_rows + (size_t)token * a.q_stride + (size_t)kvh * n_rep * hd + i) * (a.scale * LOG2E);
        cta_o[i] = 0.f;
    }
    for (int i = tid; i < n_rep; i += GEN_THREADS) { cta_ml[2 * i] = -INFINITY; cta_ml[2 * i + 1] = 0.f; }
    for (int tile = range.begin; tile < range.end; ++tile) {
        __syncthreads();
        if (tid < GT) {
            const int key = tile * GT + tid;
            int slot = 0;
            const int page = key >= lo && key <= p ? page_at(a, bt, key, slot) : -1;
            const size_t block = (size_t)max(page, 0) * a.kv_heads + kvh;
            from[tid] = page >= 0 ? (long long)((block * a.page_size + slot) * hd) : -1;
            ks[tid] = page >= 0 ? __ldg(a.k_scales + block) : 0.f;
            vs[tid] = page >= 0 ? __ldg(a.v_scales + block) : 0.f;
        }
        __syncthreads();
        if (VEC) {
            const int chunks = hd >> 4;
            for (int i = tid; i < GT * chunks; i += GEN_THREADS) {
                const int row = i / chunks, d = (i - row * chunks) * 16;
                const long long at = from[row];
                uint4 k = make_uint4(0, 0, 0, 0), v = k;
                if (at >= 0) { k = __ldg(reinterpret_cast<const uint4*>(a.k_pages + at + d)); v = __ldg(reinterpret_cast<const uint4*>(a.v_pages + at + d)); }
                const unsigned kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
                const float s = ks[row];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    *reinterpret_cast<float4*>(kt + row * ks_stride + d + 4 * j) =
                        make_float4((float)(signed char)kw[j] * s, (float)(signed char)(kw[j] >> 8) * s, (float)(signed char)(kw[j] >> 16) * s, (float)(signed char)(kw[j] >> 24) * s);
                    *reinterpret_cast<float4*>(vt + row * hd + d + 4 * j) =
                        make_float4((float)(signed char)vw[j], (float)(signed char)(vw[j] >> 8), (float)(signed char)(vw[j] >> 16), (float)(signed char)(vw[j] >> 24));
                }
            }
        } else {
#pragma unroll 4
            for (int i = tid; i < GT * hd; i += GEN_THREADS) {
                const int row = i / hd, d = i - row * hd;
                const long long at = from[row];
                kt[row * ks_stride + d] = at >= 0 ? (float)__ldg(a.k_pages + at + d) * ks[row] : 0.f;
                vt[i] = at >= 0 ? (float)__ldg(a.v_pages + at + d) : 0.f;
            }
        }
        __syncthreads();
        for (int i = tid; i < n_rep * GT; i += GEN_THREADS) {
            const int h = i / GT, row = i - h * GT, key = tile * GT + row;
            float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
            const float* x = q + h * hd;
            const float* y = kt + row * ks_stride;
            if (VEC) {
#pragma unroll 4
                for (int d = 0; d < hd; d += 4) {
                    const float4 xv = *reinterpret_cast<const float4*>(x + d), yv = *reinterpret_cast<const float4*>(y + d);
                    s0 = fmaf(xv.x, yv.x, s0); s1 = fmaf(xv.y, yv.y, s1); s2 = fmaf(xv.z, yv.z, s2); s3 = fmaf(xv.w, yv.w, s3);
                }
            } else {
                for (int d = 0; d < hd; ++d) s0 = fmaf(x[d], y[d], s0);
            }
            const bool seen = key >= lo && key <= p;
            const float v = seen ? (s0 + s1) + (s2 + s3) : -INFINITY;
            // a warp holds the 32 keys of one head
            const float top = warp_max(v + reference_log2(vs[row]));
            const float m_old = cta_ml[2 * h], m_new = fmaxf(m_old, top), m_use = m_new == -INFINITY ? 0.f : m_new - LIFT;
            const float e = exp2f(v - m_use);
            const float sum = warp_sum(e);
            __syncwarp();
            if (row == 0) {
                const float c = m_old == -INFINITY ? 0.f : exp2f(m_old - m_new);
                corr[h] = c;
                cta_ml[2 * h] = m_new;
                cta_ml[2 * h + 1] = cta_ml[2 * h + 1] * c + sum;
            }
            w[i] = e == 0.f ? 0.f : e * (vs[row] * UNLIFT);
        }
        __syncthreads();
        for (int i = tid; i < n_rep * hd; i += GEN_THREADS) {
            const int h = i / hd, d = i - h * hd;
            float acc = cta_o[i] * corr[h];
#pragma unroll 8
            for (int r = 0; r < GT; ++r) acc = fmaf(w[h * GT + r], vt[r * hd + d], acc);
            cta_o[i] = acc;
        }
    }
    __syncthreads();
    finish(cta_o, cta_ml, a, hd, out, GEN_THREADS);
}

long long any_smem(int n_rep, int hd) { return 4LL * (2LL * n_rep * hd + GT * (2LL * hd + 4) + n_rep * (GT + 3LL)); }
constexpr long long MAX_SMEM = 226 * 1024;         // (and what a CTA has besides)

template <typename T>
int launch_rows(void (*kernel)(const T*, T*, Args), const Args& a, int n_tokens, int step, int threads, long long smem, const void* q, void* out, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.span ? a.parts : a.csize, n_tokens, a.kv_heads);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)smem;
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
    NIB_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const T*)q, (T*)out, a));
    if (a.span) NIB_CUDA(launch_pdl(merge_int8_kernel<T>, dim3(a.heads, n_tokens), dim3(128), (size_t)0, stream, (T*)out, a, step));
    return 0;
}

}  // namespace

// Which kernel takes single tokens of this shape: 1 the one on the tensor cores, 0 the general one, -1 neither.
NIB_API int nib_attention_int8_decode_kind(int heads, int kv_heads, int head_dim, int page_size, int dtype) {
    if (kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return -1;
    if (dtype == NIB_BF16 && (head_dim == 64 || head_dim == 128) && heads / kv_heads <= 16 && page_size % 8 == 0) return 1;
    return any_smem(heads / kv_heads, head_dim) <= MAX_SMEM ? 0 : -1;
}

// The arguments of a call, one block of memory.
struct NibAttendInt8 {
    const void* q; void* out; const int* ctx_lens; const int* block_table; const void* k_pages; const void* v_pages; const float* k_scales;
    const float* v_scales; float* part_o; float* part_ml;
    int q_stride, bt_stride, bt_width, page_size, num_pages, n_tokens, heads, kv_heads, head_dim, window, ctas, span, parts, dtype;
    float scale; int pad;
};

// Attention of n_tokens single tokens (token i is request i, at position ctx_lens[i] - 1) whose keys and values are in the pages.
// ``span`` 0: the keys of a (token, kv head) are cut among ``ctas`` CTAs (1, 2, 4 or 8). Else a CTA takes ``span`` keys (a multiple of
// 32) and a row has at most ``parts`` of them: part_o [tokens * heads * parts * head_dim], part_ml [tokens * heads * parts * 2].
NIB_API int nib_attention_int8_decode(const void* args, cudaStream_t stream) {
    NibAttendInt8 c;
    memcpy(&c, args, sizeof c);
    const int n_tokens = c.n_tokens, heads = c.heads, kv_heads = c.kv_heads, head_dim = c.head_dim, page_size = c.page_size, dtype = c.dtype;
    const void* q = c.q;
    void* out = c.out;
    NIB_REQUIRE(n_tokens >= 0 && c.num_pages > 0 && page_size > 0 && c.bt_width >= 0 && c.window >= 0, "attention (8-bit cache): bad sizes");
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "attention (8-bit cache): unknown dtype %d", dtype);
    const int kind = nib_attention_int8_decode_kind(heads, kv_heads, head_dim, page_size, dtype);
    NIB_REQUIRE(kind >= 0, "attention (8-bit cache): %d/%d heads of %d are not supported", heads, kv_heads, head_dim);
    if (c.span) {
        NIB_REQUIRE(c.ctas == 1 && c.span > 0 && c.span % 32 == 0 && c.parts > 0 && c.part_o && c.part_ml, "attention (8-bit cache): spans of a multiple of 32 keys, and scratch memory for them");
    } else {
        NIB_REQUIRE(c.ctas == 1 || c.ctas == 2 || c.ctas == 4 || c.ctas == 8, "attention (8-bit cache): 1, 2, 4 or 8 CTAs share a row's keys, not %d", c.ctas);
    }
    NIB_REQUIRE(n_tokens <= 65535 && kv_heads <= 65535, "attention (8-bit cache): too many tokens or heads for one launch");
    if (n_tokens == 0) return 0;
    int shift = -1;
    if ((page_size & (page_size - 1)) == 0) for (shift = 0; (1 << shift) < page_size;) ++shift;
    const Args a{c.ctx_lens, c.block_table, (const signed char*)c.k_pages, (const signed char*)c.v_pages, c.k_scales, c.v_scales, c.part_o, c.part_ml,
                 c.q_stride, c.bt_stride, c.bt_width, page_size, shift, c.num_pages, heads, kv_heads, heads / kv_heads, head_dim, c.window, c.ctas, c.span, c.parts, c.scale};
    int rc;
    if (kind == 1) {
        NIB_REQUIRE((((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) == 0, "attention (8-bit cache): the pools must be 16-byte aligned");
#define CALL(KERNEL, T, STEP, THREADS, SMEM, MOST)                                                                              \
    do {                                                                                                                        \
        static const cudaError_t set = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(MOST));  \
        NIB_CUDA(set);                                                                                                          \
        rc = launch_rows<T>(KERNEL, a, n_tokens, STEP, THREADS, SMEM, q, out, stream);                                          \
    } while (0)
#define MMA(HD, NH, KU)                                                                                                                              \
    do {                                                                                                                                             \
        if (page_size % 16 == 0) CALL((attention_int8_mma_kernel<HD, NH, KU, true>), __nv_bfloat16, KU * 16, WARPS * 32, (mma_smem<HD, NH>()), (mma_smem<HD, NH>())); \
        else CALL((attention_int8_mma_kernel<HD, NH, KU, false>), __nv_bfloat16, KU * 16, WARPS * 32, (mma_smem<HD, NH>()), (mma_smem<HD, NH>()));      \
    } while (0)
        if (a.n_rep <= 8) { if (head_dim == 64) MMA(64, 1, 2); else MMA(128, 1, 1); }
        else { if (head_dim == 64) MMA(64, 2, 2); else MMA(128, 2, 1); }
    } else {
        const bool vec = head_dim % 16 == 0 && (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) == 0;
#define ANY(T, VEC) CALL((attention_int8_any_kernel<T, VEC>), T, GT, GEN_THREADS, any_smem(a.n_rep, head_dim), MAX_SMEM)
        if (dtype == NIB_F32) { if (vec) ANY(float, true); else ANY(float, false); }
        else { if (vec) ANY(__nv_bfloat16, true); else ANY(__nv_bfloat16, false); }
#undef ANY
    }
#undef MMA
#undef CALL
    return rc;
}
