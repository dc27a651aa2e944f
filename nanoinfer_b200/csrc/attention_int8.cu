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
// 8 tokens; the general one takes any shape and 32-bit rows. Both cut the keys of a (token, kv head) among the CTAs of a cluster,
// which merge their partial (max, sum, output) through distributed shared memory; more than eight CTAs are clusters of eight whose
// results a last kernel merges in order.
#include "attention_common.cuh"
#include "pipeline.cuh"
#include <cuda_fp16.h>

using namespace nibp;

namespace {

constexpr int WARPS = 8;
constexpr float LIFT = 20.f, UNLIFT = 0x1p-20f, RELIFT = 0x1p20f;

struct Args {
    const int* ctx_lens; const int* block_table; const signed char* k_pages; const signed char* v_pages;
    const float* k_scales; const float* v_scales; float* part_o; float* part_ml;
    int q_stride, bt_stride, bt_width, page_size, shift, num_pages, heads, kv_heads, n_rep, head_dim, window, splits, csize;
    float scale;
};

// Merges the CTAs of the cluster: every CTA left its output, relative to its own maximum, in cta_o [n_rep][hd] and its (max, sum)
// in cta_ml; this CTA finishes its slice of the outputs. All threads take part.
template <typename T>
__device__ __forceinline__ void finish(const float* cta_o, const float* cta_ml, const Args& a, int hd, T* __restrict__ out, int threads) {
    if (a.csize > 1) cluster_sync(); else __syncthreads();
    const int rank = a.csize > 1 ? (int)cluster_rank() : 0;
    const int outer = a.splits / a.csize, oidx = blockIdx.x / a.csize;
    const int total = a.n_rep * hd, slice = (total + a.csize - 1) / a.csize;
    const int end = min(total, (rank + 1) * slice);
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
                const float f = (mr[r] == -INFINITY) ? 0.f : exp2f(mr[r] - m_all);
                l_all += lr[r] * f;
                acc += orr[r] * f;
            }
        } else {
            m_all = cta_ml[row * 2];
            l_all = cta_ml[row * 2 + 1];
            acc = cta_o[i];
        }
        const size_t th = (size_t)blockIdx.y * a.heads + (size_t)blockIdx.z * a.n_rep + row;
        if (outer == 1) {
            Elem<T>::store(out + th * hd + d, l_all == 0.f ? 0.f : acc / l_all * RELIFT);      // a row that sees nothing is zero, an undefined one NaN
        } else {
            a.part_o[(th * outer + oidx) * hd + d] = acc;
            if (d == 0) {
                a.part_ml[(th * outer + oidx) * 2] = m_all;
                a.part_ml[(th * outer + oidx) * 2 + 1] = l_all;
            }
        }
    }
    if (a.csize > 1) cluster_sync();        // nobody leaves while a peer may still read its shared memory
}

// Merges the clusters' results of one (token, head), in order. grid: tokens * heads.
template <typename T>
__global__ void __launch_bounds__(128)
merge_int8_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, T* __restrict__ out, int parts, int hd) {
    pdl_wait();
    pdl_launch_dependents();
    const size_t th = blockIdx.x;
    float m = -INFINITY;
    for (int s = 0; s < parts; ++s) m = fmaxf(m, part_ml[(th * parts + s) * 2]);
    for (int d = threadIdx.x; d < hd; d += 128) {
        float l = 0.f, acc = 0.f;
        for (int s = 0; s < parts; ++s) {
            const float ms = part_ml[(th * parts + s) * 2];
            const float f = ms == -INFINITY ? 0.f : exp2f(ms - m);
            l += part_ml[(th * parts + s) * 2 + 1] * f;
            acc += part_o[(th * parts + s) * hd + d] * f;
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
// Codes as 16-bit floats: a code plus 128 in the low bits of 1024.0 is 1152 + code, exactly. Two codes (bytes sel) of ``biased``.
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

template <int HD, int NH, int KU>
__global__ void __launch_bounds__(WARPS * 32)
attention_int8_mma_kernel(const __nv_bfloat16* __restrict__ q_rows, __nv_bfloat16* __restrict__ out, const Args a) {
    constexpr int STEP = KU * 16, MS = HD + 4, ROWS = NH * 8;
    extern __shared__ __align__(16) float smem[];
    const int token = blockIdx.y, kvh = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();
    const int p = a.ctx_lens[token] - 1;                     // the token's own position; -1: a padding row
    const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const int* bt = a.block_table + (size_t)token * a.bt_stride;
    const int s_first = lo / STEP, n_steps = p >= 0 ? p / STEP - s_first + 1 : 0;
    const int per = (n_steps + a.splits - 1) / a.splits;
    const int begin = s_first + blockIdx.x * per, end = min(s_first + n_steps, begin + per);

    // Q^T as the column operand, its dims in the order in which the key rows' pieces hold them. A head is scaled by a power of two so
    // that its largest element lies in 2^12 .. 2^13: 16-bit floats then hold every element that counts exactly.
    unsigned qb[HD / 16][NH][2];
    float factor[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
        const int head = nh * 8 + g;
        const __nv_bfloat16* qp = q_rows + (size_t)token * a.q_stride + (size_t)(kvh * a.n_rep + head) * HD;
        float x[HD / 16][4], top = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[kk][j] = head < a.n_rep ? __bfloat162float(qp[(kk >> 2) * 64 + t * 16 + (kk & 3) * 4 + j]) : 0.f;
                top = fmaxf(top, fabsf(x[kk][j]));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (top > 0.f && top < INFINITY) ? ilogbf(top) - 12 : 0;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) qb[kk][nh][j] = pack_f16(ldexpf(x[kk][2 * j], -e), ldexpf(x[kk][2 * j + 1], -e));
        const float mine = ldexpf(a.scale * LOG2E, e);
        factor[nh][0] = __shfl_sync(0xffffffffu, mine, 8 * t);          // of the heads 2t, 2t + 1: the lanes (g = 2t, 2t + 1; t = 0)
        factor[nh][1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
    }

    float o[HD / 16][NH][4], m_ref[NH][2], l_part[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
        m_ref[nh][0] = m_ref[nh][1] = -INFINITY;
        l_part[nh][0] = l_part[nh][1] = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[d][nh][0] = o[d][nh][1] = o[d][nh][2] = o[d][nh][3] = 0.f;
    }

    auto load = [&](Codes<HD, KU>& c, int step) {
#pragma unroll
        for (int ku = 0; ku < KU; ++ku)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = step * STEP + ku * 16 + h * 8;
                int slot = 0, page = -1;
                if (key <= p && key + 8 > lo) page = page_at(a, bt, key, slot);
                const bool held = page >= 0;
                const size_t block = (size_t)max(page, 0) * a.kv_heads + kvh;
                const size_t at = (block * a.page_size + slot) * HD;
                c.ks[ku][h] = held ? __ldg(a.k_scales + block) : 0.f;
                c.vs[ku][h] = held ? __ldg(a.v_scales + block) : 0.f;
#pragma unroll
                for (int i = 0; i < HD / 64; ++i)
                    c.k[ku][h][i] = held ? __ldg(reinterpret_cast<const uint4*>(a.k_pages + at + g * HD + i * 64 + t * 16)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const signed char* vp = a.v_pages + at + (2 * t + j) * HD + g * (HD / 8);
                    if constexpr (HD == 64) {
                        const uint2 x = held ? __ldg(reinterpret_cast<const uint2*>(vp)) : make_uint2(0, 0);
                        c.v[ku][2 * h + j][0] = x.x; c.v[ku][2 * h + j][1] = x.y;
                    } else {
                        const uint4 x = held ? __ldg(reinterpret_cast<const uint4*>(vp)) : make_uint4(0, 0, 0, 0);
                        c.v[ku][2 * h + j][0] = x.x; c.v[ku][2 * h + j][1] = x.y;
                        c.v[ku][2 * h + j][2] = x.z; c.v[ku][2 * h + j][3] = x.w;
                    }
                }
            }
    };
    auto compute = [&](const Codes<HD, KU>& c, int step) {
        float s[KU][NH][4];
        // S^T = K Q^T
#pragma unroll
        for (int ku = 0; ku < KU; ++ku) {
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) s[ku][nh][0] = s[ku][nh][1] = s[ku][nh][2] = s[ku][nh][3] = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const unsigned w0[4] = {c.k[ku][0][i].x, c.k[ku][0][i].y, c.k[ku][0][i].z, c.k[ku][0][i].w};
                const unsigned w1[4] = {c.k[ku][1][i].x, c.k[ku][1][i].y, c.k[ku][1][i].z, c.k[ku][1][i].w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const unsigned u0 = w0[b] ^ 0x80808080u, u1 = w1[b] ^ 0x80808080u;
                    const unsigned a0 = two_codes(u0, 0x4140), a1 = two_codes(u1, 0x4140), a2 = two_codes(u0, 0x4342), a3 = two_codes(u1, 0x4342);
#pragma unroll
                    for (int nh = 0; nh < NH; ++nh) mma_f16(s[ku][nh], a0, a1, a2, a3, qb[i * 4 + b][nh][0], qb[i * 4 + b][nh][1]);
                }
            }
        }
        // element e of a tile: key g + 8 * (e / 2), head 2t + (e & 1)
        const int key0 = step * STEP + g;
        const bool edge = step * STEP < lo || step * STEP + STEP - 1 > p;
        float lv[KU][2];
#pragma unroll
        for (int ku = 0; ku < KU; ++ku) { lv[ku][0] = reference_log2(c.vs[ku][0]); lv[ku][1] = reference_log2(c.vs[ku][1]); }
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
                    const float corr = (m_ref[nh][q] == -INFINITY) ? 0.f : exp2f(m_ref[nh][q] - m_new);
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
                        const float w = exp2f(s[ku][nh][2 * h + q] - m_use);
                        l_part[nh][q] += w;
                        s[ku][nh][2 * h + q] = w == 0.f ? 0.f : w * (c.vs[ku][h] * UNLIFT);            // (a hidden key's block may be undefined)
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

    Codes<HD, KU> c[2];
    int step = begin + warp;
    if (step < end) load(c[0], step);
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
            const float f = (mw[w] == -INFINITY) ? 0.f : exp2f(mw[w] - m_row);
            acc += sm_o[(w * ROWS + row) * MS + d] * f;
            l_row += sm_ml[(w * ROWS + row) * 2 + 1] * f;
        }
        cta_o[i] = acc;
        if (d == 0) { cta_ml[row * 2] = m_row; cta_ml[row * 2 + 1] = l_row; }
    }
    finish(cta_o, cta_ml, a, HD, out, WARPS * 32);
}

template <int HD, int NH> constexpr int mma_smem() { return (WARPS * NH * 8 * (HD + 4 + 2) + NH * 8 * (HD + 2)) * 4; }

// ------------------------------------------------------------------------------------------ any shape
// Tiles of 32 keys, as 32-bit values in shared memory: a thread has one (query head, key) of the scores at a time, then one
// (query head, dim) of the sums.
constexpr int GT = 32, GEN_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(GEN_THREADS)
attention_int8_any_kernel(const T* __restrict__ q_rows, T* __restrict__ out, const Args a) {
    extern __shared__ __align__(16) float smem[];
    const int hd = a.head_dim, n_rep = a.n_rep, token = blockIdx.y, kvh = blockIdx.z, tid = threadIdx.x;
    float* q = smem;                            // [n_rep][hd]
    float* kt = q + n_rep * hd;                 // [GT][hd + 1]
    float* vt = kt + GT * (hd + 1);             // [GT][hd]
    float* w = vt + GT * hd;                    // [n_rep][GT]
    float* corr = w + n_rep * GT;               // [n_rep]
    float* vs = corr + n_rep;                   // [GT] value scales
    float* cta_ml = vs + GT;                    // [n_rep][2]
    float* cta_o = cta_ml + 2 * n_rep;          // [n_rep][hd]
    pdl_wait();
    pdl_launch_dependents();
    const int p = a.ctx_lens[token] - 1;
    const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const int* bt = a.block_table + (size_t)token * a.bt_stride;
    const int first = lo / GT, n_tiles = p >= 0 ? p / GT - first + 1 : 0;
    const int per = (n_tiles + a.splits - 1) / a.splits;
    const int begin = first + blockIdx.x * per, end = min(first + n_tiles, begin + per);
    for (int i = tid; i < n_rep * hd; i += GEN_THREADS) {
        q[i] = Elem<T>::load(q_rows + (size_t)token * a.q_stride + (size_t)kvh * n_rep * hd + i) * (a.scale * LOG2E);
        cta_o[i] = 0.f;
    }
    for (int i = tid; i < n_rep; i += GEN_THREADS) { cta_ml[2 * i] = -INFINITY; cta_ml[2 * i + 1] = 0.f; }
    for (int tile = begin; tile < end; ++tile) {
        __syncthreads();
        for (int i = tid; i < GT * hd; i += GEN_THREADS) {
            const int row = i / hd, d = i - row * hd, key = tile * GT + row;
            float kv = 0.f, vv = 0.f, s = 0.f;
            if (key >= lo && key <= p) {
                int slot;
                const int page = page_at(a, bt, key, slot);
                if (page >= 0) {
                    const size_t block = (size_t)page * a.kv_heads + kvh, at = (block * a.page_size + slot) * hd + d;
                    s = __ldg(a.v_scales + block);
                    kv = (float)__ldg(a.k_pages + at) * __ldg(a.k_scales + block);
                    vv = (float)__ldg(a.v_pages + at);
                }
            }
            kt[row * (hd + 1) + d] = kv;
            vt[i] = vv;
            if (d == 0) vs[row] = s;
        }
        __syncthreads();
        for (int i = tid; i < n_rep * GT; i += GEN_THREADS) {
            const int h = i / GT, row = i - h * GT, key = tile * GT + row;
            float s0 = 0.f, s1 = 0.f;
            const float* x = q + h * hd;
            const float* y = kt + row * (hd + 1);
            int d = 0;
            for (; d + 1 < hd; d += 2) { s0 = fmaf(x[d], y[d], s0); s1 = fmaf(x[d + 1], y[d + 1], s1); }
            if (d < hd) s0 = fmaf(x[d], y[d], s0);
            const bool seen = key >= lo && key <= p;
            const float v = seen ? s0 + s1 : -INFINITY;
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

long long any_smem(int n_rep, int hd) { return 4LL * (2LL * n_rep * hd + GT * (2LL * hd + 1) + n_rep * (GT + 3LL) + GT); }
constexpr long long MAX_SMEM = 227 * 1024;

template <typename T>
int launch_split(void (*kernel)(const T*, T*, Args), const Args& a, int n_tokens, int threads, long long smem, const void* q, void* out, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.splits, n_tokens, a.kv_heads);
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
    return 0;
}

template <typename T>
int merge_parts(const Args& a, T* out, int n_tokens, cudaStream_t stream) {
    const int parts = a.splits / a.csize;
    if (parts == 1) return 0;
    NIB_CUDA(launch_pdl(merge_int8_kernel<T>, dim3((unsigned)(n_tokens * a.heads)), dim3(128), (size_t)0, stream, (const float*)a.part_o,
                        (const float*)a.part_ml, out, parts, a.head_dim));
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
    int q_stride, bt_stride, bt_width, page_size, num_pages, n_tokens, heads, kv_heads, head_dim, window, splits, dtype;
    float scale; int pad;
};

// Attention of n_tokens single tokens (token i is request i, at position ctx_lens[i] - 1) whose keys and values are in the pages.
// ``splits`` CTAs share the keys of a (token, kv head): 1, 2, 4, 8 or a multiple of 8, which needs part_o [tokens * heads * splits/8
// * head_dim] and part_ml [tokens * heads * splits/8 * 2].
NIB_API int nib_attention_int8_decode(const void* args, cudaStream_t stream) {
    NibAttendInt8 c;
    memcpy(&c, args, sizeof c);
    const int n_tokens = c.n_tokens, heads = c.heads, kv_heads = c.kv_heads, head_dim = c.head_dim, page_size = c.page_size, splits = c.splits, dtype = c.dtype;
    const void* q = c.q;
    void* out = c.out;
    NIB_REQUIRE(n_tokens >= 0 && c.num_pages > 0 && page_size > 0 && c.bt_width >= 0 && c.window >= 0 && splits >= 1 && splits <= 256, "attention (8-bit cache): bad sizes");
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "attention (8-bit cache): unknown dtype %d", dtype);
    const int kind = nib_attention_int8_decode_kind(heads, kv_heads, head_dim, page_size, dtype);
    NIB_REQUIRE(kind >= 0, "attention (8-bit cache): %d/%d heads of %d are not supported", heads, kv_heads, head_dim);
    const int csize = splits >= 8 ? 8 : splits;
    NIB_REQUIRE((csize & (csize - 1)) == 0 && splits % csize == 0, "attention (8-bit cache): %d splits; 1, 2, 4, 8 or a multiple of 8 are possible", splits);
    NIB_REQUIRE(splits == csize || (c.part_o && c.part_ml), "attention (8-bit cache): more than 8 splits need scratch memory");
    NIB_REQUIRE(n_tokens <= 65535 && kv_heads <= 65535 && (long long)n_tokens * heads < (1LL << 31), "attention (8-bit cache): too many tokens or heads for one launch");
    if (n_tokens == 0) return 0;
    int shift = -1;
    if ((page_size & (page_size - 1)) == 0) for (shift = 0; (1 << shift) < page_size;) ++shift;
    const Args a{c.ctx_lens, c.block_table, (const signed char*)c.k_pages, (const signed char*)c.v_pages, c.k_scales, c.v_scales, c.part_o, c.part_ml,
                 c.q_stride, c.bt_stride, c.bt_width, page_size, shift, c.num_pages, heads, kv_heads, heads / kv_heads, head_dim, c.window, splits, csize, c.scale};
    int rc;
    if (kind == 1) {
        NIB_REQUIRE((((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) == 0, "attention (8-bit cache): the pools must be 16-byte aligned");
#define CALL(KERNEL, T, THREADS, SMEM, MOST)                                                                                    \
    do {                                                                                                                        \
        static const cudaError_t set = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(MOST));  \
        NIB_CUDA(set);                                                                                                          \
        rc = launch_split<T>(KERNEL, a, n_tokens, THREADS, SMEM, q, out, stream);                                               \
    } while (0)
#define MMA(HD, NH, KU) CALL((attention_int8_mma_kernel<HD, NH, KU>), __nv_bfloat16, WARPS * 32, (mma_smem<HD, NH>()), (mma_smem<HD, NH>()))
        if (a.n_rep <= 8) { if (head_dim == 64) MMA(64, 1, 2); else MMA(128, 1, 1); }
        else { if (head_dim == 64) MMA(64, 2, 2); else MMA(128, 2, 1); }
    } else if (dtype == NIB_F32) {
        CALL(attention_int8_any_kernel<float>, float, GEN_THREADS, any_smem(a.n_rep, head_dim), MAX_SMEM);
    } else {
        CALL(attention_int8_any_kernel<__nv_bfloat16>, __nv_bfloat16, GEN_THREADS, any_smem(a.n_rep, head_dim), MAX_SMEM);
    }
#undef MMA
#undef CALL
    if (rc) return rc;
    return dtype == NIB_F32 ? merge_parts(a, (float*)out, n_tokens, stream) : merge_parts(a, (__nv_bfloat16*)out, n_tokens, stream);
}
