// Attention of single decoded tokens over the 8-bit cache (cache_int8.cu): codes of 8 bits, a scale for each page and kv head.
//
//     s_j = scale * q . (ck_j * sk_j),  w = softmax(s),  o = sum_j w_j cv_j sv_j        (keys at positions lo..p)
//
// The key scale multiplies a score. The value scale would multiply a row of V before a tensor core sums it; it goes into the
// softmax instead: with t_j = s_j log2(e) + log2(sv_j) and a running reference M of max t,
//     w_j = 2^(s_j log2(e) - M + 20),  p_j = w_j sv_j 2^-11  (about 2^9 at most),  l = sum_j w_j,  o = 2^11 sum_j p_j cv_j / l,
// so the tensor core multiplies p_j, in 16 bits, with whole numbers that 16 bits hold exactly, and a row is right to its own
// size however much the scales of its blocks differ. l and o are summed in 32 bits; with scales of 2^-80 .. 2^121 the terms of l that
// count lie between 2^-125 and 2^106 (the 20 is what centres them). The tensor core's p_j is rounded to 11 bits, as the 16-bit caches' weights
// are to 8; the reference may lag by 2^6, and 2^15 is what a 16-bit float holds: the 2^9 is the room that is left, so that a weight 2^-23
// of the reference still has its 11 bits and one down to 2^-34 counts (with p_j of 1 at most it was 2^-25, and tens of thousands of
// keys below that were in l and not in o).
//
// Two kernels. The one on the tensor cores takes heads of 64 and 128, at most 16 query heads a kv head and pages of a multiple of
// 8 tokens; the general one takes any shape and 32-bit rows. The keys are dealt out in one of two ways. Few rows: those of a (token, kv
// head) among the CTAs of a cluster, which merge their partial (max, sum, output) through distributed shared memory and store the row.
// Many, or long ones: the chunks of all rows, in order, in equal shares to as many CTAs as find room at a time, whatever the lengths
// are; a row that lies within one CTA's share is stored, the others' parts are merged in order by a second kernel.
//
// A kernel of a chain is on its SM before the kernel ahead of it has ended, so what that one writes (queries, codes, scales, parts) is read
// behind the wait and by loads that know of other writers (no __ldg, no const __restrict__); lengths and tables are the step's inputs.
#include "attention_common.cuh"
#include "pipeline.cuh"
#include <cuda_fp16.h>
#include <type_traits>

using namespace nibp;

namespace {

constexpr int WARPS = 4;
constexpr float LIFT = 20.f, UNLIFT = 0x1p-11f, RELIFT = 0x1p11f;

struct Args {
    const int* ctx_lens; const int* block_table; const signed char* k_pages; const signed char* v_pages;
    const float* k_scales; const float* v_scales; float* part_o; float* part_ml;        // [2 * shares][n_rep][head_dim], [2 * shares][n_rep][2]
    int q_stride, bt_stride, bt_width, page_size, shift, num_pages, n_tokens, heads, kv_heads, n_rep, head_dim, window;
    int csize, shares;              // CTAs of a cluster and 0 shares, or the CTAs that all chunks are dealt to
    int early;                      // pages before the one that a token's own key lies in are no running kernel's results
    float scale;
};

__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// The root of 2^(m - to), the factor of what is relative to m on the way to a larger reference. A sum is multiplied with it twice:
// where scales differ by as much as they may, the factor itself is below 32 bits' range and the sum times it is not.
__device__ __forceinline__ float half_factor(float m, float to) { return m == -INFINITY ? 0.f : exp2_ftz(0.5f * (m - to)); }

// The keys lo..p of a token (p -1: a padding row) and the chunks of CH keys, aligned to absolute multiples, that hold them.
template <int CH> struct Keys {
    int lo, p, first, n;
    __device__ __forceinline__ Keys(const Args& a, int token) {
        p = __ldg(a.ctx_lens + token) - 1;
        lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
        first = lo / CH;
        n = p >= 0 ? p / CH - first + 1 : 0;
    }
};

// All rows' chunks in order: token by token, a token's kv heads one behind the other. A warp looks its place up together.
template <int CH> __device__ __forceinline__ int all_chunks(const Args& a, int lane) {
    int sum = 0;
    for (int t = lane; t < a.n_tokens; t += 32) sum += Keys<CH>(a, t).n;
    return __reduce_add_sync(0xffffffffu, sum) * a.kv_heads;
}
// The token whose chunks hold number ``at``, and the number of its first.
template <int CH> __device__ __forceinline__ int token_at(const Args& a, int at, int& token_first, int lane) {
    int base = 0;
    for (int t0 = 0; t0 < a.n_tokens; t0 += 32) {
        const int n = t0 + lane < a.n_tokens ? Keys<CH>(a, t0 + lane).n * a.kv_heads : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned mine = __ballot_sync(0xffffffffu, at < base + sum);
        if (mine) {
            const int src = __ffs(mine) - 1;
            token_first = base + __shfl_sync(0xffffffffu, sum - n, src);
            return t0 + src;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    token_first = base;
    return a.n_tokens;
}

// A CTA's work, piece by piece: chunks begin..end of one (token, kv head), and the place of what they leave: -1 the output itself (or
// the cluster's), else a part.
template <int CH> struct Pieces {
    int token, kvh, lo, p, begin, end, part;
    int at, stop, per;
    __device__ __forceinline__ bool first(const Args& a, int lane) {
        if (a.shares == 0) {
            token = blockIdx.y; kvh = blockIdx.z;
            const Keys<CH> k(a, token);
            lo = k.lo; p = k.p; part = -1;
            const int share = (k.n + a.csize - 1) / a.csize;
            begin = k.first + blockIdx.x * share;
            end = min(k.first + k.n, begin + share);
            at = stop = per = 0;
            return true;
        }
        const int all = all_chunks<CH>(a, lane);
        per = max(1, (all + a.shares - 1) / a.shares);
        at = min(all, (int)blockIdx.x * per);
        stop = min(all, at + per);
        return look(a, lane);
    }
    __device__ __forceinline__ bool next(const Args& a, int lane) { return a.shares != 0 && look(a, lane); }
private:
    __device__ __forceinline__ bool look(const Args& a, int lane) {
        if (at >= stop) return false;
        int token_first;
        token = token_at<CH>(a, at, token_first, lane);
        const Keys<CH> k(a, token);
        lo = k.lo; p = k.p;
        kvh = (at - token_first) / k.n;
        const int idx = at - token_first - kvh * k.n, n = min(k.n - idx, stop - at);
        begin = k.first + idx;
        end = begin + n;
        part = n == k.n ? -1 : 2 * (int)blockIdx.x + (idx == 0 ? 1 : 0);
        at += n;
        return true;
    }
};

// What a CTA leaves of a piece: its output, relative to its own maximum, in cta_o [n_rep][hd], its (max, sum) in cta_ml. All threads
// take part, and all are behind a barrier.
template <typename T>
__device__ __forceinline__ void finish(const float* cta_o, const float* cta_ml, const Args& a, int token, int kvh, int part, int hd, T* __restrict__ out, int threads) {
    const size_t th0 = (size_t)token * a.heads + (size_t)kvh * a.n_rep;
    const int total = a.n_rep * hd;
    if (part >= 0) {
        for (int i = threadIdx.x; i < total; i += threads) a.part_o[(size_t)part * total + i] = cta_o[i];
        for (int i = threadIdx.x; i < 2 * a.n_rep; i += threads) a.part_ml[(size_t)part * 2 * a.n_rep + i] = cta_ml[i];
        return;
    }
    if (a.csize > 1) cluster_sync();
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
                const float f = half_factor(mr[r], m_all);
                l_all += lr[r] * f * f;
                acc += orr[r] * (f * f);
            }
        } else {
            l_all = cta_ml[row * 2 + 1];
            acc = cta_o[i];
        }
        Elem<T>::store(out + (th0 + row) * hd + d, l_all == 0.f ? 0.f : acc / l_all * RELIFT);      // a row that sees nothing is zero, an undefined one NaN
    }
    if (a.csize > 1) cluster_sync();        // nobody leaves while a peer may still read its shared memory
}

// Merges the parts of the rows that lie in more than one share, in order, and stores the rows that see nothing. grid: (heads, tokens).
// More than eight parts are taken in turns by as many threads as there are for an element, whose sums meet in shared memory.
constexpr int MERGE_THREADS = 256;         // the most; half of them where the rows alone fill the SMs (64 x 14 rows of 64: 15.2 us with the attention, 17.5)

template <typename T, int CH>
__global__ void __launch_bounds__(MERGE_THREADS)
merge_int8_kernel(T* __restrict__ out, const Args a) {
    __shared__ float s_acc[MERGE_THREADS], s_m[MERGE_THREADS], s_l[MERGE_THREADS];
    const int token = blockIdx.y, head = blockIdx.x, kvh = head / a.n_rep, row = head - kvh * a.n_rep, lane = threadIdx.x & 31, hd = a.head_dim;
    pdl_launch_dependents();
    int all = 0, before = 0;                        // chunks of a kv head
    for (int t = lane; t < a.n_tokens; t += 32) {
        const int n = Keys<CH>(a, t).n;
        all += n;
        if (t < token) before += n;
    }
    all = __reduce_add_sync(0xffffffffu, all) * a.kv_heads;
    const int n = Keys<CH>(a, token).n, begin = __reduce_add_sync(0xffffffffu, before) * a.kv_heads + kvh * n;
    const int per = max(1, (all + a.shares - 1) / a.shares), b0 = begin / per, parts = n ? (begin + n - 1) / per - b0 + 1 : 0;
    pdl_wait();             // (the lengths are the step's inputs)
    if (parts == 1) return;
    const int threads = blockDim.x;
    const int turns = parts <= 8 ? 1 : max(1, threads / hd);
    for (int d0 = 0; d0 < hd; d0 += threads) {
        const int turn = turns > 1 ? threadIdx.x / hd : 0, d = turns > 1 ? threadIdx.x - turn * hd : d0 + threadIdx.x;
        float m = -INFINITY, l = 0.f, acc = 0.f;
        if (turn < turns && d < hd) {
            for (int s0 = turn; s0 < parts; s0 += 8 * turns) {
                float v[8];
                float2 x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int s = s0 + u * turns;
                    v[u] = 0.f;
                    x[u] = make_float2(-INFINITY, 0.f);
                    if (s < parts) {
                        const size_t at = (size_t)(s == 0 ? 2 * b0 + 1 : 2 * (b0 + s)) * a.n_rep + row;
                        v[u] = a.part_o[at * hd + d];
                        x[u] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
                    }
                }
                float top = m;
#pragma unroll
                for (int u = 0; u < 8; ++u) top = fmaxf(top, x[u].x);
                const float f0 = half_factor(m, top);
                l = l * f0 * f0;
                acc *= f0 * f0;
                m = top;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (s0 + u * turns < parts) {
                        const float f = half_factor(x[u].x, m);
                        l += x[u].y * f * f;
                        acc += v[u] * (f * f);
                    }
                }
            }
        }
        if (turns > 1) {
            s_acc[threadIdx.x] = acc; s_m[threadIdx.x] = m; s_l[threadIdx.x] = l;
            __syncthreads();
            if (turn != 0) return;
            float top = m;
            for (int u = 1; u < turns; ++u) top = fmaxf(top, s_m[u * hd + d]);
            const float f0 = half_factor(m, top);
            l = l * f0 * f0;
            acc *= f0 * f0;
            for (int u = 1; u < turns; ++u) {
                const float f = half_factor(s_m[u * hd + d], top);
                l += s_l[u * hd + d] * f * f;
                acc += s_acc[u * hd + d] * (f * f);
            }
        }
        if (d < hd) Elem<T>::store(out + ((size_t)token * a.heads + head) * hd + d, l == 0.f ? 0.f : acc / l * RELIFT);
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
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

template <int BYTES> __device__ __forceinline__ void copy_async(unsigned dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_async_or_zero(unsigned dst, const void* src, bool valid) {       // 4 bytes
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(unsigned at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

constexpr int STAGES = 3;           // steps of a warp on their way or being used

template <int HD, int NH> struct Mma {
    static constexpr int KU = HD == 64 ? 2 : 1, STEP = KU * 16, CHUNK = STEP * WARPS;
    static constexpr int STAGE = STEP * HD * 2 + 64;        // keys, values, and (key, value) scales of every 8 keys
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int ROWS = NH * 8, MS = HD + 4;
    static constexpr int MERGE = WARPS * ROWS * (MS + 2) * 4;
    static constexpr int OWN = RING > MERGE ? RING : MERGE;
    static constexpr int BYTES = OWN + ROWS * HD * 4 + 8 * ROWS * 8 + 128;      // and what the cluster's CTAs send: slices of outputs, (max, sum)
    static_assert(OWN % 16 == 0, "the slices are stored 16 bytes at a time");
};

__device__ __forceinline__ void st_peer_f32x4(unsigned addr, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void st_peer_f32x2(unsigned addr, const float2& v) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};\n" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void store_row4(__nv_bfloat16* out, const float4& acc, float l) {
    const float f = l == 0.f ? 0.f : RELIFT / l;            // a row that sees nothing is zero, an undefined one NaN
    const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x * f, acc.y * f), b = __floats2bfloat162_rn(acc.z * f, acc.w * f);
    *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// A step of a warp is 16 (heads of 128) or 32 keys, 4 KB. Thread (g, t) uses the 16-byte pieces t, t + 4 of the key rows g and g + 8,
// and the dims g * HD/8 .. of the value rows 2t, 2t + 1, 2t + 8, 2t + 9 of every 16 keys, and copies just these, asynchronously, into
// places of its own: rows of 64 or 128 bytes are read whole by one instruction, shared memory is read without conflicts, and no
// thread waits for another's copies.
//
// A key code enters the tensor core as the 16-bit number (code + 128) 2^-24, which is the code's byte, its first bit turned over, with
// zeros before it; what the 128 adds to a score, 128 2^-24 sum of the head's elements, is what the accumulator begins at.
// WHOLE: pages of a multiple of 16 tokens, so that 16 keys lie in one.
template <int HD, int NH, bool WHOLE>
__global__ void __launch_bounds__(WARPS * 32, NH == 1 ? 4 : 2)
attention_int8_mma_kernel(const __nv_bfloat16* q_rows, __nv_bfloat16* __restrict__ out, const Args a) {
    using C = Mma<HD, NH>;
    constexpr int KU = C::KU, STEP = C::STEP, MS = C::MS, ROWS = C::ROWS, H = WHOLE ? 1 : 2, IDS = KU * H, ID_KEYS = 16 / H;
    constexpr int V_AT = STEP * HD, S_AT = 2 * STEP * HD;
    extern __shared__ __align__(16) unsigned char mma_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const unsigned ring = smem_u32(mma_smem) + warp * STAGES * C::STAGE;
    if (a.csize > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");       // this CTA is there: its peers may send
    Pieces<C::CHUNK> piece;
    // The warp takes a step of every chunk. Lane i looks up the pages of its i-th step from here, 32 at a time.
    int ids[IDS];
    auto look_up = [&](int chunk) {
        const int* bt = a.block_table + (size_t)piece.token * a.bt_stride;
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
            const int key = (chunk + lane) * C::CHUNK + warp * STEP + i * ID_KEYS;
            int slot;
            ids[i] = chunk + lane < piece.end && key <= piece.p && key + ID_KEYS > piece.lo ? page_at(a, bt, key, slot) : -1;
        }
    };
    const long long page_bytes = (long long)a.kv_heads * a.page_size * HD;
    // A page that the request does not hold is read as the pool's first with scales of 0: nothing leaves the pool.
    auto send_scales = [&](int stage, int i, int page) {
        if (lane < 2) {
            const size_t block = (size_t)max(page, 0) * a.kv_heads + piece.kvh;
            copy_async_or_zero(ring + stage * C::STAGE + S_AT + i * 8 + lane * 4, (lane ? a.v_scales : a.k_scales) + block, page >= 0);
        }
    };
    auto send = [&](int chunk, int stage, auto with_scales) {
        const unsigned dst = ring + stage * C::STAGE;
        const int from = (chunk - piece.begin) & 31;
        const signed char* k_lane = a.k_pages + (size_t)piece.kvh * a.page_size * HD + g * HD + t * 16;
        const signed char* v_lane = a.v_pages + (size_t)piece.kvh * a.page_size * HD + 2 * t * HD + g * (HD / 8);
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
            const int key = chunk * C::CHUNK + warp * STEP + i * ID_KEYS;
            const int page = __shfl_sync(0xffffffffu, ids[i], from);
            const bool held = page >= 0;
            const int slot = !held ? 0 : a.shift >= 0 ? key & (a.page_size - 1) : key % a.page_size;
            const long long at = max(page, 0) * page_bytes + slot * HD;
            if (with_scales) send_scales(stage, i, page);
#pragma unroll
            for (int h = 0; h < 2 / H; ++h) {
                const int part = i * (2 / H) + h;               // 8 keys
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) copy_async<16>(dst + (part * (HD / 64) + j) * 512 + lane * 16, k_lane + at + h * 8 * HD + j * 64);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    copy_async<HD / 8>(dst + V_AT + (part * 2 + j) * (32 * HD / 8) + lane * (HD / 8), v_lane + at + (h * 8 + j) * HD);
            }
        }
    };
    bool more = piece.first(a, lane);
    if (more) look_up(piece.begin);         // lengths and tables are the step's inputs; queries, keys, values and scales are kernels' results
    // Where the caller says so, the codes of pages before the one that the token's own key goes to are sent for before the wait. Not their
    // scales: one of another page, which the kernel before this one may be writing, can lie in the same 32 bytes, and a copy of 4 bytes
    // leaves those in the SM's first cache. (Codes of 8 bytes go through it too: pools that begin on 128 bytes have pages of whole lines.)
    int sent = 0;
    if (a.early && more) {
        const int own_page = piece.p >= 0 ? piece.p - piece.p % a.page_size : 0;
        while (sent < STAGES - 1 && piece.begin + sent < piece.end && (piece.begin + sent + 1) * C::CHUNK <= own_page) {
            send(piece.begin + sent, sent, std::false_type{});
            ++sent;
        }
    }
    pdl_wait();
    // (Let in at this kernel's first instruction the one behind takes places that its own CTAs could have: 8 tokens of 4,096 keys in a chain
    // of such calls 9.4 us instead of 6.6, 64 of 200 to 4,000 24 instead of 16.)
    pdl_launch_dependents();
    while (more) {
        const int token = piece.token, kvh = piece.kvh, p = piece.p, lo = piece.lo;
        unsigned raw[HD / 16][NH][2];           // the queries, as they are stored
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            const int head = nh * 8 + g;
            const __nv_bfloat16* qp = q_rows + (size_t)token * a.q_stride + (size_t)(kvh * a.n_rep + head) * HD + t * 16;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    raw[kk][nh][j] = head < a.n_rep ? *reinterpret_cast<const unsigned*>(qp + (kk >> 2) * 64 + (kk & 3) * 4 + 2 * j) : 0u;
        }
#pragma unroll 1
        for (int i = 0; i < sent; ++i) {
#pragma unroll
            for (int j = 0; j < IDS; ++j) send_scales(i, j, __shfl_sync(0xffffffffu, ids[j], i));
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
        for (int i = sent; i < STAGES - 1; ++i) {
            if (piece.begin + i < piece.end) send(piece.begin + i, i, std::true_type{});
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
        sent = 0;

        // Q^T as the column operand, its dims in the order in which the key rows' pieces hold them. A head is scaled by a power of two
        // so that its largest element lies in 2^12 .. 2^13: 16-bit floats then hold every element that counts exactly.
        unsigned qb[HD / 16][NH][2];
        float factor[NH][2], bias[NH][2];
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            unsigned top = 0;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
                for (int j = 0; j < 2; ++j) top = max(top, max(raw[kk][nh][j] & 0x7fffu, (raw[kk][nh][j] >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the exponent field e of the largest element: 2^(139 - e) takes it to 2^12 (in two factors: the power may leave the range)
            const int e = (int)(top >> 7), up = (e == 0 || e == 255) ? 0 : 139 - e;
            const float f1 = __uint_as_float((unsigned)(127 + up / 2) << 23), f2 = __uint_as_float((unsigned)(127 + up - up / 2) << 23);
            float sum = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qb[kk][nh][j] = pack_f16(__uint_as_float(raw[kk][nh][j] << 16) * f1 * f2, __uint_as_float(raw[kk][nh][j] & 0xffff0000u) * f1 * f2);
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

        int stage = 0, ahead = STAGES - 1;
#pragma unroll 1
        for (int chunk = piece.begin; chunk < piece.end; ++chunk) {
            if (((chunk + STAGES - 1 - piece.begin) & 31) == 0) look_up(chunk + STAGES - 1);
            if (chunk + STAGES - 1 < piece.end) send(chunk + STAGES - 1, ahead, std::true_type{});
            asm volatile("cp.async.commit_group;\ncp.async.wait_group %0;\n" ::"n"(STAGES - 1) : "memory");
            __syncwarp();                           // (the scales are two lanes' copies)
            const unsigned src = ring + stage * C::STAGE;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
            float2 sc[IDS];
#pragma unroll
            for (int i = 0; i < IDS; ++i) {
                const uint2 u = lds8(src + S_AT + i * 8);
                sc[i] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
            }
            float s[KU][NH][4];
            // S^T = K Q^T
#pragma unroll
            for (int ku = 0; ku < KU; ++ku) {
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) { s[ku][nh][0] = s[ku][nh][2] = bias[nh][0]; s[ku][nh][1] = s[ku][nh][3] = bias[nh][1]; }
#pragma unroll
                for (int i = 0; i < HD / 64; ++i) {
                    const uint4 r0 = lds16(src + ((ku * 2) * (HD / 64) + i) * 512 + lane * 16), r1 = lds16(src + ((ku * 2 + 1) * (HD / 64) + i) * 512 + lane * 16);
                    const unsigned w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
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
            const int k0 = chunk * C::CHUNK + warp * STEP;
            const bool edge = k0 < lo || k0 + STEP - 1 > p;
            float lv[IDS], vs[IDS];
#pragma unroll
            for (int i = 0; i < IDS; ++i) { lv[i] = reference_log2(sc[i].y); vs[i] = sc[i].y * UNLIFT; }
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int ku = 0; ku < KU; ++ku)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int id = WHOLE ? ku : ku * 2 + (e >> 1);
                        float v = s[ku][nh][e] * (factor[nh][e & 1] * sc[id].x);
                        if (edge) {
                            const int key = k0 + g + ku * 16 + 8 * (e >> 1);
                            if (key < lo || key > p) v = -INFINITY;
                        }
                        s[ku][nh][e] = v;
                        top[e & 1] = fmaxf(top[e & 1], v + lv[id]);
                    }
                // the reference moves only where a key is 2^6 above it: p is at most 2^15 meanwhile, within 16 bits
                if (__any_sync(0xffffffffu, top[0] > m_ref[nh][0] + 6.f || top[1] > m_ref[nh][1] + 6.f)) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 4));
                        top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 8));
                        top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 16));
                        const float m_new = fmaxf(m_ref[nh][q], top[q]);
                        const float f = half_factor(m_ref[nh][q], m_new), corr = f * f;
                        m_ref[nh][q] = m_new;
                        l_part[nh][q] = l_part[nh][q] * f * f;
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
                            float pv = w * vs[WHOLE ? ku : ku * 2 + h];
                            if (edge && s[ku][nh][2 * h + q] == -INFINITY) pv = 0.f;        // (a hidden key's block may be undefined; a seen one's counts, however little it weighs)
                            s[ku][nh][2 * h + q] = pv;
                        }
                }
            }
            // O^T += V^T P^T
#pragma unroll
            for (int ku = 0; ku < KU; ++ku) {
                unsigned pb[NH][2], v[4][HD / 32];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned at = src + V_AT + (ku * 4 + j) * (32 * HD / 8) + lane * (HD / 8);
                    if constexpr (HD == 64) { const uint2 u = lds8(at); v[j][0] = u.x; v[j][1] = u.y; }
                    else { const uint4 u = lds16(at); v[j][0] = u.x; v[j][1] = u.y; v[j][2] = u.z; v[j][3] = u.w; }
                }
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    pb[nh][0] = movmatrix_trans(pack_f16(s[ku][nh][0], s[ku][nh][1]));
                    pb[nh][1] = movmatrix_trans(pack_f16(s[ku][nh][2], s[ku][nh][3]));
                }
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) {             // four dims: two row tiles of V^T
                    const unsigned x0 = v[0][w] ^ 0x80808080u, x1 = v[1][w] ^ 0x80808080u;
                    const unsigned x2 = v[2][w] ^ 0x80808080u, x3 = v[3][w] ^ 0x80808080u;
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
            __syncwarp();                           // the scales' places are free
        }
        __syncthreads();                            // every warp is through with its copies: their room is used for the merge

        // ---- the warps' results, relative to their common maximum, and their sums
        float* sm_o = reinterpret_cast<float*>(mma_smem);           // [WARPS][ROWS][MS]
        float2* sm_ml = reinterpret_cast<float2*>(sm_o + WARPS * ROWS * MS);            // [WARPS][ROWS]
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float l = l_part[nh][q];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) sm_ml[warp * ROWS + nh * 8 + 2 * t + q] = make_float2(m_ref[nh][q], l);
            }
        __syncthreads();
        auto whole_row = [&](int row) {
            float2 x[WARPS], all = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) { x[w] = sm_ml[w * ROWS + row]; all.x = fmaxf(all.x, x[w].x); }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) { const float f = half_factor(x[w].x, all.x); all.y += x[w].y * f * f; }
            return all;
        };
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = nh * 8 + 2 * t + q;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_ml[w * ROWS + row].x);
                const float f0 = half_factor(m_ref[nh][q], top), f = f0 * f0;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d)           // row g of tile d is the dim g * HD/8 + 2d, row g + 8 the one behind it
                    *reinterpret_cast<float2*>(sm_o + (warp * ROWS + row) * MS + g * (HD / 8) + 2 * d) = make_float2(o[d][nh][q] * f, o[d][nh][2 + q] * f);
            }
        __syncthreads();
        const int quads = a.n_rep * (HD / 4);
        auto sum_of = [&](int i) {
            const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
            float4 s = *reinterpret_cast<const float4*>(sm_o + row * MS + d);
#pragma unroll
            for (int w = 1; w < WARPS; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * ROWS + row) * MS + d);
                s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
            }
            return s;
        };
        __nv_bfloat16* rows = out + ((size_t)token * a.heads + (size_t)kvh * a.n_rep) * HD;
        if (piece.part >= 0) {
            float4* to = reinterpret_cast<float4*>(a.part_o) + (size_t)piece.part * quads;
            for (int i = tid; i < quads; i += WARPS * 32) to[i] = sum_of(i);
            if (tid < a.n_rep) reinterpret_cast<float2*>(a.part_ml)[(size_t)piece.part * a.n_rep + tid] = whole_row(tid);
        } else if (a.csize == 1) {
            for (int i = tid; i < quads; i += WARPS * 32) store_row4(rows + i * 4, sum_of(i), whole_row(i / (HD / 4)).y);
        } else {
            // every CTA of the cluster finishes a slice: the others send it theirs, and the (max, sum) of all rows
            const int rank = (int)cluster_rank(), slice = (quads + a.csize - 1) / a.csize;
            float4* recv = reinterpret_cast<float4*>(mma_smem + C::OWN);               // [csize][slice]
            float2* recv_ml = reinterpret_cast<float2*>(mma_smem + C::OWN + ROWS * HD * 4 + 128);         // [csize][n_rep]
            asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");               // every CTA is there
            for (int i = tid; i < quads; i += WARPS * 32) {
                const int to = i / slice;
                st_peer_f32x4(peer_smem(recv + rank * slice + (i - to * slice), to), sum_of(i));
            }
            if (tid < a.n_rep) {
                const float2 ml = whole_row(tid);
                for (int r = 0; r < a.csize; ++r) st_peer_f32x2(peer_smem(recv_ml + rank * a.n_rep + tid, r), ml);
            }
            cluster_sync();
            const int end = min(quads, (rank + 1) * slice);
            for (int i = rank * slice + tid; i < end; i += WARPS * 32) {
                const int row = i / (HD / 4);
                float top = -INFINITY, l = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int r = 0; r < a.csize; ++r) top = fmaxf(top, recv_ml[r * a.n_rep + row].x);
                for (int r = 0; r < a.csize; ++r) {
                    const float2 ml = recv_ml[r * a.n_rep + row];
                    const float4 x = recv[r * slice + (i - rank * slice)];
                    const float f0 = half_factor(ml.x, top), f = f0 * f0;
                    l += ml.y * f0 * f0;
                    acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
                }
                store_row4(rows + i * 4, acc, l);
            }
        }
        more = piece.next(a, lane);
        if (more) {
            __syncthreads();                        // the next piece's copies go where this one's results are
            look_up(piece.begin);
        }
    }
}

// ------------------------------------------------------------------------------------------ any shape
// Tiles of 32 keys, as 32-bit values in shared memory: a thread has one (query head, key) of the scores at a time, then one
// (query head, dim) of the sums. VEC: heads of a multiple of 16, whose rows are read 16 bytes at a time.
constexpr int GT = 32, GEN_THREADS = 128;

template <typename T, bool VEC>
__global__ void __launch_bounds__(GEN_THREADS)
attention_int8_any_kernel(const T* q_rows, T* __restrict__ out, const Args a) {
    extern __shared__ __align__(16) float smem[];
    const int hd = a.head_dim, n_rep = a.n_rep, tid = threadIdx.x;
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
    pdl_launch_dependents();
    Pieces<GT> piece;
    bool more = piece.first(a, tid & 31);
    pdl_wait();
    for (; more; more = piece.next(a, tid & 31)) {
    const int token = piece.token, kvh = piece.kvh, p = piece.p, lo = piece.lo;
    const int* bt = a.block_table + (size_t)token * a.bt_stride;
    for (int i = tid; i < n_rep * hd; i += GEN_THREADS) {
        q[i] = Elem<T>::load(q_rows + (size_t)token * a.q_stride + (size_t)kvh * n_rep * hd + i) * (a.scale * LOG2E);
        cta_o[i] = 0.f;
    }
    for (int i = tid; i < n_rep; i += GEN_THREADS) { cta_ml[2 * i] = -INFINITY; cta_ml[2 * i + 1] = 0.f; }
    for (int tile = piece.begin; tile < piece.end; ++tile) {
        __syncthreads();
        if (tid < GT) {
            const int key = tile * GT + tid;
            int slot = 0;
            const int page = key >= lo && key <= p ? page_at(a, bt, key, slot) : -1;
            const size_t block = (size_t)max(page, 0) * a.kv_heads + kvh;
            from[tid] = page >= 0 ? (long long)((block * a.page_size + slot) * hd) : -1;
            ks[tid] = page >= 0 ? __ldcg(a.k_scales + block) : 0.f;
            vs[tid] = page >= 0 ? __ldcg(a.v_scales + block) : 0.f;
        }
        __syncthreads();
        if (VEC) {
            const int chunks = hd >> 4;
            for (int i = tid; i < GT * chunks; i += GEN_THREADS) {
                const int row = i / chunks, d = (i - row * chunks) * 16;
                const long long at = from[row];
                uint4 k = make_uint4(0, 0, 0, 0), v = k;
                if (at >= 0) { k = __ldcg(reinterpret_cast<const uint4*>(a.k_pages + at + d)); v = __ldcg(reinterpret_cast<const uint4*>(a.v_pages + at + d)); }
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
                kt[row * ks_stride + d] = at >= 0 ? (float)a.k_pages[at + d] * ks[row] : 0.f;
                vt[i] = at >= 0 ? (float)a.v_pages[at + d] : 0.f;
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
                const float f = half_factor(m_old, m_new);
                corr[h] = f * f;
                cta_ml[2 * h] = m_new;
                cta_ml[2 * h + 1] = cta_ml[2 * h + 1] * f * f + sum;
            }
            w[i] = e * (vs[row] * UNLIFT);          // (of a hidden key both are 0)
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
    finish(cta_o, cta_ml, a, token, kvh, piece.part, hd, out, GEN_THREADS);
    if (a.shares) __syncthreads();
    }
}

long long any_smem(int n_rep, int hd) { return 4LL * (2LL * n_rep * hd + GT * (2LL * hd + 4) + n_rep * (GT + 3LL)); }
constexpr long long MAX_SMEM = 226 * 1024;         // (and what a CTA has besides)

template <typename T, int CH>
int launch_rows(void (*kernel)(const T*, T*, Args), const Args& a, int sms, int threads, long long smem, const void* q, void* out, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = a.shares ? dim3(a.shares) : dim3(a.csize, a.n_tokens, a.kv_heads);
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
    if (a.shares) NIB_CUDA(launch_pdl(merge_int8_kernel<T, CH>, dim3(a.heads, a.n_tokens), dim3(a.heads * a.n_tokens <= 2 * sms ? MERGE_THREADS : MERGE_THREADS / 2), (size_t)0, stream, (T*)out, a));
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
    int q_stride, bt_stride, bt_width, page_size, num_pages, n_tokens, heads, kv_heads, head_dim, window, ctas, shares, dtype, early;
    float scale; int sms;       // sms: SMs of the device
};

// Attention of n_tokens single tokens (token i is request i, at position ctx_lens[i] - 1) whose keys and values are in the pages.
// ``shares`` 0: the keys of a (token, kv head) are cut among ``ctas`` CTAs (1, 2, 4 or 8). Else all rows' keys are dealt to that many
// CTAs: part_o [2 * shares * heads/kv_heads * head_dim], part_ml [2 * shares * heads/kv_heads * 2].
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
    if (c.shares) {
        NIB_REQUIRE(c.ctas == 1 && c.shares > 0 && c.part_o && c.part_ml, "attention (8-bit cache): shares need scratch memory");
        // (chunks are counted in 32 bits; of 32 keys at least)
        NIB_REQUIRE(((long long)c.bt_width * page_size / GT + 1) * kv_heads * n_tokens < (1LL << 31), "attention (8-bit cache): too many keys for one launch");
    } else {
        NIB_REQUIRE(c.ctas == 1 || c.ctas == 2 || c.ctas == 4 || c.ctas == 8, "attention (8-bit cache): 1, 2, 4 or 8 CTAs share a row's keys, not %d", c.ctas);
    }
    NIB_REQUIRE(c.sms > 0 && n_tokens <= 65535 && kv_heads <= 65535, "attention (8-bit cache): too many tokens or heads for one launch");
    if (n_tokens == 0) return 0;
    int shift = -1;
    if ((page_size & (page_size - 1)) == 0) for (shift = 0; (1 << shift) < page_size;) ++shift;
    const Args a{c.ctx_lens, c.block_table, (const signed char*)c.k_pages, (const signed char*)c.v_pages, c.k_scales, c.v_scales, c.part_o, c.part_ml,
                 c.q_stride, c.bt_stride, c.bt_width, page_size, shift, c.num_pages, n_tokens, heads, kv_heads, heads / kv_heads, head_dim, c.window, c.ctas, c.shares,
                 c.early && (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 127) == 0, c.scale};
    int rc;
    // (rows and pools that lie off the pieces that a thread reads and writes at a time go to the general kernel)
    if (kind == 1 && ((uintptr_t)q & 3) == 0 && c.q_stride % 2 == 0 && ((uintptr_t)out & 7) == 0 && (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) == 0) {
#define CALL(KERNEL, T, CH, THREADS, SMEM, MOST)                                                                                \
    do {                                                                                                                        \
        NIB_CUDA((allow_smem_once<KERNEL>((int)(MOST))));                                                                       \
        rc = launch_rows<T, CH>((KERNEL), a, c.sms, THREADS, SMEM, q, out, stream);                                                      \
    } while (0)
#define MMA(HD, NH, WHOLE)                                                                                                      \
    CALL((attention_int8_mma_kernel<HD, NH, WHOLE>), __nv_bfloat16, (Mma<HD, NH>::CHUNK), WARPS * 32, (Mma<HD, NH>::BYTES), (Mma<HD, NH>::BYTES))
#define HEADS(NH)                                                                                       \
    do {                                                                                                \
        if (page_size % 16 == 0) { if (head_dim == 64) MMA(64, NH, true); else MMA(128, NH, true); }    \
        else { if (head_dim == 64) MMA(64, NH, false); else MMA(128, NH, false); }                      \
    } while (0)
        if (a.n_rep <= 8) HEADS(1); else HEADS(2);
    } else {
        const bool vec = head_dim % 16 == 0 && (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) == 0;
#define ANY(T, VEC) CALL((attention_int8_any_kernel<T, VEC>), T, GT, GEN_THREADS, any_smem(a.n_rep, head_dim), MAX_SMEM)
        if (dtype == NIB_F32) { if (vec) ANY(float, true); else ANY(float, false); }
        else { if (vec) ANY(__nv_bfloat16, true); else ANY(__nv_bfloat16, false); }
#undef ANY
    }
#undef HEADS
#undef MMA
#undef CALL
    return rc;
}
