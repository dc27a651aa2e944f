// The 8-bit cache of keys and values: appending a step's tokens with the position rotation on the way, and reading pages
// back as 16- or 32-bit numbers.
//
// A block is the page_size tokens of one page and one kv head; it has one scale for its keys and one for its values, powers
// of two held as floats, and a value is code * scale with a signed 8-bit code. code * 2^e is exact in bfloat16 (8 significant
// bits) and in 32 bits, so every reader sees the same numbers. For the tokens that a step adds to a block, of which n0 were
// held before:
//     a  = max |x|                      over the step's elements in the block (keys after the rotation)
//     s' = 2^e, e least in -80..121 with a <= 127 * 2^e;  max(s, s') where n0 > 0 and the block has a scale s already
//     code = rint(x / s')               new elements, within -127..127
//     code = rint(code * s / s')        elements held before (only where the scale grew)
// A scale grows by factors of two, so the roundings of one element add up to less than s'/2 (1 + 1/2 + 1/4 + ...) = s'; with
// scales of any value every growth could add another half step. An element that is not finite makes the block's scale NaN:
// whoever reads the block sees that it is undefined. Slots behind the last token keep their codes.
//
// A code is a rounding to whole steps, and a key that lies between two must not change its side with the order of the rotation's
// products: an element is formed as the sum of a float and what its rounding left (the products' errors by a fused multiply-add, the
// sum's by the two-sum), some 48 bits, of which the second part decides ties. (In 64 bits it was twice as slow: conversions.)
//
// What bounds it: a decode step's launch and three dependent loads (2.7 us a call in a chain, one token of 14 + 2 x 2 heads of 64); for a
// prompt's portion loads that wait for loads, and the queries' bytes (3,789 tokens of 28 + 2 x 4 heads of 128: 19.8 us, 66 MB).
#include "common.cuh"

namespace {

constexpr int E_MIN = -80, E_MAX = 121;

// 2^e with the least e in E_MIN..E_MAX that has a <= 127 * 2^e; NaN unless a is finite.
__device__ __forceinline__ float block_scale(float a) {
    const unsigned bits = __float_as_uint(a);
    if ((bits & 0x7f800000u) == 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // a = 1.f * 2^x: 127 * 2^(x - 6) = 1.984375 * 2^x is enough unless a's fraction is above 0.984375 = 126/128
    int e = (int)(bits >> 23) - 127 - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    e = max(E_MIN, min(E_MAX, e));
    return __uint_as_float((unsigned)(e + 127) << 23);
}

// Where a unit of work lies: the tokens of one request in one page. Units are counted request by request; request r has at
// most (q_len + page_size - 2) / page_size + 1 of them, whatever its position.
struct Unit { int row, count, slot, pos; long long page; };       // pos: the first token's position

__device__ __forceinline__ Unit find_unit(int u, const int* __restrict__ q_start, const int* __restrict__ ctx_lens, int n_req,
                                          const int* __restrict__ block_table, int bt_stride, int bt_width, int page_size, int num_pages, int lane) {
    Unit out{0, 0, 0, 0, -1};
    int base = 0;
    for (int r0 = 0; r0 < n_req; r0 += 32) {
        const int r = r0 + lane;
        int begin = 0, n = 0;
        if (r < n_req) { begin = __ldg(q_start + r); n = __ldg(q_start + r + 1) - begin; }
        int units = n > 0 ? (n + page_size - 2) / page_size + 1 : 0, sum = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned mine = __ballot_sync(0xffffffffu, u < base + sum);
        if (mine) {
            const int src = __ffs(mine) - 1;
            const int before = base + __shfl_sync(0xffffffffu, sum - units, src);
            const int row = __shfl_sync(0xffffffffu, begin, src), q_len = __shfl_sync(0xffffffffu, n, src);
            const int first = __ldg(ctx_lens + r0 + src) - q_len;            // position of the request's first token of the step
            if (first < 0) return out;                                      // a padding row
            const int lp = first / page_size + (u - before);
            const int lo = max(first, lp * page_size), hi = min(first + q_len, (lp + 1) * page_size);
            if (hi <= lo || lp >= bt_width) return out;
            const int page = __ldg(block_table + (size_t)(r0 + src) * bt_stride + lp);
            out.row = row + (lo - first);
            out.count = hi - lo;
            out.slot = lo - lp * page_size;
            out.pos = lo;
            out.page = page >= 0 && page < num_pages ? page : -1;
            return out;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    return out;
}

template <typename T, int V> struct Vec;
template <> struct Vec<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void load(float (&f)[8], const __nv_bfloat16* p) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&v);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Vec<float, 8> {
    static __device__ __forceinline__ void load(float (&f)[8], const float* p) {
        *reinterpret_cast<float4*>(f) = reinterpret_cast<const float4*>(p)[0];
        *reinterpret_cast<float4*>(f + 4) = reinterpret_cast<const float4*>(p)[1];
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
        reinterpret_cast<float4*>(p)[0] = *reinterpret_cast<const float4*>(f);
        reinterpret_cast<float4*>(p)[1] = *reinterpret_cast<const float4*>(f + 4);
    }
};
template <> struct Vec<__nv_bfloat16, 4> {
    static __device__ __forceinline__ void load(float (&f)[4], const __nv_bfloat16* p) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
        f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
    }
};
template <> struct Vec<float, 4> {
    static __device__ __forceinline__ void load(float (&f)[4], const float* p) { *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p); }
};
template <typename T> struct Vec<T, 1> {
    static __device__ __forceinline__ void load(float (&f)[1], const T* p) { f[0] = Elem<T>::load(p); }
    static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { Elem<T>::store(p, f[0]); }
};

template <int V> __device__ __forceinline__ void store_codes(signed char* p, const int (&c)[V]) {
    if constexpr (V > 1) {
        unsigned w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            w[i] = (unsigned)(c[4 * i] & 0xff) | ((unsigned)(c[4 * i + 1] & 0xff) << 8) | ((unsigned)(c[4 * i + 2] & 0xff) << 16) | ((unsigned)(c[4 * i + 3] & 0xff) << 24);
        if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<unsigned*>(p) = w[0];
    } else {
        p[0] = (signed char)c[0];
    }
}

// a * b + c * d as hi + lo, hi the nearest float.
struct Two { float hi, lo; };
__device__ __forceinline__ Two sum_of_products(float a, float b, float c, float d) {
    const float p = __fmul_rn(a, b), pe = __fmaf_rn(a, b, -p), q = __fmul_rn(c, d), qe = __fmaf_rn(c, d, -q);
    const float s = __fadd_rn(p, q), bb = __fsub_rn(s, p), se = __fadd_rn(__fsub_rn(p, __fsub_rn(s, bb)), __fsub_rn(q, bb));
    const float e = __fadd_rn(se, __fadd_rn(pe, qe)), hi = __fadd_rn(s, e);
    return {hi, __fsub_rn(e, __fsub_rn(hi, s))};
}
// The magnitude of hi + lo rounded up to a float, as an integer, in whose order a NaN's bits are above everything. (127 * 2^e is a
// float, so the comparison with it stays what it is.)
__device__ __forceinline__ unsigned magnitude_up(const Two& y) {
    const unsigned bits = __float_as_uint(y.hi) & 0x7fffffffu;
    return bits + ((y.lo != 0.f && (y.lo > 0.f) == (y.hi > 0.f) && bits < 0x7f800000u) ? 1u : 0u);
}
// rint((hi + lo) / s) within -127..127, inv = 1 / s, a power of two: the product with it is exact. Of a NaN: -127 (a code like any other; its
// block's scale, NaN too, is what says that it is undefined).
__device__ __forceinline__ int code_of(const Two& y, float inv) {
    const float v = fminf(fmaxf(__fmul_rn(y.hi, inv), -127.f), 127.f);
    float r = rintf(v);
    if (fabsf(v - r) == 0.5f && y.lo != 0.f) r = y.lo > 0.f ? ceilf(v) : floorf(v);
    return (int)r;
}

// rint(code * by) of four codes.
__device__ __forceinline__ unsigned smaller(unsigned w, float by) {
    unsigned r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (unsigned)(__float2int_rn((float)(signed char)(w >> (8 * i)) * by) & 0xff) << (8 * i);
    return r;
}

constexpr int KV_THREADS = 128;

// The scale of a block whose new elements' largest magnitude is ``top``, and the codes that it held before made smaller where that
// scale is larger than theirs. All threads take part.
__device__ __forceinline__ float scale_of(unsigned top, float old, int slots, signed char* codes, int hd, int tid) {
    float scale = block_scale(__uint_as_float(top));
    if (slots == 0) return scale;
    const bool undefined = scale != scale || old != old;
    scale = undefined ? __uint_as_float(0x7fc00000u) : fmaxf(old, scale);
    if (scale > old) {          // (not where it is undefined)
        const float by = old / scale;       // a power of two, or 0 where the block had no scale yet
        const int bytes = slots * hd, wide = ((uintptr_t)codes & 15) == 0 ? bytes >> 4 : 0;
        // 16 codes at a time (a byte at a time the one block of a step's whose scale grew was what the kernel's time went by: 13 us
        // for 64 tokens of 4 heads of 128)
        for (int i = tid; i < wide; i += KV_THREADS) {
            const uint4 w = reinterpret_cast<const uint4*>(codes)[i];
            reinterpret_cast<uint4*>(codes)[i] = make_uint4(smaller(w.x, by), smaller(w.y, by), smaller(w.z, by), smaller(w.w, by));
        }
        for (int i = wide * 16 + tid; i < bytes; i += KV_THREADS) codes[i] = (signed char)__float2int_rn((float)codes[i] * by);
    }
    return scale;
}

struct AppendArgs {
    const int* positions; const int* q_start; const int* ctx_lens; const float* cos_t; const float* sin_t;
    const int* block_table; signed char* k_pages; signed char* v_pages; float* k_scales; float* v_scales;
    int table_rows, rot, bt_stride, bt_width, page_size, num_pages, m, n_req, heads, kv_heads, head_dim, q_stride, out_stride;
    int units, kv_blocks;       // the first kv_blocks CTAs append, one for each (unit, kv head); the others rotate queries
};

// ---- queries: an item is a chunk of VQ pairs, or a chunk beyond the rotated width, of one head of one token.
template <typename T, int VQ>
__device__ __forceinline__ void rotate_queries(const T* qkv, T* q_out, const AppendArgs& a, long long i, bool& waited) {
    const int half = a.rot >> 1, hd = a.head_dim, pairs = half / VQ, per_head = pairs + (hd - a.rot) / VQ, per_token = a.heads * per_head;
    const int tok = (int)(i / per_token), rest = (int)(i - (long long)tok * per_token), head = rest / per_head, c = rest - head * per_head;
    const T* p = qkv + (size_t)tok * a.q_stride + (size_t)head * hd;
    T* o = q_out + (size_t)tok * a.out_stride + (size_t)head * hd;
    float x1[VQ], x2[VQ], cs[VQ], sn[VQ], y1[VQ], y2[VQ];
    if (c < pairs) {
        const int d = c * VQ, pos = a.positions[tok];         // (positions and tables are the step's inputs)
        const bool known = pos >= 0 && pos < a.table_rows;
        const size_t at = (size_t)(known ? pos : 0) * half + d;
        Vec<float, VQ>::load(cs, a.cos_t + at);
        Vec<float, VQ>::load(sn, a.sin_t + at);
        if (!waited) { pdl_wait(); pdl_launch_dependents(); waited = true; }
        Vec<T, VQ>::load(x1, p + d);
        Vec<T, VQ>::load(x2, p + d + half);
#pragma unroll
        for (int j = 0; j < VQ; ++j) {
            y1[j] = known ? x1[j] * cs[j] - x2[j] * sn[j] : NAN;
            y2[j] = known ? x2[j] * cs[j] + x1[j] * sn[j] : NAN;
        }
        Vec<T, VQ>::store(o + d, y1);
        Vec<T, VQ>::store(o + d + half, y2);
    } else {
        const int d = a.rot + (c - pairs) * VQ;
        if (!waited) { pdl_wait(); pdl_launch_dependents(); waited = true; }
        Vec<T, VQ>::load(x1, p + d);
        Vec<T, VQ>::store(o + d, x1);
    }
}

constexpr int ROTATE_THREADS = 256;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(ROTATE_THREADS)
rotate_queries_kernel(const T* qkv, T* q_out, const AppendArgs a, long long items) {
    const long long i = (long long)blockIdx.x * ROTATE_THREADS + threadIdx.x;
    bool waited = false;
    if (i < items) rotate_queries<T, WIDE ? 8 : 1>(qkv, q_out, a, i, waited);
    if (!waited) { pdl_wait(); pdl_launch_dependents(); }
}

// ---- keys and values: a CTA for each (unit, kv head), two items of keys and two of values a thread at a time, whose loads are all on
// their way before the first is used; a page of 16 tokens of 128 elements is one such turn, and its items stay in registers from the
// search for the largest magnitude to their codes. (A warp for each of keys and values took 29 us for 4,096 tokens of 4 heads of 128,
// waiting for one load after another.)
// WIDE: chunks of 8 elements of queries and values and 4 of keys; 1 where widths or addresses do not allow it.
// QUERIES: CTAs from kv_blocks on rotate a token's queries each, one launch up to ONE_LAUNCH tokens. Without, a kernel of its own rotates them
// before: its threads hold 40 registers where these hold 125, which many tokens' queries need. us, two launches / one, 16-bit rows in a chain, 300,
// 1,000, 1,500, 2,048 and 4,096 tokens: 14 + 2 x 2 heads of 64 4.7 / 3.0, 5.0 / 3.3, 5.2 / 4.1, 5.5 / 5.3, 7.0 / 9.0; 12 + 2 x 2 of 128 5.9 / 4.3, 6.5 / 4.8, 7.1 / 5.3,
// 7.7 / 6.6, 10.3 / 12.4; 28 + 2 x 4 of 128 6.1 / 4.9, 7.6 / 6.0, 9.2 / 8.9, 10.7 / 11.7, 21.8 / 24.5.
constexpr int ONE_LAUNCH = 1536;
template <typename T, int V> struct KeyRaw { float x1[V], x2[V], cs[V], sn[V]; int row, d; bool pair; };       // the second chunk only of a rotated pair
template <int V> struct KeyItem { Two y1[V], y2[V]; int row, d; bool pair; };
template <typename T, int V> struct ValueItem { float x[V]; int row, d; };

template <typename T, bool WIDE, bool QUERIES>
__global__ void __launch_bounds__(KV_THREADS)
append_int8_kernel(const T* qkv, T* q_out, const AppendArgs a) {        // (q_out may be qkv)
    constexpr int V = WIDE ? 4 : 1, VV = WIDE ? 8 : 1, B = 2, TURN = KV_THREADS * B;
    __shared__ unsigned s_top[2][KV_THREADS / 32];
    const int half = a.rot >> 1, hd = a.head_dim, tid = threadIdx.x, lane = tid & 31;
    if (QUERIES && (int)blockIdx.x >= a.kv_blocks) {
        constexpr int VQ = WIDE ? 8 : 1;
        const int per_token = a.heads * ((half + hd - a.rot) / VQ);
        bool waited = false;
        for (int i = tid; i < per_token; i += KV_THREADS)
            rotate_queries<T, VQ>(qkv, q_out, a, (long long)(blockIdx.x - a.kv_blocks) * per_token + i, waited);
        if (!waited) { pdl_wait(); pdl_launch_dependents(); }
        return;
    }
    const int u = blockIdx.x / a.kv_heads, kvh = blockIdx.x - u * a.kv_heads;
    const Unit unit = find_unit(u, a.q_start, a.ctx_lens, a.n_req, a.block_table, a.bt_stride, a.bt_width, a.page_size, a.num_pages, lane);     // (lengths and tables, too)
    // (The attention behind is let in only now: its CTAs, placed while the kernel before this one still holds its SMs, would share few of
    // them. 8 tokens of 4,096 keys, 28 heads of 128, both calls: 17 us, and 21 let in at once.)
    pdl_wait();
    pdl_launch_dependents();
    if (unit.page < 0 || unit.row < 0 || unit.row + unit.count > a.m) return;       // (never a row that the call did not bring)
    const size_t block = (size_t)unit.page * a.kv_heads + kvh;
    signed char* k_codes = a.k_pages + block * a.page_size * hd;
    signed char* v_codes = a.v_pages + block * a.page_size * hd;
    const T* k_rows = qkv + (size_t)unit.row * a.q_stride + (size_t)(a.heads + kvh) * hd;
    const T* v_rows = k_rows + (size_t)a.kv_heads * hd;
    const float k_old = unit.slot > 0 ? a.k_scales[block] : 0.f, v_old = unit.slot > 0 ? a.v_scales[block] : 0.f;
    const int pairs = half / V, k_per_token = pairs + (hd - a.rot) / V, v_per_token = hd / VV;
    const int k_items = unit.count * k_per_token, v_items = unit.count * v_per_token;
    const int k_first = tid, v_first = (tid + KV_THREADS / 2) % KV_THREADS;       // (few items: keys and values are different warps')

    auto load_key = [&](KeyRaw<T, V>& it, int i) {
        it.row = i / k_per_token;
        const int c = i - it.row * k_per_token;
        it.pair = c < pairs;
        it.d = it.pair ? c * V : a.rot + (c - pairs) * V;
        const T* p = k_rows + (size_t)it.row * a.q_stride;
        Vec<T, V>::load(it.x1, p + it.d);
        if (it.pair) {
            Vec<T, V>::load(it.x2, p + it.d + half);
            const int pos = unit.pos + it.row;
            const size_t at = (size_t)min(pos, a.table_rows - 1) * half + it.d;
            Vec<float, V>::load(it.cs, a.cos_t + at);
            Vec<float, V>::load(it.sn, a.sin_t + at);
            if (pos >= a.table_rows) {
#pragma unroll
                for (int j = 0; j < V; ++j) it.cs[j] = NAN;
            }
        }
    };
    auto load_value = [&](ValueItem<T, VV>& it, int i) {
        it.row = i / v_per_token;
        it.d = (i - it.row * v_per_token) * VV;
        Vec<T, VV>::load(it.x, v_rows + (size_t)it.row * a.q_stride + it.d);
    };
    auto turned = [&](KeyItem<V>& it, const KeyRaw<T, V>& raw) {
        it.row = raw.row; it.d = raw.d; it.pair = raw.pair;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            it.y1[j] = Two{raw.x1[j], 0.f};
            it.y2[j] = Two{0.f, 0.f};
            if (raw.pair) {
                it.y1[j] = sum_of_products(raw.x1[j], raw.cs[j], -raw.x2[j], raw.sn[j]);
                it.y2[j] = sum_of_products(raw.x2[j], raw.cs[j], raw.x1[j], raw.sn[j]);
            }
        }
    };
    // a turn's keys and values, loads first
    KeyItem<V> key[B];
    ValueItem<T, VV> value[B];
    unsigned k_top = 0, v_top = 0;
    const int turns = max((k_items + TURN - 1) / TURN, (v_items + TURN - 1) / TURN);
    auto take = [&](int turn) {
        KeyRaw<T, V> raw[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int at = turn * TURN + b * KV_THREADS;
            if (at + k_first < k_items) load_key(raw[b], at + k_first);
            if (at + v_first < v_items) load_value(value[b], at + v_first);
        }
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (turn * TURN + b * KV_THREADS + k_first < k_items) turned(key[b], raw[b]);
    };
    for (int turn = 0; turn < turns; ++turn) {
        take(turn);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int at = turn * TURN + b * KV_THREADS;
            if (at + k_first < k_items) {
#pragma unroll
                for (int j = 0; j < V; ++j) k_top = max(k_top, max(magnitude_up(key[b].y1[j]), magnitude_up(key[b].y2[j])));
            }
            if (at + v_first < v_items) {
#pragma unroll
                for (int j = 0; j < VV; ++j) v_top = max(v_top, __float_as_uint(value[b].x[j]) & 0x7fffffffu);
            }
        }
    }
    k_top = __reduce_max_sync(0xffffffffu, k_top);
    v_top = __reduce_max_sync(0xffffffffu, v_top);
    if (lane == 0) { s_top[0][tid >> 5] = k_top; s_top[1][tid >> 5] = v_top; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KV_THREADS / 32; ++w) { k_top = max(k_top, s_top[0][w]); v_top = max(v_top, s_top[1][w]); }
    const float k_scale = scale_of(k_top, k_old, unit.slot, k_codes, hd, tid), v_scale = scale_of(v_top, v_old, unit.slot, v_codes, hd, tid);
    const float k_inv = 1.0f / k_scale, v_inv = 1.0f / v_scale;
    for (int turn = 0; turn < turns; ++turn) {
        if (turns > 1) take(turn);          // (else the items are still at hand)
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int at = turn * TURN + b * KV_THREADS;
            if (at + k_first < k_items) {
                signed char* dst = k_codes + (size_t)(unit.slot + key[b].row) * hd + key[b].d;
                int c[V];
#pragma unroll
                for (int j = 0; j < V; ++j) c[j] = code_of(key[b].y1[j], k_inv);
                store_codes<V>(dst, c);
                if (key[b].pair) {
#pragma unroll
                    for (int j = 0; j < V; ++j) c[j] = code_of(key[b].y2[j], k_inv);
                    store_codes<V>(dst + half, c);
                }
            }
            if (at + v_first < v_items) {
                int c[VV];
#pragma unroll
                for (int j = 0; j < VV; ++j) c[j] = code_of(Two{value[b].x[j], 0.f}, v_inv);
                store_codes<VV>(v_codes + (size_t)(unit.slot + value[b].row) * hd + value[b].d, c);
            }
        }
    }
    if (tid == 0) { a.k_scales[block] = k_scale; a.v_scales[block] = v_scale; }
}

// ------------------------------------------------------------------------------------------ reading pages back
template <typename T> __device__ __forceinline__ void store16(T* out, const uint4& codes, float scale);
template <> __device__ __forceinline__ void store16<float>(float* out, const uint4& u, float scale) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 f;
        f.x = (float)(signed char)(w[i]) * scale; f.y = (float)(signed char)(w[i] >> 8) * scale;
        f.z = (float)(signed char)(w[i] >> 16) * scale; f.w = (float)(signed char)(w[i] >> 24) * scale;
        reinterpret_cast<float4*>(out)[i] = f;
    }
}
template <> __device__ __forceinline__ void store16<__nv_bfloat16>(__nv_bfloat16* out, const uint4& u, float scale) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
    unsigned r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 a = __floats2bfloat162_rn((float)(signed char)(w[i]) * scale, (float)(signed char)(w[i] >> 8) * scale);
        __nv_bfloat162 b = __floats2bfloat162_rn((float)(signed char)(w[i] >> 16) * scale, (float)(signed char)(w[i] >> 24) * scale);
        r[2 * i] = *reinterpret_cast<unsigned*>(&a);
        r[2 * i + 1] = *reinterpret_cast<unsigned*>(&b);
    }
    reinterpret_cast<uint4*>(out)[0] = make_uint4(r[0], r[1], r[2], r[3]);
    reinterpret_cast<uint4*>(out)[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// out = codes * scale, block by block. Wide: the block's bytes are a multiple of 16.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256)
unpack_int8_kernel(const signed char* codes, const float* scales, T* __restrict__ out, long long items, int per_block) {      // (pools are kernels' results)
    pdl_launch_dependents();
    pdl_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const float s = __ldcg(scales + i / per_block);
    if (WIDE) {
        store16<T>(out + i * 16, __ldcg(reinterpret_cast<const uint4*>(codes) + i), s);
    } else {
        Elem<T>::store(out + i, (float)codes[i] * s);
    }
}

// A step's requests as pages of GATHER tokens in the order of their positions, those that the requests' tokens read and no others: request r
// has pages first_r .. first_r + n_r - 1 of its positions, which lie one behind the other in the result and behind those of the requests before
// it, and the table says where (-1 where a request reads no such page). A CTA finds its request by the lengths, so that the result is as long
// as the step needs, whatever the table's width. A block with an undefined scale becomes undefined keys and values of zero: a score is left out
// by choosing, not by multiplying with nothing, so that a token that does not see the block is not made undefined by it.
constexpr int GATHER = 64;

__device__ __forceinline__ int gathered_pages(int n, int ctx, int window, int& first) {
    first = 0;
    if (n <= 0 || ctx <= 0) return 0;
    if (window > 0 && ctx - n >= window) first = (ctx - n - window + 1) / GATHER;
    return (ctx - 1) / GATHER - first + 1;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(128)
gather_int8_kernel(const signed char* k_pages, const signed char* v_pages, const float* k_scales, const float* v_scales,
                   T* __restrict__ k_out, T* __restrict__ v_out, int* __restrict__ table_out, const int* __restrict__ q_start, const int* __restrict__ ctx_lens,
                   const int* __restrict__ block_table, int bt_stride, int bt_width, int page_size, int num_pages, int kv_heads, int head_dim,
                   int n_req, int pages, int width, int window) {
    pdl_wait();
    pdl_launch_dependents();
    const int at = blockIdx.x, kvh = blockIdx.y, lane = threadIdx.x & 31;
    const bool row = kvh == 0 && at < n_req;            // the CTA writes row ``at`` of the table, too
    int r = -1, i = 0, ctx = 0, lo = 0;                 // page ``at`` is page i of request r's positions
    for (int r0 = 0, base = 0; r0 < n_req && (r < 0 || (row && r0 <= at)); r0 += 32) {
        int n = 0, c = 0, first = 0;
        if (r0 + lane < n_req) { n = q_start[r0 + lane + 1] - q_start[r0 + lane]; c = ctx_lens[r0 + lane]; }
        const int mine = gathered_pages(n, c, window, first);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (row && at >= r0 && at < r0 + 32) {
            const int begin = base + __shfl_sync(0xffffffffu, sum - mine, at - r0), f = __shfl_sync(0xffffffffu, first, at - r0), count = __shfl_sync(0xffffffffu, mine, at - r0);
            for (int e = threadIdx.x; e < width; e += 128)
                table_out[(size_t)at * width + e] = e >= f && e < f + count && begin + e - f < pages ? begin + e - f : -1;
        }
        const unsigned found = __ballot_sync(0xffffffffu, at < base + sum);
        if (r < 0 && found) {
            const int src = __ffs(found) - 1;
            const int q_len = __shfl_sync(0xffffffffu, n, src);
            r = r0 + src;
            i = at - base - __shfl_sync(0xffffffffu, sum - mine, src) + __shfl_sync(0xffffffffu, first, src);
            ctx = __shfl_sync(0xffffffffu, c, src);
            lo = window > 0 && ctx - q_len >= window ? ctx - q_len - window + 1 : 0;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (r < 0 || at >= pages) return;
    constexpr int E = WIDE ? 16 : 1;
    const int chunks = head_dim / E;
    const size_t to = ((size_t)at * kv_heads + kvh) * GATHER * head_dim;
    for (int j = threadIdx.x; j < GATHER * chunks; j += 128) {
        const int row = j / chunks, d = (j - row * chunks) * E;
        const int pos = i * GATHER + row, lp = pos / page_size;
        int page = -1;
        if (pos < ctx && pos >= lo && lp < bt_width) page = __ldg(block_table + (size_t)r * bt_stride + lp);
        if (page >= num_pages) page = -1;
        const size_t block = (size_t)max(page, 0) * kv_heads + kvh;
        const size_t from = (block * page_size + (pos - lp * page_size)) * head_dim + d, dst = to + (size_t)row * head_dim + d;
        float ks = page >= 0 ? __ldcg(k_scales + block) : 0.f, vs = page >= 0 ? __ldcg(v_scales + block) : 0.f;
        if (ks != ks || vs != vs) { ks = NAN; vs = 0.f; }
        if (WIDE) {
            uint4 k = make_uint4(0, 0, 0, 0), v = k;         // slots that nobody sees are finite
            if (page >= 0) { k = __ldcg(reinterpret_cast<const uint4*>(k_pages + from)); v = __ldcg(reinterpret_cast<const uint4*>(v_pages + from)); }
            store16<T>(k_out + dst, k, ks);
            store16<T>(v_out + dst, v, vs);
        } else {
            Elem<T>::store(k_out + dst, page >= 0 ? (float)k_pages[from] * ks : 0.f);
            Elem<T>::store(v_out + dst, page >= 0 ? (float)v_pages[from] * vs : 0.f);
        }
    }
}

template <typename T, bool WIDE>
int launch_append(const void* qkv, void* q_out, const AppendArgs& a, cudaStream_t stream) {
    NIB_REQUIRE((long long)a.m + a.kv_blocks < (1LL << 31) - 1, "rope_store_int8: too many tokens for one launch");
    if (a.m <= ONE_LAUNCH) {
        NIB_CUDA(launch_pdl(append_int8_kernel<T, WIDE, true>, dim3((unsigned)(a.m + a.kv_blocks)), dim3(KV_THREADS), (size_t)0, stream, (const T*)qkv, (T*)q_out, a));
        return 0;
    }
    const int vq = WIDE ? 8 : 1;
    const long long items = (long long)a.m * a.heads * (((a.rot >> 1) + a.head_dim - a.rot) / vq), grid = (items + ROTATE_THREADS - 1) / ROTATE_THREADS;
    NIB_REQUIRE(grid < (1LL << 31) - 1, "rope_store_int8: too many elements for one launch");
    NIB_CUDA(launch_pdl(rotate_queries_kernel<T, WIDE>, dim3((unsigned)grid), dim3(ROTATE_THREADS), (size_t)0, stream, (const T*)qkv, (T*)q_out, a, items));
    NIB_CUDA(launch_pdl(append_int8_kernel<T, WIDE, false>, dim3((unsigned)a.kv_blocks), dim3(KV_THREADS), (size_t)0, stream, (const T*)qkv, (T*)q_out, a));
    return 0;
}

}  // namespace

// The arguments of a call come as one block of memory (a call of thirty arguments costs the host ten microseconds to marshal).
struct NibAppendInt8 {
    const void* qkv; void* q_out; const int* positions; const int* q_start; const int* ctx_lens; const float* cos_t; const float* sin_t;
    const int* block_table; void* k_pages; void* v_pages; float* k_scales; float* v_scales;
    int q_stride, out_stride, n_req, units, table_rows, rot, bt_stride, bt_width, page_size, num_pages, m, heads, kv_heads, head_dim, dtype, pad;
};

// Rotates the queries of the rows [q heads | k heads | v heads] of ``qkv`` (row stride q_stride elements) into ``q_out`` (row
// stride out_stride; may be qkv itself), and appends the rotated keys and the values to the 8-bit pages. ``units``: the sum over
// the requests of (q_len + page_size - 2) / page_size + 1.
NIB_API int nib_rope_store_int8(const void* args, cudaStream_t stream) {
    NibAppendInt8 c;
    memcpy(&c, args, sizeof c);
    NIB_REQUIRE(c.m >= 0 && c.n_req >= 0 && c.units >= 0 && c.heads > 0 && c.kv_heads > 0 && c.head_dim > 0 && c.page_size > 0 && c.num_pages > 0,
                "rope_store_int8: bad sizes");
    NIB_REQUIRE(c.rot >= 0 && c.rot <= c.head_dim && c.rot % 2 == 0, "rope_store_int8: rotated width %d must be even and <= head_dim %d", c.rot, c.head_dim);
    NIB_REQUIRE(c.rot == 0 || (c.cos_t && c.sin_t && c.table_rows > 0), "rope_store_int8: a rotated width without tables");
    NIB_REQUIRE(c.dtype == NIB_F32 || c.dtype == NIB_BF16, "rope_store_int8: unknown dtype %d", c.dtype);
    if (c.m == 0) return 0;
    AppendArgs a{c.positions, c.q_start, c.ctx_lens, c.cos_t, c.sin_t, c.block_table, (signed char*)c.k_pages, (signed char*)c.v_pages, c.k_scales,
                 c.v_scales, c.table_rows, c.rot, c.bt_stride, c.bt_width, c.page_size, c.num_pages, c.m, c.n_req, c.heads, c.kv_heads, c.head_dim,
                 c.q_stride, c.out_stride, c.units, 0};
    const long long jobs = (long long)c.units * c.kv_heads;
    NIB_REQUIRE(jobs < (1LL << 31) - 1, "rope_store_int8: too many pages for one launch");
    a.kv_blocks = (int)jobs;
    const bool wide = (c.rot / 2) % 8 == 0 && c.head_dim % 8 == 0 && c.q_stride % 8 == 0 && c.out_stride % 8 == 0 &&
                      (((uintptr_t)c.qkv | (uintptr_t)c.q_out | (uintptr_t)c.cos_t | (uintptr_t)c.sin_t) & 15) == 0 &&
                      (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 7) == 0;
    if (c.dtype == NIB_F32) return wide ? launch_append<float, true>(c.qkv, c.q_out, a, stream) : launch_append<float, false>(c.qkv, c.q_out, a, stream);
    return wide ? launch_append<__nv_bfloat16, true>(c.qkv, c.q_out, a, stream) : launch_append<__nv_bfloat16, false>(c.qkv, c.q_out, a, stream);
}

// out = codes * scale for ``blocks`` blocks of ``per_block`` codes each.
NIB_API int nib_unpack_int8(const void* codes, const float* scales, void* out, long long blocks, int per_block, int dtype, cudaStream_t stream) {
    NIB_REQUIRE(blocks >= 0 && per_block > 0, "unpack_int8: bad sizes");
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "unpack_int8: unknown dtype %d", dtype);
    if (blocks == 0) return 0;
    const bool wide = per_block % 16 == 0 && (((uintptr_t)codes | (uintptr_t)out) & 15) == 0;
    const int per = wide ? per_block / 16 : per_block;
    const long long items = blocks * per, grid = (items + 255) / 256;
    NIB_REQUIRE(grid < (1LL << 31) - 1, "unpack_int8: too many elements for one launch");
#define CALL(T, W) NIB_CUDA(launch_pdl(unpack_int8_kernel<T, W>, dim3((unsigned)grid), dim3(256), (size_t)0, stream, (const signed char*)codes, scales, (T*)out, items, per))
    if (dtype == NIB_F32) { if (wide) CALL(float, true); else CALL(float, false); }
    else { if (wide) CALL(__nv_bfloat16, true); else CALL(__nv_bfloat16, false); }
#undef CALL
    return 0;
}

// The positions that the tokens of n_req requests read as pages of 64 tokens [pages, kv_heads, 64, head_dim] in the order of requests and
// positions, with the block table [n_req, width] that addresses them. ``pages``: at least what the requests' lengths come to; what is more is
// left as it is.
NIB_API int nib_gather_int8(const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales, void* k_out, void* v_out,
                            int* table_out, const int* q_start, const int* ctx_lens, int n_req, const int* block_table, int bt_stride,
                            int bt_width, int page_size, int num_pages, int kv_heads, int head_dim, int pages, int width, int window, int dtype,
                            cudaStream_t stream) {
    NIB_REQUIRE(n_req >= 0 && pages > 0 && width > 0 && page_size > 0 && num_pages > 0 && kv_heads > 0 && head_dim > 0 && window >= 0, "gather_int8: bad sizes");
    NIB_REQUIRE(dtype == NIB_F32 || dtype == NIB_BF16, "gather_int8: unknown dtype %d", dtype);
    NIB_REQUIRE(kv_heads <= 65535, "gather_int8: too many heads for one launch");
    if (n_req == 0) return 0;
    const bool wide = head_dim % 16 == 0 && (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
    const unsigned grid = (unsigned)(pages > n_req ? pages : n_req);        // (a request has a row of the table even if it reads no page)
#define CALL(T, W) NIB_CUDA(launch_pdl(gather_int8_kernel<T, W>, dim3(grid, kv_heads), dim3(128), (size_t)0, stream, (const signed char*)k_pages, \
                                       (const signed char*)v_pages, k_scales, v_scales, (T*)k_out, (T*)v_out, table_out, q_start, ctx_lens, block_table, \
                                       bt_stride, bt_width, page_size, num_pages, kv_heads, head_dim, n_req, pages, width, window))
    if (dtype == NIB_F32) { if (wide) CALL(float, true); else CALL(float, false); }
    else { if (wide) CALL(__nv_bfloat16, true); else CALL(__nv_bfloat16, false); }
#undef CALL
    return 0;
}
