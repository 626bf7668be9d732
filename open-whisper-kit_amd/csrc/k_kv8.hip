// Keys and values held in 8 bits (include/owk_kv8.h): filling the cache, attending over it, reading it back.
//
// Blocks of 64 tokens; for a (block, head), keys and values apart: s = max|x| / 127, c = rint(x / s).
// Codes of keys lie token-major [64][D], codes of values dimension-major [D][64]: each is then the
// operand that its matrix product reads along its sum (keys along D, values along the tokens), 16
// contiguous bytes a lane. The incomplete last block (tail) lies in 16 bits in the same two orders.
#include <algorithm>
#include <climits>

#include "kv8.h"

namespace owk {

namespace {

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int BLK = kKv8Block;

__device__ __forceinline__ const char * row_at(const Kv8Call & a, const Kv8Rows & r, const Kv8Entry & e, int b, int64_t i, int head,
                                               int bytes) {
    return r.p + ((a.b.off ? 0 : (int64_t) b * r.entry) + (e.row0 + i) * r.row + (int64_t) head * r.head) * bytes;
}

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float) x; }

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// N elements of a row, as vectors where the tensor allows it
template <typename T, int N> __device__ __forceinline__ void load_row(const T * p, bool vec, T (&x)[N]) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) *(u32x4 *) &x[i * 8] = ((const u32x4 *) p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = p[i];
    }
}
template <typename T, int N> __device__ __forceinline__ void store_row(T * p, bool vec, const T (&x)[N]) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) ((u32x4 *) p)[i] = *(const u32x4 *) &x[i * 8];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = x[i];
    }
}

// ---------------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------------
// One workgroup per (touched block, head, keys or values, entry); four threads hold a token, D / 4
// elements each. A block that the call completes is read whole (its older tokens from the tail), one
// maximum is taken over it, and its codes are written. The rest of the tokens are the new tail. The
// first touched block's workgroup reads the old tail, so that one, after its reads, also writes the
// new tail; only where the call starts on a block border (nothing is read there) does the last one.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8Call a, Kv8Rows kr, Kv8Rows vr) {
    constexpr int Q = D / 4;
    const int b = blockIdx.z, head = blockIdx.y >> 1, j = blockIdx.x;
    const bool is_v = blockIdx.y & 1;
    const Kv8Entry e = kv8_entry(a, b);
    const int end = min(e.start + e.n, a.c.max_blocks * BLK);
    const int first = e.start / BLK, blk = first + j, lo = blk * BLK;
    if (e.seq < 0 || lo >= end || e.n == 0) return;
    const Kv8Rows & r = is_v ? vr : kr;
    T * tail = (T *) (is_v ? a.c.v_tail : a.c.k_tail) + ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
    const int t = threadIdx.x / 4, d0 = (threadIdx.x % 4) * Q;
    __shared__ float amax[4];
    __shared__ __align__(16) int8_t tile[D * 68];  // codes of values on their way to [D][64]; 68: banks

    const bool full = lo + BLK <= end;
    if (full) {
        T x[Q];
        if (lo + t < e.start) {
            if (is_v) {
#pragma unroll
                for (int i = 0; i < Q; ++i) x[i] = tail[(d0 + i) * BLK + t];
            } else {
                load_row<T, Q>(tail + t * D + d0, true, x);
            }
        } else {
            load_row<T, Q>((const T *) row_at(a, r, e, b, lo + t - e.start, head, 2) + d0, r.vec, x);
        }
        float m = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const float y = fabsf(to_f32(x[i]));
            bad |= !(y <= 3.402823466e38f);
            m = fmaxf(m, y);
        }
        m = wave_max(bad ? INFINITY : m);
        if ((threadIdx.x & 63) == 0) amax[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(amax[0], amax[1]), fmaxf(amax[2], amax[3]));
        const bool whole = m <= 3.402823466e38f;
        const float scale = whole ? m / 127.0f : NAN;
        const int64_t page = kv8_page(a.c, e.seq, blk);
        alignas(16) int8_t c[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            // the quotient is rounded once and the code once: a quotient by the reciprocal would move codes at ties
            const float y = whole && scale > 0.0f ? rintf(to_f32(x[i]) / scale) : 0.0f;
            c[i] = (int8_t) fminf(fmaxf(y, -127.0f), 127.0f);
        }
        if (page >= 0) {
            if (threadIdx.x == 0) (is_v ? a.c.v_scale : a.c.k_scale)[page * a.c.n_heads + head] = scale;
            int8_t * codes = (is_v ? a.c.v : a.c.k) + (page * a.c.n_heads + head) * BLK * D;
            if (!is_v) {
#pragma unroll
                for (int i = 0; i < Q / 16; ++i) *(u32x4 *) (codes + t * D + d0 + i * 16) = *(const u32x4 *) &c[i * 16];
            } else {
#pragma unroll
                for (int i = 0; i < Q; ++i) tile[(d0 + i) * 68 + t] = c[i];
                __syncthreads();
                for (int i = threadIdx.x; i < D * 4; i += 256) {
                    const uint32_t * s = (const uint32_t *) (tile + (i / 4) * 68 + (i % 4) * 16);
                    *(u32x4 *) (codes + (i / 4) * BLK + (i % 4) * 16) = u32x4{s[0], s[1], s[2], s[3]};
                }
            }
        }
        __syncthreads();  // the old tail is read
    }
    // the new tail: tokens [max(start, block of end), end)
    const int last = end / BLK;
    if (end % BLK == 0 || (e.start % BLK ? j != 0 : blk != last)) return;
    const int pos = last * BLK + t;
    if (pos < e.start || pos >= end) return;
    T x[Q];
    load_row<T, Q>((const T *) row_at(a, r, e, b, pos - e.start, head, 2) + d0, r.vec, x);
    if (is_v) {
#pragma unroll
        for (int i = 0; i < Q; ++i) tail[(d0 + i) * BLK + t] = x[i];
    } else {
        store_row<T, Q>(tail + t * D + d0, true, x);
    }
}

// ---------------------------------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------------------------------
// One workgroup per (block of the sequence, head, keys or values, entry), four threads a token.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Call a, const int32_t * first_of, Kv8Rows kr, Kv8Rows vr) {
    constexpr int Q = D / 4;
    const int b = blockIdx.z, head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const Kv8Entry e = kv8_entry(a, b);
    const int first = first_of ? max(first_of[b], 0) : 0;
    const int64_t blk = (int64_t) first / BLK + blockIdx.x;
    const int t = threadIdx.x / 4, d0 = (threadIdx.x % 4) * Q;
    const int64_t i = blk * BLK + t - first;  // the token's place in the output
    if (i < 0 || i >= a.b.max_new) return;
    const Kv8Rows & r = is_v ? vr : kr;
    T * out = (T *) (r.p + ((int64_t) b * r.entry + i * r.row + (int64_t) head * r.head) * 2) + d0;
    T x[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) x[k] = (T) 0.0f;
    if (e.seq >= 0 && blk * BLK + t < e.start) {
        if (blk == e.start / BLK) {
            const T * tail = (const T *) (is_v ? a.c.v_tail : a.c.k_tail) + ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
            if (is_v) {
#pragma unroll
                for (int k = 0; k < Q; ++k) x[k] = tail[(d0 + k) * BLK + t];
            } else {
                load_row<T, Q>(tail + t * D + d0, true, x);
            }
        } else {
            const int64_t page = kv8_page(a.c, e.seq, (int) blk);
            if (page >= 0) {
                const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[page * a.c.n_heads + head];
                const int8_t * codes = (is_v ? a.c.v : a.c.k) + (page * a.c.n_heads + head) * BLK * D;
#pragma unroll
                for (int k = 0; k < Q; ++k) x[k] = (T) ((float) codes[is_v ? (d0 + k) * BLK + t : t * D + d0 + k] * scale);
            }
        }
    }
    store_row<T, Q>(out, r.vec, x);
}

// ---------------------------------------------------------------------------------------------------
// attend, few rows
// ---------------------------------------------------------------------------------------------------
// A tile is 16 rows of one entry and key/value head: row r of the entry's n * group is query row r / group,
// query head head * group + r % group. A wave takes every W-th block of 64 keys, straight from memory into
// registers (each byte of the cache is read once a tile, so there is nothing to stage), and keeps a running
// maximum m, sum l and accumulator of its own; the waves are joined in a fixed order at the end.
//
// Both products run on the codes themselves (16x16x64 i8 -> i32, exact): no code is ever converted. What
// meets them is fixed point in two signed digits of 7 bits, value = unit * (128 * hi + lo):
//   queries         unit = max|q| of the row / 16255: off by at most max|q| * 2^-15
//   probabilities   exp2(s - block's maximum) in (0, 1], unit 1 / 16256: off by at most 2^-15 of the block's largest
// The scale of a block multiplies the finished integer sums, in f32.
//
// Lanes: c = lane & 15 is the row (a column of S^T = K Q^T and of O^T = V^T P^T), g = lane >> 4. Key tile t
// feeds key 16 (m >> 2) + 4 t + (m & 3) as row m, so lane (c, g) ends up with the scores of keys 16 g .. 16 g + 15
// in order: exactly the 16 bytes of P^T that the second product wants of it. Nothing crosses lanes but the maximum.
constexpr float QUNIT = 16255.0f, PUNIT = 16256.0f;
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float max_over_g(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ int max_over_g(int x) {
    x = max(x, __shfl_xor(x, 16));
    return max(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_g(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// the two digits of 16 values in [0, 16256], a byte each
__device__ __forceinline__ void digits(const float (&p)[4][4], i32x4 & hi, i32x4 & lo) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (uint32_t) fmaf(p[t][i], PUNIT, 0.5f);
        const uint32_t a = x[0] | x[1] << 16, b = x[2] | x[3] << 16;
        hi[t] = __builtin_amdgcn_perm(b >> 7, a >> 7, 0x06040200);
        lo[t] = __builtin_amdgcn_perm(b, a, 0x06040200) & 0x7f7f7f7f;
    }
}

// a wave's state for its 16 rows
template <int D> struct Acc {
    float m = -INFINITY, l = 0.0f;  // m in units of log2, the same in all four lanes of a row; l a quarter
    float o[D / 16][4];             // dimension 16 dt + 4 g + i
    __device__ Acc() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    }
    // what a block brings has its own maximum mb (-inf: nothing of it is seen): the factor of its sums
    __device__ __forceinline__ float merge(float mb, float & alpha) {
        const float top = fmaxf(m, mb);
        alpha = m == -INFINITY ? 0.0f : exp2f(m - top);
        const float f = mb == -INFINITY ? 0.0f : exp2f(mb - top);
        m = top;
        l *= alpha;
        return f;
    }
};

// the tail of a sequence: the same tile on 16x16x32 products of the tail's own 16-bit type, with f32 sums. Half-precision
// probabilities are held times 2^14 (small ones stay normal), bf16 ones as a sum of two. A token whose values are not all
// finite makes the rows that see it NaN and touches no other.
__device__ __forceinline__ floatx4 mfma16(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <typename T, int D>
__device__ __forceinline__ void attend_tail(const T * kt, const T * vt, const T * qrow, bool qvec, float unit, int have, int see,
                                            Acc<D> & acc) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr bool BF = !std::is_same<T, _Float16>::value;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    float s[4][4];
    {
        vec8 q[D / 32];
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            T x[8] = {};
            if (qrow) load_row<T, 8>(qrow + j * 32 + g * 8, qvec, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[j][i] = x[i];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int key = 16 * (c >> 2) + 4 * t + (c & 3);
            floatx4 x = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                vec8 k = {};
                if (key < have) k = *(const vec8 *) (kt + key * D + j * 32 + g * 8);
                x = mfma16(k, q[j], x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = x[i];
        }
    }
    float mb = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][i] = 16 * g + 4 * t + i < see ? s[t][i] * unit : -INFINITY;
            mb = fmaxf(mb, s[t][i]);
        }
    mb = max_over_g(mb);
    float alpha;
    const float f = acc.merge(mb, alpha);
    const float base = mb == -INFINITY ? 0.0f : mb;  // a NaN score is in no maximum, and makes its probability NaN
    float ls = 0.0f;
    vec8 ph[2], pl[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = exp2f(s[t][i] - base);
            ls += p;
            const int k = t >> 1, e = 4 * (t & 1) + i;
            ph[k][e] = (T) (BF ? p : p * 16384.0f);
            if (BF) pl[k][e] = (T) (p - to_f32(ph[k][e]));
        }
    uint32_t bad = 0;  // of the lane's 16 keys
    const float fo = BF ? f : f * (1.0f / 16384.0f);
    // values, dimension-major: lane (c, g) reads keys 16 g .. 16 g + 15 of dimension 16 dt + c
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        floatx4 x = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            vec8 v = *(const vec8 *) (vt + (dt * 16 + c) * BLK + 16 * g + 8 * k);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool mine = 16 * g + 8 * k + i < have, fine = finite(to_f32(v[i]));
                bad |= mine && !fine ? 1u << (8 * k + i) : 0u;
                v[i] = mine && fine ? v[i] : (T) 0.0f;
            }
            x = mfma16(v, ph[k], x);
            if (BF) x = mfma16(v, pl[k], x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.o[dt][i] = fmaf(x[i], fo, acc.o[dt][i] * alpha);
    }
    if (__any(bad != 0)) {
        for (int o = 8; o; o >>= 1) bad |= __shfl_xor(bad, o);  // over c: the keys of group g
        const int n = min(max(see - 16 * g, 0), 16);
        if (bad & ((1u << n) - 1)) ls = NAN;
    }
    acc.l += f * ls;
}

template <typename T, int D, typename O, int W>
__global__ __launch_bounds__(W * 64) void k_kv8_attend_rows(Kv8Call a, Kv8Attend p) {
    constexpr int DT = D / 16, KC = D / 64;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits, head = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const Kv8Entry e = kv8_entry(a, b);
    const int rows = e.n * p.group - tile * 16;  // of this tile, and of those behind it
    if (rows <= 0) return;
    const int cap = a.c.max_blocks * BLK;
    const int stored = e.seq < 0 ? 0 : p.causal ? min(e.start + e.n, cap) : e.start;
    const int full = stored / BLK;
    // what this lane's row sees, and what the tile sees at most
    const int r = tile * 16 + c, qi = r / p.group;
    const int see = p.causal ? min(stored, e.start + qi + 1) : stored;
    const int last = min(tile * 16 + 15, e.n * p.group - 1) / p.group;
    const int most = p.causal ? min(stored, e.start + last + 1) : stored;
    const int first = p.causal ? min(stored, e.start + tile * 16 / p.group + 1) : stored;  // the least a row of it sees
    const int blocks = (most + BLK - 1) / BLK, per = (blocks + p.splits - 1) / p.splits;
    const int lo = split * per, hi = min(blocks, lo + per);

    const T * qrow = c < rows ? (const T *) row_at(a, p.q, e, b, qi, head * p.group + r % p.group, 2) : nullptr;
    const float sgn = p.scale < 0.0f ? -1.0f : 1.0f;
    i32x4 qh[KC], ql[KC];
    float qunit;
    {
        T x[KC][16];
        float top = 0.0f;
        bool ok = true;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            if (qrow) load_row<T, 16>(qrow + k * 64 + g * 16, p.q.vec, x[k]);
            else
#pragma unroll
                for (int i = 0; i < 16; ++i) x[k][i] = (T) 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = fabsf(to_f32(x[k][i]));
                ok &= finite(y);
                top = fmaxf(top, y);
            }
        }
        top = max_over_g(ok ? top : INFINITY);
        const float inv = finite(top) && top > 0.0f ? QUNIT / top : 0.0f;
        // a row whose largest element is so small that QUNIT / top overflows counts as zeros
        qunit = finite(top) ? (finite(inv) ? top / QUNIT : 0.0f) * fabsf(p.scale) * LOG2E : NAN;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t h = 0, l = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int y = finite(inv) ? (int) rintf(to_f32(x[k][4 * j + i]) * inv * sgn) : 0;
                    const int yh = (y + 64) >> 7;
                    h |= (uint32_t) (yh & 255) << 8 * i;
                    l |= (uint32_t) ((y - 128 * yh) & 255) << 8 * i;
                }
                qh[k][j] = h;
                ql[k][j] = l;
            }
    }

    Acc<D> acc;
    for (int blk = lo + w; blk < hi; blk += W) {
        if (blk == full) {
            const int64_t t = ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
            attend_tail<T, D>((const T *) a.c.k_tail + t, (const T *) a.c.v_tail + t, qrow, p.q.vec, p.scale * LOG2E,
                              stored - full * BLK, see - full * BLK, acc);
            continue;
        }
        const int64_t page = kv8_page(a.c, e.seq, blk);
        if (page < 0) continue;
        const int64_t at = page * a.c.n_heads + head;
        const int8_t * kc = a.c.k + at * BLK * D;
        const int8_t * vc = a.c.v + at * BLK * D;
        i32x4 kx[4][KC], vx[DT];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < KC; ++k) kx[t][k] = *(const i32x4 *) (kc + (16 * (c >> 2) + 4 * t + (c & 3)) * D + k * 64 + g * 16);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vx[dt] = *(const i32x4 *) (vc + (dt * 16 + c) * BLK + g * 16);
        const float f = qunit * a.c.k_scale[at], sv = a.c.v_scale[at];

        int s[4][4], top = INT_MIN;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 xh = {0, 0, 0, 0}, xl = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                xh = __builtin_amdgcn_mfma_i32_16x16x64_i8(kx[t][k], qh[k], xh, 0, 0, 0);
                xl = __builtin_amdgcn_mfma_i32_16x16x64_i8(kx[t][k], ql[k], xl, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = xh[i] * 128 + xl[i];
        }
        const int here = see - blk * BLK;
        if (first < blk * BLK + BLK) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = 16 * g + 4 * t + i < here ? s[t][i] : INT_MIN;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, s[t][i]);
        top = max_over_g(top);
        const bool none = here <= 0;  // this row sees nothing of the block
        const float mb = none ? -INFINITY : (float) top * f;
        float alpha;
        const float fb = acc.merge(mb, alpha);
        float pr[4][4], ls = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // the difference of the integers is exact
                pr[t][i] = s[t][i] == INT_MIN ? 0.0f : __builtin_amdgcn_exp2f((float) (s[t][i] - top) * f);
                ls += pr[t][i];
            }
        acc.l += none ? 0.0f : fb * ls;
        i32x4 ph, pl;
        digits(pr, ph, pl);
        const float fo = none ? 0.0f : fb * sv * (1.0f / PUNIT);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const i32x4 z = {0, 0, 0, 0};
            const i32x4 xh = __builtin_amdgcn_mfma_i32_16x16x64_i8(vx[dt], ph, z, 0, 0, 0);
            const i32x4 xl = __builtin_amdgcn_mfma_i32_16x16x64_i8(vx[dt], pl, z, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc.o[dt][i] = fmaf((float) (xh[i] * 128 + xl[i]), fo, acc.o[dt][i] * alpha);
        }
    }

    // join the waves, in order
    __shared__ float ml[W][16][2];
    __shared__ __align__(16) float o[W][16][D];
    const float l = sum_over_g(acc.l);
    if (c < rows) {
        if (g == 0) {
            ml[w][c][0] = acc.m;
            ml[w][c][1] = l;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *(floatx4 *) &o[w][c][dt * 16 + 4 * g] = floatx4{acc.o[dt][0], acc.o[dt][1], acc.o[dt][2], acc.o[dt][3]};
    }
    __syncthreads();
    const int n = min(rows, 16);
    float * ws = p.ws + ((((int64_t) b * a.c.n_heads + head) * (gridDim.x / p.splits) + tile) * p.splits + split) * 16 * (D + 2);
    for (int i = threadIdx.x; i < n * D; i += W * 64) {
        const int row = i / D, d = i % D;
        float top = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) top = fmaxf(top, ml[k][row][0]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = ml[k][row][0] == -INFINITY ? 0.0f : exp2f(ml[k][row][0] - top);
            // (a NaN maximum is in no fmaxf: its wave's l is NaN and is kept)
            sum += f * ml[k][row][1] + (ml[k][row][1] == ml[k][row][1] ? 0.0f : NAN);
            x += f * o[k][row][d];
        }
        if (p.splits > 1) {
            ws[row * (D + 2) + 2 + d] = x;
            if (d < 2) ws[row * (D + 2) + d] = d ? sum : top;
        } else {
            const int q = tile * 16 + row;
            ((O *) row_at(a, p.out, e, b, q / p.group, head * p.group + q % p.group, sizeof(O)))[d] = (O) (sum == 0.0f ? 0.0f : x / sum);
        }
    }
}

// joins the splits of a tile, in order
template <int D, typename O> __global__ __launch_bounds__(256) void k_kv8_attend_join(Kv8Call a, Kv8Attend p) {
    const int tile = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    const Kv8Entry e = kv8_entry(a, b);
    const int n = min(e.n * p.group - tile * 16, 16);
    const float * ws = p.ws + (((int64_t) b * a.c.n_heads + head) * gridDim.x + tile) * p.splits * 16 * (D + 2);
    for (int i = threadIdx.x; i < n * D; i += 256) {
        const int row = i / D, d = i % D;
        float top = -INFINITY, sum = 0.0f, x = 0.0f;
        for (int k = 0; k < p.splits; ++k) top = fmaxf(top, ws[(k * 16 + row) * (D + 2)]);
        for (int k = 0; k < p.splits; ++k) {
            const float * y = ws + (k * 16 + row) * (D + 2);
            const float f = y[0] == -INFINITY ? 0.0f : exp2f(y[0] - top);
            sum += f * y[1] + (y[1] == y[1] ? 0.0f : NAN);
            x += f * y[2 + d];
        }
        const int q = tile * 16 + row;
        ((O *) row_at(a, p.out, e, b, q / p.group, head * p.group + q % p.group, sizeof(O)))[d] = (O) (sum == 0.0f ? 0.0f : x / sum);
    }
}

// blocks of a sequence that n consecutive tokens can touch
int touched(int n) { return (n + BLK - 2) / BLK + 1; }

template <typename F> void with_type(const owk_kv8_cache & c, F && f) {
    if (c.dtype == OWK_KV8_F16) {
        if (c.head_dim == 64) f((_Float16) 0, std::integral_constant<int, 64>());
        else f((_Float16) 0, std::integral_constant<int, 128>());
    } else {
        if (c.head_dim == 64) f((bf16_t) 0, std::integral_constant<int, 64>());
        else f((bf16_t) 0, std::integral_constant<int, 128>());
    }
}

} // namespace

void kv8_append(hipStream_t s, const Kv8Call & call, const Kv8Rows & k, const Kv8Rows & v) {
    const dim3 grid(touched(call.b.max_new), 2 * call.c.n_heads, call.b.n);
    with_type(call.c, [&](auto t, auto d) {
        OWK_LAUNCH((k_kv8_append<decltype(t), decltype(d)::value>), grid, dim3(256), 0, s, call, k, v);
    });
}

void kv8_read(hipStream_t s, const Kv8Call & call, const int32_t * first, const Kv8Rows & k, const Kv8Rows & v) {
    const dim3 grid(touched(call.b.max_new), 2 * call.c.n_heads, call.b.n);
    with_type(call.c, [&](auto t, auto d) {
        OWK_LAUNCH((k_kv8_read<decltype(t), decltype(d)::value>), grid, dim3(256), 0, s, call, first, k, v);
    });
}

// Splits: enough workgroups to fill the card, but no more than leaves a wave a block of its own
Kv8Plan kv8_plan(const Kv8Call & call, int group, int max_len) {
    const int64_t tiles = ((int64_t) call.b.max_new * group + 15) / 16;
    const int64_t groups = tiles * call.c.n_heads * call.b.n;
    const int64_t blocks = (max_len + BLK - 1) / BLK;
    int64_t splits = 1;
    if (groups < 512) splits = std::min((1024 + groups - 1) / groups, (blocks + 3) / 4);
    if (blocks <= 32) splits = 1;
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, 256));
    Kv8Plan plan;
    plan.splits = (int) splits;
    plan.ws_bytes = splits > 1 ? (size_t) (groups * splits * 16 * (call.c.head_dim + 2)) * 4 : 0;
    return plan;
}

void kv8_attend(hipStream_t s, const Kv8Call & call, const Kv8Attend & a, int out_type) {
    const int tiles = (int) (((int64_t) call.b.max_new * a.group + 15) / 16);
    const dim3 grid(tiles * a.splits, call.c.n_heads, call.b.n), join(tiles, call.c.n_heads, call.b.n);
    with_type(call.c, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        if (out_type == OWK_KV8_F32) {
            OWK_LAUNCH((k_kv8_attend_rows<T, D, float, 4>), grid, dim3(256), 0, s, call, a);
            if (a.splits > 1) OWK_LAUNCH((k_kv8_attend_join<D, float>), join, dim3(256), 0, s, call, a);
        } else {
            OWK_LAUNCH((k_kv8_attend_rows<T, D, T, 4>), grid, dim3(256), 0, s, call, a);
            if (a.splits > 1) OWK_LAUNCH((k_kv8_attend_join<D, T>), join, dim3(256), 0, s, call, a);
        }
    });
}

} // namespace owk
