// Keys and values held in 8 bits (include/owk_kv8.h): filling the cache, attending over it, reading it back.
//
// Blocks of 64 tokens; for a (block, head), keys and values apart: s = max|x| / 127, c = rint(x / s).
// Codes of keys lie token-major [64][D], codes of values dimension-major [D][64]: each is then the
// operand that its matrix product reads along its sum (keys along D, values along the tokens), 16
// contiguous bytes a lane. The incomplete last block (tail) lies in 16 bits in the same two orders.
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv8.h"

namespace owk {

namespace {

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int BLK = kKv8Block;

__device__ __forceinline__ const char * row_at(const Kv8Call & a, const Kv8Rows & r, const Kv8Entry & e, int b, int64_t i, int head,
                                               int bytes) {
    return r.p + ((a.b.off ? 0 : (int64_t) b * r.entry) + (e.row0 + i) * r.row + (int64_t) head * r.head) * bytes;
}

// threadIdx.x & 63, counted anew: not a register that is kept through a loop
__device__ __forceinline__ int lane_again() { return (int) __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)); }

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float) x; }

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The quotient is rounded once and the code once: a quotient by the reciprocal would move codes at ties. A block without a
// finite scale has zeros (and reads as NaN), and one of zeros, too.
__device__ __forceinline__ int8_t code_of(float x, float scale) {
    const float y = scale > 0.0f ? rintf(x / scale) : 0.0f;
    return (int8_t) fminf(fmaxf(y, -127.0f), 127.0f);
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
        const float scale = finite(m) ? m / 127.0f : NAN;
        const int64_t page = kv8_page(a.c, e.seq, blk);
        alignas(16) int8_t c[Q];
        // x * (1 / scale) is within 2^-15.4 of x / scale as rounded (both below 128, three roundings): it rounds to the same code unless it is
        // about that near to a tie; where one of the wave is, all are divided (clips into an empty cache: 100 -> 89 us)
        const float inv = 1.0f / scale;
        float off = scale >= 1.17549435e-38f ? 0.0f : 1.0f;  // (normal scales only: their reciprocals are, too)
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const float y = to_f32(x[i]) * inv, z = rintf(y);
            off = fmaxf(off, fabsf(y - z));
            c[i] = (int8_t) z;
        }
        if (__any(!(off < 0.5f - 0x1p-15f))) {
#pragma unroll
            for (int i = 0; i < Q; ++i) c[i] = code_of(to_f32(x[i]), scale);
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
// One workgroup per (block of the sequence, head, keys or values, entry); a thread has eight dimensions of D / 32 tokens that
// follow each other, so that neighbours write a row as one run (13 sequences, 12 MB of codes: 17.3 -> 9.9 us against a thread
// for a quarter of a row). Values are turned round in shared memory, the codes of a dimension's tokens a word.
template <int D> struct Share {
    static constexpr int N = D / 32;       // tokens
    static constexpr int PITCH = BLK + 4;  // bytes of a dimension's codes in shared memory
    typedef std::conditional_t<N == 4, uint32_t, uint16_t> word;
    int t0 = threadIdx.x / (D / 8) * N, d0 = threadIdx.x % (D / 8) * 8;
};

template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Call a, const int32_t * first_of, Kv8Rows kr, Kv8Rows vr) {
    const Share<D> my;
    constexpr int N = Share<D>::N, PITCH = Share<D>::PITCH;
    const int b = blockIdx.z, head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const Kv8Entry e = kv8_entry(a, b);
    const int first = first_of ? max(first_of[b], 0) : 0;
    const int64_t blk = (int64_t) first / BLK + blockIdx.x;
    __shared__ __align__(16) char store[BLK * (D + 2) * sizeof(T)];
    int8_t * tile = (int8_t *) store;  // [dimension][PITCH] codes
    T * half = (T *) store;            // [token][D + 2] values of the tail
    static_assert(D * PITCH <= sizeof(store), "both forms fit");
    T x[N][8];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[n][i] = (T) 0.0f;
    if (e.seq >= 0 && blk * BLK < e.start) {
        if (blk == e.start / BLK) {
            const T * tail = (const T *) (is_v ? a.c.v_tail : a.c.k_tail) + ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
            if (is_v) {
                for (int i = threadIdx.x; i < D * 8; i += 256) {
                    T z[8];
                    load_row<T, 8>(tail + i * 8, true, z);
#pragma unroll
                    for (int k = 0; k < 8; ++k) half[(i % 8 * 8 + k) * (D + 2) + i / 8] = z[k];
                }
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int t = my.t0 + n;
                if (blk * BLK + t >= e.start) continue;
                if (is_v) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[n][i] = half[t * (D + 2) + my.d0 + i];
                } else {
                    load_row<T, 8>(tail + t * D + my.d0, true, x[n]);
                }
            }
        } else {
            const int64_t page = kv8_page(a.c, e.seq, (int) blk);
            if (page >= 0) {
                const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[page * a.c.n_heads + head];
                const int8_t * codes = (is_v ? a.c.v : a.c.k) + (page * a.c.n_heads + head) * BLK * D;
                if (is_v) {
                    for (int i = threadIdx.x; i < D * 4; i += 256) {
                        const u32x4 z = *(const u32x4 *) (codes + i * 16);
                        uint32_t * s = (uint32_t *) (tile + (i / 4) * PITCH + (i % 4) * 16);
#pragma unroll
                        for (int k = 0; k < 4; ++k) s[k] = z[k];
                    }
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t w = *(const typename Share<D>::word *) (tile + (my.d0 + i) * PITCH + my.t0);
#pragma unroll
                        for (int n = 0; n < N; ++n) x[n][i] = (T) ((float) (int8_t) (w >> 8 * n) * scale);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        alignas(8) int8_t y[8];
                        *(uint64_t *) y = *(const uint64_t *) (codes + (my.t0 + n) * D + my.d0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[n][i] = (T) ((float) y[i] * scale);
                    }
                }
            }
        }
    }
    const Kv8Rows & r = is_v ? vr : kr;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = blk * BLK + my.t0 + n - first;  // the token's place in the output
        if (i < 0 || i >= a.b.max_new) continue;
        store_row<T, 8>((T *) (r.p + ((int64_t) b * r.entry + i * r.row + (int64_t) head * r.head) * 2) + my.d0, r.vec, x[n]);
    }
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
// meets them is fixed point in two signed bytes, value = unit * (256 * hi + lo), hi in +-127, lo in -128 .. 127:
//   queries         unit = max|q| of the row / 32639: off by at most max|q| * 2^-15.99
//   probabilities   exp2(s - block's maximum) in (0, 1], unit 1 / 32639: off by at most 2^-15.99 of the block's largest
// The sums fit 32 bits: 128 * 127 * (256 * 127 + 128) < 2^30, so even the difference of two scores does.
// The scale of a block multiplies the finished integer sums, in f32.
//
// Lanes: c = lane & 15 is the row (a column of S^T = K Q^T and of O^T = V^T P^T), g = lane >> 4. Key tile t
// feeds key 16 (m >> 2) + 4 t + (m & 3) as row m, so lane (c, g) ends up with the scores of keys 16 g .. 16 g + 15
// in order: exactly the 16 bytes of P^T that the second product wants of it. Nothing crosses lanes but the maximum.
constexpr float UNIT = 32639.0f;  // 256 * 127 + 127
constexpr float LOG2E = 1.44269504088896340736f;

// over the four lanes of a row: rows of 16 lanes, then halves of the wave, change places with each other
__device__ __forceinline__ int max_over_g(int x) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((int) a[0], (int) a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((int) b[0], (int) b[1]);
}
__device__ __forceinline__ float max_over_g(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_g(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// The two bytes of four values in [-1, 1]. A float of 1.5 * 2^23 + z has the integer z in its low bits, so one fma rounds
// to the unit; with z = value + 128, byte 1 of z is hi and byte 0 of it is lo + 128.
__device__ __forceinline__ void digits(float x0, float x1, float x2, float x3, float unit, int & hi, int & lo) {
    constexpr float MAGIC = 12582912.0f + 128.0f;
    const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(fmaf(x1, unit, MAGIC)), __float_as_uint(fmaf(x0, unit, MAGIC)), 0x05040100);
    const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(fmaf(x3, unit, MAGIC)), __float_as_uint(fmaf(x2, unit, MAGIC)), 0x05040100);
    hi = __builtin_amdgcn_perm(b, a, 0x07050301);
    lo = __builtin_amdgcn_perm(b, a, 0x06040200) ^ 0x80808080;
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
        alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float f = mb == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mb - top);
        m = top;
        l *= alpha;
        return f;
    }
};

// the tail of a sequence, in both forms of attention: the same tile on 16x16x32 products of the tail's own 16-bit type, with f32
// sums, so that a token's size is nothing to the others. Half-precision probabilities are held times 2^14 (small ones stay
// normal), bf16 ones as a sum of two. A token whose values are not all finite makes the rows that see it NaN and touches no
// other; a key that is not finite does unless its score is -inf, which has no weight.
__device__ __forceinline__ floatx4 mfma16(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <typename T, int D>
__device__ __forceinline__ void attend_tail(const T * kt, const T * vt, const T * qrow, bool qvec, float unit, int have, int see,
                                            Acc<D> & acc) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr bool BF = !std::is_same<T, _Float16>::value;
    const int lane = lane_again(), c = lane & 15, g = lane >> 4;
    // values, dimension-major: lane (c, g) reads keys 16 g .. 16 g + 15 of dimension 16 dt + c
    // (asked for before the scores where the registers allow it)
    auto values = [&](int dt, int k) { return *(const u32x4 *) (vt + (dt * 16 + c) * BLK + 16 * g + 8 * k); };
    u32x4 vx[D == 64 ? 4 : 1][2];
    if (D == 64)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int k = 0; k < 2; ++k) vx[D == 64 ? dt : 0][k] = values(dt, k);
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
                // (behind the last token its own row again: the score is hidden below)
                const vec8 k = *(const vec8 *) (kt + min(key, have - 1) * D + j * 32 + g * 8);
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
            const float p = __builtin_amdgcn_exp2f(s[t][i] - base);
            const int k = t >> 1, e = 4 * (t & 1) + i;
            ph[k][e] = (T) (BF ? p : p * 16384.0f);
            if (BF) pl[k][e] = (T) (p - to_f32(ph[k][e]));
            ls += BF ? to_f32(ph[k][e]) + to_f32(pl[k][e]) : to_f32(ph[k][e]);  // what is summed is what multiplies the values
        }
    if (!BF) ls *= 1.0f / 16384.0f;
    uint32_t bad = 0;  // of the lane's 16 keys
    const float fo = BF ? f : f * (1.0f / 16384.0f);
    u32x4 keep[2];  // pairs of the lane's keys: those that are there
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = 16 * g + 8 * k + 2 * i;
            keep[k][i] = (key < have ? 0xffffu : 0u) | (key + 1 < have ? 0xffff0000u : 0u);
        }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        u32x4 v[2];
        ushort2v big = {0, 0};  // magnitudes as bits: what is not finite is on top
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            v[k] = (D == 64 ? vx[D == 64 ? dt : 0][k] : values(dt, k)) & keep[k];
#pragma unroll
            for (int i = 0; i < 4; ++i) big = __builtin_elementwise_max(big, __builtin_bit_cast(ushort2v, v[k][i] & 0x7fff7fffu));
        }
        constexpr uint32_t INF = BF ? 0x7f80 : 0x7c00;
        if (__any(max(big[0], big[1]) >= INF)) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool lo = (v[k][i] & 0x7fffu) >= INF, hi = (v[k][i] >> 16 & 0x7fffu) >= INF;
                    bad |= (lo ? 1u : 0u) << (8 * k + 2 * i) | (hi ? 2u : 0u) << (8 * k + 2 * i);
                    v[k][i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                }
        }
        floatx4 x = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            x = mfma16(__builtin_bit_cast(vec8, v[k]), ph[k], x);
            if (BF) x = mfma16(__builtin_bit_cast(vec8, v[k]), pl[k], x);
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

// Which entry and head (group) a workgroup of a one-dimensional grid works on, and which of its `parts` parts. Workgroups go
// round the eight dies: all parts of a group run on one die, and the keys they share stay in its cache (32 groups of 128-row
// tiles: 345 us, 405 without), unless that would leave the dies unevenly loaded (4 groups of 62 parts: 35 us, 22 without).
__host__ __device__ inline bool by_die(int groups) { return (groups + 7) / 8 * 56 <= groups * 8; }
struct Place {
    int group, part;  // group -1: nothing to do
};
__device__ __forceinline__ Place place_of(const Kv8Call & a, int parts) {
    const int id = blockIdx.x, groups = a.c.n_heads * a.b.n;
    if (!by_die(groups)) return Place{id / parts, id % parts};
    const int group = (id & 7) + 8 * (id / (8 * parts));
    return Place{group < groups ? group : -1, id / 8 % parts};
}
unsigned workgroups(const Kv8Call & call, int parts) {
    const unsigned groups = (unsigned) call.c.n_heads * call.b.n;
    return (by_die(groups) ? (groups + 7) / 8 * 8 : groups) * parts;
}

// ONCE: no other tile reads these codes, they need not stay in the caches (cross attention of 32 clips 29.3 -> 26.7 us;
// with more tiles of the same keys 141 -> 171 us, so then it is off)
template <bool ONCE> __device__ __forceinline__ i32x4 load_codes(const int8_t * p) {
    return ONCE ? __builtin_nontemporal_load((const i32x4 *) p) : *(const i32x4 *) p;
}

template <typename T, int D, typename O, int W, bool ONCE>
__global__ __launch_bounds__(W * 64, D == 64 ? 4 : 2) void k_kv8_attend_rows(Kv8Call a, Kv8Attend p) {
    constexpr int DT = D / 16, KC = D / 64;
    constexpr bool BF = !std::is_same<T, _Float16>::value;
    int head = blockIdx.y, b = blockIdx.z, split = 0, tile = 0;
    if (gridDim.x > 1) {
        const Place place = place_of(a, p.tiles * p.splits);
        if (place.group < 0) return;
        head = place.group % a.c.n_heads;
        b = place.group / a.c.n_heads;
        split = place.part % p.splits;
        tile = place.part / p.splits;
    }
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const Kv8Entry e = kv8_entry(a, b);
    const int64_t page0 = kv8_page(a.c, e.seq, split * p.per + w);  // asked for together with the lengths
    const int rows = e.n * p.group - tile * 16;  // of this tile, and of those behind it
    if (rows <= 0) return;
    const int cap = a.c.max_blocks * BLK;
    const int stored = e.seq < 0 ? 0 : p.causal ? min(e.start + e.n, cap) : e.start;
    const int full = stored / BLK;
    // what this lane's row sees, and what the tile sees at least and at most
    const int r = tile * 16 + c, qi = r / p.group;
    const int see = p.causal ? min(stored, e.start + qi + 1) : stored;
    const int last = min(tile * 16 + 15, e.n * p.group - 1) / p.group;
    const int most = p.causal ? min(stored, e.start + last + 1) : stored;
    const int least = p.causal ? min(stored, e.start + tile * 16 / p.group + 1) : stored;
    const int blocks = (most + BLK - 1) / BLK, lo = split * p.per;
    const int hi = split == p.splits - 1 ? blocks : min(blocks, lo + p.per);
    if (split > 0 && lo >= hi) return;  // (the join looks at as many splits as the tile has)

    const T * qrow = c < rows ? (const T *) row_at(a, p.q, e, b, qi, head * p.group + r % p.group, 2) : nullptr;
    T qx[KC][16];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
        if (qrow) load_row<T, 16>(qrow + k * 64 + g * 16, p.q.vec, qx[k]);
        else
#pragma unroll
            for (int i = 0; i < 16; ++i) qx[k][i] = (T) 0.0f;
    }

    // A block's keys are asked for as soon as the scores of the one before are made, its values when that one's are
    // added: a wave always has loads in flight, and the first block's cover the queries' conversion.
    const int koff = (16 * (c >> 2) + (c & 3)) * D + g * 16, voff = c * BLK + g * 16;
    i32x4 kx[4][KC], vx[DT];
    int64_t at = 0;
    bool held;  // false: the block's table entry leads nowhere. Block 0 of the pool is read for it, and nothing is seen of it
    float ks = 0.0f, sv = 0.0f;
    auto ask_keys = [&](int64_t page) {
        held = page >= 0;
        at = (held ? page : 0) * a.c.n_heads + head;
        const int8_t * kc = a.c.k + at * BLK * D + koff;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < KC; ++k) kx[t][k] = load_codes<ONCE>(kc + 4 * t * D + k * 64);
    };
    auto ask_values = [&]() {
        const int8_t * vc = a.c.v + at * BLK * D + voff;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vx[dt] = load_codes<ONCE>(vc + dt * 16 * BLK);
        ks = a.c.k_scale[at];
        sv = a.c.v_scale[at];
    };
    const int codes = min(hi, full);  // blocks held in codes
    int blk = lo + w;
    ask_keys(blk < codes ? page0 : -1);
    ask_values();

    i32x4 qh[KC], ql[KC];
    float qunit;
    int qex = 0;
    {
        float top = 0.0f;
        bool ok = true;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = fabsf(to_f32(qx[k][i]));
                ok &= finite(y);
                top = fmaxf(top, y);
            }
        top = max_over_g(ok ? top : INFINITY);
        const bool any = finite(top) && top > 0.0f;
        // a bf16 row is brought to [1, 2) by a power of two that goes to the blocks' scales: neither UNIT / top nor the unit
        // leaves the range of f32 then, however small or large the queries are
        if (BF && any) qex = ilogbf(top);
        const float most = BF ? ldexpf(top, -qex) : top, inv = any ? p.scale < 0.0f ? -UNIT / most : UNIT / most : 0.0f;
        qunit = finite(top) ? most / UNIT * fabsf(p.scale) * LOG2E : NAN;
        // what is not finite goes in as zero: the row's unit is NaN then
        auto q = [&](int k, int i) { return !ok ? 0.0f : BF ? ldexpf(to_f32(qx[k][i]), -qex) : to_f32(qx[k][i]); };
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int h, l;
                digits(q(k, 4 * j), q(k, 4 * j + 1), q(k, 4 * j + 2), q(k, 4 * j + 3), inv, h, l);
                qh[k][j] = h;
                ql[k][j] = l;
            }
    }

    Acc<D> acc;
    for (; blk < codes; blk += W) {
        const float f = qunit * (BF ? ldexpf(ks, qex) : ks), svl = sv;
        const int here = held ? see - blk * BLK : 0;
        const bool all = held && least >= blk * BLK + BLK;  // every row of the tile sees the whole block
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
            for (int i = 0; i < 4; ++i) s[t][i] = xh[i] * 256 + xl[i];
        }
        ask_keys(blk + W < codes ? kv8_page(a.c, e.seq, blk + W) : -1);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, all || 16 * g + 4 * t + i < here ? s[t][i] : INT_MIN);
        top = max_over_g(top);
        const bool none = here <= 0;  // this row sees nothing of the block
        const float mb = none ? -INFINITY : (float) top * f;
        float alpha;
        const float fb = acc.merge(mb, alpha);
        float pr[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[t][i] = __builtin_amdgcn_exp2f((float) (s[t][i] - top) * f);  // the difference is exact
        if (!all) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) pr[t][i] = 16 * g + 4 * t + i < here ? pr[t][i] : 0.0f;
        }
        i32x4 ph, pl;
        int lh = 0, ll = 0;  // what is summed is what multiplies the values: the digits, exactly
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            int h, l;
            digits(pr[t][0], pr[t][1], pr[t][2], pr[t][3], UNIT, h, l);
            ph[t] = h;
            pl[t] = l;
            lh = __builtin_amdgcn_sdot4(h, 0x01010101, lh, false);
            ll = __builtin_amdgcn_sdot4(l, 0x01010101, ll, false);
        }
        acc.l += none ? 0.0f : fb * (1.0f / UNIT) * (float) (lh * 256 + ll);
        const float fo = none ? 0.0f : fb * svl * (1.0f / UNIT);
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc.o[dt][i] *= alpha;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const i32x4 z = {0, 0, 0, 0};
            const i32x4 xh = __builtin_amdgcn_mfma_i32_16x16x64_i8(vx[dt], ph, z, 0, 0, 0);
            const i32x4 xl = __builtin_amdgcn_mfma_i32_16x16x64_i8(vx[dt], pl, z, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc.o[dt][i] = fmaf((float) (xh[i] * 256 + xl[i]), fo, acc.o[dt][i]);
        }
        ask_values();
    }

    if (blk == full && blk < hi) {
        const int64_t t = ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
        attend_tail<T, D>((const T *) a.c.k_tail + t, (const T *) a.c.v_tail + t, qrow, p.q.vec, qunit == qunit ? p.scale * LOG2E : NAN,
                          stored - full * BLK, see - full * BLK, acc);
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
    float * ws = p.ws + ((((int64_t) b * a.c.n_heads + head) * p.tiles + tile) * p.splits + split) * 16 * (D + 2);
    for (int i = threadIdx.x; i < n * D; i += W * 64) {
        const int row = i / D, d = i % D;
        float top = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) top = fmaxf(top, ml[k][row][0]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = ml[k][row][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k][row][0] - top);
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

// ---------------------------------------------------------------------------------------------------
// attend, many rows
// ---------------------------------------------------------------------------------------------------
// Four waves of 32 rows each go through the blocks of their entry and head together. With that many rows what counts
// is the work a score costs, so here a block's codes become half-precision floats once (exactly: they are integers up
// to 127) on their way to shared memory, and both products are 16x16x32 f16 with f32 sums: a score then costs a fused
// multiply-add, an exponential, a sum and half a conversion.
//
// The lanes hold what they hold above: S^T = K Q^T with the keys of a tile permuted so that lane (c, g) gets the scores of
// keys 16 g .. 16 g + 15, and chunk k of eight of them is what O^T = V^T P^T wants as its k-th operand.
// Probabilities are p = exp2(s - m) times 2^6 sv / 2^sig, sv the block's scale of values: the accumulator is in units of 2^(sig - 6)
// and the block's scale costs nothing. m and sig are a row's own, and stay what they are as long as the block's sum of these
// products lies in a window of half precision: at most 2^14, and at least what one product of 2^-10 makes, so that what is rounded
// below the normal range is 2^-15 of the largest. A row that leaves the window makes its products again, with m brought up to the
// running maximum and sig to what the block adds, p sv: values of any size under weights of any size keep their bits. sig
// falls to 2^-64 of the largest it was at the most, so that the accumulator cannot overflow; what a block adds below that is
// added by f32 multiply-adds. Rows are independent of each other: none sees another's m or sig.
constexpr int MR = 2;          // row tiles of a wave
constexpr int MANY_WAVES = 4;  // of a workgroup

// sixteen codes as half-precision floats: 0x6400 | x is 1024 + x
__device__ __forceinline__ void to_half(const i32x4 & c, half8 (&h)[2]) {
    const half2v off = {(_Float16) 1152.0f, (_Float16) 1152.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = (uint32_t) c[i] ^ 0x80808080;
        const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464, x, 0x04010400)) - off;
        const half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464, x, 0x04030402)) - off;
        h[i / 2][4 * (i % 2)] = a[0];
        h[i / 2][4 * (i % 2) + 1] = a[1];
        h[i / 2][4 * (i % 2) + 2] = b[0];
        h[i / 2][4 * (i % 2) + 3] = b[1];
    }
}

// a staged block: rows of keys and of value dimensions, their 16-byte chunks xor-ed with bits of the row, so that lanes that
// read the same chunk of neighbouring rows meet different banks (four bits for keys of 128 elements, whose rows all begin on
// the same bank: two fifths fewer conflicts than with three, the quickest of 100 calls of chunks 310 -> 307 us)
template <int D> struct Stage {
    half8 k[BLK * D / 8], v[D * BLK / 8];
    static constexpr int xor_k(int key) { return (key & 3) | (key >> 2 & (D == 64 ? 4 : 12)); }
    static __device__ __forceinline__ int at_k(int key, int chunk) { return key * (D / 8) + (chunk ^ xor_k(key)); }
    static __device__ __forceinline__ int at_v(int d, int chunk) { return d * (BLK / 8) + (chunk ^ (d & 7)); }
};

// the entry with the n-th most tokens (of up to 64; more are taken as they come): long ones start first, short ones fill the gaps
__device__ __forceinline__ int nth_longest(const Kv8Call & a, int n, int lane) {
    if (a.b.n > 64) return n;
    int len = -1;
    if (lane < a.b.n) {
        const Kv8Entry e = kv8_entry(a, lane);
        len = e.start + e.n;
    }
    int rank = 0;
    for (int i = 0; i < a.b.n; ++i) {
        const int other = __builtin_amdgcn_readlane(len, i);
        rank += other > len || (other == len && i < lane);
    }
    return __builtin_ctzll(__ballot(lane < a.b.n && rank == n));
}

template <typename T, int D, typename O, int MW>
__global__ __launch_bounds__(MW * 64, D == 64 ? 3 : 2) void k_kv8_attend_tiles(Kv8Call a, Kv8Attend p, int tiles) {
    constexpr int MROWS = MW * MR * 16, NT = MW * 64;
    constexpr int DT = D / 16, KC = D / 32, NC = BLK * D / 16 / NT;  // NC: 16-byte pieces of codes of a thread
    constexpr bool BF = !std::is_same<T, _Float16>::value;
    __shared__ __align__(16) Stage<D> st[2];
    const Place place = place_of(a, tiles * p.splits);
    if (place.group < 0) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int head = place.group % a.c.n_heads, b = nth_longest(a, place.group / a.c.n_heads, lane);
    const int split = place.part % p.splits, tile = tiles - 1 - place.part / p.splits;  // tiles that see the most keys first
    const Kv8Entry e = kv8_entry(a, b);
    const int nrows = e.n * p.group;
    if (tile * MROWS >= nrows) return;
    const int cap = a.c.max_blocks * BLK;
    const int stored = e.seq < 0 ? 0 : p.causal ? min(e.start + e.n, cap) : e.start;
    const int full = stored / BLK;
    auto sees = [&](int row) { return p.causal ? min(stored, e.start + min(row, nrows - 1) / p.group + 1) : stored; };
    const int row0 = tile * MROWS + w * MR * 16;
    const int most = sees(tile * MROWS + MROWS - 1);          // of the workgroup
    const int mine = row0 < nrows ? sees(row0 + MR * 16 - 1) : 0, least = sees(row0);  // of the wave
    const int blocks = (most + BLK - 1) / BLK, lo = split * p.per;
    const int hi = split == p.splits - 1 ? blocks : min(blocks, lo + p.per);
    if (split > 0 && lo >= hi) return;

    // queries
    half8 q[MR][KC];
    float unit[MR];
    int see[MR], qex[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        const int row = row0 + r * 16 + c;
        see[r] = row < nrows ? sees(row) : 0;
        const T * qr = row < nrows ? (const T *) row_at(a, p.q, e, b, row / p.group, head * p.group + row % p.group, 2) : nullptr;
        T x[KC][8];
        float top = 0.0f;
        bool ok = true;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            if (qr) load_row<T, 8>(qr + k * 32 + g * 8, p.q.vec, x[k]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) x[k][i] = (T) 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ok &= finite(to_f32(x[k][i]));
                top = fmaxf(top, fabsf(to_f32(x[k][i])));
            }
        }
        // a row that is not finite has a unit that is NaN, and zeros for queries
        top = max_over_g(ok ? top : INFINITY);
        ok = finite(top);
        // bf16 rows are brought to [1, 2) by a power of two, exact but for what is 2^-14 of the largest or less
        qex[r] = BF && ok && top > 0.0f ? ilogbf(top) : 0;
        unit[r] = ok ? fabsf(p.scale) * LOG2E : NAN;
        const float sgn = p.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) q[r][k][i] = (_Float16) (!ok ? 0.0f : BF ? ldexpf(to_f32(x[k][i]), -qex[r]) * sgn : to_f32(x[k][i]) * sgn);
    }

    // staging of block blk into s: its codes are asked for a block ahead, 16 of keys and of values a thread and piece
    const int codes = min(hi, full);  // blocks held in codes
    i32x4 nk[NC], nv[NC];
    bool held = false, nheld;  // false: block 0 of the pool is read for a block that is not there, and nothing is seen of it
    float ks = 0.0f, sv = 0.0f, nks, nsv;
    // A block's table entry is read a block ahead of its codes, and its scales with them, by vector loads: scalar loads are
    // counted with shared memory, and every wait for keys or values in there would wait for them, too.
    int zero = 0;
    asm volatile("" : "+v"(zero));
    int entry_n = -1;
    auto ask_entry = [&](int blk) {
        entry_n = blk < codes ? a.c.table ? a.c.table[(int64_t) e.seq * a.c.max_blocks + blk + zero] : e.seq * a.c.max_blocks + blk : -1;
    };
    ask_entry(lo);
    auto ask = [&](int blk) {
        const int page = __builtin_amdgcn_readfirstlane(entry_n);
        nheld = page >= 0 && page < a.c.n_blocks;
        const int64_t at = (nheld ? (int64_t) page : 0) * a.c.n_heads + head;
        ask_entry(blk + 1);
        nks = a.c.k_scale[at + zero];
        nsv = a.c.v_scale[at + zero];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            nk[i] = ((const i32x4 *) (a.c.k + at * BLK * D))[threadIdx.x + i * NT];
            nv[i] = ((const i32x4 *) (a.c.v + at * BLK * D))[threadIdx.x + i * NT];
        }
    };
    // places in a stage: of what this thread stages (piece i is NT / (D / 16) keys, NT / 4 dimensions on), and of the keys and
    // values that its lane multiplies (tile t is 4 keys on, tile d 16 dimensions: bits that no xor looks at)
    const int pk = Stage<D>::at_k(threadIdx.x / (D / 16), threadIdx.x % (D / 16) * 2), pv = Stage<D>::at_v(threadIdx.x / 4, threadIdx.x % 4 * 2);
    const int mk = 16 * (c >> 2) + (c & 3), mv[2] = {Stage<D>::at_v(c, 2 * g), Stage<D>::at_v(c, 2 * g + 1)};
    int mkk[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) mkk[k] = Stage<D>::at_k(mk, k * 4 + g);
    static_assert(NT / (D / 16) % 32 == 0 && NT / 4 % 8 == 0, "a piece changes bits of its own alone");
    auto put = [&](Stage<D> & s) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            half8 h[2];
            to_half(nk[i], h);
            const int at = (pk ^ Stage<D>::xor_k(i * NT / (D / 16))) + i * NT / (D / 16) * (D / 8);
            s.k[at] = h[0];
            s.k[at ^ 1] = h[1];
            to_half(nv[i], h);
            s.v[pv + i * NT / 4 * (BLK / 8)] = h[0];
            s.v[(pv ^ 1) + i * NT / 4 * (BLK / 8)] = h[1];
        }
        held = nheld;
        ks = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(nks)));
        sv = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(nsv)));
    };
    // the scores of a staged block, in units of the block's and the rows' scales
    auto scores = [&](const Stage<D> & s, floatx4 (&x)[MR][4]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int r = 0; r < MR; ++r) x[r][t] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                const half8 kk = s.k[mkk[k] + 4 * t * (D / 8)];
#pragma unroll
                for (int r = 0; r < MR; ++r) x[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[r][k], x[r][t], 0, 0, 0);
            }
        }
    };
    const half8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    float m[MR], l[MR];  // the same in all four lanes of a row
    floatx4 o[MR][DT];
    constexpr float NONE = -0x1p20f;
    float sig[MR], peak[MR];  // whole numbers; peak: the largest sig was, with what m moved up since taken off
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
        sig[r] = peak[r] = NONE;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] = floatx4{0, 0, 0, 0};
    }
    const bool whole = row0 + MR * 16 <= nrows;  // all rows of the wave are there

    ask(lo);
    if (lo < codes) put(st[0]);
    __syncthreads();
    for (int blk = lo; blk < codes; ++blk) {
        const Stage<D> & s = st[(blk - lo) & 1];
        const int base = blk * BLK;
        const bool there = held;
        const float cks = there ? ks : 0.0f, csv = there ? sv : 0.0f;  // (a block that is not there: its scales are block 0's)
        ask(blk + 1);
        if (mine > base) {
            const bool part = !(there && whole && least >= base + BLK);  // some row does not see all of it
            // the block's scale of values is svm 2^e2 (1 for a block of zeros, which adds to the sums alone)
            const bool zero = csv == 0.0f;
            const int e2 = __builtin_amdgcn_frexp_expf(csv);
            const float svm = zero ? 1.0f : __builtin_amdgcn_frexp_mantf(csv);
            const float inv = __builtin_amdgcn_rcpf(svm), lsv = __builtin_amdgcn_logf(svm);
            const float low = zero ? 0.0f : 0x1p-10f;
            uint32_t ph[MR][8];  // pairs of probabilities: of keys 16 g + 2 j, + 1
            int here[MR], lag[MR];  // lag: the block's products are 2^lag above the accumulator's unit
            float f[MR], by[MR], least_sum[MR];  // by: what the accumulator is multiplied by
            float mm[MR], power[MR];  // p svm 2^power = exp2(s - mm)
#pragma unroll
            for (int r = 0; r < MR; ++r) {
                here[r] = part ? there ? see[r] - base : 0 : BLK;
                f[r] = unit[r] * (BF ? ldexpf(cks, qex[r]) : cks);
                by[r] = 1.0f;
                lag[r] = 0;
                power[r] = zero ? 6.0f : (float) (e2 + 6) - sig[r];
                mm[r] = m[r] - (power[r] + lsv);
                // (no sum is large enough where p would be far above 1, or there is no sig yet)
                least_sum[r] = ((power[r] >= -24.0f) & (power[r] < 4096.0f)) ? low * (float) (part ? min(here[r], BLK) : BLK) : INFINITY;
                if (part) least_sum[r] = here[r] > 0 ? least_sum[r] : -INFINITY;
            }
            // the products by the m and sig there are, and their sum by a product with ones (what is summed is what multiplies
            // the values); rows that leave the window are made again
            floatx4 sum[MR];
#pragma clang loop unroll(disable)
            for (int again = 0;; ++again) {
                bool out[MR];
                floatx4 x[MR][4];
                // (products before other waves' softmax: chunks 348 -> 333 us, prompts the same)
                __builtin_amdgcn_s_setprio(1);
                scores(s, x);
                __builtin_amdgcn_s_setprio(0);
#pragma unroll
                for (int r = 0; r < MR; ++r) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2v y = {__builtin_amdgcn_exp2f(fmaf(x[r][j / 2][2 * j % 4], f[r], -mm[r])),
                                           __builtin_amdgcn_exp2f(fmaf(x[r][j / 2][2 * j % 4 + 1], f[r], -mm[r]))};
                        ph[r][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, half2v));
                    }
                }
                if (part) {
#pragma unroll
                    for (int r = 0; r < MR; ++r) {
                        int till = here[r] - 16 * g;
                        asm volatile("" : "+v"(till));  // (keeps the masks in here, out of every block's registers)
#pragma unroll
                        for (int j = 0; j < 8; ++j) ph[r][j] &= (2 * j < till ? 0xffffu : 0u) | (2 * j + 1 < till ? 0xffff0000u : 0u);
                    }
                }
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    sum[r] = floatx4{0, 0, 0, 0};
                    sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, *(const half8 *) &ph[r][0], sum[r], 0, 0, 0);
                    sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, *(const half8 *) &ph[r][4], sum[r], 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < MR; ++r)
                    out[r] = !((sum[r][0] <= 16384.0f) & (sum[r][0] >= least_sum[r]));
                if (again || !__any(out[0] | out[MR - 1])) break;
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    float top = -INFINITY;
                    int till = here[r] - 16 * g;
                    asm volatile("" : "+v"(till) : : "memory");  // (the scores are made again rather than kept: registers)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        floatx4 y = {0, 0, 0, 0};
#pragma unroll
                        for (int k = 0; k < KC; ++k)
                            y = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.k[mkk[k] + 4 * t * (D / 8)], q[r][k], y, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, 4 * t + i < till ? y[i] : -INFINITY);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    top = max_over_g(top);
                    if (out[r]) {
                        const float mb = top == -INFINITY ? -INFINITY : top * f[r], next = fmaxf(m[r], mb);
                        // m moves up by `steps` whole powers of two and a factor: the same in both products
                        const float up = m[r] == -INFINITY ? 0.0f : next - m[r], steps = fminf(floorf(up), 1e5f);
                        const float frac = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(steps - up);
                        m[r] = next;
                        l[r] *= ldexpf(frac, -(int) steps);
                        float shift = -steps;
                        if (sig[r] != NONE) peak[r] = fmaxf(peak[r] - steps, -1e5f);
                        if (!zero && mb > -INFINITY) {
                            const float own = (float) e2 + floorf(fmaxf(mb - next, -1e3f));  // of what the block adds
                            peak[r] = fmaxf(peak[r], own);
                            const float to = fmaxf(own, peak[r] - 64.0f);
                            if (sig[r] != NONE) shift += sig[r] - to;
                            sig[r] = to;
                            lag[r] = (int) (to - own);
                            power[r] = (float) (e2 + 6) - own;
                        }
                        by[r] = ldexpf(frac, (int) shift);
                        mm[r] = (m[r] == -INFINITY ? 0.0f : m[r]) - (power[r] + lsv);
                    }
                }
            }
            if (__any(by[0] != 1.0f || by[MR - 1] != 1.0f)) {
#pragma unroll
                for (int r = 0; r < MR; ++r)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[r][d][i] *= by[r];
            }
#pragma unroll
            for (int r = 0; r < MR; ++r)
                if (here[r] > 0) l[r] = fmaf(sum[r][0], ldexpf(inv, -(int) power[r]), l[r]);
            if (__any(lag[0] != 0 || lag[MR - 1] != 0)) {
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    const float fo = ldexpf(1.0f, -lag[r]);
                    uint32_t pf[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        pf[j] = lag[r] ? ph[r][j] : 0;
                        ph[r][j] = lag[r] ? 0 : ph[r][j];
                    }
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        floatx4 x = {0, 0, 0, 0};
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.v[mv[0] + d * 16 * (BLK / 8)], *(const half8 *) &pf[0], x, 0, 0, 0);
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.v[mv[1] + d * 16 * (BLK / 8)], *(const half8 *) &pf[4], x, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[r][d][i] = fmaf(x[i], fo, o[r][d][i]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const half8 v0 = s.v[mv[0] + d * 16 * (BLK / 8)], v1 = s.v[mv[1] + d * 16 * (BLK / 8)];
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, *(const half8 *) &ph[r][0], o[r][d], 0, 0, 0);
                    o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, *(const half8 *) &ph[r][4], o[r][d], 0, 0, 0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
        if (blk + 1 < codes) put(st[(blk + 1 - lo) & 1]);
        __syncthreads();
    }

    // lane (c, g) holds dimensions 16 d + 4 g .. + 3 of its rows
    // l is brought to [1/2, 1) by a power of two, so that sums of values near the end of f32 stay in it
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        const int up = __builtin_amdgcn_frexp_expf(l[r]), fin = (int) sig[r] - 6 - up;
        m[r] += (float) up;
        l[r] = __builtin_amdgcn_frexp_mantf(l[r]);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][d][i] = ldexpf(o[r][d][i], fin);
    }
    const bool tail = hi > full && mine > full * BLK;
    const int64_t t = ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        const int lane = lane_again(), row = row0 + r * 16 + (lane & 15), dim = 4 * (lane >> 4);
        Acc<D> acc;
        acc.m = m[r];
        acc.l = 0.25f * l[r];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc.o[d][i] = o[r][d][i];
        if (tail && row0 + r * 16 < nrows) {
            const T * qr = row < nrows ? (const T *) row_at(a, p.q, e, b, row / p.group, head * p.group + row % p.group, 2) : nullptr;
            attend_tail<T, D>((const T *) a.c.k_tail + t, (const T *) a.c.v_tail + t, qr, p.q.vec, unit[r] == unit[r] ? p.scale * LOG2E : NAN,
                              stored - full * BLK, see[r] - full * BLK, acc);
        }
        const float sum = sum_over_g(acc.l);
        if (row >= nrows) continue;
        if (p.splits > 1) {
            const int64_t t16 = (int64_t) tiles * (MROWS / 16);
            float * ws = p.ws + (((((int64_t) b * a.c.n_heads + head) * t16 + row / 16) * p.splits + split) * 16 + row % 16) * (D + 2);
            if (dim == 0) {
                ws[0] = acc.m;
                ws[1] = sum;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) ws[2 + d * 16 + dim + i] = acc.o[d][i];
        } else {
            O * out = (O *) row_at(a, p.out, e, b, row / p.group, head * p.group + row % p.group, sizeof(O));
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                typedef O vec4 __attribute__((ext_vector_type(4)));
                vec4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (O) (sum == 0.0f ? 0.0f : acc.o[d][i] * f);
                if (p.out.vec) {
                    *(vec4 *) (out + d * 16 + dim) = y;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[d * 16 + dim + i] = y[i];
                }
            }
        }
    }
}

// splits that a tile of 16 rows has: those of the workgroup that made it
__device__ __forceinline__ int splits_of(const Kv8Call & a, const Kv8Attend & p, const Kv8Entry & e, int tile) {
    const int stored = e.seq < 0 ? 0 : p.causal ? min(e.start + e.n, a.c.max_blocks * BLK) : e.start;
    const int last = min((tile / p.join + 1) * p.join * 16 - 1, e.n * p.group - 1) / p.group;
    const int most = p.causal ? min(stored, e.start + last + 1) : stored;
    return min(p.splits, max(1, ((most + BLK - 1) / BLK + p.per - 1) / p.per));
}

// joins the splits of a row, in order: a workgroup a row, its waves take every fourth split and are joined at the end
template <int D, typename O> __global__ __launch_bounds__(256) void k_kv8_attend_join(Kv8Call a, Kv8Attend p) {
    constexpr int DL = D / 64;
    const int r = blockIdx.x, tile = r / 16, row = r % 16, head = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const Kv8Entry e = kv8_entry(a, b);
    if (r >= e.n * p.group) return;
    const int n = splits_of(a, p, e, tile);
    const float * ws = p.ws + ((((int64_t) b * a.c.n_heads + head) * p.tiles + tile) * p.splits * 16 + row) * (D + 2);
    float m = -INFINITY, l = 0.0f, x[DL] = {};
#pragma unroll 4
    for (int k = w; k < n; k += 4) {
        const float * y = ws + (int64_t) k * 16 * (D + 2);
        const float mk = y[0], lk = y[1], top = fmaxf(m, mk);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top), f = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - top);
        m = top;
        l = l * alpha + (lk == lk ? f * lk : NAN);  // a split whose maximum is NaN has that l too
#pragma unroll
        for (int i = 0; i < DL; ++i) x[i] = x[i] * alpha + f * y[2 + i * 64 + lane];
    }
    __shared__ float ml[4][2], o[4][D];
    if (lane == 0) {
        ml[w][0] = m;
        ml[w][1] = l;
    }
#pragma unroll
    for (int i = 0; i < DL; ++i) o[w][i * 64 + lane] = x[i];
    __syncthreads();
    if (threadIdx.x >= D) return;
    const int d = threadIdx.x;
    const float top = fmaxf(fmaxf(ml[0][0], ml[1][0]), fmaxf(ml[2][0], ml[3][0]));
    float sum = 0.0f, v = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float f = ml[k][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k][0] - top);
        sum += ml[k][1] == ml[k][1] ? f * ml[k][1] : NAN;
        v += f * o[k][d];
    }
    ((O *) row_at(a, p.out, e, b, r / p.group, head * p.group + r % p.group, sizeof(O)))[d] = (O) (sum == 0.0f ? 0.0f : v / sum);
}

// the same for many rows of few splits: a wave a row, four after each other (a workgroup a row took 90 us for 72k rows of two
// splits, most of it to start the workgroups)
template <int D, typename O> __global__ __launch_bounds__(256) void k_kv8_attend_join_rows(Kv8Call a, Kv8Attend p) {
    constexpr int DL = D / 64;
    const int tile = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Kv8Entry e = kv8_entry(a, b);
    if (tile * 16 >= e.n * p.group) return;
    const int n = splits_of(a, p, e, tile);
    const float * ws = p.ws + (((int64_t) b * a.c.n_heads + head) * p.tiles + tile) * p.splits * 16 * (D + 2);
    for (int row = 4 * w; row < 4 * w + 4; ++row) {
        const int r = tile * 16 + row;
        if (r >= e.n * p.group) return;
        float m = -INFINITY, l = 0.0f, x[DL] = {};
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float * y = ws + (k * 16 + row) * (D + 2);
            const float mk = y[0], lk = y[1], top = fmaxf(m, mk);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top), f = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - top);
            m = top;
            l = l * alpha + (lk == lk ? f * lk : NAN);
#pragma unroll
            for (int i = 0; i < DL; ++i) x[i] = x[i] * alpha + f * y[2 + i * 64 + lane];
        }
        O * out = (O *) row_at(a, p.out, e, b, r / p.group, head * p.group + r % p.group, sizeof(O));
#pragma unroll
        for (int i = 0; i < DL; ++i) out[i * 64 + lane] = (O) (l == 0.0f ? 0.0f : x[i] / l);
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

static thread_local int g_many_rows = 0;
void kv8_set_many_rows(int rows) { g_many_rows = rows; }

// How a call is run: host arithmetic on its sizes. The keys are cut into parts of `per` blocks, a workgroup each; entries may
// differ much in length, so parts are equal in size and not in number: long entries have more of them.
Kv8Plan kv8_plan(const Kv8Call & call, int group, int max_len) {
    const int64_t rows = (int64_t) call.b.max_new * group, tiles16 = (rows + 15) / 16;
    const int64_t blocks = std::max<int64_t>(1, (max_len + BLK - 1) / BLK), pairs = (int64_t) call.c.n_heads * call.b.n;
    Kv8Plan plan;
    // Many-row tiles where there is work for them, counted in 16 rows times a block: at heads of 64, 32 clips of 64 rows (61k)
    // take 54 us either way, of 96 rows 77 us in tiles of 16 and 67 in tiles of 128, 4 clips of 300 rows (36k) 35 and 45;
    // at heads of 128, 4 chunks of 80 rows over 4000 keys (10k) 39 and 35, of 132 rows 52 and 42.
    plan.many = rows > 32 && (double) tiles16 * pairs * blocks >= (call.c.head_dim == 64 ? 56000 : 13000);
    if (const int over = g_many_rows) plan.many = rows > over;
    const int mrows = MANY_WAVES * MR * 16;
    const int64_t tiles = plan.many ? (rows + mrows - 1) / mrows : tiles16;
    const int64_t groups = tiles * pairs;
    int64_t per = blocks;
    plan.fits = rows <= 1 << 22 && groups < 1 << 24;
    if (!plan.fits) return plan;
    if (!plan.many) {
        // 256 parts fill the card; parts of more than 32 blocks leave it unevenly loaded where lengths differ (16 streams of
        // 900 to 33000 tokens: parts of 24 to 40 blocks 103 us, of 16 125, of 65 and of 129 over 140)
        if (blocks > 32) per = std::min<int64_t>(32, std::max<int64_t>(8, (int64_t) std::min(std::ceil((double) groups * blocks / 256), 32.0)));
    } else {
        // rounds of the card (two or three workgroups on each of its 256 units) times the blocks of a part, three more to begin
        // and end it, and what the parts' workspace costs, in blocks (one chunk of 128 x 4 rows over 32000 keys: 896 us in
        // one part, 145 in eight, 119 in sixteen; 8 clips of 260 rows over 3000 keys: 101 in one, 106 in two)
        const int64_t slots = call.c.head_dim == 64 ? 768 : 512;
        int64_t best = INT64_MAX;
        for (int64_t s = 1; s <= 64 && blocks >= 8 * s; ++s) {
            const int64_t part = (blocks + s - 1) / s, cost = (groups * s + slots - 1) / slots * (part + 3) + (s > 1 ? 2 + groups * s / 120 : 0);
            if (cost < best) best = cost, per = part;
        }
    }
    plan.splits = (int) ((blocks + per - 1) / per);
    plan.fits = groups * plan.splits < (1 << 24) / 8 * 7;  // a one-dimensional grid: under 2^32 threads, by_die's spare ones among them
    if (!plan.fits) return plan;
    plan.per = (int) ((blocks + plan.splits - 1) / plan.splits);
    plan.tiles = (int) (plan.many ? tiles * (mrows / 16) : tiles);
    plan.join = plan.many ? MANY_WAVES * MR : 1;
    plan.ws_bytes = plan.splits > 1 ? (size_t) plan.tiles * call.c.n_heads * call.b.n * plan.splits * 16 * (call.c.head_dim + 2) * 4 : 0;
    // few workgroups: eight waves rather than four share a tile's blocks (1 clip 9.3 us against 10.8, 8 clips of 5 rows 10.9 against 12.0)
    plan.wide = !plan.many && plan.splits == 1 && groups <= 256;
    return plan;
}

void kv8_attend(hipStream_t s, const Kv8Call & call, const Kv8Attend & a, const Kv8Plan & plan, int out_type) {
    const int rows = call.b.max_new * a.group;
    const int parts = plan.tiles * plan.splits;
    const dim3 grid = parts == 1 ? dim3(1, call.c.n_heads, call.b.n) : dim3(workgroups(call, parts));
    const dim3 join(rows, call.c.n_heads, call.b.n);
    with_type(call.c, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        auto run = [&](auto o) {
            using O = decltype(o);
            if (plan.many) {
                constexpr int MW = MANY_WAVES;
                const int tiles = plan.tiles / (MW * MR);
                OWK_LAUNCH((k_kv8_attend_tiles<T, D, O, MW>), dim3(workgroups(call, tiles * plan.splits)), dim3(MW * 64), 0, s, call, a, tiles);
            } else if (plan.wide) {
                if (plan.tiles == 1) OWK_LAUNCH((k_kv8_attend_rows<T, D, O, 8, true>), grid, dim3(512), 0, s, call, a);
                else OWK_LAUNCH((k_kv8_attend_rows<T, D, O, 8, false>), grid, dim3(512), 0, s, call, a);
            } else {
                if (plan.tiles == 1) OWK_LAUNCH((k_kv8_attend_rows<T, D, O, 4, true>), grid, dim3(256), 0, s, call, a);
                else OWK_LAUNCH((k_kv8_attend_rows<T, D, O, 4, false>), grid, dim3(256), 0, s, call, a);
            }
            if (plan.splits > 1 && plan.splits < 16 && rows >= 16)
                OWK_LAUNCH((k_kv8_attend_join_rows<D, O>), dim3(plan.tiles, call.c.n_heads, call.b.n), dim3(256), 0, s, call, a);
            else if (plan.splits > 1)
                OWK_LAUNCH((k_kv8_attend_join<D, O>), join, dim3(256), 0, s, call, a);
        };
        if (out_type == OWK_KV8_F32) run(0.0f);
        else run(t);
    });
}

} // namespace owk
