// Keys and values held in 8 bits (include/owk_kv8.h): filling the cache, attending over it, reading it back.
//
// Blocks of 64 tokens; for a (block, head), keys and values apart: s = max|x| / 127, c = rint(x / s).
// Codes of keys lie token-major [64][D], codes of values dimension-major [D][64]: each is then the
// operand that its matrix product reads along its sum (keys along D, values along the tokens), 16
// contiguous bytes a lane. The incomplete last block (tail) lies in 16 bits in the same two orders.
#include "kv8.h"

namespace owk {

namespace {

typedef __bf16 bf16_t;
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
// attend
// ---------------------------------------------------------------------------------------------------
// One workgroup per (row, query head, entry): wave w takes blocks w, w + 4, ..; a lane is a key while
// scores are made and a dimension while values are added.
template <typename T, int D, typename O>
__global__ __launch_bounds__(256) void k_kv8_attend(Kv8Call a, Kv8Attend p) {
    constexpr int DL = D / 64;  // dimensions of a lane
    const int b = blockIdx.z, qh = blockIdx.y, i = blockIdx.x, head = qh / p.group;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const Kv8Entry e = kv8_entry(a, b);
    if (i >= e.n) return;
    const int cap = a.c.max_blocks * BLK;
    const int stored = e.seq < 0 ? 0 : p.causal ? min(e.start + e.n, cap) : e.start;
    const int seen = min(stored, p.causal ? e.start + i + 1 : stored);
    __shared__ float q[D];
    __shared__ float part[4][D + 2];
    const T * qr = (const T *) row_at(a, p.q, e, b, i, qh, 2);
    for (int d = threadIdx.x; d < D; d += 256) q[d] = to_f32(qr[d]) * p.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[DL] = {};
    for (int blk = w; blk * BLK < seen; blk += 4) {
        const bool in_tail = blk == stored / BLK;
        const int64_t page = kv8_page(a.c, e.seq, blk);
        if (!in_tail && page < 0) continue;
        const int64_t hk = (page * a.c.n_heads + head);
        const int64_t tk = ((int64_t) e.seq * a.c.n_heads + head) * BLK * D;
        const bool visible = blk * BLK + lane < seen;
        float s = 0.0f;
        if (visible) {
            if (in_tail) {
                const T * k = (const T *) a.c.k_tail + tk + lane * D;
                for (int d = 0; d < D; ++d) s = fmaf(q[d], to_f32(k[d]), s);
            } else {
                const int8_t * k = a.c.k + hk * BLK * D + lane * D;
                for (int d = 0; d < D; ++d) s = fmaf(q[d], (float) k[d], s);
                s *= a.c.k_scale[hk];
            }
        }
        const bool odd = __any(visible && !(s == s));
        const float top = fmaxf(m, wave_max(visible ? s : -INFINITY));
        const float base = top == -INFINITY ? 0.0f : top;
        const float alpha = expf(m - base);
        const float pr = odd ? NAN : visible ? expf(s - base) : 0.0f;
        l = l * alpha + wave_sum(pr);
        m = top;
#pragma unroll
        for (int g = 0; g < DL; ++g) {
            const int d = g * 64 + lane;
            float sum = 0.0f;
            for (int t = 0; t < BLK; ++t) {
                const float pt = __shfl(pr, t);
                if (blk * BLK + t >= seen) continue;
                const float v = in_tail ? to_f32(((const T *) a.c.v_tail + tk)[d * BLK + t]) : (float) (a.c.v + hk * BLK * D)[d * BLK + t];
                sum = fmaf(pt, v, sum);
            }
            acc[g] = acc[g] * alpha + (in_tail ? sum : sum * a.c.v_scale[hk]);
        }
    }
    if (lane == 0) {
        part[w][D] = m;
        part[w][D + 1] = l;
    }
#pragma unroll
    for (int g = 0; g < DL; ++g) part[w][g * 64 + lane] = acc[g];
    __syncthreads();
    const float top = fmaxf(fmaxf(part[0][D], part[1][D]), fmaxf(part[2][D], part[3][D]));
    const float base = top == -INFINITY ? 0.0f : top;
    for (int d = threadIdx.x; d < D; d += 256) {
        float o = 0.0f, total = 0.0f;
        for (int k = 0; k < 4; ++k) {
            const float f = expf(part[k][D] - base);
            total += part[k][D + 1] * f;
            o += part[k][d] * f;
        }
        ((O *) row_at(a, p.out, e, b, i, qh, sizeof(O)))[d] = (O) (total == 0.0f ? 0.0f : o / total);
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

Kv8Plan kv8_plan(const Kv8Call & call, int group, int max_len) { return Kv8Plan{1, 0}; }

void kv8_attend(hipStream_t s, const Kv8Call & call, const Kv8Attend & a, int out_type) {
    const dim3 grid(call.b.max_new, call.c.n_heads * a.group, call.b.n);
    with_type(call.c, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        if (out_type == OWK_KV8_F32) OWK_LAUNCH((k_kv8_attend<T, D, float>), grid, dim3(256), 0, s, call, a);
        else OWK_LAUNCH((k_kv8_attend<T, D, T>), grid, dim3(256), 0, s, call, a);
    });
}

} // namespace owk
