// 8-bit serving operators for gfx950: rows to codes and back, RMS norm with 8-bit output, int8 product.
//
// A quantised row is 127-level symmetric: a = max_k |y_k|, scale s = a / 127, code q_k = rint(y_k * 127 / a), so that
// y_k ~ q_k * s.  All codes of a row share s; the product of two quantised matrices is then
//
//     y[m, n] = act( (sum_k q[m, k] p[n, k]) * s[m] * t[n] + b[n] )
//
// with the sum exact in 32-bit integers (K < 2^31 / 128^2 = 131072) and everything after it in fp32.
//
// Conventions
//  * Code matrices are row-major with 16-byte aligned rows: the row stride is a multiple of 16 and at least K rounded up
//    to 16, and every byte up to there is readable.  The bytes beyond K may hold anything: the product clears them in
//    the ACTIVATION operand (0 * anything = 0 in integers, so one operand suffices).
//  * A row that holds a NaN or an infinity gets scale NaN and codes 0: whatever reads it gets NaN, never a number.
//  * A row of zeros gets scale 0 and codes 0.
#include "common.h"
#include "int8_args.h"
#include <type_traits>


typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// A launch and its own status: an error that another call has left pending is neither taken for this one's nor cleared.
template <typename A>
static int enqueue(void (*kernel)(A), dim3 grid, int block, int lds, hipStream_t stream, A a) {
    void* args[] = {&a};
    const hipError_t rc = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(block), args, lds, stream);
    if (rc != hipSuccess) (void)hipGetLastError();         // reported by the return value
    return (int)rc;
}

// ---------------------------------------------------------------------------------------------------------------
// floating rows -> codes
// ---------------------------------------------------------------------------------------------------------------

// Eight neighbouring elements of a row.  Only the element's own alignment is assumed: gfx950 takes 16-byte loads and
// stores at any address, so rows of odd length need no path of their own (the last K % 8 elements aside).
template <typename T>
struct Raw8 {
    T e[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = (T)v[i];
    __builtin_memcpy(p, &r, sizeof(r));
}

__device__ __forceinline__ unsigned row16_umax(unsigned v) {       // over 16 neighbouring lanes
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
    return v;
}
// The same bits in all 16 lanes: every step adds two values that both partners hold (neighbours, pairs, quads mirrored in 8
// lanes, eights mirrored in 16).  Rotations by 4 and 8 would pair the quads differently in the two halves of the row.
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_mov<0xb1>(v);
    v += dpp_mov<0x4e>(v);
    v += dpp_mov<0x141>(v);
    v += dpp_mov<0x140>(v);
    return v;
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
    v = row16_umax(v);
    const unsigned a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
    const unsigned c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
    return max(max(a, b), max(c, d));
}

// Sum / maximum over the G threads that share a row.  G = 16 and 64: lanes of one wave, no LDS.  `red` holds a word a wave,
// and every call of a kernel has words of its own, so that one barrier a call is enough.
template <int G>
__device__ __forceinline__ float group_sum(float v, unsigned* red) {
    if constexpr (G == 16) return row16_sum(v);
    v = wave_sum(v);
    if constexpr (G == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __builtin_bit_cast(unsigned, v);
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) s += __builtin_bit_cast(float, red[w]);
    return s;
}
template <int G>
__device__ __forceinline__ unsigned group_umax(unsigned v, unsigned* red) {
    if constexpr (G == 16) return row16_umax(v);
    v = wave_umax(v);
    if constexpr (G == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned s = 0;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) s = max(s, red[w]);
    return s;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// What turns a row's values into codes.  |y| as an unsigned integer orders like the value, with infinity and NaN above
// every finite number, so one integer maximum finds the largest magnitude and whether the row is finite.
struct RowCode {
    float pre, inv, rest, scale;       // 127 / (top * pre) = inv + rest
    unsigned keep;         // all ones, or 0 for a row that is not finite
};
__device__ __forceinline__ RowCode row_code(unsigned top_bits) {
    const float top = __builtin_bit_cast(float, top_bits);
    RowCode c;
    const bool finite = top_bits < 0x7f800000u, some = top > 0.f && finite;
    // the smallest and the largest rows are moved by 2^64 first (exact), where 127 / top or its rest would leave fp32
    c.pre = top < 0x1p-62f ? 0x1p64f : top > 0x1p62f ? 0x1p-64f : 1.f;
    const float a = top * c.pre;
    c.inv = some ? 127.f / a : 0.f;
    c.rest = some ? __builtin_fmaf(-c.inv, a, 127.f) * (c.inv * (1.f / 127.f)) : 0.f;
    c.scale = finite ? top / 127.f : __builtin_nanf("");
    c.keep = finite ? ~0u : 0u;
    return c;
}
// y * 127 / a, rounded to fp32, then to the nearest whole number, halves to even, as a byte.  127 / a in one fp32 number would
// move the halves (a / 2 is 63.5 codes whatever a is): with its rest the product's error is 2^-47 before the fma rounds it,
// so that a quotient which is exactly halfway stays there.  Adding 1.5 * 2^23 leaves the whole number in the low bits.
// One instruction a value more than without the rest: 65536 x 100 fp32 8.7 -> 8.9 us, longer rows and the policy within 1 %.
__device__ __forceinline__ unsigned code_bits(float y, const RowCode& c) {
#pragma clang fp contract(off)
    const float x = y * c.pre, v = __builtin_fmaf(x, c.inv, x * c.rest);
    return __builtin_bit_cast(unsigned, v + 12582912.f);
}
__device__ __forceinline__ unsigned pack4(unsigned a, unsigned b, unsigned c, unsigned d) {
    const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return lo | hi;
}
__device__ __forceinline__ void store_codes8(signed char* p, const float (&y)[8], const RowCode& c) {
    uint2 w;
    w.x = pack4(code_bits(y[0], c), code_bits(y[1], c), code_bits(y[2], c), code_bits(y[3], c)) & c.keep;
    w.y = pack4(code_bits(y[4], c), code_bits(y[5], c), code_bits(y[6], c), code_bits(y[7], c)) & c.keep;
    *reinterpret_cast<uint2*>(p) = w;
}

// The factor of the norm.  The plain sum of squares overflows above ~1.8e19 and loses everything below ~1e-20; a row
// like that (known from the sum itself, so that ordinary rows pay nothing) is scaled by a power of two first.
struct NormFactor {
    float pre, rs;         // y = (h * pre) * rs * weight
};
__device__ __forceinline__ bool norm_is_plain(float ss, float K, float eps) {
    const float ms = ss / K + eps;
    return ms >= 0x1p-80f && ms < __builtin_inff() && ss < __builtin_inff();
}
__device__ __forceinline__ float norm_lift(unsigned top_bits, float eps) {
    int e = (int)(top_bits >> 23) - 126;
    if (top_bits < 0x00800000u) e = -126;
    if (eps > 0.f && e < -60) e = -60;         // below that the added eps decides, and must stay finite
    e = e < -120 ? -120 : (e > 126 ? 126 : e);
    return __builtin_ldexpf(1.f, -e);
}

template <typename T>
__device__ __forceinline__ float load1(const void* p, long long i) {
    return (float)reinterpret_cast<const T*>(p)[i];
}
__device__ __forceinline__ float weight1(const QuantRowsArgs& a, long long k) {
    if (a.wdtype == F_FP32) return load1<float>(a.weight, k);
    if (a.wdtype == F_BF16) return load1<__bf16>(a.weight, k);
    if (a.wdtype == F_FP16) return load1<_Float16>(a.weight, k);
    return 1.f;
}
template <typename W>
__device__ __forceinline__ void scale8(float (&y)[8], const void* weight, long long k) {
    const Raw8<W> w = load8(reinterpret_cast<const W*>(weight) + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= (float)w.e[i];
}

// What bounds it is memory: quantising 8192 x 8192 bf16 takes 40 us (5.0 TB/s read and written), 2000 x 16384 fp32 33.8 us
// (4.9), the norm with a residual of 4096 x 4096 bf16 27 us (4.4), of 16384 x 8192 175 us (5.4); a copy of 1 GiB runs at 5.2.
// Rows of odd length (16384 x 1111 bf16, loads across cache lines) get 3.4 TB/s.  (Graph of calls on three sets of operands.)
// A row stays in the registers of its G threads from the load to the codes: one read, one write, whatever is computed
// between.  Thread t holds the 8-element chunks t, t + G, ... (V of them).
template <typename T, int G, int V, bool NORM>
__global__ __launch_bounds__(G < 256 ? 256 : G) void quant_rows_kernel(const QuantRowsArgs a) {
    constexpr int BLOCK = G < 256 ? 256 : G;
    __shared__ unsigned red[4][G > 64 ? G / 64 : 1];       // one line a reduction
    const long long row = (long long)blockIdx.x * (BLOCK / G) + threadIdx.x / G;
    if (row >= a.M) return;                      // whole groups of 16 or 64 lanes only: no barrier is skipped
    const int t = threadIdx.x % G;
    const int K = (int)a.K, full = K >> 3, rem = K & 7, chunks = (int)(a.ld_q >> 3);
    const T* const x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
    const T* const r = reinterpret_cast<const T*>(a.residual) + row * a.ld_r;
    const bool add = NORM && a.residual != nullptr;

    float y[V][8];
    {
        // every thread loads from an address inside the row and drops what lies beyond it, so that all loads are in
        // flight at once
        Raw8<T> rx[V], rr[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = min(t + j * G, full - 1);
            if (full > 0) rx[j] = load8(x + 8 * c);
        }
        if (add) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = min(t + j * G, full - 1);
                if (full > 0) rr[j] = load8(r + 8 * c);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = t + j * G;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = (float)rx[j].e[i];
                if (add) v += (float)rr[j].e[i];
                y[j][i] = c < full ? v : 0.f;
            }
            if (c == full && rem) {              // the last elements of a row whose length is no multiple of 8
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < rem) y[j][i] = (float)x[8 * c + i] + (add ? (float)r[8 * c + i] : 0.f);
            }
        }
    }
    if (NORM) {
        if (a.h != nullptr) {
            T* const h = reinterpret_cast<T*>(a.h) + row * a.ld_h;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = t + j * G;
                if (c < full) store8(h + 8 * c, y[j]);
                if (c == full && rem) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < rem) h[8 * c + i] = (T)y[j][i];
                }
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += y[j][i] * y[j][i];
        ss = group_sum<G>(ss, red[0]);
        float pre = 1.f, eps = a.eps;
        if (!norm_is_plain(ss, (float)K, eps)) { // the same for the whole row
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, abs_bits(y[j][i]));
            top = group_umax<G>(top, red[1]);
            pre = norm_lift(top, eps);
            ss = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += (y[j][i] * pre) * (y[j][i] * pre);
            ss = group_sum<G>(ss, red[2]);
            eps = eps * pre * pre;
            if (top >= 0x7f800000u) ss = __builtin_nanf("");
            if (top == 0u && a.eps == 0.f) eps = 1.f;      // a row of zeros stays one
        }
        const float rs = 1.f / sqrtf(ss / (float)K + eps);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = t + j * G;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[j][i] = (y[j][i] * pre) * rs;
            if (a.wdtype != F_NONE) {
                if (c < full) {
                    if (a.wdtype == F_FP32) scale8<float>(y[j], a.weight, 8 * c);
                    else if (a.wdtype == F_BF16) scale8<__bf16>(y[j], a.weight, 8 * c);
                    else scale8<_Float16>(y[j], a.weight, 8 * c);
                } else if (c == full && rem) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < rem) y[j][i] *= weight1(a, 8 * c + i);
                }
            }
        }
    }
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, abs_bits(y[j][i]));
    const RowCode code = row_code(group_umax<G>(top, red[3]));
    signed char* const q = a.q + row * a.ld_q;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = t + j * G;
        if (c < chunks) store_codes8(q + 8 * c, y[j], code);
    }
    if (t == 0) a.scale[row] = code.scale;
}

// Rows too long for the registers of 1024 threads: the row is read again for each of the steps (it fits the L2 once).
template <typename T, bool NORM>
__global__ __launch_bounds__(1024) void quant_long_rows_kernel(const QuantRowsArgs a) {
    constexpr int G = 1024;
    __shared__ unsigned red[4][G / 64];
    const long long row = blockIdx.x;
    const T* const x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
    const T* const r = reinterpret_cast<const T*>(a.residual) + row * a.ld_r;
    T* const h = reinterpret_cast<T*>(a.h) + row * a.ld_h;
    const bool add = NORM && a.residual != nullptr;
    const int K = (int)a.K, full = K >> 3, rem = K & 7, chunks = (int)(a.ld_q >> 3);
    // chunk c of the sum x + residual, zeros beyond the row
    auto sums8 = [&](int c, float (&y)[8]) {
        if (c < full) {
            const Raw8<T> rx = load8(x + 8ll * c);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (float)rx.e[i];
            if (add) {
                const Raw8<T> rr = load8(r + 8ll * c);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] += (float)rr.e[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = c == full && i < rem ? (float)x[8ll * c + i] + (add ? (float)r[8ll * c + i] : 0.f) : 0.f;
        }
    };
    float pre = 1.f, rs = 1.f, y[8];
    if (NORM) {
        float ss = 0.f;
        for (int c = threadIdx.x; c < chunks; c += G) {
            sums8(c, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += y[i] * y[i];
            if (a.h != nullptr) {
                if (c < full) store8(h + 8ll * c, y);
                else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c == full && i < rem) h[8ll * c + i] = (T)y[i];
                }
            }
        }
        ss = group_sum<G>(ss, red[0]);
        float eps = a.eps;
        if (!norm_is_plain(ss, (float)K, eps)) {
            unsigned top = 0;
            for (int c = threadIdx.x; c < chunks; c += G) {
                sums8(c, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, abs_bits(y[i]));
            }
            top = group_umax<G>(top, red[1]);
            pre = norm_lift(top, eps);
            ss = 0.f;
            for (int c = threadIdx.x; c < chunks; c += G) {
                sums8(c, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += (y[i] * pre) * (y[i] * pre);
            }
            ss = group_sum<G>(ss, red[2]);
            eps = eps * pre * pre;
            if (top >= 0x7f800000u) ss = __builtin_nanf("");
            if (top == 0u && a.eps == 0.f) eps = 1.f;
        }
        rs = 1.f / sqrtf(ss / (float)K + eps);
    }
    auto values8 = [&](int c) {
        sums8(c, y);
        if (NORM) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (y[i] * pre) * rs;
            if (a.wdtype != F_NONE) {
                if (c < full) {
                    if (a.wdtype == F_FP32) scale8<float>(y, a.weight, 8ll * c);
                    else if (a.wdtype == F_BF16) scale8<__bf16>(y, a.weight, 8ll * c);
                    else scale8<_Float16>(y, a.weight, 8ll * c);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c == full && i < rem) y[i] *= weight1(a, 8ll * c + i);
                }
            }
        }
    };
    unsigned top = 0;
    for (int c = threadIdx.x; c < chunks; c += G) {
        values8(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, abs_bits(y[i]));
    }
    const RowCode code = row_code(group_umax<G>(top, red[3]));
    signed char* const q = a.q + row * a.ld_q;
    for (int c = threadIdx.x; c < chunks; c += G) {
        values8(c);
        store_codes8(q + 8ll * c, y, code);
    }
    if (threadIdx.x == 0) a.scale[row] = code.scale;
}

// A launch holds fewer than 2^32 threads: more rows than that are several launches.  The entries whose names end in _in take
// the limit as an argument (1024, a workgroup, at least; the product's: what 16 rows need), so that what follows the first
// launch can be had with few rows.
constexpr long long LAUNCH_THREADS = 0xffffffffll;
static bool good_limit(long long threads) { return threads >= 1024 && threads <= LAUNCH_THREADS; }

template <typename F>
static int launch_row_ranges(QuantRowsArgs a, long long threads, long long element, int block, int rows_per_block, F launch) {
    const long long most = (threads / block) * rows_per_block, M = a.M;
    for (long long done = 0; done < M; done += most) {
        QuantRowsArgs part = a;
        part.M = M - done < most ? M - done : most;
        part.x = (const char*)a.x + done * a.ld_x * element;
        if (a.residual != nullptr) part.residual = (const char*)a.residual + done * a.ld_r * element;
        if (a.h != nullptr) part.h = (char*)a.h + done * a.ld_h * element;
        part.q = a.q + done * a.ld_q, part.scale = a.scale + done;
        const int rc = launch(part, dim3((unsigned)((part.M + rows_per_block - 1) / rows_per_block)));
        if (rc != 0) return rc;
    }
    return 0;
}
template <typename T, int G, int V>
static int launch_rows(const QuantRowsArgs& a, long long threads, hipStream_t stream) {
    constexpr int BLOCK = G < 256 ? 256 : G;
    return launch_row_ranges(a, threads, sizeof(T), BLOCK, BLOCK / G, [&](const QuantRowsArgs& part, dim3 grid) {
        return enqueue(a.norm ? quant_rows_kernel<T, G, V, true> : quant_rows_kernel<T, G, V, false>, grid, BLOCK, 0, stream, part);
    });
}
template <typename T>
static int launch_rows_of(const QuantRowsArgs& a, long long threads, hipStream_t stream) {
    // c: chunks of 8 a row needs.  Short rows share a wave, long ones take as few threads as hold them in 4 chunks each (8 from
    // 8192 columns on); where the rows are no more than the CUs, 1024 threads answer sooner than 256.  Measured (us): 65536 x 100
    // fp32 8.9, 19.0 with a wave a row; bf16 with a residual, 1024 threads and 256: 1 x 16384 4.9 and 8.8, 1 x 5000 4.2 and 5.2,
    // 256 x 16384 8.8 and 13.9, 256 x 5000 5.3 and 6.2.
    const long long c = a.ld_q >> 3;
    if (c <= 16) return launch_rows<T, 16, 1>(a, threads, stream);
    if (c <= 32) return launch_rows<T, 16, 2>(a, threads, stream);
    if (c <= 64) return launch_rows<T, 64, 1>(a, threads, stream);
    if (c <= 128) return launch_rows<T, 64, 2>(a, threads, stream);
    if (c <= 256) return launch_rows<T, 64, 4>(a, threads, stream);
    if (c <= 512) return launch_rows<T, 256, 2>(a, threads, stream);
    if (c <= 2048 && a.M <= 256) return launch_rows<T, 1024, 2>(a, threads, stream);
    if (c <= 1024) return launch_rows<T, 256, 4>(a, threads, stream);
    if (c <= 2048) return launch_rows<T, 256, 8>(a, threads, stream);
    if (c <= 4096) return launch_rows<T, 1024, 4>(a, threads, stream);
    return launch_row_ranges(a, threads, sizeof(T), 1024, 1, [&](const QuantRowsArgs& part, dim3 grid) {
        return enqueue(a.norm ? quant_long_rows_kernel<T, true> : quant_long_rows_kernel<T, false>, grid, 1024, 0, stream, part);
    });
}

D4PG_API int d4pg_quant_rows_in(const QuantRowsArgs* a, long long threads, hipStream_t stream) {
    if (!good_limit(threads)) return -8;
    if (a->M < 1 || a->M > 0x7fffffffll || a->K < 1 || a->K > 0x7fffffffll) return -1;
    if (a->x == nullptr || a->q == nullptr || a->scale == nullptr) return -2;
    if ((a->ld_q & 15) || a->ld_q < a->K || a->ld_q >= a->K + 16 || ((uintptr_t)a->q & 15)) return -3;
    if (a->wdtype != F_NONE && (a->weight == nullptr || a->wdtype < 0 || a->wdtype > F_FP16)) return -4;
    if (!a->norm && (a->residual != nullptr || a->weight != nullptr || a->h != nullptr)) return -5;
    if (a->dtype == F_FP32) return launch_rows_of<float>(*a, threads, stream);
    if (a->dtype == F_BF16) return launch_rows_of<__bf16>(*a, threads, stream);
    if (a->dtype == F_FP16) return launch_rows_of<_Float16>(*a, threads, stream);
    return -6;
}
D4PG_API int d4pg_quant_rows(const QuantRowsArgs* a, hipStream_t stream) { return d4pg_quant_rows_in(a, LAUNCH_THREADS, stream); }

// ---------------------------------------------------------------------------------------------------------------
// codes -> floating rows
// ---------------------------------------------------------------------------------------------------------------

// 8192 x 8192 to bf16: 38 us (5.3 TB/s); 30 us right after quantising, with the codes in the cache.
template <typename T>
__global__ __launch_bounds__(256) void dequant_rows_kernel(const DequantRowsArgs a) {
    const int tpr = 1 << a.tpr_log;
    const long long row = (long long)blockIdx.x * (256 >> a.tpr_log) + (threadIdx.x >> a.tpr_log);
    if (row >= a.M) return;
    const float s = a.scale[row];
    const signed char* const q = a.q + row * a.ld_q;
    T* const out = reinterpret_cast<T*>(a.out) + row * a.K;
    for (long long k = 8ll * ((threadIdx.x & (tpr - 1)) + tpr * blockIdx.y); k < a.K; k += 8ll * tpr * gridDim.y) {
        if (k + 8 <= a.K) {
            const Raw8<signed char> c = load8(q + k);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)c.e[i] * s;
            store8(out + k, v);
        } else {
            for (long long i = k; i < a.K; ++i) out[i] = (T)((float)q[i] * s);
        }
    }
}

D4PG_API int d4pg_dequant_rows_in(DequantRowsArgs* a, long long threads, hipStream_t stream) {
    if (!good_limit(threads)) return -8;
    if (a->M < 1 || a->M > 0x7fffffffll || a->K < 1 || a->K > 0x7fffffffll) return -1;
    if (a->q == nullptr || a->scale == nullptr || a->out == nullptr) return -2;
    a->tpr_log = 0;
    while (a->tpr_log < 8 && (8ll << a->tpr_log) < a->K) ++a->tpr_log;
    const int rpb = 256 >> a->tpr_log;
    const long long most = (threads / 256) * rpb;
    const int bytes = a->dtype == F_FP32 ? 4 : 2;
    if (a->dtype < F_FP32 || a->dtype > F_FP16) return -6;
    for (long long done = 0; done < a->M; done += most) {
        DequantRowsArgs part = *a;
        part.M = a->M - done < most ? a->M - done : most;
        part.q = a->q + done * a->ld_q, part.scale = a->scale + done, part.out = (char*)a->out + done * a->K * bytes;
        // few long rows: several workgroups each
        const long long blocks = (part.M + rpb - 1) / rpb, pieces = (a->K + 2047) / 2048, spread = 1024 / blocks + 1;
        const dim3 grid((unsigned)blocks, (unsigned)(spread < pieces ? spread : pieces));
        const int rc = enqueue(a->dtype == F_FP32 ? dequant_rows_kernel<float> : a->dtype == F_BF16 ? dequant_rows_kernel<__bf16> : dequant_rows_kernel<_Float16>,
                               grid, 256, 0, stream, part);
        if (rc != 0) return rc;
    }
    return 0;
}
D4PG_API int d4pg_dequant_rows(DequantRowsArgs* a, hipStream_t stream) { return d4pg_dequant_rows_in(a, LAUNCH_THREADS, stream); }

// ---------------------------------------------------------------------------------------------------------------
// product of codes
// ---------------------------------------------------------------------------------------------------------------

// Four neighbouring columns n .. n + 3 of row m (those below N).  v: integer sums.
template <typename T>
__device__ __forceinline__ void store4(T* out, const float (&v)[4], int left) {
    if (left >= 4) {
        T r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
        __builtin_memcpy(out, r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) out[i] = (T)v[i];
    }
}
// What four neighbouring columns n .. n + 3 need besides their sums.
struct Columns4 {
    float scale[4], bias[4];
};
__device__ __forceinline__ Columns4 columns4(const float* wscale, const float* bias, int n, int N) {
    Columns4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ni = min(n + i, N - 1);
        c.scale[i] = wscale[ni];
        c.bias[i] = bias != nullptr ? bias[ni] : 0.f;
    }
    return c;
}
// act(scaled * t + b) of four columns, scaled = sum * s.  ONE definition, contraction off: every kernel below rounds alike.
__device__ __forceinline__ f32x4 scaled4(const i32x4 sum, float sm) {
    return f32x4{(float)sum[0] * sm, (float)sum[1] * sm, (float)sum[2] * sm, (float)sum[3] * sm};
}
// tanh for 16-bit results: sign x (1 - 2 / (e^2|x| + 1)), below 1/2, where that cancels, the Taylor series
// x - x^3 / 3 + 2 x^5 / 15 - ... to x^15.  Over every fp32 argument of [0.001, 20) against 64 bits: at most 0.79 units of the
// last place of fp32 below 1/2 and 2.6 above, which 16 bits do not hold.  fp32 results take tanhf (1.4 units over the same
// arguments), which costs more: fp32 results of 777 x 1333 x 2001 12.8 us, 12.3 with this form; of 256 x 400 x 400 3.8 and 3.6.
__device__ __forceinline__ float tanh_of(float x) {
    const float a = __builtin_fabsf(x), s = x * x;
    const float e = __builtin_amdgcn_exp2f(a * 2.8853900817779268f);       // 2 / ln 2
    const float far = __builtin_copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f), x);
    float p = -929569.f / 638512875.f;
    p = __builtin_fmaf(p, s, 21844.f / 6081075.f);
    p = __builtin_fmaf(p, s, -1382.f / 155925.f);
    p = __builtin_fmaf(p, s, 62.f / 2835.f);
    p = __builtin_fmaf(p, s, -17.f / 315.f);
    p = __builtin_fmaf(p, s, 2.f / 15.f);
    p = __builtin_fmaf(p, s, -1.f / 3.f);
    return a < 0.5f ? __builtin_fmaf(x * s, p, x) : far;
}
__device__ __forceinline__ void values4(float (&v)[4], const f32x4 scaled, const Columns4& c, bool biased, int act, int dtype) {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = scaled[i] * c.scale[i];
        if (biased) v[i] += c.bias[i];
    }
    if (act == ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];       // keeps NaN
    } else if (act == ACT_TANH && dtype == F_FP32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = tanhf(v[i]);
    } else if (act == ACT_TANH) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = tanh_of(v[i]);
    }
}
__device__ __forceinline__ void store_values4(void* out, long long at, int dtype, const float (&v)[4], int left) {
    if (dtype == F_FP32) store4(reinterpret_cast<float*>(out) + at, v, left);
    else if (dtype == F_BF16) store4(reinterpret_cast<__bf16*>(out) + at, v, left);
    else store4(reinterpret_cast<_Float16*>(out) + at, v, left);
}
__device__ __forceinline__ void finish4(const LinearInt8Args& a, int m, int n, const f32x4 scaled, const Columns4& c) {
    if (m >= a.M || n >= a.N) return;
    float v[4];
    values4(v, scaled, c, a.bias != nullptr, a.act, a.dtype);
    store_values4(a.out, (long long)m * a.ld_out + n, a.dtype, v, a.N - n);
}

enum { TOO_MANY = -7 };        // threads for one launch: the caller halves the rows (16 rows fit the real limit whatever their columns)

// All ones in the bytes k .. k + 15 that lie below K.
__device__ __forceinline__ i32x4 below(int k, int K) {
    i32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = K - (k + 4 * i);
        m[i] = left >= 4 ? -1 : (left <= 0 ? 0 : (int)((1u << (8 * left)) - 1u));
    }
    return m;
}

// Few rows or small layers: a workgroup makes 16 MT rows x 16 NT columns, its WAVES waves split K and meet in LDS.
// Operands go from memory to the matrix instruction's registers directly (v_mfma_i32_16x16x64_i8: lane 16 g + c holds
// 16 bytes of row c at k = 16 g); the weights are the A operand, so that a lane ends with four neighbouring columns.
// A wave issues the loads of U slices of 64 k before it multiplies the first: at these sizes the time is that of the
// loads' way from memory.
template <int MT, int NT, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void linear_int8_rows_kernel(const LinearInt8Args a) {
    __shared__ i32x4 part[WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int tiles_n = (a.N + 16 * NT - 1) / (16 * NT);
    const int tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    const signed char* xp[MT];
    const signed char* wp[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xp[i] = a.q + (long long)min((tm * MT + i) * 16 + c, a.M - 1) * a.ld_q;
#pragma unroll
    for (int i = 0; i < NT; ++i) wp[i] = a.w + (long long)min((tn * NT + i) * 16 + c, a.N - 1) * a.ld_w;
    const int last = ((a.K - 1) >> 4) << 4;      // the last 16 bytes of a row that hold a code
    // what the results of this wave need besides their sums: asked for before the products, not after them
    constexpr int MINE = (MT * NT + WAVES - 1) / WAVES;
    float sm[MINE];
    Columns4 col[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int u = min(wave + i * WAVES, MT * NT - 1);
        sm[i] = a.scale[min((tm * MT + u / NT) * 16 + c, a.M - 1)];
        col[i] = columns4(a.wscale, a.bias, (tn * NT + u % NT) * 16 + 4 * g, a.N);
    }
    i32x4 acc[MT][NT] = {};
    // slice s of the wave covers k = 64 (wave + s WAVES): neighbouring waves read neighbouring bytes
    for (int k0 = 64 * wave; k0 < a.K; k0 += 64 * WAVES * U) {
        i32x4 x[U][MT], w[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kc = min(k0 + 64 * WAVES * u + 16 * g, last);
#pragma unroll
            for (int i = 0; i < NT; ++i) w[u][i] = *reinterpret_cast<const i32x4*>(wp[i] + kc);
#pragma unroll
            for (int i = 0; i < MT; ++i) x[u][i] = *reinterpret_cast<const i32x4*>(xp[i] + kc);
        }
        if (k0 + 64 * WAVES * (U - 1) + 64 > a.K) {      // what lies beyond K repeats the last bytes: cleared on one side
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const i32x4 mask = below(k0 + 64 * WAVES * u + 16 * g, a.K);
#pragma unroll
                for (int i = 0; i < MT; ++i) x[u][i] &= mask;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][j], x[u][i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int u = wave + i * WAVES;
        if (u >= MT * NT) break;
        i32x4 sum = part[0][u][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum += part[w][u][lane];
        finish4(a, (tm * MT + u / NT) * 16 + c, (tn * NT + u % NT) * 16 + 4 * g, scaled4(sum, sm[i]), col[i]);
    }
}

template <int MT, int NT, int WAVES, int U>
static int launch_linear_rows(const LinearInt8Args& a, long long threads, hipStream_t stream) {
    const long long tiles = (long long)((a.M + 16 * MT - 1) / (16 * MT)) * ((a.N + 16 * NT - 1) / (16 * NT));
    if (tiles * (64 * WAVES) > threads) return TOO_MANY;
    return enqueue(linear_int8_rows_kernel<MT, NT, WAVES, U>, dim3((unsigned)tiles), 64 * WAVES, 0, stream, a);
}

// Many rows: a workgroup of WM x WN waves makes a tile of BM = 32 MI WM rows x BN = 32 NI WN columns, a wave 32 MI x 32 NI
// of it in accumulators (v_mfma_i32_32x32x32_i8: lane 32 h + r holds 16 bytes of row r at k = 16 h; the weights are the A
// operand).
//
//  * Both tiles of 128 k lie in LDS twice.  Memory moves straight into LDS (16 bytes a lane, 8 rows of 128 bytes an
//    instruction, no registers on the way); the move for step t + 2 starts as soon as every wave has read step t.
//  * A wave reads the operands of a 32-k slice from LDS while it multiplies the slice before, across the border of two
//    steps too: the one barrier of a step stands before its LAST slice, whose operands are in registers by then.
//  * 16-byte pieces of a row are stored XOR (row / 2 % 8): the 16 lanes of an LDS cycle (256 bytes) then cover all banks
//    (XOR row % 8 left every other cycle in conflict).  The move writes LDS in lane order, so each lane fetches the piece
//    that belongs at its place.
//  * Rows beyond M or N repeat the last one and are not stored; pieces beyond K repeat the last one and are cleared in the
//    activation operand of the last step.
//  * Workgroups of one XCD (blockIdx % 8) take neighbouring tiles, 2048 rows of them at a time, so that what they share is
//    in their L2 (moves alone, 8192^3 in tiles of 256: 247 us with 4 tile rows, 231 - 254 with 8, 300 with 16).
//
// What bounds it at 8192^3 (tiles of 256): power first - the matrix instruction alone does 4.9 P/s on zeros, 3.5 on random
// codes, 3.1 - 3.2 with its LDS reads - then how well the rest hides behind it.  Moves alone take 231 us.  Waves a SIMD
// decide the rest: 1 (waves of 128 x 128) 560 us, matrix pipe 52 % busy; 2 (128 x 64) 476; 4 (64 x 64) 465 us = 2.36 P/s (pipe 70 %).
enum { STEP_FULL = 0, STEP_DRAIN = 1, STEP_LAST = 2 };

template <int MI, int NI, int WM, int WN, int KW, int S>
__device__ __forceinline__ void linear_tile(const LinearInt8Args& a, signed char* const lds) {
    constexpr int BM = 32 * MI * WM, BN = 32 * NI * WN, TILE = (BM + BN) * 128, GROUP = 2048 / BM;
    constexpr int MOVES = (BM + BN) / 8 / (WM * WN * KW), SLICES = 4 / KW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN), r = lane & 31, h = lane >> 5;

    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN, total = tiles_m * tiles_n;
    const int xcd = blockIdx.x & 7, share = total >> 3, rest = total & 7;
    const int id = (xcd < rest ? xcd * (share + 1) : rest * (share + 1) + (xcd - rest) * share) + (blockIdx.x >> 3);
    const int width = GROUP * tiles_n, first = id / width * GROUP, in = id % width, rows = min(tiles_m - first, GROUP);
    const int m0 = (first + in % rows) * BM, n0 = in / rows * BN;

    // the wave's rows in LDS: the activations' are 0 .. BM - 1, the weights' follow
    static_assert(BM / 8 % MOVES == 0 && MOVES % 2 == 0, "a wave moves rows of one operand, 16 at a time");
    const int row0 = wave * MOVES * 8;
    const bool acts = row0 < BM;
    const signed char* const from = acts ? a.q + (long long)m0 * a.ld_q : a.w + (long long)n0 * a.ld_w;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, 0x7fffffff, 0x00020000);
    const int ld = (int)(acts ? a.ld_q : a.ld_w), bottom = acts ? a.M - 1 - m0 : a.N - 1 - n0, base = acts ? row0 : row0 - BM;
    int off[MOVES];                               // this lane's row of each move, in bytes from the tile's first row
#pragma unroll
    for (int i = 0; i < MOVES; ++i) off[i] = min(base + i * 8 + (lane >> 3), bottom) * ld;
    const int piece[2] = {((lane & 7) ^ (lane >> 4)) * 16, ((lane & 7) ^ (4 + (lane >> 4))) * 16}, last = ((a.K - 1) >> 4) << 4;
    auto load = [&](int t) {
        const int k[2] = {min(t * 128 + piece[0], last), min(t * 128 + piece[1], last)};
        signed char* const to = lds + (t & (S - 1)) * TILE + row0 * 128;
#pragma unroll
        for (int i = 0; i < MOVES; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(to + i * 1024), 16, off[i] + k[i & 1], 0, 0, 0);
    };
    i32x4 fx[2][MI], fw[2][NI];
    auto read = [&](int t, int sl, int b) {       // slice sl of the wave's SLICES
        const signed char* const at = lds + (t & (S - 1)) * TILE + ((2 * (wk * SLICES + sl) + h) ^ ((lane >> 1) & 7)) * 16;
#pragma unroll
        for (int i = 0; i < NI; ++i) fw[b][i] = *reinterpret_cast<const i32x4*>(at + (BM + wn * 32 * NI + i * 32 + r) * 128);
#pragma unroll
        for (int i = 0; i < MI; ++i) fx[b][i] = *reinterpret_cast<const i32x4*>(at + (wm * 32 * MI + i * 32 + r) * 128);
    };
    i32x16 acc[NI][MI] = {};
    float sm[MI];                                 // the rows' scales: here, where the moves hide their way
#pragma unroll
    for (int j = 0; j < MI; ++j) sm[j] = a.scale[min(m0 + wm * 32 * MI + j * 32 + r, a.M - 1)];
    const int steps = (a.K + 127) >> 7;
    auto step = [&](int t, auto mode_c) {
        constexpr int MODE = decltype(mode_c)::value;
#pragma unroll
        for (int sl = 0; sl < SLICES; ++sl) {
            if (sl < SLICES - 1) {
                read(t, sl + 1, (sl + 1) & 1);
            } else if (MODE != STEP_LAST) {
                // step t + 1 has arrived, step t has been read by every wave
                if (MODE == STEP_FULL) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(MOVES * (S - 2)) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                read(t + 1, 0, 0);
                if (MODE == STEP_FULL && t + S < steps) load(t + S);
            }
            if (MODE == STEP_LAST) {
                const i32x4 mask = below(t * 128 + (wk * SLICES + sl) * 32 + h * 16, a.K);
#pragma unroll
                for (int j = 0; j < MI; ++j) fx[sl & 1][j] &= mask;
            }
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[sl & 1][i], fx[sl & 1][j], acc[i][j], 0, 0, 0);
        }
    };
    for (int t = 0; t < S && t < steps; ++t) load(t);
    if (steps >= S) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(MOVES * (S - 1)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    read(0, 0, 0);
    int t = 0;
    for (; t <= steps - S; ++t) {
        if (t == steps - 1) break;                // S = 1 step
        step(t, std::integral_constant<int, STEP_FULL>());
    }
    for (; t < steps - 1; ++t) step(t, std::integral_constant<int, STEP_DRAIN>());
    step(steps - 1, std::integral_constant<int, STEP_LAST>());

    // Element 4 e + i of an accumulator is column 8 e + 4 h + i of its 32, row r.  32 rows of the wave at a time go through
    // LDS, times their scale (its own part of it; rows 16 bytes apart from a bank's multiple), so that a row's columns leave
    // side by side.
    constexpr int PITCH = 32 * NI + 4, LANES = 8 * NI;            // words of a row; lanes that write one row of 4 columns each
    __syncthreads();
    if (KW == 2) {                                // the second half of K joins the first
        i32x4* const half = reinterpret_cast<i32x4*>(lds) + wave % (WM * WN) * (NI * MI * 256) + lane;
#pragma unroll
        for (int i = 0; i < NI * MI * 4; ++i) {
            const i32x16& v = acc[i / 4 / MI][i / 4 % MI];
            if (wk == 1) half[i * 64] = i32x4{v[4 * (i % 4)], v[4 * (i % 4) + 1], v[4 * (i % 4) + 2], v[4 * (i % 4) + 3]};
        }
        __syncthreads();
        if (wk == 1) return;                      // nothing below waits for another wave
#pragma unroll
        for (int i = 0; i < NI * MI * 4; ++i) {
            const i32x4 v = half[i * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i / 4 / MI][i / 4 % MI][4 * (i % 4) + e] += v[e];
        }
    }
    // (KW == 2: behind the halves, which other waves may still be reading)
    float* const stage = reinterpret_cast<float*>(lds + (KW == 2 ? WM * WN * NI * MI * 4096 : 0)) + wave * 32 * PITCH;
    const int n = n0 + wn * 32 * NI + lane % LANES * 4;
    const Columns4 col = columns4(a.wscale, a.bias, n, a.N);
#pragma unroll
    for (int j = 0; j < MI; ++j) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f32x4 v;
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = (float)acc[i][j][4 * e + x] * sm[j];
                *reinterpret_cast<f32x4*>(stage + r * PITCH + i * 32 + 8 * e + 4 * h) = v;
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int row = lane / LANES; row < 32; row += 64 / LANES) {
            const int m = m0 + wm * 32 * MI + j * 32 + row;
            const f32x4 scaled = *reinterpret_cast<const f32x4*>(stage + row * PITCH + lane % LANES * 4);
            finish4(a, m, n, scaled, col);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int MI, int NI, int WM, int WN, int KW, int S>
__global__ __launch_bounds__(64 * WM * WN * KW, WM * WN * KW / 4 * (MI * NI * WM * WN > 32 ? 1 : 2)) void linear_int8_tiles_kernel(const LinearInt8Args a) {
    extern __shared__ __attribute__((aligned(128))) signed char tiles[];
    linear_tile<MI, NI, WM, WN, KW, S>(a, tiles);
}

template <int MI, int NI, int WM, int WN, int KW, int S>
static int launch_linear_tiles(const LinearInt8Args& a, long long threads, hipStream_t stream) {
    constexpr int BM = 32 * MI * WM, BN = 32 * NI * WN, TILES = S * (BM + BN) * 128, STAGE = WM * WN * (32 * (32 * NI + 4) * 4 + (KW == 2 ? NI * MI * 4096 : 0));
    constexpr int LDS = TILES > STAGE ? TILES : STAGE;
    const long long tiles = (long long)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
    if (tiles * (64 * WM * WN * KW) > threads) return TOO_MANY;
    return enqueue(linear_int8_tiles_kernel<MI, NI, WM, WN, KW, S>, dim3((unsigned)tiles), 64 * WM * WN * KW, LDS, stream, a);
}

// Which kernel.  Tiles are taken from the largest size that still gives most of the 256 CUs one and is not more than twice as
// tall as there are rows (17 - 32 rows: 64 x 64 only with a long K); below 128 tiles of 64 x 64 and up to 16 rows the rows
// kernel, whose workgroups split K instead.  Few tiles with a long K get more waves and four steps of moves in flight, which
// hides the way from memory; with a short K or many tiles two steps and more workgroups a CU do better.
// Measured on an MI355X, us (graph of 20 calls on three sets of operands in turn, median; tiles of that size in brackets):
//     tile, waves, steps in LDS   for                            and by the neighbouring choice
//     256 x 256, 16, 2            2048 x 8192 x 8192  (256)  124   155 with 128 x 128;  2048 x 4096 x 4096 (128)  52 / 43
//     128 x 128,  8, 2            8192 x 1024 x 1024  (512)  19.8  24.9 with 16 waves, 4 steps; 23.1 with 256 x 256
//     128 x 128, 16, 4            1024 x 4096 x 4096  (256)  25.7  28.4 with 8 waves, 2 steps;  2048 x 4096 x 4096 (512)  52 / 43
//                                 2048 x 1152 x 2048  (144)  14.2  14.5 with 64 x 64, 4 waves;  with K = 1536  12.2 / 11.9
//                                 2048 x 1536 x 2048  (192)  14.8  15.3 with 64 x 64, 4 waves;  with K = 1024  11.7 / 10.7
//                                 short K, up to 256 tiles, goes either way: 2048 x 2048 x 1024  14.2 / 12.7, x 512  9.2 / 10.8
//     64 x 64, 8 on half of K, 4  256 x 4096 x 4096   (256)  11.7  18.9 with 4 waves, 2 steps; 24.5 with rows
//                                 777 x 1333 x 2001   (273)  11.4  11.9 with 4 waves, 2 steps; 13.2 with rows
//                                 1536 x 1024 x 2048  (384)  11.8  12.8 with 4 waves, 2 steps;  2048 x 1024 x 2048 (512)  13.9 / 13.5
//                                 2048 x 1024 x 4096  (512)  20.6  21.3 with 4 waves, 2 steps
//     64 x 64,  4, 2              2048 x 1024 x 1024  (512)   9.4  10.5 with K halved; 11.7 with 128 x 128
//                                 1280 x 1024 x 512   (320)   5.7  6.1 with K halved;  with K = 1024  8.2 / 7.9
//                                 512 x 1024 x 512    (128)   4.9  5.7 with rows;  with K = 1024 (K halved)  5.8 / 5.6
//     few rows, many columns      128 x 49152 x 1024  128 x 128  16.2, 256 x 256  23.0;  128 x 65536 x 4096  81 and 85
//                                 64 x 65536 x 4096   64 x 64  62, 128 x 128  71, 256 x 256  82;  65 x 18432 x 4096  24 and 19.5, -
//                                 32 x 18432 x 4096   64 x 64  17.9, 128 x 128  19.1, rows  24.9;  32 x 16384 x 1024  7.3, -, rows  6.8
//                                 1 x 65536 x 4096    rows  59, 64 x 64  57, 128 x 128  66, 256 x 256  72;  1 x 18432 x 4096  18.2, 16.7, 18.0, -
// Between the row kernels the number of 16 x 16 tiles decides: as many columns and rows a workgroup as leave 200 - 400
// workgroups (one set of operands, 256 x 400 x 400: 3.7 with 2 x 1 tiles, 4.0 with 1 x 1, 4.2 with 2 x 2; 512 x 1024 x 1024: 6.3 with 4 x 2, 6.9
// with 2 x 2, 8.6 with 2 x 1; 1 x 16384 x 4096: 12.8 with 1 x 4, 14.6 with 1 x 1), and K is dealt to 16 waves where it is long
// and the workgroups are few (1 x 4096 x 4096: 5.5 with 16 waves, 6.5 with 4; 1 x 1333 x 2001: 4.4 and 3.6).
static int launch_linear(const LinearInt8Args& a, long long kp, long long threads, hipStream_t stream) {
    auto tiles = [&](int side) { return (long long)((a.M + side - 1) / side) * ((a.N + side - 1) / side); };
    // the tile kernel's offsets inside 256 rows are 32-bit
    if (256 * (a.M > 1 ? a.ld_q : kp) + kp < 0x7fffffffll && 256 * (a.N > 1 ? a.ld_w : kp) + kp < 0x7fffffffll) {
        if (a.M > 128 && tiles(256) >= 192) return launch_linear_tiles<2, 2, 4, 4, 1, 2>(a, threads, stream);
        if (a.M > 64 && tiles(128) > 256) return launch_linear_tiles<2, 1, 2, 4, 1, 2>(a, threads, stream);
        if (a.M > 64 && tiles(128) >= 144 && a.K >= 2048) return launch_linear_tiles<1, 1, 4, 4, 1, 4>(a, threads, stream);
        if ((a.M > 32 && tiles(64) >= 128) || (a.M > 16 && tiles(64) >= 256 && a.K >= 2048)) {
            if (a.K >= 4096 || (a.K >= 1024 && tiles(64) <= 384)) return launch_linear_tiles<1, 1, 2, 2, 2, 4>(a, threads, stream);
            return launch_linear_tiles<1, 1, 2, 2, 1, 2>(a, threads, stream);
        }
    }
    const long long t = tiles(16);
    if (a.M <= 16) {
        if (t >= 768) return launch_linear_rows<1, 4, 4, 1>(a, threads, stream);
        if (t <= 256 && a.K >= 4096) return launch_linear_rows<1, 1, 16, 4>(a, threads, stream);
        return launch_linear_rows<1, 1, 4, 2>(a, threads, stream);
    }
    if (t <= 320) return launch_linear_rows<1, 1, 4, 2>(a, threads, stream);
    if (t <= 640) return launch_linear_rows<2, 1, 8, 2>(a, threads, stream);
    if (t <= 1536) return launch_linear_rows<2, 2, 4, 4>(a, threads, stream);
    if (a.M <= 32) return launch_linear_rows<2, 4, 4, 2>(a, threads, stream);
    return launch_linear_rows<4, 2, 8, 2>(a, threads, stream);
}

static int linear_rows_of(const LinearInt8Args& a, long long kp, long long threads, hipStream_t stream) {
    int rc = a.M > 1 << 30 ? (int)TOO_MANY : launch_linear(a, kp, threads, stream);      // row numbers past M stay 32-bit
    if (rc != TOO_MANY || a.M <= 16) return rc;
    const int whole = a.M > 512 ? 255 : 15;
    const long long done = (a.M / 2 + whole) & ~whole;
    LinearInt8Args part = a;
    part.M = (int)done;
    rc = linear_rows_of(part, kp, threads, stream);
    if (rc != 0) return rc;
    part = a;
    part.M -= (int)done, part.q += done * a.ld_q, part.scale += done;
    part.out = (char*)a.out + done * a.ld_out * (a.dtype == F_FP32 ? 4 : 2);
    return linear_rows_of(part, kp, threads, stream);
}

D4PG_API int d4pg_linear_int8_in(const LinearInt8Args* a, long long threads, hipStream_t stream) {
    if (!good_limit(threads)) return -8;
    if (a->M < 1 || a->N < 1 || a->N > 1 << 29 || a->K < 1 || a->K >= 131072) return -1;
    if (a->q == nullptr || a->w == nullptr || a->scale == nullptr || a->wscale == nullptr || a->out == nullptr) return -2;
    const long long kp = (a->K + 15) & ~15;
    if (((a->M > 1 ? a->ld_q : 16) & 15) || ((a->N > 1 ? a->ld_w : 16) & 15)) return -3;
    if ((a->M > 1 && a->ld_q < kp) || (a->N > 1 && a->ld_w < kp) || (a->M > 1 && a->ld_out < a->N)) return -4;
    if (((uintptr_t)a->q | (uintptr_t)a->w) & 15) return -5;
    if (a->dtype < F_FP32 || a->dtype > F_FP16 || a->act < ACT_NONE || a->act > ACT_TANH) return -6;
    return linear_rows_of(*a, kp, threads, stream);
}
D4PG_API int d4pg_linear_int8(const LinearInt8Args* a, hipStream_t stream) { return d4pg_linear_int8_in(a, LAUNCH_THREADS, stream); }

// ---------------------------------------------------------------------------------------------------------------
// three layers on codes in one launch
// ---------------------------------------------------------------------------------------------------------------
// Everything but the weights is local to a row, so a workgroup of 16 waves takes 16 MT rows through the whole network with
// their codes in LDS: quantise the input, then per layer the product (weights straight from L2 to registers,
// v_mfma_i32_16x16x64_i8 with the weights as the A operand: lane 16 g + c ends with columns 4 g .. 4 g + 3 of row c), the
// activation, the rows' largest magnitudes (LDS integer maxima: whatever the order, the same result) and the codes of the
// next layer.  No hidden value leaves the CU.
//
// A layer whose columns make more than 8 tiles of 16 deals them to the waves (TPW each); a narrower one deals K, the waves
// of a tile meeting in LDS integer additions.  Codes lie in LDS in rows 16 bytes apart from a multiple of 64, zero from the
// layer's width up to it: the 16 lanes of an LDS cycle cover all banks, and what the weights hold beyond K meets zeros.
constexpr int MLP_WAVES = 16;

__device__ __forceinline__ float load_any(const void* p, int dtype, long long i) {
    if (dtype == F_FP32) return load1<float>(p, i);
    if (dtype == F_BF16) return load1<__bf16>(p, i);
    return load1<_Float16>(p, i);
}

// The wave's weights, layer after layer, as one stream of slices: TPW units of 16 rows x 64 k (1 KB each), moved from
// memory into the wave's own ring in LDS (no registers, no barrier) while the slices before are multiplied, across the
// borders of layers too: weights depend on nothing.  An instruction moves 16 rows of 64 neighbouring bytes in lane order;
// read straight into the matrix operand's order, lane 16 g + c row c, the same bytes keep the address path busy four times
// as long (16 rows behind every 16 lanes).  16-byte pieces of a unit's row lie XOR (row / 4): the 16 lanes of an LDS cycle
// then cover all banks.
//
// Every slice of every layer is TPW moves for every wave, so that one count says when a slice has arrived: a wide layer's
// units are the wave's tiles at one k, a narrow layer's are one tile at TPW neighbouring k of the wave's share; what lies
// beyond the layer repeats its last row or its last bytes and is not used.
__device__ __forceinline__ void lds_barrier() {          // LDS is settled for the workgroup; moves stay on their way
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
//
// Measured (GPU time, us; the layers as launches of their own behind the /): 24-400-400-4 on one state 10.2 / 12.5, on 4096
// states 12.7 / 30, on 8192 15.5 / 41; 111-1024-1024-8 on one state 18.6 / 13.8 (whose six launches cost the host 20), on 4096 27.9 / 43, on
// 8192 35.7 / 53.  At 4096 states of the latter 256 workgroups read 1.2 MB of weights each: 300 MB at the 18 TB/s that moves
// alone reach would be 16 us.  At one state the chain of phases is what is left (clock stamps of a 400-wide network, cycles:
// descriptors 2000, input 2400, layers 1200 + 4200 + 800, results and codes 1500 - 2500 each).
struct MlpShare {                  // a wave's part of a layer: tiles tile0, tile0 + 16, ...; units of 64 k from k0, k_unit apart
    int K, N, tiles, count, tile0, k0, k_unit, slices;
    bool narrow;
};
template <int TPW>
__device__ __forceinline__ MlpShare mlp_share(const Mlp3Int8Args& a, int layer, int wave) {
    MlpShare s;
    s.K = a.width[layer], s.N = a.width[layer + 1], s.tiles = (s.N + 15) >> 4;
    s.narrow = s.tiles <= MLP_WAVES / 2;
    const int units = (s.K + 63) >> 6;
    if (s.narrow) {
        const int spread_log = s.tiles <= 1 ? 0 : (s.tiles <= 2 ? 1 : (s.tiles <= 4 ? 2 : 3)), parts = MLP_WAVES >> spread_log;
        s.tile0 = wave & ((1 << spread_log) - 1);
        s.count = s.tile0 < s.tiles ? 1 : 0;
        s.k0 = 64 * (wave >> spread_log), s.k_unit = 64 * parts;
        s.slices = (units + parts * TPW - 1) >> (4 - spread_log + (TPW == 1 ? 0 : TPW == 2 ? 1 : 2));
    } else {
        s.tile0 = wave, s.count = (s.tiles - wave + MLP_WAVES - 1) >> 4;
        s.k0 = 0, s.k_unit = 0, s.slices = units;
    }
    return s;
}
template <int TPW>
struct MlpFeed {                   // the next slice to move
    __amdgpu_buffer_rsrc_t rsrc;
    int row[TPW];                  // this lane's row of each unit, in bytes
    int layer, left, k, k_unit, k_step, last, slot;
};
template <int TPW>
__device__ __forceinline__ void mlp_open(MlpFeed<TPW>& f, const Mlp3Int8Args& a, int wave, int lane) {
    const MlpShare s = mlp_share<TPW>(a, f.layer, wave);
    f.rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)a.w[f.layer], 0, 0x7fffffff, 0x00020000);
    const int ld = (int)a.ld_w[f.layer];
#pragma unroll
    for (int j = 0; j < TPW; ++j) f.row[j] = min(16 * (s.tile0 + (s.narrow ? 0 : MLP_WAVES * j)) + (lane >> 2), s.N - 1) * ld;
    f.left = s.slices, f.k = s.k0, f.k_unit = s.k_unit, f.k_step = s.narrow ? s.k_unit * TPW : 64, f.last = ((s.K - 1) >> 4) << 4;
}
// Moves units B BATCH .. B BATCH + BATCH - 1 of the next slice.
template <int TPW, int BATCH, int SLOTS, int B>
__device__ __forceinline__ bool mlp_move(MlpFeed<TPW>& f, const Mlp3Int8Args& a, signed char* ring, int wave, int lane) {
    if (f.layer >= 3) return false;
    const int piece = 16 * ((lane & 3) ^ (lane >> 4));
    signed char* const to = ring + f.slot * (BATCH * 1024);
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(f.rsrc, (__attribute__((address_space(3))) void*)(to + i * 1024), 16,
                                                 f.row[B * BATCH + i] + min(f.k + (B * BATCH + i) * f.k_unit + piece, f.last), 0, 0, 0);
    f.slot = f.slot + 1 == SLOTS ? 0 : f.slot + 1;
    if (B == TPW / BATCH - 1) {
        f.k += f.k_step;
        if (--f.left == 0 && ++f.layer < 3) mlp_open<TPW>(f, a, wave, lane);
    }
    return true;
}

// Codes of row r, columns n .. n + 3 of one lane's values.
__device__ __forceinline__ void mlp_codes(signed char* codes, int pitch, int r, int n, const float (&v)[4], const RowCode& rc) {
    *reinterpret_cast<unsigned*>(codes + r * pitch + n) =
        pack4(code_bits(v[0], rc), code_bits(v[1], rc), code_bits(v[2], rc), code_bits(v[3], rc)) & rc.keep;
}

// LDS of a workgroup: the waves' rings, their columns (64 scales and 64 biases each), codes, sums of narrow layers, tops.
// A ring holds 8 units, 6 where 32 rows of codes need the room; it is refilled BATCH units at a time.
constexpr int mlp_ring(int mt) { return mt == 1 ? 8 : 6; }
constexpr int mlp_batch(int tpw, int mt) { return tpw == 4 && mt == 2 ? 2 : tpw; }

template <int TPW, int BATCH, int SLOTS, int I>
__device__ __forceinline__ void mlp_ahead(MlpFeed<TPW>& f, const Mlp3Int8Args& a, signed char* ring, int wave, int lane) {
    if constexpr (I < SLOTS - 1) {
        mlp_move<TPW, BATCH, SLOTS, I % (TPW / BATCH)>(f, a, ring, wave, lane);
        mlp_ahead<TPW, BATCH, SLOTS, I + 1>(f, a, ring, wave, lane);
    }
}

template <int TPW, int MT>
__device__ __forceinline__ void mlp3_rows(const Mlp3Int8Args& a, signed char* const mem) {
    constexpr int ROWS = 16 * MT, BATCH = mlp_batch(TPW, MT), NB = TPW / BATCH, SLOTS = mlp_ring(MT) / BATCH, AHEAD = SLOTS - 1;
    constexpr int RING = SLOTS * BATCH * 1024, HELD = 4;          // HELD: 64-element pieces of an input row kept in registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int m0 = blockIdx.x * ROWS, pitch = a.pitch;
    signed char* const ring = mem + wave * RING;
    float* const cols = reinterpret_cast<float*>(mem + MLP_WAVES * RING) + wave * 128;
    signed char* const codes = mem + MLP_WAVES * (RING + 512);
    int* const sums = reinterpret_cast<int*>(codes + ROWS * pitch);
    unsigned* const top = reinterpret_cast<unsigned*>(sums + a.split);       // [3][ROWS] largest magnitudes, as bits
    const int unit = wave, ut = unit / MT, ui = unit % MT;                   // this wave's share of a narrow layer's results

    // scales and biases of the columns whose values this wave will make
    auto move_columns = [&](int layer) {
        const int N = a.width[layer + 1], tiles = (N + 15) >> 4;
        const int tile = tiles <= MLP_WAVES / 2 ? ut : wave + MLP_WAVES * g, n = min(16 * tile + c, N - 1);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.wscale[layer] + n),
                                         (__attribute__((address_space(3))) void*)cols, 4, 0, 0);
        if (a.bias[layer] != nullptr)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.bias[layer] + n),
                                             (__attribute__((address_space(3))) void*)(cols + 64), 4, 0, 0);
    };
    const int S = a.width[0];
    unsigned held[MT][HELD];                     // as bits, first on their way: everything waits for the input
    auto hold = [&](auto bits) {                 // one branch for all of them: a branch each would wait for each
        using B = decltype(bits);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int p = 0; p < HELD; ++p)
                held[i][p] = reinterpret_cast<const B*>(a.x)[(long long)min(m0 + wave + MLP_WAVES * i, a.M - 1) * a.ld_x + min(lane + 64 * p, S - 1)];
    };
    if (a.xdtype == F_FP32) hold(0u);
    else hold((unsigned short)0);
    MlpFeed<TPW> feed;
    feed.layer = 0, feed.slot = 0;
    mlp_open<TPW>(feed, a, wave, lane);
    move_columns(0);
    mlp_ahead<TPW, BATCH, SLOTS, 0>(feed, a, ring, wave, lane);

    for (int i = threadIdx.x; i < a.split; i += 64 * MLP_WAVES) sums[i] = 0;
    for (int i = threadIdx.x; i < 2 * ROWS; i += 64 * MLP_WAVES) top[ROWS + i] = 0u;
    const int padded = (S + 63) & ~63;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = wave + MLP_WAVES * i;
        const long long row = (long long)min(m0 + r, a.M - 1) * a.ld_x;
        unsigned t = 0;
        float x[HELD];
#pragma unroll
        for (int p = 0; p < HELD; ++p) {
            x[p] = a.xdtype == F_FP32 ? __builtin_bit_cast(float, held[i][p])
                 : a.xdtype == F_BF16 ? __builtin_bit_cast(float, held[i][p] << 16)
                                      : (float)__builtin_bit_cast(_Float16, (unsigned short)held[i][p]);
            t = max(t, abs_bits(x[p]));          // beyond S: the last element again
        }
        for (int k = lane + 64 * HELD; k < S; k += 64) t = max(t, abs_bits(load_any(a.x, a.xdtype, row + k)));
        t = wave_umax(t);
        if (lane == 0) top[r] = t;
        const RowCode rc = row_code(t);
#pragma unroll
        for (int p = 0; p < HELD; ++p) {
            const int k = lane + 64 * p;
            if (k < padded) codes[r * pitch + k] = k < S ? (signed char)(code_bits(x[p], rc) & rc.keep) : 0;
        }
        for (int k = lane + 64 * HELD; k < padded; k += 64)
            codes[r * pitch + k] = k < S ? (signed char)(code_bits(load_any(a.x, a.xdtype, row + k), rc) & rc.keep) : 0;
    }
    lds_barrier();
    const signed char* const xp = codes + c * pitch + 16 * g;
    const int wo = c * 64 + (g ^ (c >> 2)) * 16; // this lane's piece of a unit
    int slot = 0;
    for (int layer = 0; layer < 3; ++layer) {
        const MlpShare s = mlp_share<TPW>(a, layer, wave);
        const int N = s.N;
        const bool biased = a.bias[layer] != nullptr;
        const int act = layer < 2 ? ACT_RELU : a.act;
        const unsigned* const top_in = top + layer * ROWS;
        unsigned* const top_out = top + (layer + 1) * ROWS;
        i32x4 acc[TPW][MT] = {};
        for (int sl = 0; sl < s.slices; ++sl) {
            i32x4 xf[MT];
            if (!s.narrow) {
#pragma unroll
                for (int i = 0; i < MT; ++i) xf[i] = *reinterpret_cast<const i32x4*>(xp + i * 16 * pitch + 64 * sl);
            }
            auto batch = [&](auto b_c) {
                constexpr int B = decltype(b_c)::value;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the slot that is moved into has been read
                if (mlp_move<TPW, BATCH, SLOTS, (B + AHEAD) % NB>(feed, a, ring, wave, lane)) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(BATCH * AHEAD) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                const signed char* const units = ring + slot * (BATCH * 1024) + wo;
                slot = slot + 1 == SLOTS ? 0 : slot + 1;
                if (!s.narrow) {
                    i32x4 wf[BATCH];
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) wf[j] = *reinterpret_cast<const i32x4*>(units + j * 1024);
#pragma unroll
                    for (int j = 0; j < BATCH; ++j)
#pragma unroll
                        for (int i = 0; i < MT; ++i) acc[B * BATCH + j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[B * BATCH + j][i], 0, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) {
                        const int k = s.k0 + (sl * TPW + B * BATCH + j) * s.k_unit;
                        if (k >= s.K) break;     // the same for the wave
                        const i32x4 wf = *reinterpret_cast<const i32x4*>(units + j * 1024);
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            acc[0][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, *reinterpret_cast<const i32x4*>(xp + i * 16 * pitch + k), acc[0][i], 0, 0, 0);
                    }
                }
            };
            batch(std::integral_constant<int, 0>());
            if constexpr (NB == 2) batch(std::integral_constant<int, 1>());
        }
        // The columns were moved before this layer's batches but the first AHEAD: from AHEAD batches on the waits above cover them.
        if (s.slices * NB < AHEAD) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        // Values of this wave: wide layers TPW x MT tiles; narrow ones the sums of all waves, dealt out again as units
        // (tile, 16 rows), of which a wave has at most one.
        float v[TPW][MT][4], sm[MT];
        unsigned m[MT] = {};
#pragma unroll
        for (int i = 0; i < MT; ++i) sm[i] = row_code(top_in[16 * (s.narrow ? ui : i) + c]).scale;
        auto finish = [&](float (&y)[4], const i32x4 sum, float sr, int r, int n, int col, unsigned& most) {
            Columns4 cc;
            *reinterpret_cast<f32x4*>(cc.scale) = *reinterpret_cast<const f32x4*>(cols + col);
            *reinterpret_cast<f32x4*>(cc.bias) = *reinterpret_cast<const f32x4*>(cols + 64 + col);
            values4(y, scaled4(sum, sr), cc, biased, act, a.dtype);
            if (layer == 2) {
                if (m0 + r < a.M && n < N) store_values4(a.out, (long long)(m0 + r) * a.ld_out + n, a.dtype, y, N - n);
            } else {
                // beyond the layer's width the last column again (its scale and bias, some weight row's sum): no value
                if (n + 4 > N) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = n + e < N ? y[e] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, abs_bits(y[e]));
            }
        };
        if (s.narrow) {
            if (s.count) {
                int* const sum = sums + s.tile0 * MT * 256 + lane;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) atomicAdd(sum + i * 256 + e * 64, acc[0][i][e]);
            }
            lds_barrier();
            if (ut < s.tiles) {
                int* const from = sums + unit * 256 + lane;
                i32x4 sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = from[e * 64], from[e * 64] = 0;   // zeros for the next layer that needs them
                finish(v[0][0], sum, sm[0], 16 * ui + c, 16 * ut + 4 * g, 4 * g, m[0]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < TPW; ++j)
                if (j < s.count)
#pragma unroll
                    for (int i = 0; i < MT; ++i) finish(v[j][i], acc[j][i], sm[i], 16 * i + c, 16 * (s.tile0 + MLP_WAVES * j) + 4 * g, 16 * j + 4 * g, m[i]);
        }
        if (layer == 2) break;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (s.narrow && i > 0) break;
            unsigned t = m[i];
            t = max(t, (unsigned)__shfl_xor((int)t, 16, 64));
            t = max(t, (unsigned)__shfl_xor((int)t, 32, 64));
            if (g == 0) atomicMax(top_out + 16 * (s.narrow ? ui : i) + c, t);
        }
        lds_barrier();                           // every wave has read the codes of this layer and given its largest
        move_columns(layer + 1);
        // zeros from the layer's width up to the next slice (whole tiles write their own)
        if ((N & 63) && threadIdx.x < ROWS * 4) {
            const int n = (N & ~63) + 16 * (threadIdx.x & 3);
            if (n >= 16 * s.tiles) *reinterpret_cast<i32x4*>(codes + (threadIdx.x >> 2) * pitch + n) = i32x4{0, 0, 0, 0};
        }
        if (s.narrow) {
            if (ut < s.tiles) mlp_codes(codes, pitch, 16 * ui + c, 16 * ut + 4 * g, v[0][0], row_code(top_out[16 * ui + c]));
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const RowCode rc = row_code(top_out[16 * i + c]);
#pragma unroll
                for (int j = 0; j < TPW; ++j)
                    if (j < s.count) mlp_codes(codes, pitch, 16 * i + c, 16 * (s.tile0 + MLP_WAVES * j) + 4 * g, v[j][i], rc);
            }
        }
        lds_barrier();
    }
}

template <int TPW, int MT>
__global__ __launch_bounds__(64 * MLP_WAVES) void mlp3_int8_kernel(const Mlp3Int8Args a) {
    extern __shared__ __attribute__((aligned(128))) signed char net[];
    mlp3_rows<TPW, MT>(a, net);
}

// How the one launch takes a network, from its widths and rows alone.
struct MlpPlan {
    int tpw, mt;                   // tiles of 16 columns a wave, 16-row tiles a workgroup
    int pitch, split, lds;
};
// 0, NOT_TAKEN or a refusal
static int mlp_plan(int M, const int (&width)[4], MlpPlan& p) {
    if (M < 1) return -1;
    int widest = 0, wide_out = 0, few = 0;
    for (int i = 0; i < 4; ++i) {
        if (width[i] < 1 || width[i] > 1 << 29) return -1;         // as in the product; rounded up to tiles they stay 32-bit
        if (i < 3 && width[i] > widest) widest = width[i];
        const int tiles = (width[i] + 15) / 16;
        if (i > 0 && tiles > wide_out) wide_out = tiles;
        if (i > 0 && tiles <= MLP_WAVES / 2 && tiles > few) few = tiles;
    }
    if (widest > 2048 || wide_out > 64 || M > 1 << 25) return NOT_TAKEN;       // (2^25 rows: 2^31 threads)
    p.tpw = wide_out <= 16 ? 1 : wide_out <= 32 ? 2 : 4;
    p.mt = M > 4096 ? 2 : 1;       // 32 rows a workgroup, so that one round of workgroups holds them longer
    p.pitch = ((widest + 63) & ~63) + 16;
    p.split = few * p.mt * 256;
    p.lds = MLP_WAVES * (mlp_ring(p.mt) * 1024 + 512) + 16 * p.mt * p.pitch + 4 * p.split + 3 * 16 * p.mt * 4;
    return p.lds > 160 * 1024 ? (int)NOT_TAKEN : 0;
}

template <int TPW, int MT>
static int launch_mlp3(const Mlp3Int8Args& a, int lds, hipStream_t stream) {
    return enqueue(mlp3_int8_kernel<TPW, MT>, dim3((unsigned)((a.M + 16 * MT - 1) / (16 * MT))), 64 * MLP_WAVES, lds, stream, a);
}

// NOT_TAKEN: outside this kernel's range.
D4PG_API int d4pg_mlp3_int8(Mlp3Int8Args* a, hipStream_t stream) {
    if (a->x == nullptr || a->out == nullptr || a->ld_out < a->width[3]) return -1;
    if (a->dtype < F_FP32 || a->dtype > F_FP16 || a->xdtype < F_FP32 || a->xdtype > F_FP16) return -6;
    if (a->act < ACT_NONE || a->act > ACT_TANH) return -6;
    MlpPlan p;
    const int rc = mlp_plan(a->M, a->width, p);
    if (rc != 0 && rc != NOT_TAKEN) return rc;
    for (int i = 0; i < 3; ++i) {
        const long long kp = (a->width[i] + 15) & ~15;
        if (a->w[i] == nullptr || a->wscale[i] == nullptr) return -2;
        if (((uintptr_t)a->w[i] & 15) || (a->width[i + 1] > 1 && ((a->ld_w[i] & 15) || a->ld_w[i] < kp))) return -3;
        if (a->ld_w[i] >= 1 << 20) return NOT_TAKEN;        // offsets inside a matrix are 32-bit
    }
    if (rc != 0) return rc;
    a->pitch = p.pitch, a->split = p.split;
    if (p.tpw == 1) return p.mt == 2 ? launch_mlp3<1, 2>(*a, p.lds, stream) : launch_mlp3<1, 1>(*a, p.lds, stream);
    if (p.tpw == 2) return p.mt == 2 ? launch_mlp3<2, 2>(*a, p.lds, stream) : launch_mlp3<2, 1>(*a, p.lds, stream);
    return p.mt == 2 ? launch_mlp3<4, 2>(*a, p.lds, stream) : launch_mlp3<4, 1>(*a, p.lds, stream);
}

// Launches that M rows through a network of these widths (densely stored weights) take: 1, or 6, a quantisation and a product
// a layer; < 0: refused.
D4PG_API int d4pg_mlp3_int8_launches(int M, int w0, int w1, int w2, int w3) {
    MlpPlan p;
    const int rc = mlp_plan(M, {w0, w1, w2, w3}, p);
    return rc == 0 ? 1 : rc == NOT_TAKEN ? 6 : rc;
}

D4PG_SIZEOF(Mlp3Int8Args)

D4PG_SIZEOF(QuantRowsArgs)
D4PG_SIZEOF(DequantRowsArgs)
D4PG_SIZEOF(LinearInt8Args)
