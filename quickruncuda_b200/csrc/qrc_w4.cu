// qrc_w4.cu -- weight matrices in 4 bits with one scale per group of columns
// (qrc_w4_*): quantize, pack, dequantize, and the product with a few rows of
// activations.
//
//   value[n][k] = (code[n][k] - zero[g][n]) * scale[g][n],  g = k / group
//   y[m][n]     = sum_g scale[g][n] * sum_{k in g} (code - zero) * x[m][k]  (+ bias[n])
//
// Packed layout.  A row is padded to whole blocks of 128 columns, 64 bytes
// each.  Word 4*t + j of a block (t, j < 4) holds columns 32*j + 8*t + 0..7:
// column 2*i in bits 4*i, column 2*i + 1 in bits 16 + 4*i.  A lane of the
// product's matrix instruction then reads its 16 bytes of a row with one
// load, each (word >> 4*i) & 0x000f000f is a pair of neighbouring columns,
// and the four lanes of a row share one group of 32 columns at a time.
#include "qrc_host.h"
#include "../../include/qrc_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <type_traits>

namespace {

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// What the kernels need of the two 16-bit types.  kOne | code is the value
// kBias + code: the codes are the last bits of the mantissa.
template <class T> struct Half;
template <> struct Half<__nv_bfloat16> {
    static constexpr uint32_t kOne = 0x43004300u;         // 128
    static constexpr float kMax = 3.3895313892515355e38f;
    static __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hsub2(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b));
        return reinterpret_cast<const uint32_t&>(r);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct Half<__half> {
    static constexpr uint32_t kOne = 0x64006400u;         // 1024
    static constexpr float kMax = 65504.0f;
    static __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __half2 r = __hsub2(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b));
        return reinterpret_cast<const uint32_t&>(r);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};

// Column of the first code of word `word` of a row.
__device__ __forceinline__ uint64_t word_column(uint64_t word) {
    const uint32_t i = (uint32_t)word & 15;
    return (word >> 4) * 128 + (i & 3) * 32 + (i >> 2) * 8;
}

// Bit position of code e (0..7) in its word.
__device__ __forceinline__ int code_shift(int e) { return (e >> 1) * 4 + (e & 1) * 16; }

// -- quantize --------------------------------------------------------------------

// The largest and smallest of a group leave out infinities and NaN.
__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.0f; }

// d / 15 rounded once to T.  d is exact, or nearly so, in 64 bits; the only
// way rounding twice (to float, then to T) can differ is a float that lies
// right between two values of T, and that is settled by the side d lies on.
template <class T> __device__ __forceinline__ float round_once(double d) {
    const float f = (float)d;
    const float r = Half<T>::to_float(Half<T>::round(f));
    const double miss = d - (double)f;
    if (miss == 0.0) return r;
    const float nudged = __uint_as_float(__float_as_uint(f) + (miss > 0.0 ? 1 : -1));
    return Half<T>::to_float(Half<T>::round(nudged)) == r ? r
           : fabs((double)r - d) <= fabs((double)Half<T>::to_float(Half<T>::round(nudged)) - d) ? r
           : Half<T>::to_float(Half<T>::round(nudged));
}

// One warp takes 256 columns of a row at a time, eight columns per lane, so a
// group is 4 to 32 neighbouring lanes.
template <class T>
__global__ void __launch_bounds__(256)
qrc_k_w4_quant(const T* w, uint64_t ld, uint64_t n, uint64_t k, int group, int symmetric, int vec,
               uint32_t* packed, T* scales, uint8_t* zeros) {
    wait_for_previous();
    let_next_start();
    const int lane = threadIdx.x & 31;
    const uint64_t blocks128 = (k + 127) / 128, windows = (k + 255) / 256;
    const uint64_t tasks = n * windows;
    for (uint64_t task = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += (uint64_t)gridDim.x * 8) {
        const uint64_t row = task / windows, k0 = (task - row * windows) * 256 + lane * 8;
        const T* p = w + row * ld + k0;
        T v[8];
        if (vec && k0 + 8 <= k) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
        else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k0 + i < k ? p[i] : Half<T>::round(0.0f);
        }
        float x[8], most = 0.0f, least = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = Half<T>::to_float(v[i]);
            const float f = finite_or_zero(x[i]);
            most = fmaxf(most, symmetric ? fabsf(f) : f);
            least = fminf(least, f);
        }
        for (int d = group / 16; d; d >>= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
        }
        const float s = symmetric ? Half<T>::to_float(Half<T>::round(__fdiv_rn(most, 7.0f)))
                                  : round_once<T>(((double)most - (double)least) / 15.0);
        // Quotients of two 16-bit floats keep their side of every border
        // i + 1/2 in 32 bits: they are on it or 2^-16 away at least.
        float z = symmetric ? 8.0f : 0.0f;
        if (!symmetric && s > 0.0f) z = fminf(fmaxf(rintf(__fdiv_rn(-least, s)), 0.0f), 15.0f);
        const float low = symmetric ? 1.0f : 0.0f;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float c = z;
            if (s > 0.0f && x[i] == x[i]) c = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)) + z, low), 15.0f);
            word |= (uint32_t)c << code_shift(i);
        }
        const uint64_t b = k0 >> 7;
        const uint32_t i16 = lane & 15;
        if (b < blocks128) packed[(row * blocks128 + b) * 16 + (i16 & 3) * 4 + (i16 >> 2)] = word;
        if (k0 % group == 0 && k0 < k) {
            scales[k0 / group * n + row] = Half<T>::round(s);
            if (!symmetric) zeros[k0 / group * n + row] = (uint8_t)z;
        }
    }
}

// -- pack and dequantize -----------------------------------------------------------

__global__ void __launch_bounds__(256)
qrc_k_w4_pack(const uint8_t* codes, uint64_t ld, uint64_t n, uint64_t k, uint32_t* packed) {
    wait_for_previous();
    let_next_start();
    const uint64_t words = (k + 127) / 128 * 16, total = n * words;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t row = i / words, col = word_column(i - row * words);
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (col + e < k) word |= (uint32_t)(codes[row * ld + col + e] & 15) << code_shift(e);
        packed[i] = word;
    }
}

template <class TO> __device__ __forceinline__ TO round_to(float x);
// Values beyond the type's range give its largest; NaN stays.
template <> __device__ __forceinline__ float round_to<float>(float x) {
    constexpr float m = 3.402823466e38f;
    return x > m ? m : x < -m ? -m : x;
}
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float x) {
    constexpr float m = Half<__nv_bfloat16>::kMax;
    return Half<__nv_bfloat16>::round(x > m ? m : x < -m ? -m : x);
}
template <> __device__ __forceinline__ __half round_to<__half>(float x) {
    constexpr float m = Half<__half>::kMax;
    return Half<__half>::round(x > m ? m : x < -m ? -m : x);
}

template <class T, class TO>
__global__ void __launch_bounds__(256)
qrc_k_w4_dequant(const uint32_t* packed, const T* scales, const uint8_t* zeros, uint64_t n, uint64_t k, int group,
                 TO* out, uint64_t ld, int vec) {
    wait_for_previous();
    let_next_start();
    const uint64_t words = (k + 127) / 128 * 16, total = n * words;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t row = i / words, col = word_column(i - row * words);
        if (col >= k) continue;
        const uint32_t word = packed[i];
        const uint64_t at = col / group * n + row;
        const float s = Half<T>::to_float(scales[at]);
        const float z = zeros ? (float)zeros[at] : 8.0f;
        __align__(16) TO v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = round_to<TO>(((float)((word >> code_shift(e)) & 15u) - z) * s);
        TO* q = out + row * ld + col;
        if (vec && col + 8 <= k) {
#pragma unroll
            for (int e = 0; e < (int)sizeof(v) / 16; e++) reinterpret_cast<uint4*>(q)[e] = reinterpret_cast<uint4*>(v)[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) if (col + e < k) q[e] = v[e];
        }
    }
}

// -- product -----------------------------------------------------------------------

// Activations whose rows do not start on 16 bytes, copied into rows of whole
// 128-column blocks, zero behind column k.
template <class T>
__global__ void __launch_bounds__(256)
qrc_k_w4_lay_out(const T* x, uint64_t ldx, uint64_t m, uint64_t k, T* to) {
    wait_for_previous();
    let_next_start();
    const uint64_t width = (k + 127) / 128 * 128, total = m * width;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t row = i / width, col = i - row * width;
        to[i] = col < k ? x[row * ldx + col] : Half<T>::round(0.0f);
    }
}

struct W4 {
    const uint32_t* packed;
    const void* scales;
    const uint8_t* zeros;
    uint64_t n, k;
    int group_log2;
};

constexpr int kWarps = 8;

// Eight activations from column k0 of a row, zero behind column k.
template <class T>
__device__ __forceinline__ uint4 load_x(const T* row, uint64_t k0, uint64_t k) {
    if (k0 + 8 <= k) return *reinterpret_cast<const uint4*>(row + k0);
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = k0 + i < k ? row[k0 + i] : Half<T>::round(0.0f);
    return *reinterpret_cast<const uint4*>(v);
}

// A block computes 16 rows of weights times 8 * NT rows of activations; its
// warps take the 128-column blocks in turn and add their sums in a fixed
// order.  The codes, as differences code - zero, are exact in 16 bits, and
// the matrix instruction multiplies and adds them in 32; the scale of a group
// (128 / SUB columns, or a multiple of 128 with SUB = 1) multiplies its sum.
template <class T, int NT, int SUB>
__global__ void __launch_bounds__(kWarps * 32)
qrc_k_w4_matvec(const W4 w, const T* x, uint64_t ldx, uint64_t kx, uint64_t m, const T* bias, void* y, uint64_t ldy,
                int y_float) {
    wait_for_previous();
    let_next_start();
    __shared__ float s_sum[kWarps][16][8 * NT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint64_t n0 = (uint64_t)blockIdx.x * 16, m0 = (uint64_t)blockIdx.y * 8 * NT;
    const uint64_t blocks = (w.k + 127) / 128, groups = (w.k + (1ull << w.group_log2) - 1) >> w.group_log2;
    // Rows behind the last one repeat it; their sums are not stored.
    const uint64_t ra = min(n0 + g, w.n - 1), rb = min(n0 + g + 8, w.n - 1);
    const uint4* pa = reinterpret_cast<const uint4*>(w.packed) + ra * blocks * 4 + t;
    const uint4* pb = reinterpret_cast<const uint4*>(w.packed) + rb * blocks * 4 + t;
    const T* scales = static_cast<const T*>(w.scales);
    float sum[NT][4] = {};
    for (uint64_t b = warp; b < blocks; b += kWarps) {
        const uint4 qa = pa[b * 4], qb = pb[b * 4];
        const uint32_t wa[4] = {qa.x, qa.y, qa.z, qa.w}, wb[4] = {qb.x, qb.y, qb.z, qb.w};
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
            const uint64_t group = (b * 128 + sub * (128 / SUB)) >> w.group_log2;
            if (group >= groups) break;
            const float sa = Half<T>::to_float(scales[group * w.n + ra]), sb = Half<T>::to_float(scales[group * w.n + rb]);
            const uint32_t za = Half<T>::kOne + 0x10001u * (w.zeros ? w.zeros[group * w.n + ra] : 8u);
            const uint32_t zb = Half<T>::kOne + 0x10001u * (w.zeros ? w.zeros[group * w.n + rb] : 8u);
            float part[NT][4] = {};
#pragma unroll
            for (int j = sub * 4 / SUB; j < (sub + 1) * 4 / SUB; j++) {
                uint32_t a[4], c[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    a[i] = Half<T>::sub2(((wa[j] >> (4 * i)) & 0x000f000fu) | Half<T>::kOne, za);
                    c[i] = Half<T>::sub2(((wb[j] >> (4 * i)) & 0x000f000fu) | Half<T>::kOne, zb);
                }
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const uint64_t tok = m0 + i * 8 + g;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (tok < m) v = load_x(x + tok * ldx, b * 128 + j * 32 + t * 8, kx);
                    Half<T>::mma(part[i], a[0], c[0], a[1], c[1], v.x, v.y);
                    Half<T>::mma(part[i], a[2], c[2], a[3], c[3], v.z, v.w);
                }
            }
#pragma unroll
            for (int i = 0; i < NT; i++) {
                sum[i][0] = fmaf(sa, part[i][0], sum[i][0]);
                sum[i][1] = fmaf(sa, part[i][1], sum[i][1]);
                sum[i][2] = fmaf(sb, part[i][2], sum[i][2]);
                sum[i][3] = fmaf(sb, part[i][3], sum[i][3]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) {
        s_sum[warp][g][i * 8 + 2 * t] = sum[i][0];
        s_sum[warp][g][i * 8 + 2 * t + 1] = sum[i][1];
        s_sum[warp][g + 8][i * 8 + 2 * t] = sum[i][2];
        s_sum[warp][g + 8][i * 8 + 2 * t + 1] = sum[i][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += kWarps * 32) {
        const int r = i & 15, c = i >> 4;
        const uint64_t row = n0 + r, tok = m0 + c;
        if (row >= w.n || tok >= m) continue;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < kWarps; j++) v += s_sum[j][r][c];
        if (bias) v += Half<T>::to_float(bias[row]);
        if (y_float) static_cast<float*>(y)[tok * ldy + row] = v;
        else static_cast<T*>(y)[tok * ldy + row] = Half<T>::round(v);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

constexpr uint64_t kMaxSide = 1ull << 31;     // rows or columns of a matrix, rows of activations

bool valid_w4(const qrc_w4* w) {
    if (!w || (w->type != QRC_BF16 && w->type != QRC_F16)) return false;
    if (w->group != 32 && w->group != 64 && w->group != 128 && w->group != 256) return false;
    if (w->n > kMaxSide || w->k > kMaxSide) return false;
    if (w->n && w->k && (!w->d_packed || !w->d_scales)) return false;
    return !((uintptr_t)w->d_packed & 15) && !((uintptr_t)w->d_scales & 1);
}

int log2_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 8; }

inline bool rows_aligned(const void* p, uint64_t ld, uint64_t rows, uint64_t bytes) {
    return !((uintptr_t)p & 15) && (rows <= 1 || ld * bytes % 16 == 0);
}

// Bytes that rows of `cols` elements cover from the first to the last.
inline uint64_t span(uint64_t rows, uint64_t cols, uint64_t ld, uint64_t bytes) {
    return rows && cols ? ((rows - 1) * ld + cols) * bytes : 0;
}

inline bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uint64_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

// Whether [p, p + bytes) touches the matrix's own memory.
inline bool touches(const qrc_w4& w, const void* p, uint64_t bytes) {
    const uint64_t groups = (w.k + w.group - 1) / w.group;
    return overlap(p, bytes, w.d_packed, qrc_w4_words(w.n, w.k) * 4) || overlap(p, bytes, w.d_scales, groups * w.n * 2) ||
           overlap(p, bytes, w.d_zeros, groups * w.n);
}

dim3 grid_for(uint64_t items, uint64_t per_block) {
    return dim3((unsigned)std::min<uint64_t>((items + per_block - 1) / per_block, 1u << 16));
}

template <class T>
cudaError_t launch_matvec(const qrc_w4& w, const T* x, uint64_t ldx, uint64_t kx, uint64_t m, const T* bias, void* y,
                          uint64_t ldy, int y_float, cudaStream_t s) {
    const W4 a = {w.d_packed, w.d_scales, w.d_zeros, w.n, w.k, log2_of(w.group)};
    const int nt = m <= 8 ? 1 : m <= 16 ? 2 : 4;
    auto go = [&](auto kernel) {
        // grid.y has room for 65,535 slices of activations per launch
        for (uint64_t m0 = 0; m0 < m; m0 += 65535ull * 8 * nt) {
            const uint64_t rows = std::min<uint64_t>(m - m0, 65535ull * 8 * nt);
            void* to = static_cast<char*>(y) + m0 * ldy * (y_float ? 4 : 2);
            const cudaError_t e = launch_overlapped(
                kernel, dim3((unsigned)((w.n + 15) / 16), (unsigned)((rows + 8 * nt - 1) / (8 * nt))), kWarps * 32, 0, s,
                1, a, x + m0 * ldx, ldx, kx, rows, bias, to, ldy, y_float);
            if (e != cudaSuccess) return e;
        }
        return cudaSuccess;
    };
    auto by_sub = [&](auto n) {
        constexpr int NT = decltype(n)::value;
        switch (w.group) {
            case 32: return go(qrc_k_w4_matvec<T, NT, 4>);
            case 64: return go(qrc_k_w4_matvec<T, NT, 2>);
            default: return go(qrc_k_w4_matvec<T, NT, 1>);
        }
    };
    switch (nt) {
        case 1: return by_sub(std::integral_constant<int, 1>());
        case 2: return by_sub(std::integral_constant<int, 2>());
        default: return by_sub(std::integral_constant<int, 4>());
    }
}

template <class T>
cudaError_t lay_out_and_multiply(const qrc_w4& w, const void* d_x, uint64_t m, uint64_t ldx, const void* d_bias,
                                 void* d_y, uint64_t ldy, int y_float, void* d_work, cudaStream_t s) {
    const T* x = static_cast<const T*>(d_x);
    uint64_t kx = w.k;
    if (d_work) {
        const uint64_t width = (w.k + 127) / 128 * 128;
        const cudaError_t e = launch_overlapped(qrc_k_w4_lay_out<T>, grid_for(m * width, 256), 256, 0, s, 1, x, ldx, m,
                                                w.k, static_cast<T*>(d_work));
        if (e != cudaSuccess) return e;
        x = static_cast<const T*>(d_work);
        ldx = kx = width;
    }
    return launch_matvec<T>(w, x, ldx, kx, m, static_cast<const T*>(d_bias), d_y, ldy, y_float, s);
}

template <class T>
cudaError_t launch_dequant(const qrc_w4& w, void* out, uint64_t ld, int type, cudaStream_t s) {
    const uint64_t words = w.n * ((w.k + 127) / 128 * 16);
    const int vec = rows_aligned(out, ld, w.n, type == QRC_F32 ? 4 : 2);
    const T* scales = static_cast<const T*>(w.d_scales);
    auto go = [&](auto* to) {
        using TO = std::remove_pointer_t<decltype(to)>;
        return launch_overlapped(qrc_k_w4_dequant<T, TO>, grid_for(words, 256), 256, 0, s, 1,
                                 (const uint32_t*)w.d_packed, scales, (const uint8_t*)w.d_zeros, w.n, w.k, w.group, to,
                                 ld, vec);
    };
    switch (type) {
        case QRC_F32: return go(static_cast<float*>(out));
        case QRC_BF16: return go(static_cast<__nv_bfloat16*>(out));
        default: return go(static_cast<__half*>(out));
    }
}

template <class T>
cudaError_t launch_quant(const qrc_w4& w, const void* d_w, uint64_t ld, int symmetric, cudaStream_t s) {
    const int vec = rows_aligned(d_w, ld, w.n, 2);
    return launch_overlapped(qrc_k_w4_quant<T>, grid_for(w.n * ((w.k + 255) / 256), 8), 256, 0, s, 1,
                             static_cast<const T*>(d_w), ld, w.n, w.k, w.group, symmetric, vec, w.d_packed,
                             static_cast<T*>(w.d_scales), w.d_zeros);
}

}  // namespace

QRC_API uint64_t qrc_w4_words(uint64_t n, uint64_t k) { return n * ((k + 127) / 128 * 16); }

QRC_API int qrc_w4_quant(int device, const void* d_w, uint64_t ld, int symmetric, const qrc_w4* w, void* stream) {
    if (!valid_w4(w) || (w->n > 1 && ld < w->k)) return QRC_ERR_INVALID;
    if (symmetric ? w->d_zeros != nullptr : (w->n && w->k && !w->d_zeros)) return QRC_ERR_INVALID;
    if ((w->n && w->k && !d_w) || ((uintptr_t)d_w & 1)) return QRC_ERR_INVALID;
    if (touches(*w, d_w, span(w->n, w->k, ld, 2))) return QRC_ERR_INVALID;
    if (!sm100_sms(device)) return QRC_ERR_DEVICE;
    if (!w->n || !w->k) return QRC_OK;
    DeviceScope scope(device);
    if (!scope.ok) return QRC_ERR_DEVICE;
    cudaStream_t s = as_stream(stream);
    QRC_CK(w->type == QRC_BF16 ? launch_quant<__nv_bfloat16>(*w, d_w, ld, symmetric, s)
                               : launch_quant<__half>(*w, d_w, ld, symmetric, s));
    return QRC_OK;
}

QRC_API int qrc_w4_pack(int device, const uint8_t* d_codes, uint64_t ld, const qrc_w4* w, void* stream) {
    if (!valid_w4(w) || (w->n > 1 && ld < w->k) || (w->n && w->k && !d_codes)) return QRC_ERR_INVALID;
    if (!sm100_sms(device)) return QRC_ERR_DEVICE;
    if (!w->n || !w->k) return QRC_OK;
    DeviceScope scope(device);
    if (!scope.ok) return QRC_ERR_DEVICE;
    QRC_CK(launch_overlapped(qrc_k_w4_pack, grid_for(qrc_w4_words(w->n, w->k), 256), 256, 0, as_stream(stream), 1,
                             d_codes, ld, w->n, w->k, w->d_packed));
    return QRC_OK;
}

QRC_API int qrc_w4_dequant(int device, const qrc_w4* w, void* d_out, uint64_t ld, int out_type, void* stream) {
    if (!valid_w4(w) || (w->n > 1 && ld < w->k) || (w->n && w->k && !d_out)) return QRC_ERR_INVALID;
    if (out_type != QRC_F32 && out_type != QRC_BF16 && out_type != QRC_F16) return QRC_ERR_INVALID;
    if ((uintptr_t)d_out & (out_type == QRC_F32 ? 3 : 1)) return QRC_ERR_INVALID;
    if (touches(*w, d_out, span(w->n, w->k, ld, out_type == QRC_F32 ? 4 : 2))) return QRC_ERR_INVALID;
    if (!sm100_sms(device)) return QRC_ERR_DEVICE;
    if (!w->n || !w->k) return QRC_OK;
    DeviceScope scope(device);
    if (!scope.ok) return QRC_ERR_DEVICE;
    cudaStream_t s = as_stream(stream);
    QRC_CK(w->type == QRC_BF16 ? launch_dequant<__nv_bfloat16>(*w, d_out, ld, out_type, s)
                               : launch_dequant<__half>(*w, d_out, ld, out_type, s));
    return QRC_OK;
}

QRC_API size_t qrc_w4_matvec_workspace(const qrc_w4* w, const void* d_x, uint64_t m, uint64_t ldx) {
    if (!valid_w4(w) || m > kMaxSide || !m || !w->n || !w->k || rows_aligned(d_x, ldx, m, 2)) return 0;
    return m * ((w->k + 127) / 128 * 128) * 2;
}

QRC_API int qrc_w4_matvec(int device, const qrc_w4* w, const void* d_x, uint64_t m, uint64_t ldx, const void* d_bias,
                          void* d_y, uint64_t ldy, int y_type, void* d_work, void* stream) {
    if (!valid_w4(w) || m > kMaxSide || (m > 1 && (ldx < w->k || ldy < w->n))) return QRC_ERR_INVALID;
    if (y_type != QRC_F32 && y_type != w->type) return QRC_ERR_INVALID;
    if (((uintptr_t)d_x & 1) || ((uintptr_t)d_bias & 1) || ((uintptr_t)d_y & (y_type == QRC_F32 ? 3 : 1)))
        return QRC_ERR_INVALID;
    if (m && w->n && (!d_y || (w->k && !d_x))) return QRC_ERR_INVALID;
    const uint64_t y_bytes = span(m, w->n, ldy, y_type == QRC_F32 ? 4 : 2);
    if (touches(*w, d_y, y_bytes) || overlap(d_y, y_bytes, d_x, span(m, w->k, ldx, 2)) ||
        overlap(d_y, y_bytes, d_bias, w->n * 2)) return QRC_ERR_INVALID;
    const size_t need = qrc_w4_matvec_workspace(w, d_x, m, ldx);
    if (need && (!d_work || ((uintptr_t)d_work & 15))) return QRC_ERR_INVALID;
    if (!sm100_sms(device)) return QRC_ERR_DEVICE;
    if (!m || !w->n) return QRC_OK;
    DeviceScope scope(device);
    if (!scope.ok) return QRC_ERR_DEVICE;
    cudaStream_t s = as_stream(stream);
    void* work = need ? d_work : nullptr;
    const int y_float = y_type == QRC_F32;
    QRC_CK(w->type == QRC_BF16
               ? lay_out_and_multiply<__nv_bfloat16>(*w, d_x, m, ldx, d_bias, d_y, ldy, y_float, work, s)
               : lay_out_and_multiply<__half>(*w, d_x, m, ldx, d_bias, d_y, ldy, y_float, work, s));
    return QRC_OK;
}
