// Root-mean-square norm of a residual sum, as int8 rows with scales (gfx950): what the
// W8A8 product reads after a sublayer.
//
//   h = x + residual (fp32, one rounding; stored as the new residual stream)
//   y = h * weight / sqrt(mean(h^2) + eps)
//   scale = float(max|y| / 127) (1 where that is 0), code = rint(y / scale), ties to even
//
// y is never rounded: between h and the code every step is in 64 bits (the product of two
// floats is exact there). The sum of squares takes at most width / 1024 + 46 additions one
// after another, which the root halves, and six steps follow it, so the quotient that is rounded
// to a code is off by less than 127 (width / 2048 + 32) 2^-53: 6e-13 up to 16384 values a row.
// Only within that of a half does a code differ from the formula's, and, as rarely, where
// max|y| / 127 lies that close to the middle of two floats: the scale is the other one then, and
// the quotients are off by up to 127 2^-23. In 32 bits about one value in 1e5 came out a code away.
//
// Streams are bound by memory: 4 B read for x and for the residual, 4 B written for the sum, 1 B
// for the code. A row stays in registers between the two passes over it (its statistics, its
// codes), so it is read once. 8192 x 8192 with its residual (872 MB): 152 us, 5.7 TB/s, where a
// copy of 1 GiB runs at 5.1; a row leaves some 400 cycles a SIMD for every 64 values there, and the
// 64-bit steps take about 150. What fits the last-level cache is bound by issuing them: 1021 x 5003
// without a residual (25.5 MB) takes 12.7 us, 2.0 TB/s, as the eight groups of a lane are worked
// through for every width from 4097 to 8192, whether they hold values or not.
#include <cmath>

#include "reef_common.hpp"

namespace reef {
namespace {

// Rows start anywhere: 16-byte loads on 4-byte boundaries, 4-byte stores on any.
typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));

struct NormArgs {
    const float *x, *residual, *weight;  // residual, weight: may be null
    float *sum;                          // may be null; may be x or residual
    int64_t x_stride, r_stride, s_stride;
    int8_t *q;
    float *scales;
    int64_t rows;
    int32_t width;
    double eps;
    uint32_t *status;
};

template <bool NT>
__device__ __forceinline__ f32x4 load4(const float *row, int col, int width) {
    if (col + 3 < width) {
        const f32x4_at4 *p = reinterpret_cast<const f32x4_at4 *>(row + col);
        return NT ? __builtin_nontemporal_load(p) : *p;
    }
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (col + i < width) v[i] = row[col + i];
    return v;
}

template <bool NT>
__device__ __forceinline__ void store4(float *row, int col, int width, f32x4 v) {
    if (col + 3 < width) {
        f32x4_at4 *p = reinterpret_cast<f32x4_at4 *>(row + col);
        if (NT) __builtin_nontemporal_store((f32x4_at4)v, p);
        else *p = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (col + i < width) row[col + i] = v[i];
}

// A row's statistics: sum of h^2, largest |h * weight|, and whether anything is not finite.
struct RowStats {
    double squares = 0.0, top = 0.0;
    bool bad = false;

    __device__ __forceinline__ void add(f32x4 h, f32x4 w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double d = h[i], t = __builtin_fabs(d * (double)w[i]);
            squares = __builtin_fma(d, d, squares);
            top = t > top ? t : top;
            bad |= !(t < (double)INFINITY);  // an infinity or a NaN of either factor
        }
    }
    __device__ __forceinline__ void wave_reduce() {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            squares += __shfl_xor(squares, o);
            const double t = __shfl_xor(top, o);
            top = t > top ? t : top;
        }
        bad = __any(bad);
    }
};

// The factor from h * weight to the (unrounded) code, and the row's scale.
__device__ __forceinline__ double row_factor(const NormArgs &a, double squares, double top,
                                             float &scale, uint32_t &flags) {
    if (!(top > 0.0)) {  // every y is 0 (also where eps is 0 and the length with it)
        scale = 1.0f;
        return 0.0;
    }
    const double r = 1.0 / __builtin_sqrt(squares / a.width + a.eps);
    scale = (float)(top * r / 127.0);
    if (scale == 0.0f) scale = 1.0f;
    if (__builtin_isinf(scale)) flags |= REEF_STATUS_BIT_OVERFLOW;
    return r / (double)scale;
}

__device__ __forceinline__ void store_codes(int8_t *row, int col, int width, f32x4 h, f32x4 w,
                                            double factor) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        double y = __builtin_rint((double)h[i] * (double)w[i] * factor);
        // (a scale rounded down leaves the largest at 127.00001: its code is 127)
        y = y < -127.0 ? -127.0 : (y > 127.0 ? 127.0 : y);
        c[i] = (uint32_t)(int32_t)y & 0xffu;
    }
    if (col + 3 < width) {
        *reinterpret_cast<u32_at1 *>(row + col) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (col + i < width) row[col + i] = (int8_t)c[i];
}

// Rows of at most 256 WPR F4 values: WPR waves a row, F4 groups of four values a lane.
template <int WPR, int F4, bool NT>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void norm_rows(NormArgs a) {
    constexpr int ROWS = WPR >= 4 ? 1 : 4 / WPR;  // rows of a workgroup
    __shared__ double sSquares[WPR], sTop[WPR];
    __shared__ uint32_t sBad[WPR];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = linear_block() * ROWS + wave / WPR;
    const int part = wave % WPR;
    if (row >= a.rows) return;  // (all of a workgroup's waves, or waves that meet no barrier)
    const float *x = a.x + row * a.x_stride;
    f32x4 h[F4], w[F4];
    int col[F4];
#pragma unroll
    for (int i = 0; i < F4; ++i) {
        col[i] = 4 * (64 * (WPR * i + part) + lane);
        h[i] = load4<NT>(x, col[i], a.width);
    }
    if (a.residual) {
        const float *r = a.residual + row * a.r_stride;
        f32x4 v[F4];
#pragma unroll
        for (int i = 0; i < F4; ++i) v[i] = load4<NT>(r, col[i], a.width);
#pragma unroll
        for (int i = 0; i < F4; ++i) h[i] = h[i] + v[i];
    }
#pragma unroll
    for (int i = 0; i < F4; ++i)
        w[i] = a.weight ? load4<false>(a.weight, col[i], a.width) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
    RowStats s;
#pragma unroll
    for (int i = 0; i < F4; ++i) s.add(h[i], w[i]);
    if (a.sum) {
        float *o = a.sum + row * a.s_stride;
#pragma unroll
        for (int i = 0; i < F4; ++i) store4<NT>(o, col[i], a.width, h[i]);
    }
    s.wave_reduce();
    if (WPR > 1) {
        if (lane == 0) {
            sSquares[part] = s.squares;
            sTop[part] = s.top;
            sBad[part] = s.bad;
        }
        __syncthreads();
        s.squares = 0.0;
        s.top = 0.0;
        s.bad = false;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            s.squares += sSquares[i];
            s.top = sTop[i] > s.top ? sTop[i] : s.top;
            s.bad |= sBad[i] != 0;
        }
    }
    float scale;
    uint32_t flags = s.bad ? REEF_STATUS_BIT_NON_FINITE : 0;
    const double factor = row_factor(a, s.squares, s.top, scale, flags);
    if (part == 0 && lane == 0) {
        a.scales[row] = scale;
        if (flags) flag_status(a.status, flags);
    }
    int8_t *q = a.q + row * a.width;
#pragma unroll
    for (int i = 0; i < F4; ++i) store_codes(q, col[i], a.width, h[i], w[i], factor);
}

// Longer rows: a workgroup walks the row twice, the second time from the sum it stored (or
// adding x and the residual again where none is kept).
__global__ __launch_bounds__(1024) void norm_long_rows(NormArgs a) {
    constexpr int W = 16;
    __shared__ double sSquares[W], sTop[W];
    __shared__ uint32_t sBad[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = linear_block();
    if (row >= a.rows) return;
    const float *x = a.x + row * a.x_stride;
    const float *r = a.residual ? a.residual + row * a.r_stride : nullptr;
    float *o = a.sum ? a.sum + row * a.s_stride : nullptr;
    const f32x4 one = {1.0f, 1.0f, 1.0f, 1.0f};
    RowStats s;
    for (int64_t c = 4 * (int)threadIdx.x; c < a.width; c += 4096) {
        f32x4 h = load4<false>(x, (int)c, a.width);
        if (r) h = h + load4<false>(r, (int)c, a.width);
        s.add(h, a.weight ? load4<false>(a.weight, (int)c, a.width) : one);
        if (o) store4<false>(o, (int)c, a.width, h);
    }
    s.wave_reduce();
    if (lane == 0) {
        sSquares[wave] = s.squares;
        sTop[wave] = s.top;
        sBad[wave] = s.bad;
    }
    __syncthreads();
    s.squares = 0.0;
    s.top = 0.0;
    s.bad = false;
    for (int i = 0; i < W; ++i) {
        s.squares += sSquares[i];
        s.top = sTop[i] > s.top ? sTop[i] : s.top;
        s.bad |= sBad[i] != 0;
    }
    float scale;
    uint32_t flags = s.bad ? REEF_STATUS_BIT_NON_FINITE : 0;
    const double factor = row_factor(a, s.squares, s.top, scale, flags);
    if (threadIdx.x == 0) {
        a.scales[row] = scale;
        if (flags) flag_status(a.status, flags);
    }
    int8_t *q = a.q + row * a.width;
    for (int64_t c = 4 * (int)threadIdx.x; c < a.width; c += 4096) {
        // (each thread reads the groups that it stored)
        f32x4 h = load4<false>(o ? o : x, (int)c, a.width);
        if (r && !o) h = h + load4<false>(r, (int)c, a.width);
        store_codes(q, (int)c, a.width, h, a.weight ? load4<false>(a.weight, (int)c, a.width) : one,
                    factor);
    }
}

template <int WPR, int F4>
void launch_rows(const NormArgs &a, bool nt, hipStream_t stream) {
    const dim3 grid = linear_grid(WPR >= 4 ? a.rows : ceil_div(a.rows, 4 / WPR));
    const dim3 block(WPR > 4 ? 64 * WPR : 256);
    if (nt) hipLaunchKernelGGL((norm_rows<WPR, F4, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((norm_rows<WPR, F4, false>), grid, block, 0, stream, a);
}

}  // namespace
}  // namespace reef

using namespace reef;

extern "C" reef_status reef_rmsnorm_quantize_int8(const float *x, int64_t rows, int64_t width,
                                                  int64_t x_row_stride, const float *residual,
                                                  int64_t residual_row_stride, const float *weight,
                                                  double eps, int8_t *q, float *scales, float *sum,
                                                  int64_t sum_row_stride, uint32_t *status_word,
                                                  hipStream_t stream) {
    if (!x || !q || !scales || rows <= 0 || width <= 0 || x_row_stride < width ||
        (residual && residual_row_stride < width) || (sum && (sum_row_stride < width || !residual)) ||
        !std::isfinite(eps) || eps < 0.0 || !aligned(x, 4) || !aligned(residual, 4) ||
        !aligned(weight, 4) || !aligned(sum, 4) || !aligned(scales, 4))
        return REEF_INVALID_ARGUMENT;
    if (rows >= (int64_t(1) << 31) || width >= (int64_t(1) << 30)) return REEF_UNSUPPORTED;
    NormArgs a;
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.sum = sum;
    a.x_stride = x_row_stride;
    a.r_stride = residual_row_stride;
    a.s_stride = sum_row_stride;
    a.q = q;
    a.scales = scales;
    a.rows = rows;
    a.width = (int32_t)width;
    a.eps = eps;
    a.status = status_word;
    // Streams beyond the 256 MB last-level cache pass it by: nothing of them is found in it
    // again (8192 x 8192 with its residual: 152 us against 175, 5.7 TB/s).
    const bool nt = rows * width * (residual ? (sum ? 13 : 9) : 5) > (int64_t(256) << 20);
    // With many rows a wave takes rows of up to 2048 values alone: no barrier, and the lanes'
    // loads in flight fill the memory (65536 x 1024: 147 us against 182 with four waves a row,
    // 4096 x 2048 21.3 against 25.0). With few, four waves share a row's latency (512 x 1024:
    // 4.7 against 5.3, 16 x 2048: 4.4 against 6.5); at 2048 rows of 2048 both take 14.6.
    // A lane holds as few groups as cover the row (4096 rows of 256 values: 5.0 us with one, 5.5
    // with two, 10.5 with four waves a row; of 512: 6.6 with two, 8.0 with four, 11.0 with four
    // waves; of 1024 in four waves: 15.0 with one, 17.0 with two). Four waves or eight, for 512 and
    // for 4096 rows: of 4096 values 7.0 or 7.3 and 37.5 or 38.6 us, of 8192 12.9 or 12.6 and 77.6 or
    // 77.0. Eight, sixteen, or the walk of longer rows: of 16384 22.2, 23.7, 24.4 and 146, 151, 179.
    const bool many = rows >= 2048;
    if (width <= 256) launch_rows<1, 1>(a, nt, stream);
    else if (width <= 512) launch_rows<1, 2>(a, nt, stream);
    else if (width <= 1024 && many) launch_rows<1, 4>(a, nt, stream);
    else if (width <= 1024) launch_rows<4, 1>(a, nt, stream);
    else if (width <= 2048 && many) launch_rows<1, 8>(a, nt, stream);
    else if (width <= 2048) launch_rows<4, 2>(a, nt, stream);
    else if (width <= 4096) launch_rows<4, 4>(a, nt, stream);
    else if (width <= 8192) launch_rows<4, 8>(a, nt, stream);
    else if (width <= 16384) launch_rows<8, 8>(a, nt, stream);
    else hipLaunchKernelGGL(norm_long_rows, linear_grid(rows), dim3(1024), 0, stream, a);
    return launch_status();
}
