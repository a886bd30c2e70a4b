/* Row by row work of a decoder layer: rows into 8 bits (with a SwiGLU's gate),
 * the root-mean-square norm, rotary positions.  All three are one pass over
 * memory: a few operations to an element, bound by bytes where there are many
 * rows and by the latency of one load, one reduction and one store where there
 * are few. */
#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

constexpr auto up = layer_up;

/* ---- rows into 8 bits ------------------------------------------------------ */

/* x * g / (1 + e^-g) for g below kFarGate, where e^-g is all of the divisor: e^g leaves fp32's range long before the product
 * does, so its power of two is applied in two halves.  Nothing is left below -256 for any x. */
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ float times_far_silu(float x, float g)
{
    if (g == -INFINITY) return g - g;                        /* -infinity / infinity */
    int n;
    const float a = fminf(-g, 256.0f), part = exp_fraction(a, n);
    return ldexpf(x * ldexpf(-a * part, n / 2), n - n / 2);
}

/* A thread takes eight neighbours, 16 lanes a block.  A row has `parts`
 * workgroups of 256 threads.  Bound by bytes: SwiGLU of 4096 bf16 rows of 17408 moves 357
 * MB in 61 us, 5.8 TB/s; 48 rows 3 us, a launch's latency. */
template <typename T, bool kGate, bool kWhole>
__global__ void __launch_bounds__(256) quantize_kernel(QuantizeRows a, uint32_t parts)
{
    const uint32_t row = blockIdx.x / parts, part = blockIdx.x - row * parts;
    const uint32_t chunk = part * 256 + threadIdx.x, at = chunk * 8;
    const uint32_t some = at < a.width ? min(8u, a.width - at) : 0;
    const T *x = static_cast<const T *>(a.x) + row * a.x_row + at;
    float v[8] = {};
    if (some) {
        layer_load8<T, kWhole>(v, x, some);
        if constexpr (kGate) {
            float g[8];
            layer_load8<T, kWhole>(g, static_cast<const T *>(a.gate) + row * a.gate_row + at, some);
            float least = g[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) least = fminf(least, g[i]);
            if (least < kFarGate) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = g[i] < kFarGate ? times_far_silu(v[i], g[i]) : v[i] * (g[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-g[i])));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= g[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-g[i]));
            }
            if constexpr (!kWhole) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (uint32_t)i < some ? v[i] : 0.0f;
            }
        }
    }
    layer_u32x2 codes;
    const uint32_t byte = e4m3_encode8(codes, v);
    if (!some) return;
    e4m3_store8<kWhole>(a.codes + (uint64_t)row * a.width + at, codes, some);
    if (chunk % 16 == 0) e4m3_store_scale(a.scales + (uint64_t)row * a.pitch, chunk / 16, byte, up(a.width, kE4M3Block), a.pitch);
}

/* ---- root-mean-square norm ------------------------------------------------- */

template <typename T>
__device__ __forceinline__ float rounded(float v)
{
    return static_cast<float>(static_cast<T>(v));
}

/* A workgroup takes a row, a thread eight neighbours of every THREADS * 8.
 * With N > 0 the row (up to N * THREADS * 8 elements) stays in registers
 * between its sum and its result; with N = 0 it is read again.  The squares
 * are summed in fp64: no square leaves its range, and what that costs is hidden
 * behind the loads.  Bound by bytes: 4096 bf16 rows of 5120 with an addend, into 8 bits, move 147 MB
 * in 30 us, 4.9 TB/s; one row takes 3.6 us: a load, a sum over the workgroup, a store. */
template <typename T, int THREADS, int N, bool kWhole>
__global__ void __launch_bounds__(THREADS) norm_kernel(NormRows a)
{
    __shared__ double partial[THREADS / 64];
    const uint64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_row;
    const T *addend = static_cast<const T *>(a.addend) + row * a.addend_row;
    T *total = static_cast<T *>(a.total) + row * a.total_row;
    float kept[N ? N : 1][8];
    double sum = 0.0;
    const auto take = [&](float v[8], uint32_t at, uint32_t some) {
        layer_load8<T, kWhole>(v, x + at, some);
        if (a.addend) {
            float add[8];
            layer_load8<T, kWhole>(add, addend + at, some);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = rounded<T>(v[i] + add[i]);
        }
    };
    const auto squares = [&](const float v[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fma((double)v[i], (double)v[i], sum);
    };
    if constexpr (N > 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t at = (n * THREADS + threadIdx.x) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) kept[n][i] = 0.0f;
            if (at < a.width) take(kept[n], at, min(8u, a.width - at));
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t at = (n * THREADS + threadIdx.x) * 8;
            if (a.addend && at < a.width) layer_store8<T, kWhole>(total + at, kept[n], min(8u, a.width - at));
            squares(kept[n]);
        }
    } else {
        for (uint32_t at = threadIdx.x * 8; at < a.width; at += THREADS * 8) {
            const uint32_t some = min(8u, a.width - at);
            float v[8];
            take(v, at, some);
            if (a.addend) layer_store8<T, kWhole>(total + at, v, some);
            squares(v);
        }
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) sum += partial[w];
    /* in two factors: the inverse of a row near the ends of fp32's range is outside of it, or subnormal */
    int power;
    const float inverse = (float)frexp(1.0 / sqrt(sum / (double)a.width + (double)a.eps), &power);

    const auto finish = [&](float v[8], uint32_t at) {
        const uint32_t some = at < a.width ? min(8u, a.width - at) : 0;
        if (some) {
            float w[8];
            /* `whole` speaks for the weight too: the launcher looked */
            if (a.weight_type == kLayerF32)
                layer_load8<float, kWhole>(w, static_cast<const float *>(a.weight) + at, some);
            else if (a.weight_type == kLayerF16)
                layer_load8<_Float16, kWhole>(w, static_cast<const _Float16 *>(a.weight) + at, some);
            else
                layer_load8<__bf16, kWhole>(w, static_cast<const __bf16 *>(a.weight) + at, some);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (uint32_t)i < some ? ldexpf(v[i], power) * inverse * (w[i] + a.offset) : 0.0f;
            if (a.output) layer_store8<T, kWhole>(static_cast<T *>(a.output) + row * a.output_row + at, v, some);
        }
        if (a.codes) {
            layer_u32x2 codes;
            const uint32_t byte = e4m3_encode8(codes, v);
            if (some) {
                e4m3_store8<kWhole>(a.codes + row * a.width + at, codes, some);
                if (at % kE4M3Block == 0)
                    e4m3_store_scale(a.scales + row * a.pitch, at / kE4M3Block, byte, up(a.width, kE4M3Block), a.pitch);
            }
        }
    };
    if constexpr (N > 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) finish(kept[n], (n * THREADS + threadIdx.x) * 8);
    } else {
        /* whole rounds of the workgroup: the lanes of a block stay together */
        for (uint32_t at = threadIdx.x * 8; at < up(a.width, THREADS * 8) * (THREADS * 8); at += THREADS * 8) {
            const uint32_t some = at < a.width ? min(8u, a.width - at) : 0;
            float v[8] = {};
            if (some && a.addend)
                layer_load8<T, kWhole>(v, total + at, some);
            else if (some)
                layer_load8<T, kWhole>(v, x + at, some);
            finish(v, at);
        }
    }
}

/* ---- rotary positions ------------------------------------------------------ */

/* A workgroup takes a row, `parts` of them share one, or it takes `group` short rows.  Their angles are
 * formed once, in fp64, reduced to a turn and their sines and cosines, times the magnitude, rounded to fp32 and kept in
 * LDS for all heads (all of it in fp64: 12.2 us instead of 10.5 for 60000 rows of one head of 80, else no time); a thread then
 * takes eight pairs (or eight channels that are copied) of a head at a time.  Bound by bytes:
 * 8192 bf16 rows of 40 heads of 128 move 168 MB in 33 us, 5.1 TB/s; few rows by the latency of their
 * angles (16 rows 2.7 us). */
template <typename T, bool kInterleaved, bool kWhole, bool kGroup>
__global__ void __launch_bounds__(256) rotary_kernel(Rotary a, uint32_t parts, uint32_t group, uint32_t items, uint32_t turned_items, uint32_t pass_items)
{
    __shared__ float cosine[512], sine[512];
    const uint32_t part = blockIdx.x % parts, row0 = blockIdx.x / parts * group, rows = kGroup ? min(group, a.rows - row0) : 1;
    for (uint32_t i = threadIdx.x; i < rows * a.pairs; i += blockDim.x) {
        const uint32_t r = kGroup ? i / a.pairs : 0;
        const double turns = (double)a.positions[row0 + r] * (double)a.frequencies[i - r * a.pairs] * 0.15915494309189533577;
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        sine[i] = (float)(s * (double)a.magnitude);
        cosine[i] = (float)(c * (double)a.magnitude);
    }
    __syncthreads();
    const uint32_t per_head = turned_items + pass_items;
    for (uint32_t i = part * blockDim.x + threadIdx.x; i < rows * items; i += parts * blockDim.x) {
        const uint32_t r = kGroup ? i / items : 0, item = i - r * items, angles = r * a.pairs;
        const uint32_t head = item / per_head, place = item - head * per_head;
        const T *from = static_cast<const T *>(a.x) + (uint64_t)(row0 + r) * a.x_row + head * a.x_head;
        T *to = static_cast<T *>(a.output) + (uint64_t)(row0 + r) * a.output_row + head * a.output_head;
        if (place >= turned_items) {
            const uint32_t at = 2 * a.pairs + (place - turned_items) * 8, some = min(8u, a.head_dim - at);
            float v[8];
            layer_load8<T, kWhole>(v, from + at, some);
            layer_store8<T, kWhole>(to + at, v, some);
        } else if constexpr (kInterleaved) {
            const uint32_t at = place * 8, some = min(8u, 2 * a.pairs - at);
            float v[8], u[8];
            layer_load8<T, kWhole>(v, from + at, some);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t pair = angles + min(at / 2 + i, a.pairs - 1);
                const float c = cosine[pair], s = sine[pair];
                u[2 * i] = v[2 * i] * c - v[2 * i + 1] * s;
                u[2 * i + 1] = v[2 * i + 1] * c + v[2 * i] * s;
            }
            layer_store8<T, kWhole>(to + at, u, some);
        } else {
            const uint32_t at = place * 8, some = min(8u, a.pairs - at);
            float v[8], w[8], p[8], q[8];
            layer_load8<T, kWhole>(v, from + at, some);
            layer_load8<T, kWhole>(w, from + a.pairs + at, some);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t pair = angles + min(at + i, a.pairs - 1);
                const float c = cosine[pair], s = sine[pair];
                p[i] = v[i] * c - w[i] * s;
                q[i] = w[i] * c + v[i] * s;
            }
            layer_store8<T, kWhole>(to + at, p, some);
            layer_store8<T, kWhole>(to + a.pairs + at, q, some);
        }
    }
}

/* ---- launches -------------------------------------------------------------- */

/* rows that wide accesses can take: 16-byte aligned, whole groups of eight */
template <typename T>
bool whole(const void *p, uint64_t stride, uint32_t rows)
{
    return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || stride * sizeof(T) % 16 == 0));
}

template <typename T>
bool quantize(const QuantizeRows &a, hipStream_t stream)
{
    const uint32_t parts = quantize_parts(a.width);
    const bool wide = a.width % 8 == 0 && whole<T>(a.x, a.x_row, a.rows) && whole<T>(a.gate, a.gate_row, a.rows) &&
                      (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0;
    const auto kernel = a.gate ? (wide ? quantize_kernel<T, true, true> : quantize_kernel<T, true, false>)
                               : (wide ? quantize_kernel<T, false, true> : quantize_kernel<T, false, false>);
    return launch_kernel(kernel, dim3(a.rows * parts), dim3(256), stream, a, parts);
}

template <typename T, bool kWhole>
bool norm(const NormRows &a, hipStream_t stream)
{
    const auto go = [&](void (*kernel)(NormRows), uint32_t threads) {
        return launch_kernel(kernel, dim3(a.rows), dim3(threads), stream, a);
    };
    switch (up(a.width, 2048)) {
    case 1: return go(norm_kernel<T, 256, 1, kWhole>, 256);
    case 2: return go(norm_kernel<T, 256, 2, kWhole>, 256);
    case 3: return go(norm_kernel<T, 256, 3, kWhole>, 256);
    case 4: return go(norm_kernel<T, 256, 4, kWhole>, 256);
    }
    switch (up(a.width, 8192)) {
    case 2: return go(norm_kernel<T, 1024, 2, kWhole>, 1024);
    case 3: return go(norm_kernel<T, 1024, 3, kWhole>, 1024);
    }
    return go(norm_kernel<T, 1024, 0, kWhole>, 1024);
}

template <typename T>
bool norm(const NormRows &a, hipStream_t stream)
{
    const bool wide = a.width % 8 == 0 && whole<T>(a.x, a.x_row, a.rows) && whole<T>(a.addend, a.addend_row, a.rows) &&
                      whole<T>(a.total, a.total_row, a.rows) && whole<T>(a.output, a.output_row, a.rows) &&
                      whole<T>(a.weight, 0, 1) && (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0;
    return wide ? norm<T, true>(a, stream) : norm<T, false>(a, stream);
}

template <typename T>
bool rotary(const Rotary &a, hipStream_t stream)
{
    /* in place, what is not turned stays where it is */
    const uint32_t pass = a.output == a.x ? 0 : up(a.head_dim - 2 * a.pairs, 8);
    const uint32_t turned = a.interleaved ? up(2 * a.pairs, 8) : up(a.pairs, 8);
    const uint32_t items = a.heads * (turned + pass);
    const bool wide = a.head_dim % 8 == 0 && a.pairs % (a.interleaved ? 4 : 8) == 0 && whole<T>(a.x, a.x_row, a.rows) &&
                      whole<T>(a.output, a.output_row, a.rows) && whole<T>(a.x, a.x_head, a.heads) &&
                      whole<T>(a.output, a.output_head, a.heads);
    const uint32_t threads = items >= 256 ? 256 : up(items, 64) * 64;
    /* Rows that leave units idle have a workgroup for each 256 of their items, each with angles of its own: 16 fp32
     * rows of 28 heads of 256 2.7 us against 4.2, 200 rows 4.4 against 4.7, 300 bf16 rows of 40 heads of 128 no
     * different. */
    const uint32_t parts = a.rows < 256 ? up(items, 256) : 1;
    /* Short rows by as many to a workgroup as it has threads and room for angles, while four workgroups to a unit are
     * left: 60000 fp32 rows of one head of 80 23 us against 54; with 64 items a row (8192 bf16 rows of 8 heads of 128)
     * 6.9 against 6.3. */
    uint32_t group = items <= 32 ? 256 / items : 1;
    if (group > 512 / a.pairs) group = 512 / a.pairs;
    if (group > a.rows / 1024) group = a.rows / 1024;
    const auto go = [&](auto kernel, uint32_t workgroups, uint32_t size) {
        return launch_kernel(kernel, dim3(workgroups), dim3(size), stream, a, parts, group, items, turned, pass);
    };
    if (group > 1) {
        const auto kernel = a.interleaved ? (wide ? rotary_kernel<T, true, true, true> : rotary_kernel<T, true, false, true>)
                                          : (wide ? rotary_kernel<T, false, true, true> : rotary_kernel<T, false, false, true>);
        return go(kernel, up(a.rows, group), 256);
    }
    group = 1;
    const auto kernel = a.interleaved ? (wide ? rotary_kernel<T, true, true, false> : rotary_kernel<T, true, false, false>)
                                      : (wide ? rotary_kernel<T, false, true, false> : rotary_kernel<T, false, false, false>);
    return go(kernel, a.rows * parts, threads);
}

}  // namespace

bool launch_quantize_e4m3(const QuantizeRows &a, int type, hipStream_t stream)
{
    return type == kLayerF32 ? quantize<float>(a, stream) : type == kLayerF16 ? quantize<_Float16>(a, stream)
                                                                              : quantize<__bf16>(a, stream);
}

bool launch_rms_norm(const NormRows &a, int type, hipStream_t stream)
{
    return type == kLayerF32 ? norm<float>(a, stream) : type == kLayerF16 ? norm<_Float16>(a, stream)
                                                                          : norm<__bf16>(a, stream);
}

bool launch_rotary(const Rotary &a, int type, hipStream_t stream)
{
    return type == kLayerF32 ? rotary<float>(a, stream) : type == kLayerF16 ? rotary<_Float16>(a, stream)
                                                                            : rotary<__bf16>(a, stream);
}

}  // namespace q38
