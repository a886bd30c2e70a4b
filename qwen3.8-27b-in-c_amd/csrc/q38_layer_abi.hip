/* C ABI of a decoder layer's operators (declared in include/q38hip.h): checks
 * of what the host can see, then the launch. */
#include <cmath>
#include <initializer_list>

#include "q38_kernels.h"
#include "q38_layer.h"

namespace {

using q38::abi_fail;

constexpr uint32_t kMost = 1u << 24;      /* rows, and elements of a row */

bool element_type(uint32_t type)
{
    return type == (uint32_t)q38::kLayerF32 || type == (uint32_t)q38::kLayerF16 || type == (uint32_t)q38::kLayerBF16;
}

bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

/* elements of whole numbers of bytes */
bool element_aligned(const void *p, uint32_t type) { return aligned(p, type == (uint32_t)q38::kLayerF32 ? 4 : 2); }

/* an output or a workspace that begins where another tensor of the call does */
bool among(const void *p, std::initializer_list<const void *> others)
{
    for (const void *other : others)
        if (p && p == other) return true;
    return false;
}

const char *rows_fault(uint64_t width, uint32_t rows)
{
    if (!width || !rows) return "empty rows";
    if (width > kMost || rows > kMost) return "more than 2^24 rows or elements of a row";
    if (width * rows > 1ull << 40) return "more than 2^40 elements";
    return nullptr;
}

}  // namespace

extern "C" uint32_t q38hip_e4m3_scale_pitch(uint64_t width)
{
    if (!width || width > kMost) {
        abi_fail("width must be 1 to 2^24");
        return 0;
    }
    return q38::e4m3_pitch(width);
}

extern "C" int q38hip_quantize_e4m3(uint8_t *codes, uint8_t *scales, const void *x, uint64_t x_row_stride,
                                    const void *gate, uint64_t gate_row_stride, uint32_t type, uint64_t width,
                                    uint32_t rows, void *stream)
{
    if (const char *fault = rows_fault(width, rows)) return abi_fail(fault);
    if (!codes || !scales || !x) return abi_fail("bad quantize arguments");
    if (!element_type(type)) return abi_fail("rows must be F32, F16 or BF16");
    if (rows > 1 && (x_row_stride < width || (gate && gate_row_stride < width))) return abi_fail("row stride too small");
    if (!element_aligned(x, type) || !element_aligned(gate, type)) return abi_fail("rows must be aligned to their elements");
    if (among(codes, {x, gate}) || among(scales, {x, gate, codes})) return abi_fail("codes and scales must not be an input or each other");
    if (!q38::layer_launch_holds((uint64_t)rows * q38::quantize_parts(width), 256)) return abi_fail("more rows than a launch holds");
    const q38::QuantizeRows a = {codes, scales, x, gate, x_row_stride, gate_row_stride, (uint32_t)width,
                                 q38::e4m3_pitch(width), rows};
    return q38::launch_quantize_e4m3(a, (int)type, static_cast<hipStream_t>(stream)) ? 1
                                                                                     : abi_fail("quantize kernel failed");
}

extern "C" int q38hip_rms_norm(void *output, uint64_t output_row_stride, uint8_t *codes, uint8_t *scales, void *total,
                               uint64_t total_row_stride, const void *x, uint64_t x_row_stride, const void *addend,
                               uint64_t addend_row_stride, uint32_t type, const void *weight, uint32_t weight_type,
                               float weight_offset, float eps, uint64_t width, uint32_t rows, void *stream)
{
    if (const char *fault = rows_fault(width, rows)) return abi_fail(fault);
    if (!x || !weight || (!output && !codes) || (!codes != !scales) || (!addend != !total))
        return abi_fail("bad norm arguments");
    if (!element_type(type) || !element_type(weight_type)) return abi_fail("rows and weight must be F32, F16 or BF16");
    if (rows > 1 && (x_row_stride < width || (output && output_row_stride < width) ||
                     (addend && (addend_row_stride < width || total_row_stride < width))))
        return abi_fail("row stride too small");
    if (!element_aligned(x, type) || !element_aligned(output, type) || !element_aligned(addend, type) ||
        !element_aligned(total, type) || !element_aligned(weight, weight_type))
        return abi_fail("rows must be aligned to their elements");
    if (among(output, {total, weight}) || among(total, {weight})) return abi_fail("total and output must differ, and not be the weight");
    if (among(codes, {x, addend, total, output, weight}) || among(scales, {x, addend, total, output, weight, codes}))
        return abi_fail("codes and scales must not be an input or another output");
    if (rows > 1 && ((total && ((total == x && total_row_stride != x_row_stride) ||
                                (total == addend && total_row_stride != addend_row_stride))) ||
                     (output && ((output == x && output_row_stride != x_row_stride) ||
                                 (output == addend && output_row_stride != addend_row_stride)))))
        return abi_fail("rows written in place must keep their stride");
    if (!(eps >= 0.0f) || !std::isfinite(eps) || !std::isfinite(weight_offset))
        return abi_fail("eps must be finite and not negative, the weight's offset finite");
    if (!q38::layer_launch_holds(rows, q38::norm_threads(width))) return abi_fail("more rows than a launch holds");
    const q38::NormRows a = {output, total, codes, scales, x, addend, weight, output_row_stride, total_row_stride,
                             x_row_stride, addend_row_stride, (uint32_t)width, q38::e4m3_pitch(width), rows,
                             (int)weight_type, weight_offset, eps};
    return q38::launch_rms_norm(a, (int)type, static_cast<hipStream_t>(stream)) ? 1 : abi_fail("norm kernel failed");
}

namespace {

const char *product_fault(uint32_t batch_size, uint64_t input_length, uint32_t rows)
{
    if (!batch_size || !input_length || !rows) return "empty product";
    if (input_length % 16) return "input_length must be a multiple of 16";
    if (batch_size > kMost || input_length > kMost || rows > kMost) return "more than 2^24 rows or elements of a row";
    if ((uint64_t)batch_size * rows > 1ull << 36) return "more than 2^36 outputs";
    return nullptr;
}

}  // namespace

extern "C" uint64_t q38hip_gemm_e4m3_workspace_bytes(uint32_t batch_size, uint64_t input_length, uint32_t rows)
{
    if (const char *fault = product_fault(batch_size, input_length, rows)) {
        abi_fail(fault);
        return 0;
    }
    return q38::product_e4m3_workspace_bytes(batch_size, input_length, rows);
}

extern "C" int q38hip_gemm_e4m3(void *output, uint32_t type, uint64_t output_row_stride, const uint8_t *codes,
                                const uint8_t *scales, uint32_t batch_size, uint64_t input_length, const uint8_t *weight,
                                const float *weight_scales, uint32_t rows, void *workspace, void *stream)
{
    if (const char *fault = product_fault(batch_size, input_length, rows)) return abi_fail(fault);
    if (!output || !codes || !scales || !weight || !weight_scales) return abi_fail("bad product arguments");
    if (!element_type(type)) return abi_fail("output must be F32, F16 or BF16");
    if (batch_size > 1 && output_row_stride < rows) return abi_fail("output row stride too small");
    if (!aligned(codes, 16) || !aligned(weight, 16)) return abi_fail("codes must be 16-byte aligned");
    if (!aligned(scales, 4) || !aligned(weight_scales, 4)) return abi_fail("scales must be 4-byte aligned");
    if (!element_aligned(output, type)) return abi_fail("output must be aligned to its elements");
    if (among(output, {codes, scales, weight, weight_scales})) return abi_fail("output must not be an input");
    if (among(workspace, {output, codes, scales, weight, weight_scales})) return abi_fail("workspace must be memory of its own");
    if (q38::product_e4m3_workspace_bytes(batch_size, input_length, rows) && !workspace)
        return abi_fail("this product needs a workspace");
    if (!aligned(workspace, 16)) return abi_fail("workspace must be 16-byte aligned");
    const q38::ProductE4M3 a = {output, output_row_stride, codes, scales, weight, weight_scales,
                                static_cast<float *>(workspace), batch_size, (uint32_t)input_length, rows,
                                q38::e4m3_blocks(input_length), q38::e4m3_pitch(input_length), (int)type};
    return q38::launch_product_e4m3(a, static_cast<hipStream_t>(stream)) ? 1 : abi_fail("product kernel failed");
}

extern "C" int q38hip_rotary(void *output, uint64_t output_row_stride, uint64_t output_head_stride, const void *x,
                             uint64_t x_row_stride, uint64_t x_head_stride, uint32_t type, uint32_t rows, uint32_t heads,
                             uint32_t head_dim, const int32_t *positions, const float *frequencies, uint32_t pairs,
                             int interleaved, float magnitude, void *stream)
{
    if (!rows || !heads || !head_dim || !pairs) return abi_fail("empty rows");
    if (!output || !x || !positions || !frequencies) return abi_fail("bad rotary arguments");
    if (!element_type(type)) return abi_fail("rows must be F32, F16 or BF16");
    if (rows > kMost) return abi_fail("more than 2^24 rows");
    if (head_dim > 1024 || (uint64_t)heads * head_dim > 1u << 20) return abi_fail("heads of more than 1024 or rows of more than 2^20 elements");
    if (2ull * pairs > head_dim) return abi_fail("more pairs than the head holds");
    if (heads > 1 && (x_head_stride < head_dim || output_head_stride < head_dim)) return abi_fail("head stride too small");
    if (rows > 1 && (x_row_stride < head_dim || output_row_stride < head_dim)) return abi_fail("row stride too small");
    if (!element_aligned(x, type) || !element_aligned(output, type)) return abi_fail("rows must be aligned to their elements");
    if (!aligned(positions, 4) || !aligned(frequencies, 4)) return abi_fail("positions and frequencies must be 4-byte aligned");
    if (output == x && ((rows > 1 && output_row_stride != x_row_stride) || (heads > 1 && output_head_stride != x_head_stride)))
        return abi_fail("rows turned in place must keep their strides");
    if (among(output, {positions, frequencies})) return abi_fail("output must not be the positions or frequencies");
    if (!std::isfinite(magnitude)) return abi_fail("magnitude must be finite");
    if (!q38::layer_launch_holds(rows, 256)) return abi_fail("more rows than a launch holds");
    const q38::Rotary a = {output, x, output_row_stride, output_head_stride, x_row_stride, x_head_stride, rows, heads,
                           head_dim, pairs, positions, frequencies, magnitude, interleaved != 0};
    return q38::launch_rotary(a, (int)type, static_cast<hipStream_t>(stream)) ? 1 : abi_fail("rotary kernel failed");
}

extern "C" int q38hip_prompt_attention(void *output, uint64_t output_row_stride, const void *query, const void *gate,
                                       uint64_t query_row_stride, uint64_t query_head_stride, const void *key,
                                       uint64_t key_row_stride, const void *value, uint64_t value_row_stride, uint32_t type,
                                       uint32_t heads, uint32_t kv_heads, uint32_t head_dim, float scale,
                                       const int32_t *row_starts, uint32_t count, uint32_t total_rows, void *stream)
{
    if (!count || !total_rows) return abi_fail("no sequences or no rows");
    if (!output || !query || !key || !value || !row_starts) return abi_fail("bad attention arguments");
    if (!element_type(type)) return abi_fail("rows must be F32, F16 or BF16");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return abi_fail("head_dim must be 64, 128 or 256");
    if (!heads || !kv_heads || heads % kv_heads) return abi_fail("heads must be a multiple of kv_heads");
    if (heads > 65535) return abi_fail("more than 65535 heads");
    if (count > kMost || total_rows > kMost || (uint64_t)total_rows * heads > 1u << 30)
        return abi_fail("more than 2^24 rows or sequences, or 2^30 query rows");
    if (heads > 1 && query_head_stride < head_dim) return abi_fail("query head stride too small");
    if (total_rows > 1 && (query_row_stride < head_dim || key_row_stride < (uint64_t)kv_heads * head_dim ||
                           value_row_stride < (uint64_t)kv_heads * head_dim || output_row_stride < (uint64_t)heads * head_dim))
        return abi_fail("row stride too small");
    if (!element_aligned(output, type) || !element_aligned(query, type) || !element_aligned(gate, type) ||
        !element_aligned(key, type) || !element_aligned(value, type) || !aligned(row_starts, 4))
        return abi_fail("rows must be aligned to their elements");
    if (among(output, {query, gate, key, value, row_starts})) return abi_fail("output must not be an input");
    /* weights are equal where the scale is 0 (and where it is so small); a product with
     * -infinity must not become NaN there */
    const float factor = scale * 1.44269504088896340736f;
    if (!std::isfinite(factor)) return abi_fail("scale must be finite, at most 2^127");
    const q38::PromptAttention a = {output, query, gate, key, value, output_row_stride, query_row_stride,
                                    query_head_stride, key_row_stride, value_row_stride, row_starts, count, total_rows,
                                    heads, kv_heads, head_dim, std::fabs(factor) < 0x1p-126f ? 0x1p-126f : factor,
                                    (int)type};
    return q38::launch_prompt_attention(a, static_cast<hipStream_t>(stream)) ? 1
                                                                             : abi_fail("prompt attention kernel failed");
}
