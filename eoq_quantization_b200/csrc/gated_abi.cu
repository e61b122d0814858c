// C entry points of the gated feed-forward block on packed weights and of 8-bit activation storage (include/eoq_b200.h): checks,
// scratch, and which form takes a call.
#include "../../include/eoq_b200.h"

#include <algorithm>
#include <cstdio>
#include <cuda_runtime.h>

#include "gated.h"

namespace eoq {
namespace {

bool have_device()
{
    int n = 0;
    return cudaGetDeviceCount(&n) == cudaSuccess && n > 0;
}

eoq_error_t launched(int e, const char *where)
{
    if (e == 0) return EOQ_OK;
    std::fprintf(stderr, "%s: launch failed: %s\n", where, cudaGetErrorString((cudaError_t)e));
    return EOQ_ERR_CUDA;
}

// Parts of the caller's scratch, one behind the other.
struct Carve {
    uint8_t *base;
    size_t at = 0;
    template <class T> T *take(size_t bytes)
    {
        T *p = base ? reinterpret_cast<T *>(base + at) : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    }
};

bool fine(uint32_t rows, uint32_t cols, uint32_t bits, uint32_t group) { return rows && cols && bits >= 2 && bits <= 8 && group; }
uint32_t row_bytes(uint32_t cols, uint32_t bits) { return bits == 4 ? (cols + 1) / 2 : bits == 2 ? (cols + 3) / 4 : cols; }

PackedPair pair_of(const eoq_b200_gated_t *w)
{
    return PackedPair{{w->gate, w->up}, {w->gate_scales, w->up_scales}, w->rows, w->cols, w->bits, w->group, row_bytes(w->cols, w->bits)};
}
Kept kept_of(const eoq_b200_kept_t *k)
{
    if (!k || k->form == kKeepNone) return Kept{kKeepNone, {nullptr, nullptr}, {nullptr, nullptr}};
    return Kept{k->form, {k->gate, k->up}, {k->gate_scales, k->up_scales}};
}
size_t values(uint32_t batch, uint32_t n) { return (size_t)batch * n; }

// fp32 activations: both products by the kernel that multiplies the codes exactly with two fp16 halves of each activation.
bool exact_products(const PackedPair &w, int dtype, const void *codes, const void *x)
{
    return dtype == EOQ_B200_F32 && qmm_takes(w.K, w.bits, w.group, codes, x) && split_rows_takes(w.K, 1);
}

// Up to 32 rows of 16-bit activations: one pass over the codes.
bool few_rows(const PackedPair &w, int dtype, uint32_t batch) { return dtype != EOQ_B200_F32 && gated_rows_takes(w, batch); }

// 16-bit activations on the tensor cores: fp16 rows as they are, where copies of them can be aligned; others as fp16 times a
// power of two a row.
uint32_t pitch_of(uint32_t n) { return (n + 7u) & ~7u; }
bool as_it_is(const void *x, int dtype, uint32_t n) { return dtype == EOQ_B200_F16 && n % 8u == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0; }
size_t half_bytes(uint32_t batch, uint32_t n) { return values(batch, pitch_of(n)) * 2; }

}  // namespace
}  // namespace eoq

using namespace eoq;

extern "C" size_t eoq_b200_gated_scratch(const eoq_b200_gated_t *w, const eoq_b200_kept_t *kept, int dtype, uint32_t batch)
{
    if (!w || !fine(w->rows, w->cols, w->bits, w->group)) return 0;
    const int form = kept ? kept->form : kKeepNone;
    Carve c{nullptr};
    if (dtype == EOQ_B200_F32) {
        c.take<float>(values(batch, w->cols + 1) * 4);
        if (form != kKeepFull) c.take<float>(2 * values(batch, w->rows) * 4);
        return c.at;
    }
    if (product_takes(pair_of(w), 2)) {
        c.take<void>(half_bytes(batch, w->cols));
        c.take<float>((size_t)batch * 4);
        c.take<void>(gated_product_scratch(pair_of(w), batch).bytes);
        if (!few_rows(pair_of(w), dtype, batch)) return c.at;
    }
    const size_t sums = form == kKeep8bit ? 2 * values(batch, w->rows) * 4 : 0;
    return std::max(c.at, sums);
}

extern "C" eoq_error_t eoq_b200_gated_packed(const eoq_b200_gated_t *w, const void *x, int dtype, uint32_t batch, void *d_scratch, void *h,
                                             const eoq_b200_kept_t *kept, void *stream)
{
    if (!w || !w->gate || !w->up || !w->gate_scales || !w->up_scales || !x || !h) return EOQ_ERR_NULL_PTR;
    const int form = kept ? kept->form : kKeepNone;
    if (form != kKeepNone && (!kept->gate || !kept->up || (form == kKeep8bit && (!kept->gate_scales || !kept->up_scales)))) return EOQ_ERR_NULL_PTR;
    if (batch == 0 || w->rows == 0) return EOQ_OK;
    if (dtype < 0 || dtype > 2 || w->bias_dtype < 0 || w->bias_dtype > 2 || form < 0 || form > kKeep8bit || w->activation < 0 || w->activation > kActGeluTanh) return EOQ_ERR_UNSUPPORTED;
    if (!fine(w->rows, w->cols, w->bits, w->group)) return EOQ_ERR_INVALID_HEADER;
    if (eoq_b200_gated_scratch(w, kept, dtype, batch) && !d_scratch) return EOQ_ERR_NULL_PTR;
    if (!have_device()) return EOQ_ERR_CUDA;
    const char *where = "eoq_b200_gated_packed";
    GatedCall c = {pair_of(w), {w->gate_bias, w->up_bias}, x, h, batch, dtype, w->activation, w->bias_dtype, kept_of(kept)};
    Carve scratch{static_cast<uint8_t *>(d_scratch)};
    const size_t n = values(batch, w->rows);
    int e = 0;
    const Kept keep = c.keep;
    if (few_rows(c.w, dtype, batch) && (reinterpret_cast<uintptr_t>(x) & 15u) == 0) {
        if (form == kKeep8bit) {
            float *g = scratch.take<float>(2 * n * 4);
            c.keep = Kept{kKeepF32, {g, g + n}, {nullptr, nullptr}};
        }
        e = launch_gated_rows(c, stream);
        for (int i = 0; i < 2 && e == 0 && form == kKeep8bit; i++)
            e = launch_store_8bit(c.keep.v[i], EOQ_B200_F32, batch, w->rows, static_cast<int8_t *>(keep.v[i]), keep.scale[i], stream);
        return launched(e, where);
    }
    if (dtype != EOQ_B200_F32 && product_takes(c.w, 2)) {
        uint16_t *half = scratch.take<uint16_t>(half_bytes(batch, w->cols));
        float *factor = scratch.take<float>((size_t)batch * 4);
        const Scratch s = gated_product_scratch(c.w, batch);
        uint32_t *parts = scratch.take<uint32_t>(s.bytes);
        if (as_it_is(x, dtype, w->cols)) {
            half = static_cast<uint16_t *>(const_cast<void *>(x));
            factor = nullptr;
            e = launch_zeros(Zeros{parts, s.zeros}, stream);
        } else {
            e = launch_rows_to_half(x, dtype, batch, w->cols, pitch_of(w->cols), half, factor, Zeros{parts, s.zeros}, stream);
        }
        if (e == 0) e = launch_gated_product(c, half, factor, parts, stream);
        return launched(e, where);
    }
    const bool bf_bias = w->bias_dtype == EOQ_B200_BF16 && (w->gate_bias || w->up_bias);       // (that kernel has fp32 and fp16 biases)
    if (!bf_bias && exact_products(c.w, dtype, w->gate, d_scratch) && exact_products(c.w, dtype, w->up, d_scratch)) {
        void *planes = scratch.take<void>(values(batch, w->cols + 1) * 4);
        float *factors = reinterpret_cast<float *>(static_cast<uint8_t *>(planes) + values(batch, w->cols) * 4);
        float *out[2] = {static_cast<float *>(c.keep.v[0]), static_cast<float *>(c.keep.v[1])};
        if (form != kKeepFull) { out[0] = scratch.take<float>(2 * n * 4); out[1] = out[0] + n; }
        e = launch_split_rows(x, dtype, w->cols, batch, 1, planes, factors, stream);
        for (int i = 0; i < 2 && e == 0; i++) {
            QmmCall q = {};
            q.packed = c.w.codes[i]; q.scales = c.w.scales[i]; q.bias = c.bias[i]; q.tok_scale = factors; q.x = planes; q.y = out[i];
            q.N = w->rows; q.K = w->cols; q.M = batch; q.bits = w->bits; q.group = w->group; q.split_x = 1; q.bias_half = w->bias_dtype == EOQ_B200_F16; q.y_dtype = EOQ_B200_F32;
            e = launch_qmm(q, stream);
        }
        if (e != (int)cudaErrorNotSupported) {
            if (e == 0) e = launch_gate_apply(out[0], out[1], n, w->activation, h, dtype, stream);
            for (int i = 0; i < 2 && e == 0 && form == kKeep8bit; i++)
                e = launch_store_8bit(out[i], EOQ_B200_F32, batch, w->rows, static_cast<int8_t *>(c.keep.v[i]), c.keep.scale[i], stream);
            return launched(e, where);
        }
        scratch.at = 0;
    }
    if (dtype == EOQ_B200_F32) scratch.take<void>(values(batch, w->cols + 1) * 4);
    if (form == kKeep8bit) {
        float *g = scratch.take<float>(2 * n * 4);
        c.keep = Kept{kKeepF32, {g, g + n}, {nullptr, nullptr}};
    }
    e = launch_gated_general(c, stream);
    for (int i = 0; i < 2 && e == 0 && form == kKeep8bit; i++)
        e = launch_store_8bit(c.keep.v[i], EOQ_B200_F32, batch, w->rows, static_cast<int8_t *>(keep.v[i]), keep.scale[i], stream);
    return launched(e, where);
}

extern "C" size_t eoq_b200_gated_grad_scratch(const eoq_b200_gated_t *w, const eoq_b200_kept_t *, int dtype, uint32_t batch)
{
    if (!w || !fine(w->rows, w->cols, w->bits, w->group)) return 0;
    Carve c{nullptr};
    if (dtype != EOQ_B200_F32 && product_takes(pair_of(w), 2)) {
        c.take<void>(2 * half_bytes(batch, w->rows));
        c.take<float>((size_t)batch * 4);
        c.take<void>(input_grad_product_scratch(pair_of(w), 2, batch).bytes);
        c.take<void>(column_sums_scratch(batch, w->rows));
        return c.at;
    }
    c.take<float>(2 * values(batch, w->rows) * 4);
    c.take<void>(std::max(column_sums_scratch(batch, w->rows), input_grad_general_scratch(pair_of(w), batch)));
    return c.at;
}

extern "C" eoq_error_t eoq_b200_gated_grad(const eoq_b200_gated_t *w, const eoq_b200_kept_t *kept, const void *dh, int dtype, uint32_t batch,
                                           void *d_scratch, void *dx, void *d_gate_bias, void *d_up_bias, void *stream)
{
    if (!w || !w->gate || !w->up || !w->gate_scales || !w->up_scales || !kept || !kept->gate || !kept->up || !dh || !d_scratch) return EOQ_ERR_NULL_PTR;
    if (kept->form == kKeep8bit && (!kept->gate_scales || !kept->up_scales)) return EOQ_ERR_NULL_PTR;
    if (dtype < 0 || dtype > 2 || w->bias_dtype < 0 || w->bias_dtype > 2 || (kept->form != kKeepFull && kept->form != kKeep8bit) || w->activation < 0 || w->activation > kActGeluTanh) return EOQ_ERR_UNSUPPORTED;
    if (batch == 0 || w->rows == 0 || (!dx && !d_gate_bias && !d_up_bias)) return EOQ_OK;
    if (!fine(w->rows, w->cols, w->bits, w->group)) return EOQ_ERR_INVALID_HEADER;
    if (!have_device()) return EOQ_ERR_CUDA;
    const size_t n = values(batch, w->rows);
    const PackedPair pair = pair_of(w);
    Carve scratch{static_cast<uint8_t *>(d_scratch)};
    const char *where = "eoq_b200_gated_grad";
    void *const to[2] = {d_gate_bias, d_up_bias};
    if (dtype != EOQ_B200_F32 && product_takes(pair, 2)) {
        const uint32_t pitch = pitch_of(w->rows);
        uint16_t *half = scratch.take<uint16_t>(2 * half_bytes(batch, w->rows));
        float *factor = scratch.take<float>((size_t)batch * 4);
        const Scratch s = input_grad_product_scratch(pair, 2, batch);
        uint32_t *parts = scratch.take<uint32_t>(s.bytes);
        float *sums = scratch.take<float>(0);
        int e = launch_gate_grad(kept_of(kept), dh, dtype, w->activation, batch, w->rows, nullptr, half, pitch, factor, Zeros{parts, s.zeros}, stream);
        if (e == 0 && (d_gate_bias || d_up_bias)) e = launch_column_sums(nullptr, half, pitch, factor, batch, w->rows, sums, to, w->bias_dtype, stream);
        if (e == 0 && dx) e = launch_input_grad_product(pair, 2, half, pitch, factor, batch, dx, dtype, parts, stream);
        return launched(e, where);
    }
    float *d = scratch.take<float>(2 * n * 4), *out[2] = {d, d + n};
    void *sums = scratch.take<void>(0);
    int e = launch_gate_grad(kept_of(kept), dh, dtype, w->activation, batch, w->rows, out, nullptr, 0, nullptr, Zeros{nullptr, 0}, stream);
    if (e == 0 && (d_gate_bias || d_up_bias)) e = launch_column_sums(out, nullptr, 0, nullptr, batch, w->rows, static_cast<float *>(sums), to, w->bias_dtype, stream);
    if (e == 0 && dx) {
        const void *dy[2] = {out[0], out[1]};
        e = launch_input_grad_general(pair, 2, dy, EOQ_B200_F32, batch, sums, dx, dtype, stream);
    }
    return launched(e, where);
}

extern "C" size_t eoq_b200_packed_input_grad_scratch(uint32_t rows, uint32_t cols, uint32_t bits, uint32_t group, int dtype, uint32_t batch)
{
    if (!fine(rows, cols, bits, group)) return 0;
    const PackedPair p = {{nullptr, nullptr}, {nullptr, nullptr}, rows, cols, bits, group, row_bytes(cols, bits)};
    const size_t any = input_grad_general_scratch(p, batch);        // (codes that are not aligned)
    if (dtype == EOQ_B200_F32 || !product_takes(p, 1)) return any;
    Carve c{nullptr};
    c.take<void>(half_bytes(batch, rows));
    c.take<float>((size_t)batch * 4);
    c.take<void>(input_grad_product_scratch(p, 1, batch).bytes);
    return std::max(c.at, any);
}

extern "C" eoq_error_t eoq_b200_packed_input_grad(const uint8_t *d_packed, const uint16_t *d_scales_fp16, uint32_t rows, uint32_t cols, uint32_t bits,
                                                  uint32_t group, const void *dy, int dtype, uint32_t batch, void *d_scratch, void *dx, void *stream)
{
    if (!d_packed || !d_scales_fp16 || !dy || !dx || !d_scratch) return EOQ_ERR_NULL_PTR;
    if (dtype < 0 || dtype > 2) return EOQ_ERR_UNSUPPORTED;
    if (batch == 0 || cols == 0) return EOQ_OK;
    if (!fine(rows, cols, bits, group)) return EOQ_ERR_INVALID_HEADER;
    if (!have_device()) return EOQ_ERR_CUDA;
    const PackedPair p = {{d_packed, d_packed}, {d_scales_fp16, d_scales_fp16}, rows, cols, bits, group, row_bytes(cols, bits)};
    if (dtype != EOQ_B200_F32 && product_takes(p, 1)) {
        Carve scratch{static_cast<uint8_t *>(d_scratch)};
        uint16_t *half = scratch.take<uint16_t>(half_bytes(batch, rows));
        float *factor = scratch.take<float>((size_t)batch * 4);
        const Scratch s = input_grad_product_scratch(p, 1, batch);
        uint32_t *parts = scratch.take<uint32_t>(s.bytes);
        int e = 0;
        if (as_it_is(dy, dtype, rows)) {
            half = static_cast<uint16_t *>(const_cast<void *>(dy));
            factor = nullptr;
            e = launch_zeros(Zeros{parts, s.zeros}, stream);
        } else {
            e = launch_rows_to_half(dy, dtype, batch, rows, pitch_of(rows), half, factor, Zeros{parts, s.zeros}, stream);
        }
        if (e == 0) e = launch_input_grad_product(p, 1, half, pitch_of(rows), factor, batch, dx, dtype, parts, stream);
        return launched(e, "eoq_b200_packed_input_grad");
    }
    const void *d[2] = {dy, dy};
    return launched(launch_input_grad_general(p, 1, d, dtype, batch, d_scratch, dx, dtype, stream), "eoq_b200_packed_input_grad");
}

extern "C" eoq_error_t eoq_b200_store_8bit(const void *x, int dtype, size_t rows, uint32_t cols, int8_t *d_codes, float *d_scales, void *stream)
{
    if (!x || !d_codes || !d_scales) return EOQ_ERR_NULL_PTR;
    if (dtype < 0 || dtype > 2) return EOQ_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return EOQ_OK;
    if (!have_device()) return EOQ_ERR_CUDA;
    return launched(launch_store_8bit(x, dtype, rows, cols, d_codes, d_scales, stream), "eoq_b200_store_8bit");
}

extern "C" eoq_error_t eoq_b200_load_8bit(const int8_t *d_codes, const float *d_scales, size_t rows, uint32_t cols, void *y, int dtype, void *stream)
{
    if (!d_codes || !d_scales || !y) return EOQ_ERR_NULL_PTR;
    if (dtype < 0 || dtype > 2) return EOQ_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return EOQ_OK;
    if (!have_device()) return EOQ_ERR_CUDA;
    return launched(launch_load_8bit(d_codes, d_scales, rows, cols, y, dtype, stream), "eoq_b200_load_8bit");
}
