// The gated feed-forward block on packed weights and what its backward pass takes: between abi.cu, gated.cu (the forms for any
// shape and type, the passes over activations) and gated_product.cu (the tensor-core forms).
#pragma once

#include <cstddef>
#include <cstdint>

#include "eoq_internal.h"

namespace eoq {

constexpr uint32_t kStoreBlock = 64;       // values of a row that share a scale in 8-bit storage

enum { kActSilu = 0, kActGelu = 1, kActGeluTanh = 2 };
enum { kKeepNone = 0, kKeepFull = 1, kKeep8bit = 2, kKeepF32 = 3 };      // (F32: the forms for any shape, on the way to 8 bits)

// One or two packed weights of one shape (core/quantized_linear.py:49-66), scales indexed over the flattened matrix.
struct PackedPair {
    const uint8_t *codes[2];
    const uint16_t *scales[2];
    uint32_t N, K, bits, group, row_bytes;
};

// What the forward pass leaves for the backward one, per projection (0: gate, 1: up).
struct Kept {
    int form;
    void *v[2];                  // [M][N] in the activations' type, or signed codes
    float *scale[2];             // 8 bits: [M][ceil(N / 64)]
};

struct GatedCall {
    PackedPair w;
    const void *bias[2];         // of bias_dtype, or null
    const void *x;               // [M][K]
    void *h;                     // [M][N]
    uint32_t M;
    int dtype, act, bias_dtype;
    Kept keep;
};

int launch_gated_general(const GatedCall &c, void *stream);
// dx[m][k] = sum over n of dy[0][m][n] w[0][n][k] + dy[1][m][n] w[1][n][k]; nw: one weight or two; dy fp32 or 16-bit, [M][N].
// scratch: partial sums, input_grad_general_scratch() bytes.
int launch_input_grad_general(const PackedPair &w, int nw, const void *const dy[2], int dy_dtype, uint32_t M, void *scratch, void *dx, int dtype, void *stream);
size_t input_grad_general_scratch(const PackedPair &w, uint32_t M);

// dg = dh u act'(g), du = dh act(g): fp32 [M][N] each, or (half) fp16 [2][M][pitch] times a power of two of the row, whose inverse
// goes to factor[m]; the pad of a row is zero.
// zeros: words that are set to zero besides (a later kernel's counters).
struct Zeros { uint32_t *p; uint32_t n; };
int launch_gate_grad(const Kept &k, const void *dh, int dtype, int act, uint32_t M, uint32_t N, float *out32[2], uint16_t *half, uint32_t pitch, float *factor,
                     Zeros zeros, void *stream);
int launch_zeros(Zeros zeros, void *stream);
// Sums over the rows, to values of dtype: of fp32 [M][N] x 2, or of the form above.  scratch: column_sums_scratch() bytes.
int launch_column_sums(const float *const in32[2], const uint16_t *half, uint32_t pitch, const float *factor, uint32_t M, uint32_t N, float *scratch,
                       void *const out[2], int dtype, void *stream);
size_t column_sums_scratch(uint32_t M, uint32_t N);
// Rows to fp16, pitch values apart (a multiple of 8; the pad is zero), times a power of two that brings the largest to 2^14 .. 2^15.
int launch_rows_to_half(const void *x, int dtype, uint32_t M, uint32_t K, uint32_t pitch, uint16_t *out, float *factor, Zeros zeros, void *stream);

// h = act(g) u of fp32 [M][N].
int launch_gate_apply(const float *g, const float *u, size_t count, int act, void *h, int dtype, void *stream);
// The tensor-core forms (gated_product.cu): whole groups per row, groups of 32 columns and their multiples, rows of codes that are
// multiples of 16 bytes, everything 16-byte aligned.  x, dy: fp16, [M][K] and [nw][M][pitch], pitch a multiple of 8.  Scratch: bytes,
// of which the first `zeros` words are zero when the kernel before has ended.
struct Scratch { size_t bytes; uint32_t zeros; };
bool product_takes(const PackedPair &w, int nw);
Scratch gated_product_scratch(const PackedPair &w, uint32_t M);
Scratch input_grad_product_scratch(const PackedPair &w, int nw, uint32_t M);
int launch_gated_product(const GatedCall &c, const uint16_t *x, const float *factor, void *scratch, void *stream);
int launch_input_grad_product(const PackedPair &w, int nw, const uint16_t *dy, uint32_t pitch, const float *factor, uint32_t M, void *dx, int dtype, void *scratch,
                              void *stream);
// Up to 32 rows of 16-bit activations, 16-byte aligned; kept in full or in fp32 (gated_rows.cu).
bool gated_rows_takes(const PackedPair &w, uint32_t batch);
int launch_gated_rows(const GatedCall &c, void *stream);
long long gated_wait_limit();
uint32_t *gated_status_word();       // of the current device
uint32_t gated_status();
void set_gated_wait_us(int v);

int launch_store_8bit(const void *x, int dtype, size_t M, uint32_t N, int8_t *codes, float *scales, void *stream);
int launch_load_8bit(const int8_t *codes, const float *scales, size_t M, uint32_t N, void *y, int dtype, void *stream);

}  // namespace eoq
