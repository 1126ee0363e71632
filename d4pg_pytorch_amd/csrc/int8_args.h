// Launch descriptors of the 8-bit operators: shared by their kernels (int8.hip) and the tensor binding (int8_bind.cpp),
// mirrored in ops/hip.py.
#pragma once

enum { F_FP32 = 0, F_BF16 = 1, F_FP16 = 2, F_NONE = -1 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_TANH = 2 };
// What the entries return: 0, enqueued; a hipError_t (positive), the launch's own; negative, refused and nothing enqueued.
enum { NOT_TAKEN = -100 };         // mlp3: good arguments, outside the one launch's range

// floating rows -> codes
struct QuantRowsArgs {
    const void* x;         // [M, K] rows of ld_x elements
    const void* residual;  // [M, K] added to x, or null                       (norm only)
    const void* weight;    // [K] factor after the norm, or null               (norm only)
    void* h;               // [M, K] x + residual in x's type, or null         (norm only)
    signed char* q;        // [M, ld_q] codes, zero from K to ld_q
    float* scale;          // [M]
    long long M, K;
    long long ld_x, ld_r, ld_h, ld_q;   // elements (bytes for ld_q, a multiple of 16)
    int dtype, wdtype;     // F_*: of x, residual and h; of weight
    int norm;              // 0: quantise x; 1: RMS norm first
    float eps;
};

// codes -> floating rows
struct DequantRowsArgs {
    const signed char* q;  // [M, K] rows of ld_q bytes
    const float* scale;    // [M]
    void* out;             // [M, K] contiguous
    long long M, K, ld_q;
    int dtype, tpr_log;    // threads a row = 2^tpr_log (set by the host entry)
};

// product of codes
struct LinearInt8Args {
    const signed char* q;  // [M, K] activations' codes, rows of ld_q bytes
    const float* scale;    // [M]
    const signed char* w;  // [N, K] weights' codes, rows of ld_w bytes
    const float* wscale;   // [N]
    const float* bias;     // [N] or null
    void* out;             // [M, N], rows of ld_out elements
    long long ld_q, ld_w, ld_out;
    int M, N, K;
    int act, dtype, pad_;
};

// three layers on codes
struct Mlp3Int8Args {
    const void* x;                 // [M, width[0]] rows of ld_x elements
    void* out;                     // [M, width[3]] rows of ld_out elements
    const signed char* w[3];       // [width[i + 1], width[i]] codes, rows of ld_w[i] bytes
    const float* wscale[3];
    const float* bias[3];          // or null
    long long ld_x, ld_out, ld_w[3];
    int M, width[4];
    int xdtype, dtype, act;        // F_* of x and out; ACT_* of the last layer (the others: ReLU)
    int pitch, split;              // bytes of a row of codes in LDS, words of the split layers' sums (set by the host entry)
};
