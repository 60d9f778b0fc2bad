// A call of the grouped products (product.hip)
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace frt {

struct ProductArgs {
    const void* x;           // the operand along the output's rows: a (product), dout (both gradients)
    int64_t ldx;
    const void* y;           // the one along its columns: w (product, grad), a (wgrad; in 8 bits with scales)
    int64_t ldy;             // (of a; w is contiguous)
    const uint8_t* scales;   // a's, where it is in 8 bits
    int a_rows;              // rows of a
    const int32_t* rows;
    const int32_t* bounds;
    int E, M, N, C;
    void* out;
    int64_t ldout;
    int out_type;            // ggml type id
    int add;                 // wgrad: to what is there
};
int moe_product(int type, const ProductArgs& p, hipStream_t stream);
int moe_product_grad(int type, const ProductArgs& p, hipStream_t stream);
int moe_product_wgrad(int type, const ProductArgs& p, hipStream_t stream);

}  // namespace frt
