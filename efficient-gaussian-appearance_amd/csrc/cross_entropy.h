// What the sources of the cross entropy share: the products' arguments and tiles.
#pragma once
#include "internal.h"

namespace efgs {

constexpr uint32_t entropy_none = 0xffffffffu;
constexpr uint32_t entropy_row_tile = 256;     // packed rows come in multiples of it
constexpr uint32_t entropy_column_tile = 64;   // so do their columns
constexpr float entropy_half_range = 32768.0f; // float16: what upstream gradients of the logits are held times

// The log sum of a row's exponentials (log 2) is held in two parts, the first near the largest logit and the second small: a probability is
// exp2(z - first) exp2(-second), exact to the rounding of z alone also where z and the sum are large.

// C(i, j) = sum_k A(i, k) B(k, j); i is the table row in the first two products and the column in the gradients, j the packed row and, in
// the table's gradient, the table row.
enum EntropyProduct { entropy_logits, entropy_upstream, entropy_features_gradient, entropy_table_gradient };

struct EntropyProductArgs {
    const void* a;
    const void* b;
    uint64_t a_stride, b_stride;   // elements from row to row as they lie in memory
    uint32_t i_end, j_end, k_end;  // (j of all but the table's gradient, and its k: at most *count)
    uint32_t a_columns;            // of a's rows in memory (a multiple of 8)
    uint32_t a_plane, b_plane;     // floats: elements from one part of a row to the next
    uint32_t i_tiles;
    uint32_t j_first;              // of the launch
    uint32_t splits;               // of k
    const uint32_t* count;         // packed rows
    float to_log2;                 // scale log2 e
    float2* partial;               // logits: i_tiles x slab_rows (maximum, sum of exponentials), from row j_first on
    float* target_logit;
    const uint32_t* target;
    const float2* lse;
    const float* weight;
    uint32_t first_row;            // of the piece in the table
    void* piece;                   // upstream gradients of the logits: padded rows x piece_stride, floats in three parts piece_plane apart
    uint64_t piece_stride;
    uint32_t piece_plane;
    bool apart;                    // residuals go into the table's gradient; floats: there are any
    float* residual;               // of a row's own target's gradient, what is not in the piece: what was lost as it was rounded; floats: all of it
    float* slab;                   // splits x slab_rows x slab_stride
    uint64_t slab_stride, slab_rows;
    bool add;
    void* out;                     // table's gradient without splits: its rows from the piece's first
    uint64_t out_stride;
    const float* factor;
};

// More columns, tiles of side x side (256 or 128): rows of 16-byte aligned memory, strides in multiples of 8 elements; j of them at most. Floats come as
// three bfloat16 parts, one after the other in each row, and are multiplied by pairs of parts.
void launch_entropy_wide(EntropyProduct product, int type, uint32_t side, const EntropyProductArgs& a, uint32_t j, hipStream_t s);

// eight consecutive values, those from `valid` on zero
template <typename T>
__device__ __forceinline__ void entropy_load8(float (&x)[8], const T* p, int32_t valid) {
    typedef T Eight __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (valid >= 8) {
        const Eight v = *reinterpret_cast<const Eight*>(p);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = static_cast<float>(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = k < valid ? static_cast<float>(p[k]) : 0.0f;
    }
}

// bfloat16 parts of values whose sum is each value (three of a float: to 2^-26 of it; two of a float16: exactly). Two values at a time: one conversion, and its
// halves back as floats by a shift and a mask (five instructions a pair and part).
template <uint32_t PARTS, int N, typename V>
__device__ __forceinline__ void entropy_split(V (&parts)[PARTS], const float (&x)[N]) {
    typedef uint32_t Words __attribute__((ext_vector_type(N / 2)));
    Words words[PARTS];
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        float low = x[k], high = x[k + 1];
#pragma unroll
        for (uint32_t part = 0; part < PARTS; part++) {
            typedef float Floats __attribute__((ext_vector_type(2)));
            typedef __bf16 Halves __attribute__((ext_vector_type(2)));
            const uint32_t word = __builtin_bit_cast(uint32_t, __builtin_convertvector(Floats{low, high}, Halves));
            words[part][k / 2] = word;
            if (part + 1 < PARTS) {
                low -= __builtin_bit_cast(float, word << 16);
                high -= __builtin_bit_cast(float, word & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (uint32_t part = 0; part < PARTS; part++) parts[part] = __builtin_bit_cast(V, words[part]);
}

// few columns: products and exponentials of a tile in one kernel
struct EntropyNarrowArgs {
    const void* packed;
    const void* table;
    uint64_t packed_stride, table_stride;
    uint32_t table_rows, columns, padded;
    uint32_t own_waves;            // of a block's four that own different rows
    const uint32_t* count;
    const uint32_t* target;        // of packed rows, as the next two
    const float2* lse;
    const float* weight;
    float to_log2;
    float2* partial;               // logits: splits x padded (reference, sum of exponentials)
    float* target_logit;
    float* slab;                   // gradients: splits x slab_rows x slab_stride
    uint64_t slab_rows, slab_stride;
};
struct EntropyNarrowPlan {
    uint32_t own_waves, blocks, stream_blocks;
    uint32_t splits;               // partial results of an owned row
};
constexpr uint32_t entropy_narrow_most = 64;  // columns
EntropyNarrowPlan entropy_narrow_plan(uint32_t own, uint32_t stream, uint32_t columns, int type);
void launch_entropy_narrow(EntropyProduct product, int type, const EntropyNarrowArgs& a, const EntropyNarrowPlan& p, hipStream_t s);

// up to 64 rows without a gradient (n, rows and columns at least 1)
constexpr uint32_t entropy_few_most = 64;
size_t entropy_few_bytes(const EntropyArgs& a);
void launch_entropy_few(const EntropyArgs& a, float* loss, void* scratch, hipStream_t s);

}  // namespace efgs
