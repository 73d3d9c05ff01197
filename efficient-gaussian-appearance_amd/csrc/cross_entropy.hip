// Softmax cross entropy of rows x_n against every row w_v of a table, without the logits in memory, and its gradients:
//
//   z_nv = scale x_n . w_v,  loss_n = log sum_v exp z_nv - z_n,target(n)
//   g_nv = upstream_n (p_nv - [v = target(n)]),  dx_n = scale sum_v g_nv w_v,  dw_v = scale sum_n g_nv x_n
//
// A target outside the table leaves its row out. The rows that count are packed first (in their order, columns padded with
// zeros), so that rows left out cost nothing behind that and nothing that stands in them reaches a sum. The forward is one
// matrix product whose tiles leave, for each row, the maximum and the sum of exponentials over the tile's part of the table; a
// second kernel joins them. The backward computes the logits again by pieces of the table, writes g of a piece, and multiplies
// it by the piece and, transposed, by the rows. Statistics and sums are in 32 bits (logits in units of log 2), the sum over rows in 64.
#include <algorithm>
#include <type_traits>

#include "internal.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float log2_e = 1.4426950408889634f, ln_2 = 0.6931471805599453f, infinity = __builtin_inff();
constexpr uint32_t none = 0xffffffffu;
constexpr uint32_t row_tile = 256;        // packed rows come in multiples of it
constexpr uint32_t column_tile = 64;      // so do their columns
constexpr uint32_t rank_block = 1024;
constexpr uint32_t count_alone = 16384;   // largest list that every block counts by itself

template <typename T, int W> using Part = T __attribute__((ext_vector_type(W), aligned(sizeof(T))));

uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// ---- the rows that count ---------------------------------------------------------------------------------------------

struct Packing {
    const void* targets;
    const void* features;
    uint64_t feature_stride;
    uint32_t n, padded, rows, columns, padded_columns, target_bytes;
    uint32_t* chunk_counts;  // null: short lists
    uint32_t* count;         // rows that count
    uint32_t* row_of;        // packed row -> row
    uint32_t* packed_of;     // row -> packed row, or none
    uint32_t* target;        // of a packed row; none past them
    void* packed;            // padded x padded_columns
};

__device__ __forceinline__ uint32_t target_at(const Packing& a, uint32_t i) {
    const int64_t t = a.target_bytes == 8 ? static_cast<const int64_t*>(a.targets)[i] : static_cast<const int32_t*>(a.targets)[i];
    return static_cast<uint64_t>(t) < a.rows ? static_cast<uint32_t>(t) : none;
}

__device__ __forceinline__ uint32_t block_total(uint32_t v, uint32_t* lds) {
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t w = 0; w < rank_block / 64; w++) sum += lds[w];
    return sum;
}

__global__ __launch_bounds__(rank_block) void entropy_count_kernel(Packing a) {
    __shared__ uint32_t lds[rank_block / 64];
    const uint32_t i = blockIdx.x * rank_block + threadIdx.x;
    const uint32_t total = block_total(i < a.n && target_at(a, i) != none, lds);
    if (threadIdx.x == 0) a.chunk_counts[blockIdx.x] = total;
}

// a block a chunk of rank_block rows
__global__ __launch_bounds__(rank_block) void entropy_rank_kernel(Packing a) {
    __shared__ uint32_t lds[rank_block / 64], waves[rank_block / 64];
    uint32_t before = 0, all = 0;
    if (a.chunk_counts) {
        for (uint32_t c = threadIdx.x; c < gridDim.x; c += rank_block) {
            const uint32_t k = a.chunk_counts[c];
            all += k;
            before += c < blockIdx.x ? k : 0u;
        }
    } else {
        for (uint32_t i = threadIdx.x; i < a.n; i += rank_block) {
            const bool counts = target_at(a, i) != none;
            all += counts;
            before += counts && i < blockIdx.x * rank_block;
        }
    }
    before = block_total(before, lds);
    all = block_total(all, lds);
    const uint32_t i = blockIdx.x * rank_block + threadIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t target = i < a.n ? target_at(a, i) : none;
    const uint64_t ballot = __ballot(target != none);
    if (lane == 0) waves[wave] = static_cast<uint32_t>(__popcll(ballot));
    __syncthreads();
    uint32_t at = before + static_cast<uint32_t>(__popcll(ballot & ((1ull << lane) - 1ull)));
    for (uint32_t w = 0; w < wave; w++) at += waves[w];
    if (i < a.n) a.packed_of[i] = target == none ? none : at;
    if (target != none) {
        a.row_of[at] = i;
        a.target[at] = target;
    }
    if (i >= all && i < a.padded) {
        a.row_of[i] = none;
        a.target[i] = none;
    }
    if (i == 0) *a.count = all;
}

// Sixteen bytes a thread; rows past those that count are zeros, up to a whole tile.
template <typename T>
__global__ __launch_bounds__(256) void entropy_pack_kernel(Packing a) {
    constexpr uint32_t W = 16 / sizeof(T);
    const uint32_t parts = a.padded_columns / W, end = (*a.count + row_tile - 1) / row_tile * row_tile;
    const uint64_t items = static_cast<uint64_t>(end) * parts, step = static_cast<uint64_t>(gridDim.x) * 256u;
    for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < items; t += step) {
        const uint32_t m = static_cast<uint32_t>(t / parts), column = static_cast<uint32_t>(t - static_cast<uint64_t>(m) * parts) * W;
        const uint32_t row = a.row_of[m];
        Part<T, W> v{};
        if (row != none && column < a.columns) {
            const T* const p = static_cast<const T*>(a.features) + row * a.feature_stride + column;
            if (column + W <= a.columns) v = *reinterpret_cast<const Part<T, W>*>(p);
            else
#pragma unroll
                for (uint32_t k = 0; k < W; k++)
                    if (column + k < a.columns) v[k] = p[k];
        }
        *reinterpret_cast<Part<T, W>*>(static_cast<T*>(a.packed) + t * W) = v;
    }
}

// ---- matrix products in 32 bits ----------------------------------------------------------------------------------------
// C(i, j) = sum_k A(i, k) B(k, j), 128 x 128 to a block of four waves (64 x 64 each), v_mfma_f32_16x16x4_f32. A lane's results are
// four consecutive i at one j: i is the table row in the logits, so that a row's maximum and sum stay mostly in
// registers, and the column in the gradients, which are stored along it.

constexpr uint32_t tile = 128, tile_k = 16, tile_pitch = tile + 4, tile_block = 256;

enum Product { logits, upstream_piece, features_gradient, table_gradient };

struct ProductArgs {
    const void* a;
    const void* b;
    uint64_t a_stride, b_stride;   // elements from row to row as they lie in memory
    uint32_t i_end, j_end, k_end;  // (j of the logits and of the rows' gradient, k of the table's: at most *count)
    uint32_t i_tiles;
    uint32_t j_first;              // of the launch
    uint32_t splits;               // of k, over gridDim.y
    const uint32_t* count;
    float to_log2;                 // scale log2 e
    float2* partial;               // logits: i_tiles x slab_rows (maximum, sum of exponentials), from row j_first on
    float* target_logit;
    const uint32_t* target;
    const float* lse;
    const float* weight;
    uint32_t first_row;            // of the piece in the table
    float* piece;                  // upstream_piece: padded x piece_stride
    uint64_t piece_stride;
    float* slab;                   // splits x j_slab x slab_stride
    uint64_t slab_stride, slab_rows;
    bool add;
    void* out;                     // table_gradient without splits: the gradient's rows from the piece's first
    uint64_t out_stride;
    const float* factor;
};

// eight consecutive values, those from `valid` on zero
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, int64_t valid) {
    if (valid >= 8) {
        const Part<T, 8> v = *reinterpret_cast<const Part<T, 8>*>(p);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = static_cast<float>(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = k < valid ? static_cast<float>(p[k]) : 0.0f;
    }
}

// A tile of an operand: ALONG_K where its memory runs along k, else along i (or j).
template <typename T, bool ALONG_K>
__device__ __forceinline__ void load_tile(float (&x)[8], const void* base, uint64_t stride, uint32_t first, uint32_t end, uint32_t k, uint32_t k_end) {
    const uint32_t t = threadIdx.x;
    const uint32_t row = ALONG_K ? first + t / 2 : k + t / 16, column = ALONG_K ? k + t % 2 * 8 : first + t % 16 * 8;
    const uint32_t rows = ALONG_K ? end : k_end, columns = ALONG_K ? k_end : end;
    const int64_t valid = row < rows ? static_cast<int64_t>(columns) - column : 0;
    load8<T>(x, static_cast<const T*>(base) + static_cast<uint64_t>(row) * stride + column, valid);
}

template <bool ALONG_K>
__device__ __forceinline__ void store_tile(float (*lds)[tile_pitch], const float (&x)[8]) {
    const uint32_t t = threadIdx.x;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if constexpr (ALONG_K) lds[t % 2 * 8 + k][t / 2] = x[k];
        else lds[t / 16][t % 16 * 8 + k] = x[k];
    }
}

template <typename T, Product P>
__global__ __launch_bounds__(tile_block) void entropy_product_kernel(ProductArgs a) {
    using B = std::conditional_t<P == logits || P == upstream_piece, T, float>;
    constexpr bool a_along_k = P == logits || P == upstream_piece, b_along_k = P != table_gradient;
    __shared__ float lds_a[tile_k][tile_pitch], lds_b[tile_k][tile_pitch];
    __shared__ float2 joined[2][tile];
    const uint32_t i0 = blockIdx.x % a.i_tiles * tile, j0 = a.j_first + blockIdx.x / a.i_tiles * tile;
    const uint32_t count = *a.count;
    const uint32_t j_end = P == table_gradient ? a.j_end : count;
    if (j0 >= (P == upstream_piece ? (count + row_tile - 1) / row_tile * row_tile : j_end)) return;
    const uint32_t k_all = P == table_gradient ? count : a.k_end;
    const uint32_t k_each = (k_all / a.splits + tile_k) / tile_k * tile_k, k_first = min(blockIdx.y * k_each, k_all), k_end = min(k_first + k_each, k_all);
    const uint32_t lane = threadIdx.x & 63u, e = lane & 15u, q = lane >> 4, wave = threadIdx.x >> 6, wi = wave & 1u, wj = wave >> 1;
    floatx4 acc[4][4] = {};
    float xa[8], xb[8];
    if (k_first < k_end) {
        load_tile<T, a_along_k>(xa, a.a, a.a_stride, i0, a.i_end, k_first, k_end);
        load_tile<B, b_along_k>(xb, a.b, a.b_stride, j0, j_end, k_first, k_end);
    }
    for (uint32_t k = k_first; k < k_end; k += tile_k) {
        __syncthreads();
        store_tile<a_along_k>(lds_a, xa);
        store_tile<b_along_k>(lds_b, xb);
        __syncthreads();
        if (k + tile_k < k_end) {
            load_tile<T, a_along_k>(xa, a.a, a.a_stride, i0, a.i_end, k + tile_k, k_end);
            load_tile<B, b_along_k>(xb, a.b, a.b_stride, j0, j_end, k + tile_k, k_end);
        }
#pragma unroll
        for (uint32_t s = 0; s < tile_k / 4; s++) {
            float fa[4], fb[4];
#pragma unroll
            for (uint32_t t = 0; t < 4; t++) {
                fa[t] = lds_a[4 * s + q][wi * 64 + t * 16 + e];
                fb[t] = lds_b[4 * s + q][wj * 64 + t * 16 + e];
            }
#pragma unroll
            for (uint32_t ti = 0; ti < 4; ti++)
#pragma unroll
                for (uint32_t tj = 0; tj < 4; tj++) acc[ti][tj] = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[ti], fb[tj], acc[ti][tj], 0, 0, 0);
        }
    }
    const uint32_t i_lane = i0 + wi * 64 + 4 * q, j_lane = j0 + wj * 64 + e;  // results: i_lane + 16 ti + r, j_lane + 16 tj
    if constexpr (P == logits) {
#pragma unroll
        for (uint32_t tj = 0; tj < 4; tj++) {
            const uint32_t j = j_lane + tj * 16, target = a.target[j];
            float top = -infinity, sum = 0.0f;
#pragma unroll
            for (uint32_t ti = 0; ti < 4; ti++)
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    const uint32_t i = i_lane + ti * 16 + r;
                    const float z = i < a.i_end ? acc[ti][tj][r] * a.to_log2 : -infinity;
                    acc[ti][tj][r] = z;
                    if (i == target) a.target_logit[j] = z;
                    top = fmaxf(top, z);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top == -infinity ? 0.0f : top;
#pragma unroll
            for (uint32_t ti = 0; ti < 4; ti++)
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f(acc[ti][tj][r] - from);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (q == 0) joined[wi][wj * 64 + tj * 16 + e] = make_float2(top, sum);
        }
        __syncthreads();
        if (threadIdx.x < tile) {
            const float2 x = joined[0][threadIdx.x], y = joined[1][threadIdx.x];
            const float top = fmaxf(x.x, y.x), from = top == -infinity ? 0.0f : top;
            const float sum = x.y * __builtin_amdgcn_exp2f(x.x - from) + y.y * __builtin_amdgcn_exp2f(y.x - from);
            a.partial[(i0 / tile) * a.slab_rows + (j0 - a.j_first) + threadIdx.x] = make_float2(top, sum);
        }
    } else if constexpr (P == upstream_piece) {
#pragma unroll
        for (uint32_t tj = 0; tj < 4; tj++) {
            const uint32_t j = j_lane + tj * 16, target = a.target[j];
            const bool counts = target != none;
            const float lse = counts ? a.lse[j] : 0.0f, weight = counts ? a.weight[j] : 0.0f;
#pragma unroll
            for (uint32_t ti = 0; ti < 4; ti++) {
                const uint32_t i = i_lane + ti * 16;
                floatx4 g;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    const float p = __builtin_amdgcn_exp2f(acc[ti][tj][r] * a.to_log2 - lse) - (a.first_row + i + r == target ? 1.0f : 0.0f);
                    g[r] = counts && i + r < a.i_end ? p * weight : 0.0f;
                }
                *reinterpret_cast<floatx4*>(a.piece + j * a.piece_stride + i) = g;
            }
        }
    } else {
        const bool direct = P == table_gradient && a.out;
        const float factor = direct ? *a.factor : 1.0f;
#pragma unroll
        for (uint32_t tj = 0; tj < 4; tj++) {
            const uint32_t j = j_lane + tj * 16;
            if (j >= j_end) continue;
#pragma unroll
            for (uint32_t ti = 0; ti < 4; ti++) {
                const uint32_t i = i_lane + ti * 16;
                if (direct) {
                    T* const out = static_cast<T*>(a.out) + j * a.out_stride + i;
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++)
                        if (i + r < a.i_end) out[r] = static_cast<T>(acc[ti][tj][r] * factor);
                } else if (i < a.slab_stride) {
                    floatx4* const out = reinterpret_cast<floatx4*>(a.slab + (blockIdx.y * a.slab_rows + j) * a.slab_stride + i);
                    *out = a.add ? *out + acc[ti][tj] : acc[ti][tj];
                }
            }
        }
    }
}

// ---- joins -----------------------------------------------------------------------------------------------------------

struct JoinArgs {
    const float2* partial;
    uint32_t tiles;
    uint32_t first_row, rows;  // of packed rows: a launch's
    uint32_t n;
    const uint32_t* count;
    const uint32_t* row_of;
    const uint32_t* packed_of;
    const float* target_logit;
    float* lse;
    float* losses;         // of each row, or null
    double* sums;          // of each block's rows
};

constexpr uint32_t join_rows = 64, join_parts = 16;

// 64 packed rows a block, the tiles of the table in sixteen parts
__global__ __launch_bounds__(join_rows * join_parts) void entropy_join_kernel(JoinArgs a) {
    __shared__ float2 parts[join_parts][join_rows];
    const uint32_t lane = threadIdx.x & (join_rows - 1u), part = threadIdx.x / join_rows, at = blockIdx.x * join_rows + lane, row = a.first_row + at;
    const uint32_t count = *a.count;
    const bool counts = row < count;
    float top = -infinity, sum = 0.0f;
    if (counts)
        for (uint32_t t = part; t < a.tiles; t += join_parts) {
            const float2 x = a.partial[static_cast<uint64_t>(t) * a.rows + at];
            const float higher = fmaxf(top, x.x), from = higher == -infinity ? 0.0f : higher;
            sum = sum * __builtin_amdgcn_exp2f(top - from) + x.y * __builtin_amdgcn_exp2f(x.x - from);
            top = higher;
        }
    parts[part][lane] = make_float2(top, sum);
    __syncthreads();
    if (part != 0) return;
    for (uint32_t k = 1; k < join_parts; k++) {
        const float2 x = parts[k][lane];
        const float higher = fmaxf(top, x.x), from = higher == -infinity ? 0.0f : higher;
        sum = sum * __builtin_amdgcn_exp2f(top - from) + x.y * __builtin_amdgcn_exp2f(x.x - from);
        top = higher;
    }
    const float lse = top + log2f(sum);
    const float loss = counts ? (lse - a.target_logit[row]) * ln_2 : 0.0f;
    if (counts) a.lse[row] = lse;
    if (a.losses) {
        if (counts) a.losses[a.row_of[row]] = loss;
        if (row < a.n && a.packed_of[row] == none) a.losses[row] = 0.0f;
        return;
    }
    double total = loss;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    if (lane == 0) a.sums[row / join_rows] = total;
}

__global__ __launch_bounds__(256) void entropy_total_kernel(const double* sums, uint32_t blocks, const uint32_t* count, bool mean, float* loss) {
    __shared__ double lds[4];
    double total = 0.0;
    for (uint32_t b = threadIdx.x; b < blocks; b += 256) total += sums[b];
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        total = (lds[0] + lds[1]) + (lds[2] + lds[3]);
        *loss = static_cast<float>(mean ? total / max(*count, 1u) : total);
    }
}

// ---- backward's ends ---------------------------------------------------------------------------------------------------

struct WeightArgs {
    const float* upstream;   // one, or one for each row
    const uint32_t* count;
    const uint32_t* row_of;
    uint32_t padded;
    bool each, mean;
    float scale;
    float* weight;           // of packed rows
    float* factor;           // of the sums
};

__global__ __launch_bounds__(256) void entropy_weights_kernel(WeightArgs a) {
    const uint32_t m = blockIdx.x * 256 + threadIdx.x, count = *a.count;
    if (m < a.padded) a.weight[m] = m >= count ? 0.0f : a.each ? a.upstream[a.row_of[m]] : 1.0f;
    if (m == 0) *a.factor = a.each ? a.scale : a.scale * *a.upstream / (a.mean ? static_cast<float>(max(count, 1u)) : 1.0f);
}

// sums of the splits, scaled; rows without a packed one are zeros
template <typename T>
__global__ __launch_bounds__(256) void entropy_gather_kernel(const float* slab, uint64_t slab_rows, uint64_t slab_stride, uint32_t splits,
                                                             const uint32_t* packed_of, uint32_t rows, uint32_t columns, const float* factor, T* out) {
    const uint64_t items = static_cast<uint64_t>(rows) * columns, step = static_cast<uint64_t>(gridDim.x) * 256u;
    const float f = *factor;
    for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < items; t += step) {
        const uint32_t row = static_cast<uint32_t>(t / columns), column = static_cast<uint32_t>(t - static_cast<uint64_t>(row) * columns);
        const uint32_t m = packed_of ? packed_of[row] : row;
        float sum = 0.0f;
        if (m != none)
            for (uint32_t s = 0; s < splits; s++) sum += slab[(s * slab_rows + m) * slab_stride + column];
        out[t] = static_cast<T>(m == none ? 0.0f : sum * f);
    }
}

// ---- sizes and buffers -------------------------------------------------------------------------------------------------

// hands out 256-byte aligned parts of a buffer, or, without one, counts them
class Carver {
  public:
    explicit Carver(void* base) : base_(static_cast<char*>(base)) {}
    template <typename T>
    T* take(uint64_t n) {
        char* const p = base_ ? base_ + used_ : nullptr;
        used_ += round_up(std::max<uint64_t>(n, 1) * sizeof(T), 256);
        return reinterpret_cast<T*>(p);
    }
    size_t used() const { return used_; }

  private:
    char* base_;
    size_t used_ = 0;
};

uint32_t type_bytes(int type) { return type == type_float ? 4 : 2; }

struct Saved {
    uint32_t* count;
    uint32_t* row_of;
    uint32_t* packed_of;
    uint32_t* target;
    float* lse;
    void* packed;
    uint32_t padded, padded_columns;
    size_t bytes;
    Saved(const EntropyArgs& a, void* base) {
        Carver c(base);
        padded = static_cast<uint32_t>(round_up(std::max(a.n, 1u), row_tile));
        padded_columns = static_cast<uint32_t>(round_up(a.columns, column_tile));
        count = c.take<uint32_t>(1);
        row_of = c.take<uint32_t>(padded);
        packed_of = c.take<uint32_t>(padded);
        target = c.take<uint32_t>(padded);
        lse = c.take<float>(padded);
        packed = c.take<char>(static_cast<uint64_t>(padded) * padded_columns * type_bytes(a.type));
        bytes = c.used();
    }
};

constexpr uint64_t partial_bytes = 256ull << 20;  // of the tiles' statistics at once
constexpr uint64_t piece_bytes = 256ull << 20;    // of a piece's upstream gradients
constexpr uint64_t most_blocks = 1ull << 23;      // of a launch of 256 threads (32 bits of threads)

struct ForwardScratch {
    uint32_t* chunk_counts;
    float2* partial;
    float* target_logit;
    double* sums;
    uint32_t tiles, rows_at_once;
    size_t bytes;
    ForwardScratch(const EntropyArgs& a, const Saved& s, void* base) {
        Carver c(base);
        tiles = div_up(a.rows, tile);
        chunk_counts = c.take<uint32_t>(div_up(s.padded, rank_block));
        const uint64_t most = std::min(partial_bytes / sizeof(float2), most_blocks * tile) / std::max(tiles, 1u);
        rows_at_once = static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(most / row_tile * row_tile, row_tile), s.padded));
        partial = c.take<float2>(static_cast<uint64_t>(tiles) * rows_at_once);
        target_logit = c.take<float>(s.padded);
        sums = c.take<double>(s.padded / join_rows);
        bytes = c.used();
    }
};

// how often a product's k is split so that its blocks fill the GPU
uint32_t splits_for(uint64_t tiles, uint64_t k) {
    const uint64_t wanted = tiles >= 512 ? 1 : (1024 + tiles - 1) / std::max<uint64_t>(tiles, 1);
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min({wanted, k / 256, static_cast<uint64_t>(64)})));
}

struct BackwardScratch {
    float* weight;
    float* factor;
    float* piece;
    float* features_slab;
    float* table_slab;
    uint32_t piece_rows, pieces;
    uint32_t features_splits, table_splits;
    size_t bytes;
    BackwardScratch(const EntropyArgs& a, const Saved& s, void* base) {
        Carver c(base);
        const uint64_t most = std::max<uint64_t>(piece_bytes / (static_cast<uint64_t>(s.padded) * sizeof(float)) / 256 * 256, 256);
        const uint64_t all = round_up(std::max(a.rows, 1u), 256);
        pieces = div_up(all, std::min(most, all));
        piece_rows = static_cast<uint32_t>(round_up(div_up(all, pieces), 256));
        pieces = div_up(all, piece_rows);
        const uint64_t column_tiles = div_up(std::max(a.columns, 1u), tile);
        features_splits = splits_for(s.padded / tile * column_tiles, piece_rows);
        table_splits = splits_for(piece_rows / tile * column_tiles, s.padded);
        weight = c.take<float>(s.padded);
        factor = c.take<float>(1);
        piece = c.take<float>(static_cast<uint64_t>(s.padded) * piece_rows);
        features_slab = c.take<float>(static_cast<uint64_t>(features_splits) * s.padded * s.padded_columns);
        table_slab = table_splits > 1 ? c.take<float>(static_cast<uint64_t>(table_splits) * piece_rows * s.padded_columns) : nullptr;
        bytes = c.used();
    }
};

template <typename F>
void with_type(int type, F&& f) {
    if (type == type_float) f(float{});
    else if (type == type_bfloat16) f(__bf16{});
    else f(static_cast<_Float16>(0.0f));
}

constexpr uint32_t copy_blocks = 1u << 16;

uint32_t copy_grid(uint64_t items) { return static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>((items + 255) / 256, 1), copy_blocks)); }

void launch_packing(const EntropyArgs& a, const Saved& s, uint32_t* chunk_counts, hipStream_t stream) {
    Packing p{};
    p.targets = a.targets;
    p.features = a.features;
    p.feature_stride = a.feature_stride;
    p.n = a.n;
    p.padded = s.padded;
    p.rows = a.rows;
    p.columns = a.columns;
    p.padded_columns = s.padded_columns;
    p.target_bytes = static_cast<uint32_t>(a.target_bytes);
    p.chunk_counts = a.n > count_alone ? chunk_counts : nullptr;
    p.count = s.count;
    p.row_of = s.row_of;
    p.packed_of = s.packed_of;
    p.target = s.target;
    p.packed = s.packed;
    const dim3 chunks(div_up(s.padded, rank_block));
    if (p.chunk_counts) hipLaunchKernelGGL(entropy_count_kernel, chunks, dim3(rank_block), 0, stream, p);
    hipLaunchKernelGGL(entropy_rank_kernel, chunks, dim3(rank_block), 0, stream, p);
    if (a.columns == 0) return;
    const uint32_t blocks = copy_grid(static_cast<uint64_t>(s.padded) * s.padded_columns * type_bytes(a.type) / 16);
    with_type(a.type, [&](auto t) { hipLaunchKernelGGL(entropy_pack_kernel<decltype(t)>, dim3(blocks), dim3(256), 0, stream, p); });
}

}  // namespace

bool entropy_fits(const EntropyArgs& a) {
    const Saved s(a, nullptr);
    const uint64_t row_tiles = s.padded / tile, column_tiles = div_up(std::max(a.columns, 1u), tile);
    const uint64_t most_tiles = std::max<uint64_t>(row_tiles, div_up(a.rows, tile));
    return most_tiles * std::max<uint64_t>(column_tiles, row_tile / tile) <= most_blocks;
}

size_t entropy_saved_bytes(const EntropyArgs& a) { return Saved(a, nullptr).bytes; }
size_t entropy_forward_bytes(const EntropyArgs& a) { return ForwardScratch(a, Saved(a, nullptr), nullptr).bytes; }
size_t entropy_backward_bytes(const EntropyArgs& a) { return BackwardScratch(a, Saved(a, nullptr), nullptr).bytes; }

bool launch_entropy_forward(const EntropyArgs& a, float* loss, void* saved, void* scratch, hipStream_t stream) {
    const Saved s(a, saved);
    const ForwardScratch f(a, s, scratch);
    launch_packing(a, s, f.chunk_counts, stream);
    for (uint32_t first = 0; first < s.padded; first += f.rows_at_once) {
        const uint32_t rows = std::min(s.padded - first, f.rows_at_once);
        if (a.rows > 0) {
            ProductArgs p{};
            p.a = a.table;
            p.a_stride = a.table_stride;
            p.b = s.packed;
            p.b_stride = s.padded_columns;
            p.i_end = a.rows;
            p.k_end = a.columns;
            p.i_tiles = f.tiles;
            p.j_first = first;
            p.splits = 1;
            p.count = s.count;
            p.to_log2 = a.scale * log2_e;
            p.partial = f.partial;
            p.slab_rows = rows;
            p.target_logit = f.target_logit;
            p.target = s.target;
            with_type(a.type, [&](auto t) {
                hipLaunchKernelGGL((entropy_product_kernel<decltype(t), logits>), dim3(f.tiles * (rows / tile)), dim3(tile_block), 0, stream, p);
            });
        }
        const JoinArgs j{f.partial, f.tiles, first, rows, a.n, s.count, s.row_of, s.packed_of, f.target_logit, s.lse, a.each ? loss : nullptr, f.sums};
        hipLaunchKernelGGL(entropy_join_kernel, dim3(rows / join_rows), dim3(join_rows * join_parts), 0, stream, j);
    }
    if (!a.each) hipLaunchKernelGGL(entropy_total_kernel, dim3(1), dim3(256), 0, stream, f.sums, s.padded / join_rows, s.count, a.mean, loss);
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

bool launch_entropy_backward(const EntropyArgs& a, const float* upstream, const void* saved, void* grad_features, void* grad_table, void* scratch,
                             hipStream_t stream) {
    if (a.columns == 0) return true;
    const Saved s(a, const_cast<void*>(saved));
    const BackwardScratch w(a, s, scratch);
    const WeightArgs weights{upstream, s.count, s.row_of, s.padded, a.each, a.mean, a.scale, w.weight, w.factor};
    hipLaunchKernelGGL(entropy_weights_kernel, dim3(div_up(s.padded, 256)), dim3(256), 0, stream, weights);
    const uint32_t row_tiles = s.padded / tile, column_tiles = div_up(a.columns, tile);
    for (uint32_t piece = 0; piece < w.pieces && a.rows > 0; piece++) {
        const uint32_t first = piece * w.piece_rows, rows = std::min(a.rows - first, w.piece_rows);
        with_type(a.type, [&](auto t) {
            using T = decltype(t);
            const T* const table = static_cast<const T*>(a.table) + first * a.table_stride;
            ProductArgs p{};
            p.a = table;
            p.a_stride = a.table_stride;
            p.b = s.packed;
            p.b_stride = s.padded_columns;
            p.i_end = rows;
            p.k_end = a.columns;
            p.i_tiles = w.piece_rows / tile;
            p.splits = 1;
            p.count = s.count;
            p.to_log2 = a.scale * log2_e;
            p.target = s.target;
            p.lse = s.lse;
            p.weight = w.weight;
            p.first_row = first;
            p.piece = w.piece;
            p.piece_stride = w.piece_rows;
            hipLaunchKernelGGL((entropy_product_kernel<T, upstream_piece>), dim3(p.i_tiles * row_tiles), dim3(tile_block), 0, stream, p);
            ProductArgs x{};
            x.count = s.count;
            x.i_end = a.columns;
            x.i_tiles = column_tiles;
            x.slab_stride = s.padded_columns;
            if (grad_features) {
                x.a = table;
                x.a_stride = a.table_stride;
                x.b = w.piece;
                x.b_stride = w.piece_rows;
                x.k_end = rows;
                x.splits = w.features_splits;
                x.slab = w.features_slab;
                x.slab_rows = s.padded;
                x.add = piece > 0;
                hipLaunchKernelGGL((entropy_product_kernel<T, features_gradient>), dim3(column_tiles * row_tiles, x.splits), dim3(tile_block), 0, stream, x);
            }
            if (grad_table) {
                T* const out = static_cast<T*>(grad_table) + static_cast<uint64_t>(first) * a.columns;
                x.a = s.packed;
                x.a_stride = s.padded_columns;
                x.b = w.piece;
                x.b_stride = w.piece_rows;
                x.j_end = rows;
                x.splits = w.table_splits;
                x.slab = w.table_slab;
                x.slab_rows = w.piece_rows;
                x.add = false;
                x.out = x.splits > 1 ? nullptr : out;
                x.out_stride = a.columns;
                x.factor = w.factor;
                hipLaunchKernelGGL((entropy_product_kernel<T, table_gradient>), dim3(column_tiles * div_up(rows, tile), x.splits), dim3(tile_block), 0,
                                   stream, x);
                if (x.splits > 1)
                    hipLaunchKernelGGL(entropy_gather_kernel<T>, dim3(copy_grid(static_cast<uint64_t>(rows) * a.columns)), dim3(256), 0, stream,
                                       w.table_slab, w.piece_rows, s.padded_columns, x.splits, nullptr, rows, a.columns, w.factor, out);
            }
        });
    }
    if (grad_features && a.n > 0)
        with_type(a.type, [&](auto t) {
            using T = decltype(t);
            hipLaunchKernelGGL(entropy_gather_kernel<T>, dim3(copy_grid(static_cast<uint64_t>(a.n) * a.columns)), dim3(256), 0, stream, w.features_slab,
                               s.padded, s.padded_columns, w.features_splits, s.packed_of, a.n, a.columns, w.factor, static_cast<T*>(grad_features));
        });
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
