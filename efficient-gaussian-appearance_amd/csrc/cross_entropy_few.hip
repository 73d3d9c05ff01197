// The cross entropy of a few rows (up to 64) without a gradient: what answering asks for. The table's bytes bound it, so a wave takes 16 rows of the table straight
// from memory to registers, operands of v_mfma_f32_16x16x32 (floats: x4) as they come, with eight steps' loads under way at once, and multiplies them by every one of
// the few, which the block holds in LDS, 1 KB of each row at a time: nothing is packed or copied. Lane (e, q) holds 32 consecutive bytes of row e
// from 32 q on, so that a row's four lanes take a whole line; which k a lane's values have does not matter while both sides have the
// same. A second kernel joins the blocks' statistics and makes the losses.
//
// 1 row against 49,999 of 4,096 bfloat16: 96 us, 4.3 TB/s (a copy reaches 5.1); blocks that begin at different columns 102, loads past the caches 105, a row's
// columns shared by the block's waves 103. 37 against 30,011 of 1,000 float16: 21 us, where each block stages 74 KB of rows for 128 KB of the table (28 past the caches, which hold this table; with the few rows through the
// caches instead of LDS 36).
#include <algorithm>
#include <type_traits>

#include "cross_entropy.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

constexpr uint32_t block = 256, waves = 4;
constexpr float infinity = __builtin_inff(), ln_2 = 0.6931471805599453f;

struct FewArgs {
    const void* features;
    const void* table;
    const void* targets;
    uint64_t feature_stride, table_stride;
    uint32_t n, rows, columns, target_bytes;
    float to_log2;
    float2* partial;       // blocks x entropy_few_most (maximum, sum of exponentials)
    float* target_logit;   // of each row
    uint32_t blocks;
    bool each, mean;
    float* loss;
};

__device__ __forceinline__ uint32_t target_at(const FewArgs& a, uint32_t i) {
    const int64_t t = a.target_bytes == 8 ? static_cast<const int64_t*>(a.targets)[i] : static_cast<const int32_t*>(a.targets)[i];
    return static_cast<uint64_t>(t) < a.rows ? static_cast<uint32_t>(t) : entropy_none;
}

template <typename T> constexpr uint32_t width = 16 / sizeof(T);   // values of 16 bytes
template <typename T> using Piece = T __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));

template <typename T>
__device__ __forceinline__ Piece<T> guarded(const T* p, int32_t valid) {
    Piece<T> x{};
#pragma unroll
    for (int32_t k = 0; k < static_cast<int32_t>(width<T>); k++)
        if (k < valid) x[k] = p[k];
    return x;
}

template <typename T>
__device__ __forceinline__ floatx4 multiply(const Piece<T>& a, const Piece<T>& b, floatx4 c) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int k = 0; k < 4; k++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    }
}

// NT: tiles of 16 of the few rows
template <typename T, int NT>
__global__ __launch_bounds__(block) void entropy_few_kernel(FewArgs a) {
    constexpr uint32_t step = 8 * width<T>, depth = 8, chunk = depth * step, pitch = chunk + width<T>;  // columns; a step is a line
    __shared__ __attribute__((aligned(16))) T few[NT * 16 * pitch];
    __shared__ float2 joined[waves][NT * 16];
    const uint32_t lane = threadIdx.x & 63u, e = lane & 15u, q = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t first = (blockIdx.x * waves + wave) * 16;
    const T* const row = static_cast<const T*>(a.table) + min(first + e, a.rows - 1) * a.table_stride + q * 2 * width<T>;
    uint32_t at[NT];
#pragma unroll
    for (uint32_t t = 0; t < NT; t++) at[t] = min(t * 16 + e, a.n - 1) * pitch + q * 2 * width<T>;
    floatx4 acc[NT] = {};
    Piece<T> x[depth][2];
    const uint32_t steps = a.columns / step, chunks = (a.columns + chunk - 1) / chunk, whole = a.columns / chunk;
    const auto load = [&](uint32_t d, uint32_t s) {
        const T* const p = row + min(s, steps - 1) * step;   // (past the end the last step's again, not multiplied)
        x[d][0] = *reinterpret_cast<const Piece<T>*>(p);
        x[d][1] = *reinterpret_cast<const Piece<T>*>(p + width<T>);
    };
    const auto multiply_step = [&](uint32_t d) {
#pragma unroll
        for (uint32_t h = 0; h < 2; h++)
#pragma unroll
            for (uint32_t t = 0; t < NT; t++)
                acc[t] = multiply<T>(x[d][h], *reinterpret_cast<const Piece<T>*>(few + at[t] + d * step + h * width<T>), acc[t]);
    };
    // the few rows' columns of a chunk; zeros past them
    const auto stage = [&](uint32_t c) {
        __syncthreads();
        constexpr uint32_t pieces = chunk / width<T>;
        for (uint32_t i = threadIdx.x; i < a.n * pieces; i += block) {
            const uint32_t n = i / pieces, column = i % pieces * width<T>;
            const T* const p = static_cast<const T*>(a.features) + n * a.feature_stride + c * chunk + column;
            const int32_t valid = static_cast<int32_t>(a.columns) - static_cast<int32_t>(c * chunk + column);
            Piece<T> v;
            if (valid >= static_cast<int32_t>(width<T>)) v = *reinterpret_cast<const Piece<T>*>(p);
            else v = guarded<T>(p, valid);
            *reinterpret_cast<Piece<T>*>(few + n * pitch + column) = v;
        }
        __syncthreads();
    };
    if (steps > 0) {
#pragma unroll
        for (uint32_t d = 0; d < depth; d++) load(d, d);
    }
    for (uint32_t c = 0; c < whole; c++) {
        stage(c);
#pragma unroll
        for (uint32_t d = 0; d < depth; d++) {
            multiply_step(d);
            load(d, (c + 1) * depth + d);
        }
    }
    if (whole < chunks) {
        stage(whole);
#pragma unroll
        for (uint32_t d = 0; d < depth; d++) {
            const uint32_t s = whole * depth + d;
            if (s == steps) {
                const int32_t valid = static_cast<int32_t>(a.columns) - static_cast<int32_t>(s * step + q * 2 * width<T>);
                x[d][0] = guarded<T>(row + s * step, valid);
                x[d][1] = guarded<T>(row + s * step + width<T>, valid - static_cast<int32_t>(width<T>));
            }
            if (s * step < a.columns) multiply_step(d);
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < NT; j++) {
        const uint32_t n = j * 16 + e, target = n < a.n ? target_at(a, n) : entropy_none;
        float z[4], top = -infinity, sum = 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) {
            const uint32_t v = first + 4 * q + r;
            z[r] = v < a.rows ? acc[j][r] * a.to_log2 : -infinity;
            if (v == target) a.target_logit[n] = z[r];
            top = fmaxf(top, z[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float from = top == -infinity ? 0.0f : top;
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f(z[r] - from);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (q == 0) joined[wave][n] = make_float2(top, sum);
    }
    __syncthreads();
    if (threadIdx.x < NT * 16) {
        float top = -infinity, sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < waves; w++) top = fmaxf(top, joined[w][threadIdx.x].x);
        const float from = top == -infinity ? 0.0f : top;
#pragma unroll
        for (uint32_t w = 0; w < waves; w++) sum += joined[w][threadIdx.x].y * __builtin_amdgcn_exp2f(joined[w][threadIdx.x].x - from);
        a.partial[blockIdx.x * entropy_few_most + threadIdx.x] = make_float2(top, sum);
    }
}

__device__ __forceinline__ float2 join(float2 x, float2 y) {
    const float top = fmaxf(x.x, y.x), from = top == -infinity ? 0.0f : top;
    return make_float2(top, x.y * __builtin_amdgcn_exp2f(x.x - from) + y.y * __builtin_amdgcn_exp2f(y.x - from));
}

constexpr uint32_t join_block = 1024;

// `lanes` (a power of two) of the few rows side by side, the blocks' statistics in as many parts as are left; one block where it adds up the losses
__global__ __launch_bounds__(join_block) void entropy_few_join_kernel(FewArgs a, uint32_t lanes) {
    __shared__ float2 parts[join_block];
    __shared__ double losses[entropy_few_most];
    const uint32_t lane = threadIdx.x & (lanes - 1u), part = threadIdx.x / lanes, step = join_block / lanes, n = blockIdx.x * lanes + lane;
    constexpr uint32_t at_once = 4;
    float2 x = make_float2(-infinity, 0.0f);
    for (uint32_t b = part; b < a.blocks; b += at_once * step) {
        float2 y[at_once];
#pragma unroll
        for (uint32_t k = 0; k < at_once; k++) y[k] = a.partial[min(b + k * step, a.blocks - 1) * entropy_few_most + min(n, a.n - 1)];
#pragma unroll
        for (uint32_t k = 0; k < at_once; k++)
            if (b + k * step < a.blocks) x = join(x, y[k]);
    }
    parts[threadIdx.x] = x;
    for (uint32_t half = join_block / 2; half >= lanes; half /= 2) {
        __syncthreads();
        if (threadIdx.x < half) parts[threadIdx.x] = join(parts[threadIdx.x], parts[threadIdx.x + half]);
    }
    __syncthreads();
    if (threadIdx.x < lanes) {
        const bool counts = n < a.n && target_at(a, n) != entropy_none;
        const float2 s = parts[threadIdx.x];
        const float loss = counts ? ((s.x - a.target_logit[n]) + log2f(s.y)) * ln_2 : 0.0f;
        if (a.each && n < a.n) a.loss[n] = loss;
        losses[threadIdx.x] = loss;
    }
    __syncthreads();
    if (threadIdx.x == 0 && !a.each) {
        double total = 0.0;
        uint32_t count = 0;
        for (uint32_t k = 0; k < a.n; k++) {
            total += losses[k];
            count += target_at(a, k) != entropy_none;
        }
        *a.loss = static_cast<float>(a.mean ? total / max(count, 1u) : total);
    }
}

uint32_t tiles_of(uint32_t n) { return (n + 15) / 16; }
uint32_t blocks_of(uint32_t rows) { return div_up(rows, waves * 16); }

template <typename T>
void launch(const FewArgs& a, hipStream_t s) {
    const dim3 grid(a.blocks);
    switch (tiles_of(a.n)) {
        case 1: hipLaunchKernelGGL((entropy_few_kernel<T, 1>), grid, dim3(block), 0, s, a); break;
        case 2: hipLaunchKernelGGL((entropy_few_kernel<T, 2>), grid, dim3(block), 0, s, a); break;
        case 3: hipLaunchKernelGGL((entropy_few_kernel<T, 3>), grid, dim3(block), 0, s, a); break;
        default: hipLaunchKernelGGL((entropy_few_kernel<T, 4>), grid, dim3(block), 0, s, a); break;
    }
}

}  // namespace

size_t entropy_few_bytes(const EntropyArgs& a) {
    return (static_cast<size_t>(blocks_of(a.rows)) * sizeof(float2) + sizeof(float)) * entropy_few_most;
}

void launch_entropy_few(const EntropyArgs& e, float* loss, void* scratch, hipStream_t s) {
    FewArgs a{};
    a.features = e.features;
    a.table = e.table;
    a.targets = e.targets;
    a.feature_stride = e.feature_stride;
    a.table_stride = e.table_stride;
    a.n = e.n;
    a.rows = e.rows;
    a.columns = e.columns;
    a.target_bytes = static_cast<uint32_t>(e.target_bytes);
    a.to_log2 = e.scale * 1.4426950408889634f;
    a.blocks = blocks_of(e.rows);
    a.partial = static_cast<float2*>(scratch);
    a.target_logit = reinterpret_cast<float*>(a.partial + static_cast<size_t>(a.blocks) * entropy_few_most);
    a.each = e.each;
    a.mean = e.mean;
    a.loss = loss;
    if (e.type == type_float) launch<float>(a, s);
    else if (e.type == type_bfloat16) launch<__bf16>(a, s);
    else launch<_Float16>(a, s);
    uint32_t lanes = 1;
    while (lanes < e.n && !(e.each && lanes == 4)) lanes *= 2;
    hipLaunchKernelGGL(entropy_few_join_kernel, dim3(div_up(e.n, lanes)), dim3(join_block), 0, s, a, lanes);
}

}  // namespace efgs
