// Dropout by a counter-based generator: out = keep x / (1 - t / 2^16) (+ residual), t = round(2^16 p).
//
// Philox4x32-10 of the counter (i / 8, offset) and the key seed gives eight elements 16 bits each (element i the bits
// 16 (i mod 8) of its four words); bits below t drop the element, so that p is met to 2^-17 and the expectation of out is
// x whatever t is. Nothing of the mask is stored: the backward draws it again from the same numbers, its input the upstream gradient.
// A dropped element is zero whatever x held (an infinity or NaN too). Products and the sum are in 32 bits, rounded once.
//
// HBM bounds it: 16,383 x 4,096 bfloat16 74 us with a residual (three arrays, 5.4 TB/s), 43 without (two, 6.2 TB/s, where a copy reaches 5.1: half of it stays in
// the memory-side cache); 1,000,000 x 8 float32 12 us (5.3 TB/s). The ten rounds are 40 products of 32 bits for eight elements, under the loads.
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "philox.h"

namespace efgs {

namespace {

constexpr uint32_t dropout_block = 256, dropout_group = 8, dropout_max_blocks = 1u << 23;

template <typename T> using Group = T __attribute__((ext_vector_type(dropout_group), aligned(sizeof(T))));

struct DropoutKernelArgs {
    const void* x;
    const void* residual;
    void* out;
    uint64_t n;
    uint64_t seed, offset;
    const uint64_t* seed_at;  // on the device, or null: `seed`
    uint32_t threshold;       // 0 to 2^16
    float scale;
};

// a float32 product, a float32 sum, then rounded to T: the compiler would make one float16 instruction of the last two (as of
// the lookup's product, embedding.hip), whose one rounding now and then gives another value
template <typename T, bool RESIDUAL>
__device__ __forceinline__ T dropped_or_scaled(float x, uint32_t bits, const DropoutKernelArgs& a, float residual) {
    float y = bits < a.threshold ? 0.0f : x * a.scale;
    if constexpr (RESIDUAL) y += residual;
    if constexpr (std::is_same_v<T, _Float16>) asm("" : "+v"(y));
    return static_cast<T>(y);
}

// One group of eight elements a thread: 16 bytes of 16-bit types, 32 of floats.
template <typename T, bool RESIDUAL>
__global__ __launch_bounds__(dropout_block) void dropout_kernel(DropoutKernelArgs a) {
    const uint64_t seed = a.seed_at ? *a.seed_at : a.seed;
    const uint64_t groups = (a.n + dropout_group - 1) / dropout_group, step = static_cast<uint64_t>(gridDim.x) * dropout_block;
    for (uint64_t g = static_cast<uint64_t>(blockIdx.x) * dropout_block + threadIdx.x; g < groups; g += step) {
        const uint64_t first = g * dropout_group;
        const T* const x = static_cast<const T*>(a.x) + first;
        const T* const residual = static_cast<const T*>(a.residual) + (RESIDUAL ? first : 0);
        T* const out = static_cast<T*>(a.out) + first;
        const uint4 words = philox4x32_10(make_uint4(static_cast<uint32_t>(g), static_cast<uint32_t>(g >> 32), static_cast<uint32_t>(a.offset),
                                                     static_cast<uint32_t>(a.offset >> 32)),
                                          make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32)));
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
        if (first + dropout_group <= a.n) {
            const Group<T> v = *reinterpret_cast<const Group<T>*>(x);
            Group<T> r{}, y;
            if constexpr (RESIDUAL) r = *reinterpret_cast<const Group<T>*>(residual);
#pragma unroll
            for (uint32_t k = 0; k < dropout_group; k++)
                y[k] = dropped_or_scaled<T, RESIDUAL>(static_cast<float>(v[k]), k & 1 ? word[k / 2] >> 16 : word[k / 2] & 0xffffu, a,
                                            RESIDUAL ? static_cast<float>(r[k]) : 0.0f);
            *reinterpret_cast<Group<T>*>(out) = y;
        } else {
            for (uint32_t k = 0; first + k < a.n; k++)
                out[k] = dropped_or_scaled<T, RESIDUAL>(static_cast<float>(x[k]), word[k / 2] >> (16 * (k & 1)) & 0xffffu, a,
                                              RESIDUAL ? static_cast<float>(residual[k]) : 0.0f);
        }
    }
}

template <typename T>
void launch(const DropoutKernelArgs& a, hipStream_t s) {
    const uint64_t groups = (a.n + dropout_group - 1) / dropout_group;
    const uint32_t blocks = static_cast<uint32_t>(std::min<uint64_t>((groups + dropout_block - 1) / dropout_block, dropout_max_blocks));
    if (a.residual) hipLaunchKernelGGL((dropout_kernel<T, true>), dim3(blocks), dim3(dropout_block), 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<T, false>), dim3(blocks), dim3(dropout_block), 0, s, a);
}

}  // namespace

bool launch_dropout(const DropoutArgs& d, hipStream_t s) {
    DropoutKernelArgs a{d.x, d.residual, d.out, d.n, d.seed, d.offset, d.seed_at, d.threshold, 0.0f};
    if (d.threshold < 65536u) a.scale = static_cast<float>(65536.0 / (65536.0 - d.threshold));
    if (d.type == type_float) launch<float>(a, s);
    else if (d.type == type_bfloat16) launch<__bf16>(a, s);
    else launch<_Float16>(a, s);
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
