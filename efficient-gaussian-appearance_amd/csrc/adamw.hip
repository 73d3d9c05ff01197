// AdamW over many tensors at once, with states in 32 or in 8 bits, the decoding of 8-bit states, and the gradient norm
// over many tensors that clips a step. A launch takes the descriptors of up to 40 tensors as kernel arguments (nothing is
// copied to the device and nothing has to outlive the call); a block finds its tensor from the first blocks of all.
//
// Per element, t the step, c the clipping coefficient min(1, max_norm / (norm + 1e-6)):
//   g = c grad, m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps), lr cycled by element index
//
// 8-bit states hold r = sqrt(v) against the maximum of its block of 256 elements, and u = m / r. By Cauchy-Schwarz
// |m| <= B sqrt(v) with B = (1 - beta1) / sqrt((1 - beta2) (1 - beta1^2 / beta2)) while beta1^2 < beta2, step by step: if
// it holds before one, |beta1 m| + (1 - beta1) |g| <= sqrt(beta1^2 B^2 / beta2 + (1 - beta1)^2 / (1 - beta2)) sqrt(v') =
// B sqrt(v'). So u needs no scale, and an element whose gradients are small against its block's keeps the relative
// precision of its m (with m against a block maximum, an m that rounds to the least code over a small r is a large step).
//
// A value y >= 0 is held as the top bits, four of the mantissa, of the float y + c, counted from those of c: steps of c / 16
// up to c, 16 steps to an octave above. c = 2^-16 makes 256 codes of r (top 31/32 - c), c = 2^-8 128 codes of |u|; the sign
// is u's top bit. Codes are rounded up or down by a dither of 16 bits, in the mean to the value itself: beta2 = 0.999 moves
// r by 0.05 % of itself a step, and rounding to the nearest of steps of 3 to 6 % would never move it. The dither is a hash
// of the element's index, the step and the seed, so that a step's result depends on nothing else.
//
// An element whose new r is not finite (a gradient that is not, or whose square overflows) gets the update that the formula
// gives and a zero state, and does not count in its block's maximum: its neighbours keep theirs. Contraction is off for
// this file: every operation of the 8-bit state is rounded by itself, so that the codes follow from the formulas above.
#include "internal.h"

namespace efgs {

namespace {

constexpr uint32_t adamw_block = 256;

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bfloat4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t uint32u __attribute__((aligned(1)));

template <typename T> struct Vector4;
template <> struct Vector4<float> { using type = float4u; };
template <> struct Vector4<_Float16> { using type = half4u; };
template <> struct Vector4<__bf16> { using type = bfloat4u; };

// x[0..3] = p[0..3] in 32 bits; past `count` zeros
template <typename T>
__device__ __forceinline__ void load4(const T* p, uint32_t count, float* x) {
    if (count >= 4) {
        const typename Vector4<T>::type v = *reinterpret_cast<const typename Vector4<T>::type*>(p);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = static_cast<float>(v[k]);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = k < count ? static_cast<float>(p[k]) : 0.0f;
    }
}

// rounded to nearest even, what a cast of a tensor does
template <typename T>
__device__ __forceinline__ void store4(T* p, uint32_t count, const float* x) {
    if (count >= 4) {
        typename Vector4<T>::type v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = static_cast<T>(x[k]);
        *reinterpret_cast<typename Vector4<T>::type*>(p) = v;
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (k < count) p[k] = static_cast<T>(x[k]);
    }
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, uint32_t count) {
    if (count >= 4) return *reinterpret_cast<const uint32u*>(p);
    uint32_t v = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (k < count) v |= static_cast<uint32_t>(p[k]) << (8 * k);
    return v;
}

__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t count, uint32_t v) {
    if (count >= 4) {
        *reinterpret_cast<uint32u*>(p) = v;
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (k < count) p[k] = static_cast<uint8_t>(v >> (8 * k));
}

// maximum over the wave's lanes
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x121, 0xf, 0xf, false)));  // row_ror:1
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x122, 0xf, 0xf, false)));  // row_ror:2
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x124, 0xf, 0xf, false)));  // row_ror:4
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xf, 0xf, false)));  // row_ror:8
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(static_cast<uint32_t>(a[0]), static_cast<uint32_t>(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(static_cast<uint32_t>(b[0]), static_cast<uint32_t>(b[1]));
}

// the last of the n (<= 64) tensors whose first block is at most `block`
__device__ __forceinline__ uint32_t tensor_of_block(const uint32_t* first_block, uint32_t n, uint32_t block) {
    const uint32_t lane = threadIdx.x & 63u;
    const bool at_most = lane < n && first_block[lane] <= block;
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(__popcll(__ballot(at_most)))) - 1u;
}

struct AdamWLaunch {
    uint32_t first_block[adamw_max_tensors];
    AdamWTensorDevice tensors[adamw_max_tensors];
    AdamWGroupDevice groups[adamw_max_groups];
    const float* grad_norm;  // null: gradients as they are
    float max_grad_norm;
    uint32_t n_tensors;
};
static_assert(sizeof(AdamWLaunch) <= 4096, "kernel arguments");

// the clipping coefficient; false where the norm is not finite (the step is left out)
__device__ __forceinline__ bool clipping(const AdamWLaunch& L, float& coefficient) {
    coefficient = 1.0f;
    if (!L.grad_norm) return true;
    const float norm = *L.grad_norm;
    coefficient = fminf(L.max_grad_norm / (norm + 1e-6f), 1.0f);
    return norm < INFINITY;
}

// learning rate and decay of element i, whose position in the cycle of learning rates is `column`
__device__ __forceinline__ float updated(const AdamWGroupDevice& G, const AdamWTensorDevice& T, float p, float m, float root, uint32_t column) {
    const float update = m / (root * T.root_factor + G.eps);
    return p * G.decays[column] - G.lrs[column] * T.step_factor * update;
}

// position in the cycle of learning rates of the thread's first element
__device__ __forceinline__ uint32_t first_column(const AdamWGroupDevice& G, uint64_t block_base, uint32_t offset) {
    if (G.n_lrs == 1) return 0;
    return (static_cast<uint32_t>(block_base % G.n_lrs) + offset) % G.n_lrs;
}

__device__ __forceinline__ uint32_t next_column(const AdamWGroupDevice& G, uint32_t column) { return column + 1 == G.n_lrs ? 0 : column + 1; }

template <typename P, typename D>
__device__ __forceinline__ void step32(const AdamWTensorDevice& T, const AdamWGroupDevice& G, uint32_t block, float coefficient) {
    const uint64_t base = static_cast<uint64_t>(block) * adamw_block * 4, i = base + threadIdx.x * 4u;
    if (i >= T.n) return;
    const uint32_t count = T.n - i >= 4 ? 4u : static_cast<uint32_t>(T.n - i);
    float p[4], g[4], m[4], v[4];
    load4(static_cast<const D*>(T.grad) + i, count, g);
    load4(static_cast<const float*>(T.m) + i, count, m);
    load4(static_cast<const float*>(T.v) + i, count, v);
    load4(static_cast<const P*>(T.param) + i, count, p);
    uint32_t column = first_column(G, base, threadIdx.x * 4u);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float gk = g[k] * coefficient;
        m[k] = G.beta1 * m[k] + G.beta1_rest * gk;
        v[k] = G.beta2 * v[k] + G.beta2_rest * (gk * gk);
        p[k] = updated(G, T, p[k], m[k], sqrtf(v[k]), column);
        column = next_column(G, column);
    }
    store4(static_cast<float*>(T.m) + i, count, m);
    store4(static_cast<float*>(T.v) + i, count, v);
    store4(static_cast<P*>(T.param) + i, count, p);
}

// ---- 8-bit codes -----------------------------------------------------------------------------------------------------

constexpr uint32_t root_base = 111u * 16, ratio_base = 119u * 16;  // top bits of 2^-16 and of 2^-8
constexpr float root_c = 0x1p-16f, ratio_c = 0x1p-8f;
constexpr float root_top = 0.96875f - root_c, ratio_top = 0.96875f - ratio_c;
constexpr float least_scale = 0x1p-100f;  // (below it the reciprocal is no float: such a block's r is zero)

__device__ __forceinline__ float decode_root(uint32_t code, float scale) { return (__uint_as_float((code + root_base) << 19) - root_c) * scale; }
__device__ __forceinline__ float decode_ratio(uint32_t code, float factor) {
    const float u = (__uint_as_float(((code & 127u) + ratio_base) << 19) - ratio_c) * factor;
    return code & 128u ? -u : u;
}
__device__ __forceinline__ uint32_t encode(float y, float c, uint32_t dither, uint32_t base, uint32_t top) {
    return min(((__float_as_uint(y + c) + (dither << 3)) >> 19) - base, top);
}

__device__ __forceinline__ uint32_t dither_of(uint32_t element, uint32_t key) { return adamw_mix(element * 0x9E3779B1u + key); }

// One wave per block of 256 elements, four to a lane.
template <typename P, typename D>
__device__ __forceinline__ void step8(const AdamWTensorDevice& T, const AdamWGroupDevice& G, uint32_t block, float coefficient) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t group = static_cast<uint64_t>(block) * (adamw_block / 64) + (threadIdx.x >> 6), base = group * 256;
    if (base >= T.n) return;
    const uint64_t i = base + lane * 4u;
    const uint32_t count = i >= T.n ? 0u : T.n - i >= 4 ? 4u : static_cast<uint32_t>(T.n - i);
    uint8_t* const ratios = static_cast<uint8_t*>(T.m) + i;
    uint8_t* const roots = static_cast<uint8_t*>(T.v) + i;
    float p[4], g[4], r[4], u[4];
    load4(static_cast<const D*>(T.grad) + i, count, g);
    const uint32_t ratio_codes = load_codes(ratios, count), root_codes = load_codes(roots, count);
    load4(static_cast<const P*>(T.param) + i, count, p);
    const float scale = T.scale[group];
    uint32_t column = first_column(G, base, lane * 4u);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float gk = g[k] * coefficient;
        const float old = decode_root((root_codes >> (8 * k)) & 255u, scale);
        const float m = G.beta1 * (decode_ratio((ratio_codes >> (8 * k)) & 255u, T.ratio_decode) * old) + G.beta1_rest * gk;
        r[k] = sqrtf(G.beta2 * (old * old) + G.beta2_rest * (gk * gk));
        p[k] = updated(G, T, p[k], m, r[k], column);
        column = next_column(G, column);
        r[k] = r[k] < INFINITY && static_cast<uint32_t>(k) < count ? r[k] : 0.0f;
        u[k] = r[k] > 0.0f ? m / r[k] : 0.0f;
        top = max(top, __float_as_uint(r[k]));
    }
    float new_scale = __uint_as_float(wave_max(top)) * (1.0f / root_top);
    if (new_scale < least_scale) new_scale = 0.0f;
    const float inverse = new_scale > 0.0f ? 1.0f / new_scale : 0.0f;
    uint32_t new_ratios = 0, new_roots = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t h = dither_of(static_cast<uint32_t>(i) + k, T.key);
        new_roots |= encode(r[k] * inverse, root_c, h & 0xffffu, root_base, 255u) << (8 * k);
        const float y = fminf(fabsf(u[k]) * G.ratio_encode, ratio_top);
        new_ratios |= (encode(y, ratio_c, h >> 16, ratio_base, 127u) | (u[k] < 0.0f ? 128u : 0u)) << (8 * k);
    }
    store4(static_cast<P*>(T.param) + i, count, p);
    store_codes(ratios, count, new_ratios);
    store_codes(roots, count, new_roots);
    if (lane == 0) T.scale[group] = new_scale;
}

template <int BITS, typename P, typename D>
__device__ __forceinline__ void step_block(const AdamWTensorDevice& T, const AdamWGroupDevice& G, uint32_t block, float coefficient) {
    if constexpr (BITS == 32) step32<P, D>(T, G, block, coefficient);
    else step8<P, D>(T, G, block, coefficient);
}

template <int BITS, typename P>
__device__ __forceinline__ void step_gradient(const AdamWTensorDevice& T, const AdamWGroupDevice& G, uint32_t block, float coefficient) {
    if (T.grad_type == type_float) step_block<BITS, P, float>(T, G, block, coefficient);
    else if (T.grad_type == type_bfloat16) step_block<BITS, P, __bf16>(T, G, block, coefficient);
    else step_block<BITS, P, _Float16>(T, G, block, coefficient);
}

template <int BITS>
__global__ __launch_bounds__(adamw_block) void adamw_kernel(AdamWLaunch L) {
    float coefficient;
    if (!clipping(L, coefficient)) return;
    const uint32_t k = tensor_of_block(L.first_block, L.n_tensors, blockIdx.x);
    const AdamWTensorDevice& T = L.tensors[k];
    const AdamWGroupDevice& G = L.groups[T.group];
    const uint32_t block = blockIdx.x - L.first_block[k];
    if (T.param_type == type_float) step_gradient<BITS, float>(T, G, block, coefficient);
    else if (T.param_type == type_bfloat16) step_gradient<BITS, __bf16>(T, G, block, coefficient);
    else step_gradient<BITS, _Float16>(T, G, block, coefficient);
}

// ---- decoding ----------------------------------------------------------------------------------------------------------

struct MomentsLaunch {
    uint32_t first_block[moments_max_tensors];
    AdamWMomentsDevice tensors[moments_max_tensors];
    uint32_t n_tensors;
};
static_assert(sizeof(MomentsLaunch) <= 4096, "kernel arguments");

__global__ __launch_bounds__(adamw_block) void adamw_moments_kernel(MomentsLaunch L) {
    const uint32_t k = tensor_of_block(L.first_block, L.n_tensors, blockIdx.x);
    const AdamWMomentsDevice& T = L.tensors[k];
    const uint64_t i = static_cast<uint64_t>(blockIdx.x - L.first_block[k]) * adamw_block * 4 + threadIdx.x * 4u;
    if (i >= T.n) return;
    const uint32_t count = T.n - i >= 4 ? 4u : static_cast<uint32_t>(T.n - i);
    const uint32_t ratio_codes = load_codes(T.ratios + i, count), root_codes = load_codes(T.roots + i, count);
    const float scale = T.scale[i / 256];
    float m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float r = decode_root((root_codes >> (8 * j)) & 255u, scale);
        m[j] = decode_ratio((ratio_codes >> (8 * j)) & 255u, T.ratio_decode) * r;
        v[j] = r * r;
    }
    store4(T.m + i, count, m);
    store4(T.v + i, count, v);
}

// ---- gradient norm -----------------------------------------------------------------------------------------------------

constexpr uint32_t norm_chunk = adamw_block * 16;

struct NormLaunch {
    uint32_t first_block[norm_max_tensors];
    NormTensorDevice tensors[norm_max_tensors];
    double* partials;
    uint32_t n_tensors;
};
static_assert(sizeof(NormLaunch) <= 4096, "kernel arguments");

// sum over the block's threads in a fixed order (thread 0's result counts)
template <uint32_t BLOCK>
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double parts[BLOCK / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_down(x, o);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = x;
    __syncthreads();
    double sum = parts[0];
#pragma unroll
    for (uint32_t w = 1; w < BLOCK / 64; w++) sum += parts[w];
    return sum;
}

template <typename T>
__device__ __forceinline__ double squares(const T* data, uint64_t n, uint64_t base) {
    double sum = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint64_t i = base + j * adamw_block * 4 + threadIdx.x * 4u;
        float x[4];
        load4(data + i, i >= n ? 0u : n - i >= 4 ? 4u : static_cast<uint32_t>(n - i), x);
#pragma unroll
        for (int k = 0; k < 4; k++) sum = __builtin_fma(static_cast<double>(x[k]), static_cast<double>(x[k]), sum);
    }
    return sum;
}

__global__ __launch_bounds__(adamw_block) void norm_partials_kernel(NormLaunch L) {
    const uint32_t k = tensor_of_block(L.first_block, L.n_tensors, blockIdx.x);
    const NormTensorDevice& T = L.tensors[k];
    const uint64_t base = static_cast<uint64_t>(blockIdx.x - L.first_block[k]) * norm_chunk;
    const uint64_t n = T.n_and_type >> 2;
    const uint32_t type = static_cast<uint32_t>(T.n_and_type & 3u);
    double sum;
    if (type == type_float) sum = squares(static_cast<const float*>(T.data), n, base);
    else if (type == type_bfloat16) sum = squares(static_cast<const __bf16*>(T.data), n, base);
    else sum = squares(static_cast<const _Float16*>(T.data), n, base);
    sum = block_sum<adamw_block>(sum);
    if (threadIdx.x == 0) L.partials[blockIdx.x] = sum;
}

__global__ __launch_bounds__(1024) void norm_kernel(const double* __restrict__ partials, uint32_t n, float* __restrict__ norm) {
    double sum = 0.0;
    for (uint32_t k = threadIdx.x; k < n; k += 1024) sum += partials[k];
    sum = block_sum<1024>(sum);
    if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(sum));
}

}  // namespace

bool launch_adamw(const AdamWTensorDevice* tensors, uint64_t n_tensors, const AdamWGroupDevice* groups, int bits, const float* grad_norm,
                  float max_grad_norm, hipStream_t s) {
    AdamWLaunch L;
    L.grad_norm = grad_norm;
    L.max_grad_norm = max_grad_norm;
    uint64_t at = 0;
    while (at < n_tensors) {
        uint32_t blocks = 0, n_groups = 0;
        uint32_t of_group[adamw_max_groups];
        L.n_tensors = 0;
        for (; at < n_tensors && L.n_tensors < adamw_max_tensors; at++) {
            const uint32_t more = div_up(tensors[at].n, adamw_block * 4);
            if (blocks + more > adamw_max_blocks && L.n_tensors > 0) break;
            uint32_t g = 0;
            while (g < n_groups && of_group[g] != tensors[at].group) g++;
            if (g == n_groups) {
                if (n_groups == adamw_max_groups) break;
                of_group[n_groups++] = tensors[at].group;
                L.groups[g] = groups[tensors[at].group];
            }
            L.tensors[L.n_tensors] = tensors[at];
            L.tensors[L.n_tensors].group = g;
            L.first_block[L.n_tensors++] = blocks;
            blocks += more;
        }
        if (bits == 32) adamw_kernel<32><<<blocks, adamw_block, 0, s>>>(L);
        else adamw_kernel<8><<<blocks, adamw_block, 0, s>>>(L);
        EFGS_HIP_CHECK(hipGetLastError());
    }
    return true;
}

bool launch_adamw_moments(const AdamWMomentsDevice* tensors, uint64_t n_tensors, hipStream_t s) {
    MomentsLaunch L;
    uint64_t at = 0;
    while (at < n_tensors) {
        uint32_t blocks = 0;
        L.n_tensors = 0;
        for (; at < n_tensors && L.n_tensors < moments_max_tensors; at++) {
            const uint32_t more = div_up(tensors[at].n, adamw_block * 4);
            if (blocks + more > adamw_max_blocks && L.n_tensors > 0) break;
            L.tensors[L.n_tensors] = tensors[at];
            L.first_block[L.n_tensors++] = blocks;
            blocks += more;
        }
        adamw_moments_kernel<<<blocks, adamw_block, 0, s>>>(L);
        EFGS_HIP_CHECK(hipGetLastError());
    }
    return true;
}

uint64_t norm_partials_of(uint64_t n) { return (n + norm_chunk - 1) / norm_chunk; }

bool launch_grad_norm(const NormTensorDevice* tensors, uint64_t n_tensors, double* partials, float* norm, hipStream_t s) {
    NormLaunch L;
    uint64_t at = 0;
    uint32_t done = 0;
    while (at < n_tensors) {
        uint32_t blocks = 0;
        L.n_tensors = 0;
        L.partials = partials + done;
        for (; at < n_tensors && L.n_tensors < norm_max_tensors; at++) {
            const uint32_t more = static_cast<uint32_t>(norm_partials_of(tensors[at].n_and_type >> 2));
            if (blocks + more > adamw_max_blocks && L.n_tensors > 0) break;
            L.tensors[L.n_tensors] = tensors[at];
            L.first_block[L.n_tensors++] = blocks;
            blocks += more;
        }
        norm_partials_kernel<<<blocks, adamw_block, 0, s>>>(L);
        EFGS_HIP_CHECK(hipGetLastError());
        done += blocks;
    }
    norm_kernel<<<1, 1024, 0, s>>>(partials, done, norm);
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
