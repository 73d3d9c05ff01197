// AdamW over many tensors at once, with states in 32 or in 8 bits, the decoding of 8-bit states, and the gradient norm
// over many tensors that clips a step. A launch takes the descriptors of 60 to 72 tensors as kernel arguments (nothing is
// copied to the device and nothing has to outlive the call); a block finds its tensor from the first blocks of all. What tensors
// of one group and step share is held once.
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
#include <type_traits>

#include "internal.h"

namespace efgs {

namespace {

constexpr uint32_t adamw_block = 256, adamw_piece = adamw_block * 4;

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bfloat4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t uint32u __attribute__((aligned(1)));

template <typename T> struct Vector4;
template <> struct Vector4<float> { using type = float4u; };
template <> struct Vector4<_Float16> { using type = half4u; };
template <> struct Vector4<__bf16> { using type = bfloat4u; };

// x[0..3] = p[0..3] in 32 bits, and zeros past `count`. WHOLE: the block lies within its tensor, and every count is 4. At a tensor's
// end each value is loaded by itself, from the last one's place past it: whatever its count, no lane waits for a load before all are
// sent, as it would with one in a branch. (p + 0 has to be in the tensor: callers clamp it.)
//
// The step streams its tensors once each way, with nontemporal loads and stores: 59M float32 elements 325 -> 309 us, 30M bfloat16
// ones 120 -> 106, 22M with 8-bit states 64 -> 56 (loads or stores alone gain nothing).
template <bool WHOLE, typename T>
__device__ __forceinline__ void load4(const T* p, uint32_t count, float* x) {
    if constexpr (WHOLE) {
        const typename Vector4<T>::type v = __builtin_nontemporal_load(reinterpret_cast<const typename Vector4<T>::type*>(p));
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = static_cast<float>(v[k]);
    } else {
        const uint32_t last = count > 0 ? count - 1 : 0u;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = static_cast<float>(p[min(k, last)]);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = k < count ? x[k] : 0.0f;
    }
}

// rounded to nearest even, what a cast of a tensor does
template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(T* p, uint32_t count, const float* x) {
    if constexpr (WHOLE) {
        typename Vector4<T>::type v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = static_cast<T>(x[k]);
        __builtin_nontemporal_store(v, reinterpret_cast<typename Vector4<T>::type*>(p));
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (k < count) p[k] = static_cast<T>(x[k]);
    }
}

template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, uint32_t count) {
    if constexpr (WHOLE) return *reinterpret_cast<const uint32u*>(p);
    const uint32_t last = count > 0 ? count - 1 : 0u;
    uint32_t code[4], v = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) code[k] = p[min(k, last)];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) v |= k < count ? code[k] << (8 * k) : 0u;
    return v;
}

template <bool WHOLE>
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t count, uint32_t v) {
    if constexpr (WHOLE) {
        *reinterpret_cast<uint32u*>(p) = v;
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (k < count) p[k] = static_cast<uint8_t>(v >> (8 * k));
}

// a thread's first element and how many of four from there lie in the tensor; past its end 0 of its last element
struct Four {
    uint64_t at;
    uint32_t count;
};
template <bool WHOLE>
__device__ __forceinline__ Four four_from(uint64_t i, uint64_t n) {
    if constexpr (WHOLE) return {i, 4u};
    return {i < n ? i : n - 1, i >= n ? 0u : n - i >= 4 ? 4u : static_cast<uint32_t>(n - i)};
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

// A tensor's first block, and in the top bits the launch's group that it belongs to: the descriptors of both are then loaded
// at once, where the group's number in the tensor's made a load wait for another (arguments are slow to read the first time).
__host__ __device__ inline uint32_t pack_first_block(uint32_t block, uint32_t group) { return group << 28 | block; }
__host__ __device__ inline uint32_t first_block_of(uint32_t packed) { return packed & 0x0fffffffu; }
__host__ __device__ inline uint32_t first_block_group(uint32_t packed) { return packed >> 28; }

// the last of the n tensors whose first block is at most `block`: its index and packed first block
template <uint32_t MAX>
__device__ __forceinline__ uint2 tensor_of_block(const uint32_t* first_blocks, uint32_t n, uint32_t block) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t packed[(MAX + 63) / 64];
#pragma unroll
    for (uint32_t k = 0; k < MAX; k += 64) packed[k / 64] = first_blocks[min(k + lane, n - 1)];
    uint32_t count = 0, found = 0;
#pragma unroll
    for (uint32_t k = 0; k < MAX; k += 64) {
        const uint64_t at_most = __ballot(k + lane < n && first_block_of(packed[k / 64]) <= block);
        if (at_most) found = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(packed[k / 64]), 63 - __clzll(at_most)));
        count += static_cast<uint32_t>(__popcll(at_most));
    }
    return make_uint2(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(count))) - 1u, found);
}

template <int BITS>
struct AdamWLaunch {
    static constexpr uint32_t max_tensors = BITS == 32 ? 72 : 60;
    using Tensor = std::conditional_t<BITS == 32, AdamWTensor, AdamWTensor8>;
    uint32_t first_block[max_tensors];
    Tensor tensors[max_tensors];
    AdamWGroupDevice groups[adamw_max_groups];
    const float* grad_norm;  // null: gradients as they are
    float max_grad_norm;
    uint32_t n_tensors;
};
static_assert(sizeof(AdamWLaunch<32>) <= 4096 && sizeof(AdamWLaunch<8>) <= 4096, "kernel arguments");

// The clipping coefficient; not a number where the norm is not finite (the step then leaves parameters and moments).
__device__ __forceinline__ float clipping(float norm, float max_grad_norm) {
    return norm < INFINITY ? fminf(max_grad_norm / (norm + 1e-6f), 1.0f) : NAN;
}

// The parameter after the step. The reciprocal is the hardware's (1 ulp): the division's last bit would be
// 6e-8 of the update, for about ten operations an element. root is 0 or at least 3e-23, a float's least square root, and eps, as
// the host hands it over, 0 or a normal float, so that the sum is no denormal.
__device__ __forceinline__ float updated(const AdamWGroupDevice& G, float p, float m, float root, float rate, float decay) {
    const float update = m * __builtin_amdgcn_rcpf(root * G.root_factor + G.eps);
    return p * decay - rate * update;
}

// Learning rates of four consecutive elements: the group's one, or from the table of its cycle (in LDS, rate and decay).
struct Rates {
    float2 of[4];
};

// What the gradients are multiplied with. The norm was loaded before the tensors, and is waited for with them.
struct Clip {
    bool on;
    float norm, max_grad_norm;
    __device__ __forceinline__ float coefficient() const { return on ? clipping(norm, max_grad_norm) : 1.0f; }
};
template <bool CYCLE>
__device__ __forceinline__ Rates rates_of(const AdamWGroupDevice& G, const float2* cycle, uint32_t first_column) {
    Rates r;
    uint32_t column = first_column;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (CYCLE) {
            r.of[k] = cycle[column];
            column = column + 1 == G.n_lrs ? 0 : column + 1;
        } else {
            r.of[k] = make_float2(G.rates[0], G.decays[0]);
        }
    }
    return r;
}

// PIECES pieces of four elements a thread, 1,024 apart, all loaded before the first is worked on. Memory bounds it: 59M float32
// elements, 1,652 MB, in 280 us (5.9 TB/s; a large copy reaches 5.1, a sum of two arrays 5.9). 590k, 17 MB, take 6 us, of which
// 3.2 would be memory at a large copy's rate.
template <bool WHOLE, bool CYCLE, int PIECES, typename P, typename D>
__device__ __forceinline__ void step_block(const AdamWTensor& T, const AdamWGroupDevice& G, const float2* cycle, uint64_t base, uint64_t n, uint32_t column,
                                           Clip clip) {
    float p[PIECES][4], g[PIECES][4], m[PIECES][4], v[PIECES][4];
    Four four[PIECES];
#pragma unroll
    for (int q = 0; q < PIECES; q++) {
        four[q] = four_from<WHOLE>(base + q * adamw_piece + threadIdx.x * 4u, n);
        load4<WHOLE>(static_cast<const D*>(T.grad) + four[q].at, four[q].count, g[q]);
        load4<WHOLE>(static_cast<const float*>(T.m) + four[q].at, four[q].count, m[q]);
        load4<WHOLE>(static_cast<const float*>(T.v) + four[q].at, four[q].count, v[q]);
        load4<WHOLE>(static_cast<const P*>(T.param) + four[q].at, four[q].count, p[q]);
    }
    const float coefficient = clip.coefficient();
    if (coefficient != coefficient) return;
#pragma unroll
    for (int q = 0; q < PIECES; q++) {
        const Rates rates = rates_of<CYCLE>(G, cycle, column);
        if constexpr (CYCLE) column = (column + adamw_piece) % G.n_lrs;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float gk = g[q][k] * coefficient;
            m[q][k] = G.beta1 * m[q][k] + G.beta1_rest * gk;
            v[q][k] = G.beta2 * v[q][k] + G.beta2_rest * (gk * gk);
            p[q][k] = updated(G, p[q][k], m[q][k], sqrtf(v[q][k]), rates.of[k].x, rates.of[k].y);
        }
        store4<WHOLE>(static_cast<float*>(T.m) + four[q].at, four[q].count, m[q]);
        store4<WHOLE>(static_cast<float*>(T.v) + four[q].at, four[q].count, v[q]);
        store4<WHOLE>(static_cast<P*>(T.param) + four[q].at, four[q].count, p[q]);
    }
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
    return min((__float_as_uint(y + c) + (dither << 3) - (base << 19)) >> 19, top);
}

__device__ __forceinline__ uint32_t dither_of(uint32_t element, uint32_t key) { return adamw_mix(element * 0x9E3779B1u + key); }

// sqrt(x) and its reciprocal's approximation for x = 0 or x >= 2^-100, rounded to nearest: one step from the hardware's reciprocal
// square root (s = x y, s + (x - s^2) y / 2, the residual exact by the fused operation).
__device__ __forceinline__ float rounded_sqrt(float x, float& reciprocal) {
    reciprocal = __builtin_amdgcn_rsqf(__uint_as_float(max(__float_as_uint(x), __float_as_uint(0x1p-100f))));
    const float s = x * reciprocal;
    return __builtin_fmaf(__builtin_fmaf(-s, s, x), 0.5f * reciprocal, s);
}

// a / b rounded to nearest from an approximation of 1 / b (the quotient's residual exact by the fused operation)
__device__ __forceinline__ float rounded_quotient(float a, float b, float reciprocal) {
    const float q = a * reciprocal;
    return __builtin_fmaf(__builtin_fmaf(-q, b, a), reciprocal, q);
}

// Codes of u for another bound, where a step that is left out was given other betas: its caller counts the state as one of these.
// Values past the new bound become the bound, as they do in a step.
__device__ __forceinline__ uint32_t recoded_ratios(uint32_t codes, const AdamWGroupDevice& G, uint32_t element) {
    uint32_t out = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t code = (codes >> (8 * k)) & 255u;
        const float y = fminf(decode_ratio(code & 127u, G.ratio_decode) * G.ratio_encode, ratio_top);
        out |= (encode(y, ratio_c, dither_of(element + k, G.key) >> 16, ratio_base, 127u) | (code & 128u)) << (8 * k);
    }
    return out;
}

// One wave per block of 256 elements, four to a lane: the block's maximum is one reduction of the wave, and nothing crosses waves.
// float32 elements are bound by memory (22M, 353 MB, in 60 us, 5.9 TB/s), bfloat16 ones by the vector units (13.4M, 134 MB, in
// 35 us, 3.8 TB/s, at about 90 vector operations an element). A square root and a quotient with the library's full range would be 30 more, so they
// are done in five and three where every element's v is zero, or at least 2^-100 and finite (a gradient of 3e-14 after one step),
// and by the library where the wave holds another one; both round to nearest. Two or four blocks a wave, loaded together, gained
// nothing (33.6M float32 86, 86 and 87 us, bfloat16 75, 75 and 74).
template <bool WHOLE, bool CYCLE, int PIECES, typename P, typename D>
__device__ __forceinline__ void step_block(const AdamWTensor8& T, const AdamWGroupDevice& G, const float2* cycle, uint64_t base, uint64_t n, uint32_t column,
                                           Clip clip) {
    static_assert(PIECES == 1, "a wave takes one block of 256");
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t first = base + (threadIdx.x - lane) * 4u;  // of the wave's block
    if (!WHOLE && first >= n) return;
    const Four four = four_from<WHOLE>(first + lane * 4u, n);
    const uint64_t i = four.at;
    const uint32_t count = four.count;
    uint8_t* const ratios = static_cast<uint8_t*>(T.m) + i;
    uint8_t* const roots = static_cast<uint8_t*>(T.v) + i;
    float p[4], g[4], m[4], v[4], r[4], u[4];
    load4<WHOLE>(static_cast<const D*>(T.grad) + i, count, g);
    const uint32_t ratio_codes = load_codes<WHOLE>(ratios, count), root_codes = load_codes<WHOLE>(roots, count);
    load4<WHOLE>(static_cast<const P*>(T.param) + i, count, p);
    const float scale = T.scale[first / 256];
    const Rates rates = rates_of<CYCLE>(G, cycle, column);
    const float coefficient = clip.coefficient();
    if (coefficient != coefficient) {
        // (for one bound the factors' product is 1 to two roundings)
        if (fabsf(G.ratio_decode * G.ratio_encode - 1.0f) > 1e-6f) store_codes<WHOLE>(ratios, count, recoded_ratios(ratio_codes, G, static_cast<uint32_t>(i)));
        return;
    }
    uint32_t least = 0xffffffffu, most = 0;  // of v's bits less one (which makes zeros the largest), and of v's bits
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float gk = g[k] * coefficient;
        const float old = decode_root((root_codes >> (8 * k)) & 255u, scale);
        m[k] = G.beta1 * (decode_ratio((ratio_codes >> (8 * k)) & 255u, G.ratio_decode) * old) + G.beta1_rest * gk;
        v[k] = G.beta2 * (old * old) + G.beta2_rest * (gk * gk);
        // (past the tensor's end: code 0 and gradient 0 make 0)
        least = min(least, __float_as_uint(v[k]) - 1u);
        most = max(most, __float_as_uint(v[k]));
    }
    const bool plain = least >= __float_as_uint(0x1p-100f) - 1u && most < __float_as_uint(INFINITY);
    if (__ballot(!plain) == 0) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float reciprocal;
            r[k] = rounded_sqrt(v[k], reciprocal);
            u[k] = rounded_quotient(m[k], r[k], reciprocal);  // (v = 0: whatever it is, r's code is 0)
            p[k] = updated(G, p[k], m[k], r[k], rates.of[k].x, rates.of[k].y);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            r[k] = sqrtf(v[k]);
            p[k] = updated(G, p[k], m[k], r[k], rates.of[k].x, rates.of[k].y);
            r[k] = r[k] < INFINITY ? r[k] : 0.0f;
            u[k] = r[k] > 0.0f ? m[k] / r[k] : 0.0f;
        }
    }
    const uint32_t top = max(max(__float_as_uint(r[0]), __float_as_uint(r[1])), max(__float_as_uint(r[2]), __float_as_uint(r[3])));
    float new_scale = __uint_as_float(wave_max(top)) * (1.0f / root_top);
    if (new_scale < least_scale) new_scale = 0.0f;
    const float inverse = new_scale > 0.0f ? rounded_quotient(1.0f, new_scale, __builtin_amdgcn_rcpf(new_scale)) : 0.0f;
    uint32_t new_ratios = 0, new_roots = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t h = dither_of(static_cast<uint32_t>(i) + k, G.key);  // (past the end nothing is stored)
        new_roots |= encode(r[k] * inverse, root_c, h & 0xffffu, root_base, 255u) << (8 * k);
        const float y = fminf(fabsf(u[k]) * G.ratio_encode, ratio_top);
        new_ratios |= (encode(y, ratio_c, h >> 16, ratio_base, 127u) | ((__float_as_uint(u[k]) >> 24) & 128u)) << (8 * k);
    }
    store4<WHOLE>(static_cast<P*>(T.param) + i, count, p);
    store_codes<WHOLE>(ratios, count, new_ratios);
    store_codes<WHOLE>(roots, count, new_roots);
    if (lane == 0) T.scale[first / 256] = new_scale;
}

template <bool WHOLE, bool CYCLE, int PIECES, typename P, typename T>
__device__ __forceinline__ void step_gradient(const T& tensor, const AdamWGroupDevice& G, const float2* cycle, uint64_t base, uint64_t n, uint32_t column,
                                              Clip clip) {
    const uint32_t type = tensor.grad_type();
    if (type == type_float) step_block<WHOLE, CYCLE, PIECES, P, float>(tensor, G, cycle, base, n, column, clip);
    else if (type == type_bfloat16) step_block<WHOLE, CYCLE, PIECES, P, __bf16>(tensor, G, cycle, base, n, column, clip);
    else step_block<WHOLE, CYCLE, PIECES, P, _Float16>(tensor, G, cycle, base, n, column, clip);
}

template <bool WHOLE, bool CYCLE, int PIECES, typename T>
__device__ __forceinline__ void step_tensor(const T& tensor, const AdamWGroupDevice& G, const float2* cycle, uint64_t base, uint64_t n, uint32_t column,
                                            Clip clip) {
    const uint32_t type = tensor.param_type();
    if (type == type_float) step_gradient<WHOLE, CYCLE, PIECES, float>(tensor, G, cycle, base, n, column, clip);
    else if (type == type_bfloat16) step_gradient<WHOLE, CYCLE, PIECES, __bf16>(tensor, G, cycle, base, n, column, clip);
    else step_gradient<WHOLE, CYCLE, PIECES, _Float16>(tensor, G, cycle, base, n, column, clip);
}

template <int BITS, int PIECES>
__global__ __launch_bounds__(adamw_block) void adamw_kernel(AdamWLaunch<BITS> L) {
    __shared__ float2 cycle[adam_max_lrs];
    const Clip clip = {L.grad_norm != nullptr, L.grad_norm ? *L.grad_norm : 0.0f, L.max_grad_norm};
    const uint2 found = tensor_of_block<AdamWLaunch<BITS>::max_tensors>(L.first_block, L.n_tensors, blockIdx.x);
    // (copies: with references the whole argument was copied to scratch memory)
    const auto T = L.tensors[found.x];
    const AdamWGroupDevice G = L.groups[first_block_group(found.y)];
    const uint64_t base = static_cast<uint64_t>(blockIdx.x - first_block_of(found.y)) * adamw_piece * PIECES, n = T.n();
    const bool whole = base + adamw_piece * PIECES <= n;
    if (G.n_lrs == 1) {
        if (whole) step_tensor<true, false, PIECES>(T, G, cycle, base, n, 0u, clip);
        else step_tensor<false, false, PIECES>(T, G, cycle, base, n, 0u, clip);
        return;
    }
    if (threadIdx.x < G.n_lrs) cycle[threadIdx.x] = make_float2(L.groups[first_block_group(found.y)].rates[threadIdx.x], L.groups[first_block_group(found.y)].decays[threadIdx.x]);
    __syncthreads();
    const uint32_t column = (static_cast<uint32_t>(base % G.n_lrs) + threadIdx.x * 4u) % G.n_lrs;
    if (whole) step_tensor<true, true, PIECES>(T, G, cycle, base, n, column, clip);
    else step_tensor<false, true, PIECES>(T, G, cycle, base, n, column, clip);
}

// ---- decoding ----------------------------------------------------------------------------------------------------------

struct MomentsLaunch {
    uint32_t first_block[moments_max_tensors];
    AdamWMomentsDevice tensors[moments_max_tensors];
    uint32_t n_tensors;
};
static_assert(sizeof(MomentsLaunch) <= 4096, "kernel arguments");

// bound by memory: 22M elements, 10 bytes each, in 32 us (6.8 TB/s)
template <bool WHOLE>
__device__ __forceinline__ void decode_block(const AdamWMomentsDevice& T, uint64_t base) {
    const Four four = four_from<WHOLE>(base + threadIdx.x * 4u, T.n);
    const uint32_t ratio_codes = load_codes<WHOLE>(T.ratios + four.at, four.count), root_codes = load_codes<WHOLE>(T.roots + four.at, four.count);
    const float scale = T.scale[four.at / 256];
    float m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float r = decode_root((root_codes >> (8 * j)) & 255u, scale);
        m[j] = decode_ratio((ratio_codes >> (8 * j)) & 255u, T.ratio_decode) * r;
        v[j] = r * r;
    }
    store4<WHOLE>(T.m + four.at, four.count, m);
    store4<WHOLE>(T.v + four.at, four.count, v);
}

__global__ __launch_bounds__(adamw_block) void adamw_moments_kernel(MomentsLaunch L) {
    const uint2 found = tensor_of_block<moments_max_tensors>(L.first_block, L.n_tensors, blockIdx.x);
    const AdamWMomentsDevice T = L.tensors[found.x];
    const uint64_t base = static_cast<uint64_t>(blockIdx.x - found.y) * adamw_piece;
    if (base + adamw_piece <= T.n) decode_block<true>(T, base);
    else decode_block<false>(T, base);
}

// ---- gradient norm -----------------------------------------------------------------------------------------------------

constexpr uint32_t norm_loads = 8, norm_step = adamw_block * 4 * norm_loads;  // loads of a thread at once, and a block's elements

struct NormLaunch {
    uint32_t first_block[norm_max_tensors];
    NormTensorDevice tensors[norm_max_tensors];
    double* partials;
    uint32_t n_tensors;
    uint32_t steps;  // of a block
};
static_assert(sizeof(NormLaunch) <= 4096, "kernel arguments");

__host__ __device__ inline uint32_t norm_blocks(uint64_t n, uint32_t steps) {
    return static_cast<uint32_t>((n + static_cast<uint64_t>(norm_step) * steps - 1) / (static_cast<uint64_t>(norm_step) * steps));
}

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

// Eight loads `stride` elements apart. WHOLE: all of them lie in the tensor; else one that does not takes the tensor's last four
// elements (there are four) and counts those from its own place on.
template <bool WHOLE, typename T>
__device__ __forceinline__ void add_squares(const T* data, uint64_t n, uint64_t base, uint64_t stride, double* sum) {
    typename Vector4<T>::type x[norm_loads];
#pragma unroll
    for (uint32_t j = 0; j < norm_loads; j++) {
        const uint64_t i = base + j * stride + threadIdx.x * 4u;
        x[j] = *reinterpret_cast<const typename Vector4<T>::type*>(data + (WHOLE ? i : min(i, n - 4)));
    }
#pragma unroll
    for (uint32_t j = 0; j < norm_loads; j++) {
        const uint64_t i = base + j * stride + threadIdx.x * 4u;
        const uint32_t skipped = WHOLE || i + 4 <= n ? 0u : i >= n ? 4u : static_cast<uint32_t>(i + 4 - n);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const double value = k >= skipped ? static_cast<double>(static_cast<float>(x[j][k])) : 0.0;
            sum[k] = __builtin_fma(value, value, sum[k]);
        }
    }
}

// A tensor's blocks take its 1,024-element pieces in turn, so that at any time they read one stretch of memory: with a stretch
// of its own for each block (32 to 128 KB apart) they met on few memory channels (70M float32 values 98 us, interleaved 86). Now
// 50 us, 5.6 TB/s, with the step's accesses nontemporal. Reading is what bounds it.
template <typename T>
__device__ __forceinline__ double squares(const T* data, uint64_t n, uint32_t block, uint32_t blocks) {
    double sum[4] = {};
    if (n < 4) {
        const double value = threadIdx.x < n ? static_cast<double>(static_cast<float>(data[threadIdx.x])) : 0.0;
        return value * value;
    }
    const uint64_t stride = static_cast<uint64_t>(blocks) * adamw_block * 4;
    for (uint64_t base = static_cast<uint64_t>(block) * adamw_block * 4; base < n; base += norm_loads * stride) {
        if (base + (norm_loads - 1) * stride + adamw_block * 4 <= n) add_squares<true>(data, n, base, stride, sum);
        else add_squares<false>(data, n, base, stride, sum);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__global__ __launch_bounds__(adamw_block) void norm_partials_kernel(NormLaunch L) {
    const uint2 found = tensor_of_block<norm_max_tensors>(L.first_block, L.n_tensors, blockIdx.x);
    const NormTensorDevice T = L.tensors[found.x];
    const uint64_t n = T.n_and_type >> 2;
    const uint32_t type = static_cast<uint32_t>(T.n_and_type & 3u), block = blockIdx.x - found.y, blocks = norm_blocks(n, L.steps);
    double sum;
    if (type == type_float) sum = squares(static_cast<const float*>(T.data), n, block, blocks);
    else if (type == type_bfloat16) sum = squares(static_cast<const __bf16*>(T.data), n, block, blocks);
    else sum = squares(static_cast<const _Float16*>(T.data), n, block, blocks);
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

template <int BITS, int PIECES, typename T>
bool launch_steps(const T* tensors, const uint32_t* of_tensor, uint64_t n_tensors, const AdamWGroupDevice* groups, const float* grad_norm,
                  float max_grad_norm, hipStream_t s) {
    AdamWLaunch<BITS> L;
    L.grad_norm = grad_norm;
    L.max_grad_norm = max_grad_norm;
    uint64_t at = 0;
    while (at < n_tensors) {
        uint32_t blocks = 0, n_groups = 0;
        uint32_t group_of[adamw_max_groups];
        L.n_tensors = 0;
        for (; at < n_tensors && L.n_tensors < AdamWLaunch<BITS>::max_tensors; at++) {
            const uint32_t more = div_up(tensors[at].n(), adamw_piece * PIECES);
            if (blocks + more > adamw_max_blocks && L.n_tensors > 0) break;
            uint32_t g = 0;
            while (g < n_groups && group_of[g] != of_tensor[at]) g++;
            if (g == n_groups) {
                if (n_groups == adamw_max_groups) break;
                group_of[n_groups++] = of_tensor[at];
                L.groups[g] = groups[of_tensor[at]];
            }
            L.tensors[L.n_tensors] = tensors[at];
            L.first_block[L.n_tensors++] = pack_first_block(blocks, g);
            blocks += more;
        }
        adamw_kernel<BITS, PIECES><<<blocks, adamw_block, 0, s>>>(L);
        EFGS_HIP_CHECK(hipGetLastError());
    }
    return true;
}

bool launch_adamw(const AdamWTensor* tensors, const uint32_t* of_tensor, uint64_t n_tensors, const AdamWGroupDevice* groups, const float* grad_norm,
                  float max_grad_norm, hipStream_t s) {
    // Two pieces a thread from about a million elements on (one, two and four: 590k elements 5.9 and 7.5 us, 1M 6.8, 6.5 and 7.6, 4M 22.0, 21.0
    // and 21.3, 67M 341, 317 and 316; bfloat16 67M 255, 248 and 244): below, the blocks of a launch would not fill the GPU.
    uint64_t total = 0;
    for (uint64_t k = 0; k < n_tensors; k++) total += tensors[k].n();
    const uint64_t launches = (n_tensors + AdamWLaunch<32>::max_tensors - 1) / AdamWLaunch<32>::max_tensors;
    if (total < (launches << 20)) return launch_steps<32, 1>(tensors, of_tensor, n_tensors, groups, grad_norm, max_grad_norm, s);
    return launch_steps<32, 2>(tensors, of_tensor, n_tensors, groups, grad_norm, max_grad_norm, s);
}

bool launch_adamw8(const AdamWTensor8* tensors, const uint32_t* of_tensor, uint64_t n_tensors, const AdamWGroupDevice* groups, const float* grad_norm,
                   float max_grad_norm, hipStream_t s) {
    return launch_steps<8, 1>(tensors, of_tensor, n_tensors, groups, grad_norm, max_grad_norm, s);
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

// Steps of a block: one, until that makes as many blocks as the GPU holds (2,048), then more, which keeps the partial sums few.
static uint32_t norm_steps(const NormTensorDevice* tensors, uint64_t n_tensors) {
    uint64_t total = 0;
    for (uint64_t k = 0; k < n_tensors; k++) total += tensors[k].n_and_type >> 2;
    const uint64_t steps = total / (2048ull * norm_step);
    return static_cast<uint32_t>(steps < 1 ? 1 : steps > 4096 ? 4096 : steps);
}

uint64_t norm_partials(const NormTensorDevice* tensors, uint64_t n_tensors) {
    const uint32_t steps = norm_steps(tensors, n_tensors);
    uint64_t partials = 0;
    for (uint64_t k = 0; k < n_tensors; k++) partials += norm_blocks(tensors[k].n_and_type >> 2, steps);
    return partials;
}

bool launch_grad_norm(const NormTensorDevice* tensors, uint64_t n_tensors, double* partials, float* norm, hipStream_t s) {
    NormLaunch L;
    L.steps = norm_steps(tensors, n_tensors);
    uint64_t at = 0;
    uint32_t done = 0;
    while (at < n_tensors) {
        uint32_t blocks = 0;
        L.n_tensors = 0;
        L.partials = partials + done;
        for (; at < n_tensors && L.n_tensors < norm_max_tensors; at++) {
            const uint32_t more = norm_blocks(tensors[at].n_and_type >> 2, L.steps);
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
