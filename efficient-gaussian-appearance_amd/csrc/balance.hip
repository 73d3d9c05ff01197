// The loss that balances how often codes (or experts) are chosen, and their counts.
//
//   count_e = choices of e, share_e = count_e / all choices, p_n = softmax(z_n), P_e = mean of p_ne over the rows that count
//   loss = E sum_e share_e P_e,  d loss / d z_ne = E / rows p_ne (share_e - sum_j share_j p_nj)
//
// The probabilities of a row sum to one, so the gradient takes shares less the even one, 1 / E: even choices give zeros and not what the rounded sum of
// probabilities leaves.
//
// A choice outside [0, E) counts nowhere, a row without any other is left out. Rows of nothing but -inf have no
// probabilities and no gradient. One pass over the logits either way: TPR lanes share a row (a wave takes several short rows, a
// block one long row), each holds the same columns of every row that it meets, so that the sums over rows stay in registers until
// the block's end. The forward leaves a table of the blocks' sums, which a second kernel adds up in the blocks' order
// (64 bits) and a third makes the loss of: no atomics on floats, the same bits from call to call.
//
// 1,000,000 x 64 float32, one choice each: forward 74 us (3.6 TB/s of logits and choices; a group of rows is loaded when the one before is summed), sums 11,
// loss 4.3, backward 85 (6.1 TB/s of what it moves, the logits partly from the memory-side cache). A pass took 213 us instead of 173 before the loads of several rows were under way together, choices came beside the logits
// and the lanes' exchanges went past LDS. 16,383 x 250 bfloat16, eight choices: 8.4, 7.1, 2.9 and 8.8, each at its latency.
#include <algorithm>

#include "internal.h"

namespace efgs {

namespace {

constexpr uint32_t balance_block = 256, balance_waves = balance_block / 64;
constexpr uint32_t balance_max_blocks = 2048;   // eight to a CU; of the forward: rows of the table of sums
constexpr float log2_e = 1.4426950408889634f;

template <typename T, int W> struct Part { typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T)))); };
template <typename T> struct Part<T, 1> { using type = T; };

struct BalanceKernelArgs {
    const void* logits;
    const void* indices;
    uint64_t n;
    uint32_t experts, chosen, index_bytes;
    float* sums;          // blocks x experts
    uint32_t* counts;     // blocks x (experts + 1): choices of each, then rows that count
    const float* share;   // backward: of each expert, less 1 / E; then E / rows
    const float* upstream;
    void* gradient;
};

// v of another lane, without LDS: its neighbour, the other pair of its four, its mirror image in eight or in sixteen lanes
template <int CONTROL>
__device__ __forceinline__ float exchanged(float v) {
    const int x = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, CONTROL, 0xf, 0xf, true));
}

template <uint32_t TPR, typename F>
__device__ __forceinline__ float across(float v, float* lds, F&& join) {
    if constexpr (TPR >= 2) v = join(v, exchanged<0xb1>(v));
    if constexpr (TPR >= 4) v = join(v, exchanged<0x4e>(v));
    if constexpr (TPR >= 8) v = join(v, exchanged<0x141>(v));
    if constexpr (TPR >= 16) v = join(v, exchanged<0x140>(v));
    if constexpr (TPR >= 32) v = join(v, __shfl_xor(v, 16));
    if constexpr (TPR >= 64) v = join(v, __shfl_xor(v, 32));
    if constexpr (TPR > 64) {  // (a row to the block: a slot for each wave, one set of slots for each reduction of a row)
        if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (uint32_t w = 1; w < balance_waves; w++) v = join(v, lds[w]);
    }
    return v;
}

__device__ __forceinline__ int64_t choice_at(const BalanceKernelArgs& a, uint64_t i) {
    return a.index_bytes == 8 ? static_cast<const int64_t*>(a.indices)[i] : static_cast<const int32_t*>(a.indices)[i];
}

// the lane's columns of a row; what lies past the row is -inf
template <typename T, int W, uint32_t TPR, int ITEMS>
__device__ __forceinline__ void load_row(const BalanceKernelArgs& a, uint64_t row, uint32_t lane, float (&z)[ITEMS][W]) {
    const T* const p = static_cast<const T*>(a.logits) + row * a.experts;
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const uint32_t column = (k * TPR + lane) * W;
        const typename Part<T, W>::type v = *reinterpret_cast<const typename Part<T, W>::type*>(p + min(column, a.experts - W));
#pragma unroll
        for (int j = 0; j < W; j++) {
            float x;
            if constexpr (W == 1) x = static_cast<float>(v);
            else x = static_cast<float>(v[j]);
            z[k][j] = column < a.experts ? x : -__builtin_inff();
        }
    }
}

// z becomes exp(z - max); the reciprocal of their sum, 0 for a row of nothing but -inf
template <int W, uint32_t TPR, int ITEMS>
__device__ __forceinline__ float exponentials(float (&z)[ITEMS][W], float (*lds)[balance_waves]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
#pragma unroll
        for (int j = 0; j < W; j++) top = fmaxf(top, z[k][j]);
    top = across<TPR>(top, lds[0], [](float x, float y) { return fmaxf(x, y); });
    if (top == -__builtin_inff()) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            z[k][j] = __builtin_amdgcn_exp2f((z[k][j] - top) * log2_e);
            sum += z[k][j];
        }
    sum = across<TPR>(sum, lds[1], [](float x, float y) { return x + y; });
    return sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum);  // (to a step of the last place)
}

// The lane's first choice of a row (-1 where it has none). Loaded beside the logits: a load that only follows them costs their latency again.
template <uint32_t TPR>
__device__ __forceinline__ int64_t first_choice(const BalanceKernelArgs& a, uint64_t row, uint32_t lane) {
    if (a.chosen == 0) return -1;
    const int64_t e = choice_at(a, row * a.chosen + min(lane, a.chosen - 1));
    return lane < a.chosen ? e : -1;
}

// whether the row has a choice; counts its choices in `histogram`, if there is one
template <uint32_t TPR>
__device__ __forceinline__ bool row_counts(const BalanceKernelArgs& a, uint64_t row, uint32_t lane, bool active, int64_t first, uint32_t* histogram) {
    bool any = false;
    int64_t e = first;
    for (uint32_t k = lane;;) {
        const bool valid = active && static_cast<uint64_t>(e) < a.experts;
        if (valid && histogram) atomicAdd(&histogram[e], 1u);
        any |= valid;
        k += TPR;
        if (k >= a.chosen) break;
        e = choice_at(a, row * a.chosen + k);
    }
    if constexpr (TPR > 64) return __syncthreads_or(any);
    const uint64_t ballot = __ballot(any), mask = TPR >= 64 ? ~0ull : (1ull << (TPR & 63u)) - 1ull;
    return (ballot >> (threadIdx.x & 63u & ~(TPR - 1u)) & mask) != 0;
}

struct BalanceTotals {
    const float* sums;
    const uint32_t* counts;
    uint32_t blocks, experts;
    double* totals;       // experts + 1: sums of probabilities; rows
    int64_t* count;       // experts
    float* share;         // of each expert, less 1 / E; then E / rows
    float* loss;
};

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < balance_waves; w++) sum += lds[w];
    return sum;
}

// one block: shares and the loss from the totals
__device__ __forceinline__ void loss_of_totals(const BalanceTotals& a) {
    __shared__ double lds[balance_waves];
    double choices = 0.0;
    for (uint32_t e = threadIdx.x; e < a.experts; e += balance_block) choices += static_cast<double>(a.count[e]);
    choices = block_sum(choices, lds);
    const double rows = a.totals[a.experts], per_choice = choices > 0.0 ? 1.0 / choices : 0.0, per_row = rows > 0.0 ? a.experts / rows : 0.0;
    double loss = 0.0;
    for (uint32_t e = threadIdx.x; e < a.experts; e += balance_block) {
        const double count = static_cast<double>(a.count[e]);
        a.share[e] = static_cast<float>((count * a.experts - choices) * per_choice / a.experts);
        if (a.count[e] > 0) loss += count * per_choice * a.totals[e];
    }
    loss = block_sum(loss, lds);
    if (threadIdx.x == 0) {
        a.share[a.experts] = static_cast<float>(per_row);
        *a.loss = static_cast<float>(loss * per_row);
    }
}

// rows of a group of lanes whose loads are under way at once: several where a lane has few values of each
template <int W, uint32_t TPR, int ITEMS>
constexpr uint32_t rows_under_way = TPR > 64 || ITEMS * W > 8 ? 1 : ITEMS * W > 4 ? 2 : 4;

// LDS: choices of each expert (experts x 4 bytes), then, where several groups share the block, their sums (waves x experts x 4)
template <typename T, int W, uint32_t TPR, int ITEMS>
__global__ __launch_bounds__(balance_block) void balance_forward_kernel(BalanceKernelArgs a, BalanceTotals totals) {
    extern __shared__ uint32_t histogram[];
    __shared__ float slots[2][balance_waves];
    __shared__ uint32_t rows_of_wave[balance_waves];
    constexpr uint32_t groups = balance_block / TPR;
    const uint32_t lane = threadIdx.x & (TPR - 1u), group = threadIdx.x / TPR, wave = threadIdx.x >> 6;
    for (uint32_t e = threadIdx.x; e < a.experts; e += balance_block) histogram[e] = 0;
    __syncthreads();
    float sums[ITEMS][W] = {};
    uint32_t rows = 0;
    constexpr uint32_t at_once = rows_under_way<W, TPR, ITEMS>;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * groups;
    for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups; first < a.n; first += at_once * step) {
        float z[at_once][ITEMS][W];
        int64_t choice[at_once];
#pragma unroll
        for (uint32_t u = 0; u < at_once; u++) {
            const uint64_t row = min(first + u * step + group, a.n - 1);
            choice[u] = first_choice<TPR>(a, row, lane);
            load_row<T, W, TPR, ITEMS>(a, row, lane, z[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < at_once; u++) {
            const uint64_t row = first + u * step + group;
            const bool counts = row_counts<TPR>(a, min(row, a.n - 1), lane, row < a.n, choice[u], histogram);
            const float inverse = exponentials<W, TPR, ITEMS>(z[u], slots);
            rows += counts && lane == 0;
#pragma unroll
            for (int k = 0; k < ITEMS; k++)
#pragma unroll
                for (int j = 0; j < W; j++) sums[k][j] += counts ? z[u][k][j] * inverse : 0.0f;
        }
        if constexpr (TPR > 64) __syncthreads();  // (the slots are written again)
    }
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) rows += __shfl_xor(rows, o);
    if ((threadIdx.x & 63u) == 0) rows_of_wave[wave] = rows;
    float* const out = a.sums + static_cast<uint64_t>(blockIdx.x) * a.experts;
    float* const shared = reinterpret_cast<float*>(histogram + a.experts);
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            float x = sums[k][j];
#pragma unroll
            for (uint32_t o = TPR; o < 64; o <<= 1) x += __shfl_xor(x, o);
            const uint32_t column = (k * TPR + lane) * W + j;
            if (column >= a.experts) continue;
            if constexpr (TPR > 64) out[column] = x;
            else if ((threadIdx.x & 63u) < TPR) shared[wave * a.experts + column] = x;
        }
    __syncthreads();
    uint32_t* const counts = a.counts + static_cast<uint64_t>(blockIdx.x) * (a.experts + 1);
    for (uint32_t e = threadIdx.x; e < a.experts; e += balance_block) {
        counts[e] = histogram[e];
        if constexpr (TPR <= 64) {
            float x = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < balance_waves; w++) x += shared[w * a.experts + e];
            out[e] = x;
        }
    }
    if (threadIdx.x == 0) {
        uint32_t all = 0;
#pragma unroll
        for (uint32_t w = 0; w < balance_waves; w++) all += rows_of_wave[w];
        counts[a.experts] = all;
    }
    if (gridDim.x > 1) return;
    // few rows: the only block's sums are the totals, which spares two launches
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= a.experts; e += balance_block) {
        totals.totals[e] = e < a.experts ? static_cast<double>(out[e]) : static_cast<double>(counts[e]);
        if (e < a.experts) totals.count[e] = static_cast<int64_t>(counts[e]);
    }
    __syncthreads();
    loss_of_totals(totals);
}

constexpr uint32_t totals_block = 1024, totals_columns = 16, totals_parts = totals_block / totals_columns;

// sixteen columns a block, the table's rows in 64 parts, joined in their order; column `experts` is the number of rows
__global__ __launch_bounds__(totals_block) void balance_totals_kernel(BalanceTotals a) {
    __shared__ double sums[totals_parts][totals_columns];
    __shared__ uint64_t counts[totals_parts][totals_columns];
    const uint32_t c = threadIdx.x & (totals_columns - 1u), part = threadIdx.x / totals_columns, column = blockIdx.x * totals_columns + c;
    const uint32_t each = (a.blocks + totals_parts - 1) / totals_parts, last = min(a.blocks, (part + 1) * each);
    double sum = 0.0;
    uint64_t count = 0;
    if (column <= a.experts) {
        const uint32_t sum_column = min(column, a.experts - 1);
        constexpr uint32_t at_once = 4;
        for (uint32_t b = part * each; b < last; b += at_once) {
            float x[at_once];
            uint32_t n[at_once];
#pragma unroll
            for (uint32_t k = 0; k < at_once; k++) {
                const uint64_t row = min(b + k, last - 1);
                x[k] = a.sums[row * a.experts + sum_column];
                n[k] = a.counts[row * (a.experts + 1) + column];
            }
#pragma unroll
            for (uint32_t k = 0; k < at_once; k++) {
                sum += b + k < last ? static_cast<double>(x[k]) : 0.0;
                count += b + k < last ? n[k] : 0u;
            }
        }
    }
    sums[part][c] = sum;
    counts[part][c] = count;
    __syncthreads();
    if (part != 0 || column > a.experts) return;
    for (uint32_t p = 1; p < totals_parts; p++) {
        sum += sums[p][c];
        count += counts[p][c];
    }
    a.totals[column] = column < a.experts ? sum : static_cast<double>(count);
    if (column < a.experts) a.count[column] = static_cast<int64_t>(count);
}

__global__ __launch_bounds__(balance_block) void balance_loss_kernel(BalanceTotals a) { loss_of_totals(a); }

template <typename T, int W, uint32_t TPR, int ITEMS>
__global__ __launch_bounds__(balance_block) void balance_backward_kernel(BalanceKernelArgs a) {
    __shared__ float slots[3][balance_waves];
    constexpr uint32_t groups = balance_block / TPR;
    const uint32_t lane = threadIdx.x & (TPR - 1u), group = threadIdx.x / TPR;
    const float factor = a.share[a.experts] * *a.upstream;
    float share[ITEMS][W];
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
#pragma unroll
        for (int j = 0; j < W; j++) share[k][j] = a.share[min((k * TPR + lane) * W + j, a.experts - 1)];
    constexpr uint32_t at_once = rows_under_way<W, TPR, ITEMS>;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * groups;
    for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups; first < a.n; first += at_once * step) {
        float z[at_once][ITEMS][W];
        int64_t choice[at_once];
#pragma unroll
        for (uint32_t u = 0; u < at_once; u++) {
            const uint64_t row = min(first + u * step + group, a.n - 1);
            choice[u] = first_choice<TPR>(a, row, lane);
            load_row<T, W, TPR, ITEMS>(a, row, lane, z[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < at_once; u++) {
            const uint64_t row = first + u * step + group;
            const bool active = row < a.n, counts = row_counts<TPR>(a, min(row, a.n - 1), lane, active, choice[u], nullptr);
            const float inverse = exponentials<W, TPR, ITEMS>(z[u], slots);
            float mean = 0.0f;
#pragma unroll
            for (int k = 0; k < ITEMS; k++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    z[u][k][j] *= inverse;
                    mean += z[u][k][j] * share[k][j];
                }
            mean = across<TPR>(mean, slots[2], [](float x, float y) { return x + y; });
            T* const out = static_cast<T*>(a.gradient) + row * a.experts;
#pragma unroll
            for (int k = 0; k < ITEMS; k++) {
                const uint32_t column = (k * TPR + lane) * W;
                typename Part<T, W>::type v;
#pragma unroll
                for (int j = 0; j < W; j++) {
                    const T y = static_cast<T>(counts ? z[u][k][j] * (share[k][j] - mean) * factor : 0.0f);
                    if constexpr (W == 1) v = y;
                    else v[j] = y;
                }
                if (active && column < a.experts) *reinterpret_cast<typename Part<T, W>::type*>(out + column) = v;
            }
        }
        if constexpr (TPR > 64) __syncthreads();
    }
}

// calls f with a part's width, the lanes of a row and the parts of a lane; the last shape of each width holds balance_max_experts, so that f is always called
template <typename T, int W, typename F>
void with_shape(uint32_t experts, F&& f) {
    const uint32_t parts = (experts + W - 1) / W;
    constexpr uint32_t most_parts = (balance_max_experts + W - 1) / W;
    static_assert(most_parts <= 8192, "the longest shape is 256 x 32 parts");
    auto lanes = [&](auto tpr, auto items) { f(std::integral_constant<int, W>{}, tpr, items); };
#define EFGS_LANES(TPR, ITEMS) lanes(std::integral_constant<uint32_t, TPR>{}, std::integral_constant<int, ITEMS>{})
    if (parts <= 1) EFGS_LANES(1, 1);
    else if (parts <= 2) EFGS_LANES(2, 1);
    else if (parts <= 4) EFGS_LANES(4, 1);
    else if (parts <= 8) EFGS_LANES(8, 1);
    else if (parts <= 16) EFGS_LANES(16, 1);
    else if (parts <= 32) EFGS_LANES(32, 1);
    else if (parts <= 64) EFGS_LANES(64, 1);
    else if (parts <= 128) EFGS_LANES(64, 2);
    else if (parts <= 256) EFGS_LANES(64, 4);
    else if (parts <= 512) EFGS_LANES(256, 2);
    else if (parts <= 1024) EFGS_LANES(256, 4);
    else if constexpr (most_parts <= 2048) EFGS_LANES(256, 8);
    else if (parts <= 2048) EFGS_LANES(256, 8);
    else if constexpr (most_parts <= 4096) EFGS_LANES(256, 16);
    else if (parts <= 4096) EFGS_LANES(256, 16);
    else EFGS_LANES(256, 32);
#undef EFGS_LANES
}

template <typename T, typename F>
void with_type(uint32_t experts, F&& f) {
    constexpr int widest = 16 / sizeof(T);
    if (experts % widest == 0) with_shape<T, widest>(experts, [&](auto w, auto tpr, auto items) { f(T{}, w, tpr, items); });
    else if (sizeof(T) == 2 && experts % 2 == 0) with_shape<T, 2>(experts, [&](auto w, auto tpr, auto items) { f(T{}, w, tpr, items); });
    else with_shape<T, 1>(experts, [&](auto w, auto tpr, auto items) { f(T{}, w, tpr, items); });
}

template <typename F>
void dispatch(int type, uint32_t experts, F&& f) {
    if (type == type_float) with_type<float>(experts, f);
    else if (type == type_bfloat16) with_type<__bf16>(experts, f);
    else with_type<_Float16>(experts, f);
}

BalanceKernelArgs kernel_args(const BalanceArgs& a) {
    BalanceKernelArgs k{};
    k.logits = a.logits;
    k.indices = a.indices;
    k.n = a.n;
    k.experts = a.experts;
    k.chosen = a.chosen;
    k.index_bytes = static_cast<uint32_t>(a.index_bytes);
    return k;
}

// blocks whose groups all have the rows that they take at once, but enough of them where there are few rows
uint32_t blocks_for(const BalanceArgs& a) {
    uint64_t rows = 1, at_once = 1;
    dispatch(a.type, a.experts, [&](auto, auto w, auto tpr, auto items) {
        rows = balance_block / decltype(tpr)::value;
        at_once = rows_under_way<decltype(w)::value, decltype(tpr)::value, decltype(items)::value>;
    });
    if (a.n <= rows * at_once) return 1;
    const uint64_t full = (a.n + rows * at_once - 1) / (rows * at_once), most = (a.n + rows - 1) / rows;
    return static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>({full, std::min<uint64_t>(most, 512), 1}), balance_max_blocks));
}

}  // namespace

size_t balance_scratch_bytes(const BalanceArgs& a) {
    const uint64_t blocks = blocks_for(a);
    return (a.experts + 1ull) * sizeof(double) + blocks * a.experts * sizeof(float) + blocks * (a.experts + 1ull) * sizeof(uint32_t);
}

bool launch_balance_forward(const BalanceArgs& a, int64_t* counts, float* share, float* loss, void* scratch, hipStream_t s) {
    const uint32_t blocks = blocks_for(a);
    BalanceTotals t{};
    t.totals = static_cast<double*>(scratch);
    float* const sums = reinterpret_cast<float*>(t.totals + a.experts + 1);
    uint32_t* const table = reinterpret_cast<uint32_t*>(sums + static_cast<uint64_t>(blocks) * a.experts);
    t.sums = sums;
    t.counts = table;
    t.blocks = blocks;
    t.experts = a.experts;
    t.count = counts;
    t.share = share;
    t.loss = loss;
    BalanceKernelArgs k = kernel_args(a);
    k.sums = sums;
    k.counts = table;
    if (a.n > 0) {
        dispatch(a.type, a.experts, [&](auto type, auto w, auto tpr, auto items) {
            constexpr uint32_t lanes = decltype(tpr)::value;
            const size_t lds = a.experts * sizeof(uint32_t) * (lanes > 64 ? 1 : 1 + balance_waves);
            hipLaunchKernelGGL((balance_forward_kernel<decltype(type), decltype(w)::value, lanes, decltype(items)::value>), dim3(blocks),
                               dim3(balance_block), lds, s, k, t);
        });
        if (blocks == 1) {
            EFGS_HIP_CHECK(hipGetLastError());
            return true;
        }
    } else {
        t.blocks = 0;
    }
    hipLaunchKernelGGL(balance_totals_kernel, dim3(div_up(a.experts + 1ull, totals_columns)), dim3(totals_block), 0, s, t);
    hipLaunchKernelGGL(balance_loss_kernel, dim3(1), dim3(balance_block), 0, s, t);
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

bool launch_balance_backward(const BalanceArgs& a, const float* share, const float* upstream, void* gradient, hipStream_t s) {
    if (a.n == 0) return true;
    const uint32_t blocks = blocks_for(a);
    BalanceKernelArgs k = kernel_args(a);
    k.share = share;
    k.upstream = upstream;
    k.gradient = gradient;
    dispatch(a.type, a.experts, [&](auto type, auto w, auto tpr, auto items) {
        constexpr uint32_t lanes = decltype(tpr)::value;
        hipLaunchKernelGGL((balance_backward_kernel<decltype(type), decltype(w)::value, lanes, decltype(items)::value>), dim3(blocks),
                           dim3(balance_block), 0, s, k);
    });
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
