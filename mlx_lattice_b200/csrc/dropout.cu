// Dropout whose mask is a function of a counter and is never stored.
//
//   word(i) = word i % 4 of Philox4x32-10(counter = (i / 4, offset), key = seed)
//   y[i] = word(i) >= threshold ? x[i] * scale : 0   (+ residual[i])
//   threshold = round(p 2^32), scale = 1 / (1 - p)
//
// Philox4x32 with ten rounds is the generator of Salmon, Moraes, Dror and Shaw ("Parallel
// random numbers: as easy as 1, 2, 3", 2011). The backward pass is the same kernel over the
// gradient: it draws the same words again. A dropped element is selected away, not multiplied
// by zero, so an infinity or a NaN in a dropped place is gone.
//
// One read of x (and of the residual), one write of y. A thread takes 16 bytes: one counter for
// four floats, two for eight halves. 960,000 x 64 float16: 57 us, 4.3 TB/s; with a residual 61 us,
// 6.0 TB/s of the 6.55 that a copy moves; 240,000 x 96 float32: 32 us, 5.8 TB/s. Without a residual
// nothing is used up: the issue slots are 63 per cent busy, the memory 43 per cent of its nominal
// rate. Of the 19 or 20 instructions an element ten are the generator's (20 wide products and 20
// xors for four words), the others loads, conversions, selects and addresses.
#include <algorithm>

#include "common.cuh"
#include "pairs.cuh"
#include "vector_io.cuh"

namespace lat {

namespace {

constexpr int kThreads = 256;

constexpr int kRounds = 10;

// The keys of the rounds. They are the same for every element, so the host makes them; from a
// seed on the device every thread makes them, for all its elements.
struct Keys {
    uint32_t k0[kRounds], k1[kRounds];
};

__host__ __device__ inline Keys round_keys(unsigned long long seed) {
    Keys keys;
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        keys.k0[round] = k0;
        keys.k1[round] = k1;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return keys;
}

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ void multiply(uint32_t a, uint32_t b, uint32_t& low, uint32_t& high) {
    asm("{\n.reg .b64 p;\nmul.wide.u32 p, %2, %3;\nmov.b64 {%0, %1}, p;\n}" : "=r"(low), "=r"(high) : "r"(a), "r"(b));
}

__device__ __forceinline__ Words philox(uint32_t low, uint32_t high, unsigned long long offset, const Keys& keys) {
    uint32_t c0 = low, c1 = high;
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        uint32_t a_low, a_high, b_low, b_high;
        multiply(c0, 0xD2511F53u, a_low, a_high);
        multiply(c2, 0xCD9E8D57u, b_low, b_high);
        c0 = b_high ^ c1 ^ keys.k0[round];
        c1 = b_low;
        c2 = a_high ^ c3 ^ keys.k1[round];
        c3 = a_low;
    }
    return {{c0, c1, c2, c3}};
}

// Element i of the words, kept or dropped, plus the residual.
template <typename T, bool Residual>
__device__ __forceinline__ float drop(float x, float add, uint32_t word, uint32_t threshold, float scale) {
    const float kept = word >= threshold ? x * scale : 0.0f;
    return Residual ? kept + add : kept;
}

// V elements a thread, a multiple of four; the last ones of an odd total one by one. Aligned:
// V elements can be moved at once.
template <typename T, int V, bool Aligned, bool Residual, bool DeviceSeed>
__global__ void __launch_bounds__(kThreads) dropout_kernel(
    const T* x, const T* residual, long long total, uint32_t threshold, float scale, Keys keys,
    const unsigned long long* seed, unsigned long long offset, T* out
) {
    const long long first = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * V;
    if (first >= total) {
        return;
    }
    // the loads are on their way while the words are computed
    const bool whole = Aligned && first + V <= total;
    Pack<T, V> in, add, y;
    if (whole) {
        in = load_pack<T, V>(x + first);
        if (Residual) {
            add = load_pack<T, V>(residual + first);
        }
    }
    if (DeviceSeed) {
        keys = round_keys(__ldg(seed));
    }
    // A block's counters share their upper word, as a block has a power of two of them: two of the
    // 20 products are then the same for the whole block.
    const unsigned long long counter = blockIdx.x * static_cast<unsigned long long>(kThreads * V / 4);
    const uint32_t low = static_cast<uint32_t>(counter) + threadIdx.x * (V / 4);
    Words words[V / 4];
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        words[q] = philox(low + q, static_cast<uint32_t>(counter >> 32), offset, keys);
    }
    if (whole) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const Pair v = get_pair(in, i / 2);
            const Pair more = Residual ? get_pair(add, i / 2) : both(0.0f);
            set_pair(y, i / 2, {drop<T, Residual>(v.x, more.x, words[i / 4].w[i % 4], threshold, scale),
                                drop<T, Residual>(v.y, more.y, words[i / 4].w[i % 4 + 1], threshold, scale)});
        }
        store_pack<T, V>(out + first, y);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (first + i < total) {
                out[first + i] = narrow<T>(drop<T, Residual>(
                    widen<T>(x[first + i]), Residual ? widen<T>(residual[first + i]) : 0.0f, words[i / 4].w[i % 4],
                    threshold, scale));
            }
        }
    }
}

template <typename T, int V, bool Aligned, bool Residual>
void launch_dropout(const T* x, const T* residual, long long total, uint32_t threshold, float scale,
                    unsigned long long seed, const unsigned long long* seed_device, unsigned long long offset, T* out,
                    unsigned blocks, cudaStream_t stream) {
    if (seed_device != nullptr) {
        dropout_kernel<T, V, Aligned, Residual, true><<<blocks, kThreads, 0, stream>>>(
            x, residual, total, threshold, scale, Keys{}, seed_device, offset, out);
    } else {
        dropout_kernel<T, V, Aligned, Residual, false><<<blocks, kThreads, 0, stream>>>(
            x, residual, total, threshold, scale, round_keys(seed), nullptr, offset, out);
    }
}

template <typename T>
int run_dropout(const T* x, const T* residual, long long total, uint32_t threshold, float scale,
                unsigned long long seed, const unsigned long long* seed_device, unsigned long long offset, T* out,
                cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const bool aligned = aligned_to(x, 16) && aligned_to(residual, 16) && aligned_to(out, 16);
    const long long per_block = static_cast<long long>(kThreads) * V;
    const long long blocks = (total + per_block - 1) / per_block;
    LAT_REQUIRE(blocks <= 0x7fffffffLL, "dropout supports at most 2^31 blocks of elements.");
    const unsigned grid = static_cast<unsigned>(blocks);
    if (aligned && residual != nullptr) {
        launch_dropout<T, V, true, true>(x, residual, total, threshold, scale, seed, seed_device, offset, out, grid, stream);
    } else if (aligned) {
        launch_dropout<T, V, true, false>(x, residual, total, threshold, scale, seed, seed_device, offset, out, grid, stream);
    } else if (residual != nullptr) {
        launch_dropout<T, V, false, true>(x, residual, total, threshold, scale, seed, seed_device, offset, out, grid, stream);
    } else {
        launch_dropout<T, V, false, false>(x, residual, total, threshold, scale, seed, seed_device, offset, out, grid, stream);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

} // namespace

} // namespace lat

using namespace lat;

extern "C" {

int lat_dropout(
    int32_t dtype, const void* feats, const void* residual, int64_t elements, double p, uint64_t seed,
    const uint64_t* seed_device, uint64_t offset, void* out, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "dropout supports float32 and float16 tensors.");
    LAT_REQUIRE(p >= 0.0 && p < 1.0, "p must satisfy 0 <= p < 1.");
    LAT_REQUIRE(elements >= 0, "feats must have shape (N, C).");
    LAT_REQUIRE(aligned_to(seed_device, 8), "the device seed must be an aligned 64-bit word.");
    if (elements == 0) {
        return LAT_OK;
    }
    // p just below one may round to 2^32, which no word reaches: the largest word stays
    const uint32_t threshold = static_cast<uint32_t>(std::min(p * 4294967296.0 + 0.5, 4294967295.0));
    const float scale = static_cast<float>(1.0 / (1.0 - p));
    cudaStream_t stream = as_stream(stream_ptr);
    auto* words = reinterpret_cast<const unsigned long long*>(seed_device);
    if (dtype == LAT_F32) {
        return run_dropout<float>(static_cast<const float*>(feats), static_cast<const float*>(residual), elements,
                                  threshold, scale, seed, words, offset, static_cast<float*>(out), stream);
    }
    return run_dropout<__half>(static_cast<const __half*>(feats), static_cast<const __half*>(residual), elements,
                               threshold, scale, seed, words, offset, static_cast<__half*>(out), stream);
}

} // extern "C"
