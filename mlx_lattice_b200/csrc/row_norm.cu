// Layer and RMS normalisation of sparse rows for training: the forward pass that also
// leaves the row statistics, and the backward pass with the gradients of x, weight and bias.
//
//   m = mean(x) (0 for RMS), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r
//   y = xh w + b
//   g = dy w:  dx = r (g - mean(g) [layer only] - xh mean(g xh))
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// The forward pass reads x and writes y, the backward pass reads x and dy and writes dx. A group
// of L lanes (a power of two) holds a row in registers or in its own part of shared memory, so
// every element is read once and the variance is taken about the mean in a second pass over what
// is held. All sums are float32; results are rounded once.
//
// Against the 6.55 TB/s that a copy moves:
//   960,000 x 64 float16, layer   forward 41 us, 5.9 TB/s   backward 64 us + sums 3 us, 5.7 TB/s
//   240,001 x 192 float16, RMS    forward 28 us, 6.5 TB/s   backward 49 us + sums 3 us, 5.6 TB/s
//   30,011 x 1000 float32, layer  forward 43 us, 5.6 TB/s   backward 61 us + sums 3 us, 5.9 TB/s
// The RMS forward pass is bound by the memory. The layer form of narrow rows keeps the issue slots
// 74 per cent busy forward and 59 backward: two shuffle trees a row, and the sums down the rows.
//
// The gradients of weight and bias are sums down the rows. Every lane keeps the sums of the
// channels it owns over all rows it visits, a block adds its lanes' sums up in a fixed order
// and writes one partial row, and a second kernel adds the partial rows in a fixed order: no
// atomics, bitwise repeatable.
#include <algorithm>

#include "common.cuh"
#include "pairs.cuh"
#include "vector_io.cuh"

namespace lat {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int d = lanes >> 1; d > 0; d >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    return v;
}

template <typename T> struct NormArgs {
    const T* x;
    long long x_stride;
    const T* dy;
    long long dy_stride;
    long long rows;
    int channels;
    int lanes;        // lanes per row
    const T* weight;
    const T* bias;
    float eps;
    T* out;           // y, or dx
    float* mean;
    float* rstd;
    float* partial;   // [gridDim.x][2][channels]
};

// Rows that a group of lanes has in flight where a lane takes so many bytes of each: enough of
// them that a thread waits for about 64 bytes of x at once (the memory needs some 50 KB in flight
// per SM).
template <int Bytes> constexpr int kRowsInFlight = Bytes <= 8 ? 8 : Bytes <= 16 ? 4 : Bytes <= 48 ? 2 : 1;

// How a lane's part of a row moves: vectors of V elements, every L-th of the row, one a step; for
// V = 1 two elements a step, L apart, which are computed as one pair.
template <typename T, int V> struct Columns {
    static constexpr int kWidth = V == 1 ? 2 : V;   // elements of a step
    using Raw = Pack<T, kWidth>;
    int first, lanes, channels;

    __device__ __forceinline__ Columns(int sub, int lanes, int channels) : first(sub * V), lanes(lanes), channels(channels) {}
    // element i of step k
    __device__ __forceinline__ int at(int k, int i) const { return first + k * lanes * kWidth + (V == 1 ? i * lanes : i); }
    __device__ __forceinline__ bool has(int k, int i = 0) const { return at(k, i) < channels; }
    __device__ __forceinline__ Raw load(const T* row, int k) const {
        if constexpr (V == 1) {
            Raw raw = zero_pack<T, kWidth>();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (has(k, i)) {
                    raw.v[i] = row[at(k, i)];
                }
            }
            return raw;
        } else {
            return has(k) ? load_pack<T, V>(row + at(k, 0)) : zero_pack<T, V>();
        }
    }
    __device__ __forceinline__ void store(T* row, int k, const Raw& raw) const {
        if constexpr (V == 1) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (has(k, i)) {
                    row[at(k, i)] = raw.v[i];
                }
            }
        } else if (has(k)) {
            store_pack<T, V>(row + at(k, 0), raw);
        }
    }
    // a step of a vector of the row's length, or `value` without one
    __device__ __forceinline__ void vector(const T* from, int k, float value, Pair (&to)[kWidth / 2]) const {
        if (from != nullptr) {
            const Raw raw = load(from, k);
#pragma unroll
            for (int i = 0; i < kWidth / 2; ++i) {
                to[i] = get_pair(raw, i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWidth / 2; ++i) {
                to[i] = both(value);
            }
        }
    }
    // a pair of a step that the row has, with a zero behind the row's end
    __device__ __forceinline__ Pair within(int k, Pair value) const {
        return {value.x, V > 1 || has(k, 1) ? value.y : 0.0f};
    }
};

// sum / count by the rounded reciprocal and one correction of the quotient with its remainder
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990),
// a third of the instructions of a division. The remainder is exact, so the quotient is within one
// unit in the last place.
struct Count {
    float n, inverse;

    __device__ __forceinline__ explicit Count(int channels) : n(static_cast<float>(channels)), inverse(1.0f / n) {}
    __device__ __forceinline__ float mean(float sum) const {
        const float q = sum * inverse;
        return fmaf(fmaf(-q, n, sum), inverse, q);
    }
};

// The sums of all rows in flight over the lanes of a row, side by side.
template <int U> __device__ __forceinline__ void group_sums(float (&v)[U], int lanes) {
    for (int d = lanes >> 1; d > 0; d >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] += __shfl_xor_sync(0xffffffffu, v[u], d);
        }
    }
}

// All rows of a thread are loaded before the first is used. For float32, and element by element
// (V = 1) for rows of no vectors that lie apart or off a 16-byte boundary.
template <typename T, int V, int K, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_forward_kernel(NormArgs<T> p) {
    using Lane = Columns<T, V>;
    constexpr int U = kRowsInFlight<Lane::kWidth * K * sizeof(T)>, P = Lane::kWidth / 2;
    const int lane = threadIdx.x & 31;
    const int sub = lane & (p.lanes - 1);
    const int rows_per_warp = 32 / p.lanes;
    const Lane columns(sub, p.lanes, p.channels);
    const Count count(p.channels);
    const long long warp = blockIdx.x * static_cast<long long>(kWarps) + (threadIdx.x >> 5);
    const long long row0 = warp * rows_per_warp * U + lane / p.lanes;
    const int left = static_cast<int>(min(p.rows - row0, static_cast<long long>(U) * 32));   // rows from row0 on
    const T* from = p.x + row0 * p.x_stride;
    const long long step = rows_per_warp * p.x_stride;
    Pair x[U][K][P];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const auto raw = u * rows_per_warp < left ? columns.load(from + u * step, k) : zero_pack<T, Lane::kWidth>();
#pragma unroll
            for (int i = 0; i < P; ++i) {
                x[u][k][i] = get_pair(raw, i);
            }
        }
    }
    float mean[U], r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Pair sum = both(0.0f);
        if (!Rms) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    sum = sum + x[u][k][i];
                }
            }
        }
        mean[u] = sum.x + sum.y;
    }
    if (!Rms) {
        group_sums(mean, p.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = count.mean(mean[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Pair squares = both(0.0f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (columns.has(k)) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    if (!Rms) {
                        x[u][k][i] = columns.within(k, minus(x[u][k][i], both(mean[u])));
                    }
                    squares = fma(x[u][k][i], x[u][k][i], squares);
                }
            }
        }
        r[u] = squares.x + squares.y;
    }
    group_sums(r, p.lanes);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        r[u] = rsqrtf(fmaf(r[u], count.inverse, p.eps));
        const long long row = row0 + u * rows_per_warp;
        if (sub == 0 && u * rows_per_warp < left) {
            p.rstd[row] = r[u];
            if (!Rms) {
                p.mean[row] = mean[u];
            }
        }
    }
    T* to = p.out + row0 * p.channels;
    const long long down = static_cast<long long>(rows_per_warp) * p.channels;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!columns.has(k)) {
            break;
        }
        Pair w[P], b[P];
        columns.vector(p.weight, k, 1.0f, w);
        columns.vector(p.bias, k, 0.0f, b);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            typename Lane::Raw y;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const Pair xh = x[u][k][i] * both(r[u]);
                set_pair(y, i, Rms ? xh * w[i] : fma(xh, w[i], b[i]));
            }
            if (u * rows_per_warp < left) {
                columns.store(to + u * down, k, y);
            }
        }
    }
}

// The sums of a block: lanes of a warp that own the same channels; the upper warps' sums to the
// lower ones; then the four sums of each channel, as a partial row, or as the result of the only
// block.
template <typename T, int V, int K, int P>
__device__ __forceinline__ void finish_sums(
    const NormArgs<T>& p, Pair (&dw)[K][P], Pair (&db)[K][P], float* sums, T* dw_out, T* db_out
) {
    using Lane = Columns<T, V>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Lane columns(lane & (p.lanes - 1), p.lanes, p.channels);
    if (dw_out == nullptr && db_out == nullptr) {
        return;
    }
    for (int d = p.lanes; d < 32; d <<= 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                dw[k][i].x += __shfl_xor_sync(0xffffffffu, dw[k][i].x, d);
                dw[k][i].y += __shfl_xor_sync(0xffffffffu, dw[k][i].y, d);
                db[k][i].x += __shfl_xor_sync(0xffffffffu, db[k][i].x, d);
                db[k][i].y += __shfl_xor_sync(0xffffffffu, db[k][i].y, d);
            }
        }
    }
    constexpr int kHalf = kWarps / 2;
    float* mine = sums + static_cast<size_t>(warp % kHalf) * 2 * p.channels;
#pragma unroll
    for (int phase = 0; phase < 2; ++phase) {
        if ((warp >= kHalf) == (phase == 0) && lane < p.lanes) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < Lane::kWidth; ++i) {
                    const int c = columns.at(k, i);
                    if (c < p.channels) {
                        const float w_sum = i % 2 == 0 ? dw[k][i / 2].x : dw[k][i / 2].y;
                        const float b_sum = i % 2 == 0 ? db[k][i / 2].x : db[k][i / 2].y;
                        mine[c] = phase == 0 ? w_sum : w_sum + mine[c];
                        mine[p.channels + c] = phase == 0 ? b_sum : b_sum + mine[p.channels + c];
                    }
                }
            }
        }
        __syncthreads();
    }
    float* partial = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.channels;
    for (int c = threadIdx.x; c < 2 * p.channels; c += kThreads) {
        float total = 0.0f;
#pragma unroll
        for (int q = 0; q < kHalf; ++q) {
            total += sums[static_cast<size_t>(q) * 2 * p.channels + c];
        }
        if (gridDim.x > 1) {
            partial[c] = total;
        } else if (c < p.channels ? dw_out != nullptr : db_out != nullptr) {
            (c < p.channels ? dw_out : db_out)[c < p.channels ? c : c - p.channels] = narrow<T>(total);
        }
    }
}

// The backward pass for rows of 16-byte vectors. The rows on their way lie in a ring in shared
// memory that asynchronous copies fill, a thread copying what it reads itself: nothing is
// synchronised, and rows in flight cost no registers, of which the sums take up to 128.
template <int K> constexpr int kRingRows = K == 1 ? 2 : 1;   // rows of a thread in a stage
template <int K> constexpr int kRingStages = K <= 2 ? 4 : K <= 4 ? 3 : 2;
template <int K> constexpr int kRingVectors = kRingRows<K> * K * 2;   // of a thread in a stage
// blocks of an SM, by the registers that the sums of V * K channels leave
template <int V, int K> constexpr int kRingBlocks = V * K <= 4 || (V == 4 && K == 2) ? 3 : V * K <= 16 ? 2 : 1;

template <int K> constexpr size_t ring_bytes() {
    return static_cast<size_t>(kRingStages<K>) * kThreads * (kRingVectors<K> * 16 + kRingRows<K> * 8);
}

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy_vector(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_word(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_address(to)), "l"(from) : "memory");
}

template <typename T, int K, bool Rms>
__global__ void __launch_bounds__(kThreads, kRingBlocks<16 / sizeof(T), K>) norm_backward_ring_kernel(NormArgs<T> p, T* dw_out, T* db_out) {
    constexpr int V = 16 / static_cast<int>(sizeof(T)), P = V / 2, U = kRingRows<K>, S = kRingStages<K>;
    extern __shared__ __align__(16) unsigned char memory[];
    using Vector = Pack<T, V>;
    // [stage][row][vector][x, dy][thread], then [stage][row][rstd, mean][thread]
    Vector* vectors = reinterpret_cast<Vector*>(memory) + threadIdx.x;
    float* stats = reinterpret_cast<float*>(memory + static_cast<size_t>(S) * kRingVectors<K> * kThreads * 16) + threadIdx.x;
    const auto vector_at = [&](int stage, int u, int k, int array) -> Vector* {
        return vectors + (((stage * U + u) * K + k) * 2 + array) * kThreads;
    };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & (p.lanes - 1), rows_per_warp = 32 / p.lanes;
    const Count count(p.channels);
    Pair dw[K][P], db[K][P], w[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (sub + k * p.lanes) * V;
        const bool weighted = p.weight != nullptr && c < p.channels;
        Vector raw;
        if (weighted) {
            raw = load_pack<T, V>(p.weight + c);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            dw[k][i] = db[k][i] = both(0.0f);
            w[k][i] = weighted ? get_pair(raw, i) : both(1.0f);
        }
        if (c >= p.channels) {   // zeros for good: with dy every term is zero there
#pragma unroll
            for (int at = 0; at < S * U; ++at) {
                *vector_at(at / U, at % U, k, 0) = *vector_at(at / U, at % U, k, 1) = zero_pack<T, V>();
            }
        }
    }
    const int step_rows = static_cast<int>(gridDim.x) * kWarps * rows_per_warp * U;   // of all blocks in a turn
    long long left = p.rows - (blockIdx.x * static_cast<long long>(kWarps) + warp) * rows_per_warp * U - lane / p.lanes;
    const long long row0 = p.rows - left;
    const T* x_from = p.x + row0 * p.x_stride + sub * V;
    const T* dy_from = p.dy + row0 * p.dy_stride + sub * V;
    const float* rstd_from = p.rstd + row0;
    const float* mean_from = Rms ? nullptr : p.mean + row0;
    T* to = p.out + row0 * p.channels + sub * V;
    const long long x_step = rows_per_warp * p.x_stride, dy_step = rows_per_warp * p.dy_stride;
    long long to_fetch = left;
    const auto fetch = [&](int stage) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = u * rows_per_warp < to_fetch;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if ((sub + k * p.lanes) * V < p.channels) {
                    if (live) {
                        copy_vector(vector_at(stage, u, k, 0), x_from + u * x_step + k * p.lanes * V);
                        copy_vector(vector_at(stage, u, k, 1), dy_from + u * dy_step + k * p.lanes * V);
                    } else {
                        *vector_at(stage, u, k, 0) = *vector_at(stage, u, k, 1) = zero_pack<T, V>();
                    }
                }
            }
            float* stat = stats + (stage * U + u) * 2 * kThreads;
            if (live) {
                copy_word(stat, rstd_from + u * rows_per_warp);
                if (!Rms) {
                    copy_word(stat + kThreads, mean_from + u * rows_per_warp);
                }
            } else {
                stat[0] = stat[kThreads] = 0.0f;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        x_from += step_rows * p.x_stride;
        dy_from += step_rows * p.dy_stride;
        rstd_from += step_rows;
        mean_from += Rms ? 0 : step_rows;
        to_fetch -= step_rows;
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        fetch(s);
    }
    int stage = 0;
    // the warp goes on as long as its first row exists
    for (long long first_left = left + lane / p.lanes; first_left > 0; first_left -= step_rows) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        fetch((stage + S - 1) % S);
        float r[U], mean[U], c1[U], c2[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* stat = stats + (stage * U + u) * 2 * kThreads;
            r[u] = stat[0];
            mean[u] = Rms ? 0.0f : stat[kThreads];
            Pair s1 = both(0.0f), s2 = both(0.0f);
            const Pair scale = both(r[u]), shift = both(mean[u]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Vector x_raw = *vector_at(stage, u, k, 0), dy_raw = *vector_at(stage, u, k, 1);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const Pair d = get_pair(dy_raw, i), x = get_pair(x_raw, i);
                    const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                    const Pair g = d * w[k][i];
                    if (!Rms) {
                        s1 = s1 + g;
                        db[k][i] = db[k][i] + d;
                    }
                    s2 = fma(g, xh, s2);
                    dw[k][i] = fma(d, xh, dw[k][i]);
                }
            }
            c1[u] = s1.x + s1.y;
            c2[u] = s2.x + s2.y;
        }
        if (!Rms) {
            group_sums(c1, p.lanes);
        }
        group_sums(c2, p.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // r (g - c1 - xh c2) with xh = (x - m) r
            const Pair scale = both(r[u]), shift = both(mean[u]);
            const Pair minus_c1 = both(-count.mean(c1[u])), minus_c2 = both(-count.mean(c2[u]));
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Vector x_raw = *vector_at(stage, u, k, 0), dy_raw = *vector_at(stage, u, k, 1);
                Vector dx;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const Pair d = get_pair(dy_raw, i), x = get_pair(x_raw, i);
                    const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                    const Pair g = Rms ? d * w[k][i] : fma(d, w[k][i], minus_c1);
                    set_pair(dx, i, scale * fma(xh, minus_c2, g));
                }
                if (u * rows_per_warp < left && (sub + k * p.lanes) * V < p.channels) {
                    store_pack<T, V>(to + static_cast<long long>(u * rows_per_warp) * p.channels + k * p.lanes * V, dx);
                }
            }
        }
        to += static_cast<long long>(step_rows) * p.channels;
        left -= step_rows;
        stage = (stage + 1) % S;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();   // the ring's memory takes the sums
    finish_sums<T, V, K, P>(p, dw, db, reinterpret_cast<float*>(memory), dw_out, db_out);
}

// The forward pass for rows of 16-byte vectors, the same way.
template <int K> constexpr int kForwardRows = K <= 2 ? 2 : 1;   // of a thread in a stage
template <int K> constexpr int kForwardStages = K <= 2 ? 4 : 3;
template <int V, int K> constexpr int kForwardBlocks = V * K <= 8 ? 4 : 2;
// The ring pays where the kernel is bound by its instructions, for float16 (45 to 54 us against 52
// to 55 with every row loaded before the first is used, 120 MB of rows of 16 to 768 channels);
// float32 is faster without (41 to 44 us against 43 to 49).
template <typename T> constexpr bool kForwardRing = sizeof(T) == 2;

template <typename T, int K, bool Rms>
__global__ void __launch_bounds__(kThreads, kForwardBlocks<16 / sizeof(T), K>) norm_forward_ring_kernel(NormArgs<T> p) {
    constexpr int V = 16 / static_cast<int>(sizeof(T)), P = V / 2, U = kForwardRows<K>, S = kForwardStages<K>;
    extern __shared__ __align__(16) unsigned char memory[];
    using Vector = Pack<T, V>;
    Vector* vectors = reinterpret_cast<Vector*>(memory) + threadIdx.x;   // [stage][row][vector][thread]
    const auto vector_at = [&](int stage, int u, int k) -> Vector* { return vectors + ((stage * U + u) * K + k) * kThreads; };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & (p.lanes - 1), rows_per_warp = 32 / p.lanes;
    const Count count(p.channels);
    Pair w[K][P], b[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (sub + k * p.lanes) * V;
        const bool in = c < p.channels;
        Vector w_raw, b_raw;
        if (in && p.weight != nullptr) {
            w_raw = load_pack<T, V>(p.weight + c);
        }
        if (in && p.bias != nullptr) {
            b_raw = load_pack<T, V>(p.bias + c);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            w[k][i] = in && p.weight != nullptr ? get_pair(w_raw, i) : both(1.0f);
            b[k][i] = in && p.bias != nullptr ? get_pair(b_raw, i) : both(0.0f);
        }
        if (!in) {
#pragma unroll
            for (int at = 0; at < S * U; ++at) {
                *vector_at(at / U, at % U, k) = zero_pack<T, V>();
            }
        }
    }
    const int step_rows = static_cast<int>(gridDim.x) * kWarps * rows_per_warp * U;
    long long left = p.rows - (blockIdx.x * static_cast<long long>(kWarps) + warp) * rows_per_warp * U - lane / p.lanes;
    const long long row0 = p.rows - left;
    const T* from = p.x + row0 * p.x_stride + sub * V;
    T* to = p.out + row0 * p.channels + sub * V;
    float* mean_to = p.mean + row0;
    float* rstd_to = p.rstd + row0;
    const long long step = rows_per_warp * p.x_stride;
    long long to_fetch = left;
    const auto fetch = [&](int stage) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * rows_per_warp < to_fetch) {   // a row that does not exist is computed from what lies there
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if ((sub + k * p.lanes) * V < p.channels) {
                        copy_vector(vector_at(stage, u, k), from + u * step + k * p.lanes * V);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        from += step_rows * p.x_stride;
        to_fetch -= step_rows;
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        fetch(s);
    }
    int stage = 0;
    for (long long first_left = left + lane / p.lanes; first_left > 0; first_left -= step_rows) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        fetch((stage + S - 1) % S);
        Pair x[U][K][P];
        float mean[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Pair sum = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Vector raw = *vector_at(stage, u, k);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    x[u][k][i] = get_pair(raw, i);
                    if (!Rms) {
                        sum = sum + x[u][k][i];
                    }
                }
            }
            mean[u] = sum.x + sum.y;
        }
        if (!Rms) {
            group_sums(mean, p.lanes);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = Rms ? 0.0f : count.mean(mean[u]);
            Pair squares = both(0.0f);
            const Pair shift = both(mean[u]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if ((sub + k * p.lanes) * V < p.channels) {
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        if (!Rms) {
                            x[u][k][i] = minus(x[u][k][i], shift);
                        }
                        squares = fma(x[u][k][i], x[u][k][i], squares);
                    }
                }
            }
            r[u] = squares.x + squares.y;
        }
        group_sums(r, p.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r[u] = rsqrtf(fmaf(r[u], count.inverse, p.eps));
            if (u * rows_per_warp < left) {
                if (sub == 0) {
                    rstd_to[u * rows_per_warp] = r[u];
                    if (!Rms) {
                        mean_to[u * rows_per_warp] = mean[u];
                    }
                }
                const Pair scale = both(r[u]);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    Vector y;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const Pair xh = x[u][k][i] * scale;
                        set_pair(y, i, Rms ? xh * w[k][i] : fma(xh, w[k][i], b[k][i]));
                    }
                    if ((sub + k * p.lanes) * V < p.channels) {
                        store_pack<T, V>(to + static_cast<long long>(u * rows_per_warp) * p.channels + k * p.lanes * V, y);
                    }
                }
            }
        }
        to += static_cast<long long>(step_rows) * p.channels;
        mean_to += Rms ? 0 : step_rows;
        rstd_to += step_rows;
        left -= step_rows;
        stage = (stage + 1) % S;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// For rows of no vectors that lie apart or off a 16-byte boundary, element by element.
template <int Bytes> constexpr int kBackwardRows = Bytes <= 8 ? 4 : Bytes <= 16 ? 2 : 1;

template <typename T, int K, bool Rms>
__global__ void __launch_bounds__(kThreads, K <= 6 ? 2 : 1) norm_backward_kernel(NormArgs<T> p, T* dw_out, T* db_out) {
    constexpr int V = 1;
    using Lane = Columns<T, V>;
    constexpr int U = kBackwardRows<Lane::kWidth * K * sizeof(T)>, P = Lane::kWidth / 2;
    extern __shared__ float sums[];  // [kWarps / 2][2][channels]
    const int lane = threadIdx.x & 31;
    const int sub = lane & (p.lanes - 1);
    const int rows_per_warp = 32 / p.lanes;
    const Lane columns(sub, p.lanes, p.channels);
    const Count count(p.channels);
    const int warp = threadIdx.x >> 5;
    Pair dw[K][P], db[K][P], w[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        columns.vector(p.weight, k, 1.0f, w[k]);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            dw[k][i] = db[k][i] = both(0.0f);
        }
    }
    const long long stride = static_cast<long long>(gridDim.x) * kWarps * rows_per_warp * U;
    const long long x_step = rows_per_warp * p.x_stride, dy_step = rows_per_warp * p.dy_stride;
    const long long down = static_cast<long long>(rows_per_warp) * p.channels;
    for (long long base = (blockIdx.x * static_cast<long long>(kWarps) + warp) * rows_per_warp * U; base < p.rows;
         base += stride) {
        const long long row0 = base + lane / p.lanes;
        const int left = static_cast<int>(min(p.rows - row0, static_cast<long long>(U) * 32));
        const T* x_from = p.x + row0 * p.x_stride;
        const T* dy_from = p.dy + row0 * p.dy_stride;
        T* to = p.out + row0 * p.channels;
        typename Lane::Raw x_raw[U][K], dy_raw[U][K];
        float r[U], mean[U], c1[U], c2[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = u * rows_per_warp < left;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                x_raw[u][k] = live ? columns.load(x_from + u * x_step, k) : zero_pack<T, Lane::kWidth>();
                dy_raw[u][k] = live ? columns.load(dy_from + u * dy_step, k) : zero_pack<T, Lane::kWidth>();
            }
            r[u] = live ? p.rstd[row0 + u * rows_per_warp] : 0.0f;
            mean[u] = !Rms && live ? p.mean[row0 + u * rows_per_warp] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Pair s1 = both(0.0f), s2 = both(0.0f);
            const Pair scale = both(r[u]), shift = both(mean[u]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    // zeros beyond the row's end: dy and with it every term is zero there
                    const Pair d = get_pair(dy_raw[u][k], i), x = get_pair(x_raw[u][k], i);
                    const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                    const Pair g = d * w[k][i];
                    if (!Rms) {
                        s1 = s1 + g;
                        db[k][i] = db[k][i] + d;
                    }
                    s2 = fma(g, xh, s2);
                    dw[k][i] = fma(d, xh, dw[k][i]);
                }
            }
            c1[u] = s1.x + s1.y;
            c2[u] = s2.x + s2.y;
        }
        if (!Rms) {
            group_sums(c1, p.lanes);
        }
        group_sums(c2, p.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // r (g - c1 - xh c2) with xh = (x - m) r
            const Pair scale = both(r[u]), shift = both(mean[u]);
            const Pair minus_c1 = both(-count.mean(c1[u])), minus_c2 = both(-count.mean(c2[u]));
#pragma unroll
            for (int k = 0; k < K; ++k) {
                typename Lane::Raw dx;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const Pair d = get_pair(dy_raw[u][k], i), x = get_pair(x_raw[u][k], i);
                    const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                    const Pair g = Rms ? d * w[k][i] : fma(d, w[k][i], minus_c1);
                    set_pair(dx, i, scale * fma(xh, minus_c2, g));
                }
                if (u * rows_per_warp < left) {
                    columns.store(to + u * down, k, dx);
                }
            }
        }
    }
    finish_sums<T, V, K, P>(p, dw, db, sums, dw_out, db_out);
}

// Rows that lie one behind the other but do not come in 16-byte vectors. A warp takes a batch of
// them, which is one range of memory: 16-byte copies bring it to shared memory, a lane computes
// its elements in place there, and 16-byte stores take the batch away; a 16-byte word that two
// batches share is stored by elements. A batch is on its way while the one before it is computed.
// 120 MB of rows, forward and backward, against every element loaded from global memory: 62 float16
// 74 / 120 us (206 / 412), 63 float16 97 / 164 (133 / 176), 191 float16 102 / 173 (144 / 395), 97
// float32 97 / 130 (98 / 283), 999 float32 88 / 120 (81 / 278). Bound by the instructions that take
// one or two elements at a time.
constexpr int kBatchStages = 2;
constexpr int kBatchBytes = 2560;   // of a batch, at least; 1536 bytes take 63 float16 105 / 175 us

struct Batches {
    int rows;                     // of a batch
    int bytes;                    // of its range in shared memory, whatever its start
    int stage;                    // bytes of a stage: the ranges of x and, backward, dy, rstd and mean
};

template <typename T> inline Batches batches_of(int channels, int lanes, bool backward) {
    const int at_once = 32 / lanes, row = channels * static_cast<int>(sizeof(T));
    Batches b;
    const int group = at_once * (row + 8);   // with the statistics, which outweigh the narrowest rows
    b.rows = at_once * ((kBatchBytes + group - 1) / group);
    b.bytes = (b.rows * row + 15) / 16 * 16 + 16;
    b.stage = backward ? 2 * b.bytes + (2 * 4 * b.rows + 15) / 16 * 16 : b.bytes;
    return b;
}

// blocks of an SM, by the registers that a lane's elements of a row take
template <int Elements, bool Backward>
constexpr int kBatchBlocks = Backward ? (Elements <= 4 ? 4 : Elements <= 8 ? 3 : Elements <= 12 ? 2 : 1)
                                      : (Elements <= 8 ? 4 : Elements <= 12 ? 3 : Elements <= 24 ? 2 : 1);

// A batch of a warp: `row` and the rows behind it, as far as the array goes.
template <typename T> struct Range {
    long long begin, end, total;   // bytes of the array

    __device__ __forceinline__ Range(const NormArgs<T>& p, const Batches& b, long long row) {
        const long long bytes = static_cast<long long>(p.channels) * sizeof(T);
        total = p.rows * bytes;
        begin = min(row, p.rows) * bytes;
        end = min(begin + b.rows * bytes, total);
    }
    __device__ __forceinline__ int shift() const { return static_cast<int>(begin & 15); }
    // 16-byte words that hold a byte of the range, not past the array's end
    __device__ __forceinline__ void fetch(unsigned char* to, const T* from) const {
        const long long base = begin - shift();
        const unsigned char* bytes = reinterpret_cast<const unsigned char*>(from);
        for (long long at = base + (threadIdx.x & 31) * 16; at < end; at += 512) {
            const int size = static_cast<int>(min(total - at, 16LL));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(to + (at - base))),
                         "l"(bytes + at), "r"(size) : "memory");
        }
    }
    __device__ __forceinline__ void store(const unsigned char* from, T* to) const {
        const int lane = threadIdx.x & 31;
        const long long base = begin - shift();
        unsigned char* bytes = reinterpret_cast<unsigned char*>(to);
        const long long first = min((begin + 15) / 16 * 16, end), last = max(end / 16 * 16, first);
        for (long long at = first + lane * 16; at < last; at += 512) {
            *reinterpret_cast<uint4*>(bytes + at) = *reinterpret_cast<const uint4*>(from + (at - base));
        }
        // up to 16 / sizeof(T) - 1 elements before the first whole word, and behind the last
        constexpr int kEdge = 16 / static_cast<int>(sizeof(T));
        const long long at = lane < kEdge ? begin + lane * static_cast<int>(sizeof(T))
                                          : last + (lane - kEdge) * static_cast<int>(sizeof(T));
        if (lane < kEdge ? at < first : lane < 2 * kEdge && at < end) {
            *reinterpret_cast<T*>(bytes + at) = *reinterpret_cast<const T*>(from + (at - base));
        }
    }
};

template <typename T, int V, int K, bool Rms>
__global__ void __launch_bounds__(kThreads, kBatchBlocks<Columns<T, V>::kWidth * K, false>) norm_forward_batch_kernel(NormArgs<T> p, Batches batches) {
    using Lane = Columns<T, V>;
    constexpr int W = Lane::kWidth, P = W / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & (p.lanes - 1), rows_per_warp = 32 / p.lanes;
    unsigned char* mine = memory + warp * kBatchStages * batches.stage;
    const Lane columns(sub, p.lanes, p.channels);
    const Count count(p.channels);
    Pair w[K][P], b[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        columns.vector(p.weight, k, 1.0f, w[k]);
        columns.vector(p.bias, k, 0.0f, b[k]);
    }
    const long long step = static_cast<long long>(gridDim.x) * kWarps * batches.rows;
    long long row = (blockIdx.x * static_cast<long long>(kWarps) + warp) * batches.rows;
    Range<T>(p, batches, row).fetch(mine, p.x);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int stage = 0; row < p.rows; row += step, stage ^= 1) {
        Range<T>(p, batches, row + step).fetch(mine + (stage ^ 1) * batches.stage, p.x);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const Range<T> range(p, batches, row);
        unsigned char* data = mine + stage * batches.stage;
        const int rows = static_cast<int>(min(p.rows - row, static_cast<long long>(batches.rows)));
        for (int first = 0; first < rows; first += rows_per_warp) {
            const int at = first + lane / p.lanes;
            T* values = reinterpret_cast<T*>(data + range.shift()) + at * p.channels;
            Pair x[K][P], sum = both(0.0f), squares = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const auto raw = at < rows ? columns.load(values, k) : zero_pack<T, W>();
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    x[k][i] = get_pair(raw, i);
                    sum = sum + x[k][i];
                }
            }
            float mean[1] = {0.0f}, r[1];
            if (!Rms) {
                mean[0] = sum.x + sum.y;
                group_sums(mean, p.lanes);
                mean[0] = count.mean(mean[0]);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (columns.has(k)) {
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        if (!Rms) {
                            x[k][i] = columns.within(k, minus(x[k][i], both(mean[0])));
                        }
                        squares = fma(x[k][i], x[k][i], squares);
                    }
                }
            }
            r[0] = squares.x + squares.y;
            group_sums(r, p.lanes);
            r[0] = rsqrtf(fmaf(r[0], count.inverse, p.eps));
            if (at < rows) {
                if (sub == 0) {
                    p.rstd[row + at] = r[0];
                    if (!Rms) {
                        p.mean[row + at] = mean[0];
                    }
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    typename Lane::Raw y;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const Pair xh = x[k][i] * both(r[0]);
                        set_pair(y, i, Rms ? xh * w[k][i] : fma(xh, w[k][i], b[k][i]));
                    }
                    columns.store(values, k, y);
                }
            }
        }
        __syncwarp();
        range.store(data, p.out);
        __syncwarp();   // the next turn's copies overwrite this stage
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, int V, int K, bool Rms>
__global__ void __launch_bounds__(kThreads, kBatchBlocks<Columns<T, V>::kWidth * K, true>) norm_backward_batch_kernel(
    NormArgs<T> p, Batches batches, T* dw_out, T* db_out
) {
    using Lane = Columns<T, V>;
    constexpr int W = Lane::kWidth, P = W / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & (p.lanes - 1), rows_per_warp = 32 / p.lanes;
    unsigned char* mine = memory + warp * kBatchStages * batches.stage;
    const Lane columns(sub, p.lanes, p.channels);
    const Count count(p.channels);
    Pair dw[K][P], db[K][P], w[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        columns.vector(p.weight, k, 1.0f, w[k]);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            dw[k][i] = db[k][i] = both(0.0f);
        }
    }
    const long long step = static_cast<long long>(gridDim.x) * kWarps * batches.rows;
    long long row = (blockIdx.x * static_cast<long long>(kWarps) + warp) * batches.rows;
    const auto fetch = [&](long long from, int stage) {
        const Range<T> range(p, batches, from);
        unsigned char* data = mine + stage * batches.stage;
        range.fetch(data, p.x);
        range.fetch(data + batches.bytes, p.dy);
        float* stats = reinterpret_cast<float*>(data + 2 * batches.bytes);
        for (long long i = lane; i < batches.rows && from + i < p.rows; i += 32) {
            copy_word(stats + i, p.rstd + from + i);
            if (!Rms) {
                copy_word(stats + batches.rows + i, p.mean + from + i);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(row, 0);
    for (int stage = 0; row < p.rows; row += step, stage ^= 1) {
        fetch(row + step, stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const Range<T> range(p, batches, row);
        unsigned char* data = mine + stage * batches.stage;
        const float* stats = reinterpret_cast<const float*>(data + 2 * batches.bytes);
        const int rows = static_cast<int>(min(p.rows - row, static_cast<long long>(batches.rows)));
        for (int first = 0; first < rows; first += rows_per_warp) {
            const int at = first + lane / p.lanes;
            const bool live = at < rows;
            const T* x_values = reinterpret_cast<const T*>(data + range.shift()) + at * p.channels;
            T* dy_values = reinterpret_cast<T*>(data + batches.bytes + range.shift()) + at * p.channels;
            const Pair scale = both(live ? stats[at] : 0.0f), shift = both(!Rms && live ? stats[batches.rows + at] : 0.0f);
            Pair s1 = both(0.0f), s2 = both(0.0f);
            typename Lane::Raw x_raw[K], dy_raw[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                x_raw[k] = live ? columns.load(x_values, k) : zero_pack<T, W>();
                dy_raw[k] = live ? columns.load(dy_values, k) : zero_pack<T, W>();
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const Pair d = get_pair(dy_raw[k], i), x = get_pair(x_raw[k], i);
                    const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                    const Pair g = d * w[k][i];
                    if (!Rms) {
                        s1 = s1 + g;
                        db[k][i] = db[k][i] + d;
                    }
                    s2 = fma(g, xh, s2);
                    dw[k][i] = fma(d, xh, dw[k][i]);
                }
            }
            float c1[1] = {s1.x + s1.y}, c2[1] = {s2.x + s2.y};
            if (!Rms) {
                group_sums(c1, p.lanes);
            }
            group_sums(c2, p.lanes);
            const Pair minus_c1 = both(-count.mean(c1[0])), minus_c2 = both(-count.mean(c2[0]));
            if (live) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    typename Lane::Raw dx;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const Pair d = get_pair(dy_raw[k], i), x = get_pair(x_raw[k], i);
                        const Pair xh = (Rms ? x : minus(x, shift)) * scale;
                        const Pair g = Rms ? d * w[k][i] : fma(d, w[k][i], minus_c1);
                        set_pair(dx, i, scale * fma(xh, minus_c2, g));
                    }
                    columns.store(dy_values, k, dx);
                }
            }
        }
        __syncwarp();
        range.store(data + batches.bytes, p.out);
        __syncwarp();   // the next turn's copies overwrite this stage
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();   // the batches' memory takes the sums
    finish_sums<T, V, K, P>(p, dw, db, reinterpret_cast<float*>(memory), dw_out, db_out);
}

// Rows wider than the registers of a warp: one block per row, element by element, three passes
// over a row that stays in L1 / L2, and the sums down the rows by another kernel that reads x and dy
// again. Far from the memory's rate: 30,000 x 2048 forward 115 us float16, 111 float32 (38 and
// 75 at 6.55 TB/s), backward with its sums 278 and 304 (56 and 112).
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = group_sum(v, 32);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        scratch[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
        total += scratch[w];
    }
    return total;
}

template <typename T, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_forward_wide_kernel(NormArgs<T> p) {
    __shared__ float scratch[kWarps];
    const float count = static_cast<float>(p.channels);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = p.x + row * p.x_stride;
        float mean = 0.0f;
        if (!Rms) {
            float sum = 0.0f;
            for (int c = threadIdx.x; c < p.channels; c += kThreads) {
                sum += widen<T>(x[c]);
            }
            mean = block_sum(sum, scratch) / count;
        }
        float squares = 0.0f;
        for (int c = threadIdx.x; c < p.channels; c += kThreads) {
            const float d = widen<T>(x[c]) - mean;
            squares = fmaf(d, d, squares);
        }
        const float r = rsqrtf(block_sum(squares, scratch) / count + p.eps);
        if (threadIdx.x == 0) {
            p.rstd[row] = r;
            if (!Rms) {
                p.mean[row] = mean;
            }
        }
        T* y = p.out + row * p.channels;
        for (int c = threadIdx.x; c < p.channels; c += kThreads) {
            float v = (widen<T>(x[c]) - mean) * r;
            if (p.weight != nullptr) {
                v *= widen<T>(p.weight[c]);
            }
            if (p.bias != nullptr) {
                v += widen<T>(p.bias[c]);
            }
            y[c] = narrow<T>(v);
        }
    }
}

template <typename T, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_backward_wide_kernel(NormArgs<T> p) {
    __shared__ float scratch[kWarps];
    const float count = static_cast<float>(p.channels);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = p.x + row * p.x_stride;
        const T* dy = p.dy + row * p.dy_stride;
        const float r = p.rstd[row];
        const float mean = Rms ? 0.0f : p.mean[row];
        float c1 = 0.0f, c2 = 0.0f;
        for (int c = threadIdx.x; c < p.channels; c += kThreads) {
            const float g = widen<T>(dy[c]) * (p.weight != nullptr ? widen<T>(p.weight[c]) : 1.0f);
            c1 += g;
            c2 = fmaf(g, (widen<T>(x[c]) - mean) * r, c2);
        }
        c1 = Rms ? 0.0f : block_sum(c1, scratch) / count;
        c2 = block_sum(c2, scratch) / count;
        T* dx = p.out + row * p.channels;
        for (int c = threadIdx.x; c < p.channels; c += kThreads) {
            const float g = widen<T>(dy[c]) * (p.weight != nullptr ? widen<T>(p.weight[c]) : 1.0f);
            const float xh = (widen<T>(x[c]) - mean) * r;
            dx[c] = narrow<T>(r * (g - c1 - xh * c2));
        }
    }
}

// Partial sums of the wide form: a thread per channel walks a range of rows.
template <typename T, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_sums_wide_kernel(NormArgs<T> p, long long rows_per_block) {
    const int c = blockIdx.y * kThreads + threadIdx.x;
    if (c >= p.channels) {
        return;
    }
    const long long begin = blockIdx.x * rows_per_block;
    const long long end = begin + rows_per_block < p.rows ? begin + rows_per_block : p.rows;
    float dw = 0.0f, db = 0.0f;
    for (long long row = begin; row < end; ++row) {
        const float d = widen<T>(p.dy[row * p.dy_stride + c]);
        const float mean = Rms ? 0.0f : p.mean[row];
        dw = fmaf(d, (widen<T>(p.x[row * p.x_stride + c]) - mean) * p.rstd[row], dw);
        db += d;
    }
    float* partial = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.channels;
    partial[c] = dw;
    partial[p.channels + c] = db;
}

// Sum of the partial rows, 32 channels a block: 32 threads of a channel walk every 32nd partial
// row, then their sums are added in order.
constexpr int kReduceParts = 32;

template <typename T>
__global__ void __launch_bounds__(32 * kReduceParts) norm_reduce_kernel(
    const float* partial, int blocks, int channels, T* dw, T* db
) {
    __shared__ float tile[kReduceParts][33];
    const int lane = threadIdx.x & 31;
    const int part = threadIdx.x >> 5;
    const int at = blockIdx.x * 32 + lane;  // over [2][channels]
    float sum = 0.0f;
    if (at < 2 * channels) {
#pragma unroll 8
        for (int b = part; b < blocks; b += kReduceParts) {
            sum += partial[static_cast<size_t>(b) * 2 * channels + at];
        }
    }
    tile[part][lane] = sum;
    __syncthreads();
    if (part == 0 && at < 2 * channels) {
        float total = 0.0f;
#pragma unroll
        for (int q = 0; q < kReduceParts; ++q) {
            total += tile[q][lane];
        }
        T* out = at < channels ? dw : db;
        if (out != nullptr) {
            out[at < channels ? at : at - channels] = narrow<T>(total);
        }
    }
}

constexpr int kMaxLaneElements = 32;   // values of a row that a lane holds
constexpr int kMaxNarrow = 32 * kMaxLaneElements;

// Lanes per row and vectors per lane: among the splits that leave the fewest idle slots, the one
// with the fewest lanes, but not fewer than `least` (from global memory eight, which read whole
// 128-byte lines) and with at most `most` vectors each. Fewer lanes take fewer steps to add a row
// up: 256 float16 channels backward, 120 MB of rows, 107 us with 32
// lanes, 66 with 16 or 8; 32 float16 channels 66 us with 4 lanes, 79 with 2.
inline void split_row(int vectors, int elements, int least, int most, int& lanes, int& per_lane) {
    long long best_slots = -1;
    for (int l = 32; l >= 1; l >>= 1) {
        const int k = (vectors + l - 1) / l;
        if (k * elements > kMaxLaneElements) {
            break;
        }
        const long long slots = static_cast<long long>(l) * k;
        if (best_slots < 0 || slots < best_slots || (slots == best_slots && l >= least && k <= most)) {
            best_slots = slots;
            lanes = l;
            per_lane = k;
        }
    }
}

inline long long blocks_of(long long rows, int lanes, int in_flight) {
    const long long per_block = static_cast<long long>(kWarps) * (32 / lanes) * in_flight;
    return (rows + per_block - 1) / per_block;
}

template <typename T, int V, int K>
int launch_forward(const NormArgs<T>& p, bool rms, bool batches, cudaStream_t stream) {
    constexpr bool kVectors = V == 16 / static_cast<int>(sizeof(T));
    if constexpr (!kVectors) {
        if (batches || V > 1) {
            const Batches b = batches_of<T>(p.channels, p.lanes, false);
            const int bytes = kWarps * kBatchStages * b.stage;
            const long long blocks = std::min<long long>((p.rows - 1) / (kWarps * b.rows) + 1, 148 * 8);
            auto* kernel = rms ? norm_forward_batch_kernel<T, V, K, true> : norm_forward_batch_kernel<T, V, K, false>;
            LAT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
            kernel<<<static_cast<unsigned>(blocks), kThreads, bytes, stream>>>(p, b);
            LAT_LAUNCH_CHECK();
            return LAT_OK;
        }
    }
    if constexpr (V == 1 || (kVectors && !kForwardRing<T>)) {
        const long long blocks = blocks_of(p.rows, p.lanes, kRowsInFlight<Columns<T, V>::kWidth * K * sizeof(T)>);
        LAT_REQUIRE(blocks <= 0x7fffffffLL, "normalisation supports at most 2^31 blocks of rows.");
        auto* kernel = rms ? norm_forward_kernel<T, V, K, true> : norm_forward_kernel<T, V, K, false>;
        kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
    } else if constexpr (kVectors) {
        constexpr int kBytes = kForwardStages<K> * kForwardRows<K> * K * kThreads * 16;
        const long long blocks = std::min<long long>(blocks_of(p.rows, p.lanes, kForwardRows<K>), 148 * kForwardBlocks<V, K>);
        auto* kernel = rms ? norm_forward_ring_kernel<T, K, true> : norm_forward_ring_kernel<T, K, false>;
        LAT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
        kernel<<<static_cast<unsigned>(blocks), kThreads, kBytes, stream>>>(p);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

constexpr int kMaxBackwardBlocks = 148 * 4;
constexpr int kMaxChannels = 65535 * kThreads;   // of the sums' grid

template <typename T> int launch_reduce(const NormArgs<T>& p, int blocks, T* dw, T* db, cudaStream_t stream) {
    norm_reduce_kernel<T><<<(2 * p.channels + 31) / 32, 32 * kReduceParts, 0, stream>>>(
        p.partial, blocks, p.channels, dw, db);
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

template <typename T, int V, int K>
int launch_backward(const NormArgs<T>& p, bool rms, bool batches, T* dw, T* db, cudaStream_t stream) {
    const size_t sums = sizeof(float) * kWarps * p.channels;
    int grid = 1;
    constexpr bool kVectors = V == 16 / static_cast<int>(sizeof(T));
    if constexpr (!kVectors) {
        if (batches || V > 1) {
            const Batches b = batches_of<T>(p.channels, p.lanes, true);
            const size_t smem = std::max<size_t>(kWarps * kBatchStages * b.stage, sums);
            grid = static_cast<int>(std::min<long long>((p.rows - 1) / (kWarps * b.rows) + 1, kMaxBackwardBlocks));
            auto* kernel = rms ? norm_backward_batch_kernel<T, V, K, true> : norm_backward_batch_kernel<T, V, K, false>;
            LAT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
            kernel<<<grid, kThreads, smem, stream>>>(p, b, dw, db);
            LAT_LAUNCH_CHECK();
            return grid > 1 && (dw != nullptr || db != nullptr) ? launch_reduce(p, grid, dw, db, stream) : LAT_OK;
        }
    }
    if constexpr (V == 1) {
        constexpr int kRows = kBackwardRows<Columns<T, V>::kWidth * K * sizeof(T)>;
        grid = static_cast<int>(std::min<long long>(blocks_of(p.rows, p.lanes, kRows), kMaxBackwardBlocks));
        if (rms) {
            norm_backward_kernel<T, K, true><<<grid, kThreads, sums, stream>>>(p, dw, db);
        } else {
            norm_backward_kernel<T, K, false><<<grid, kThreads, sums, stream>>>(p, dw, db);
        }
    } else if constexpr (kVectors) {
        grid = static_cast<int>(std::min<long long>(blocks_of(p.rows, p.lanes, kRingRows<K>), 148 * kRingBlocks<V, K>));
        const size_t smem = std::max(ring_bytes<K>(), sums);
        auto* kernel = rms ? norm_backward_ring_kernel<T, K, true> : norm_backward_ring_kernel<T, K, false>;
        LAT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        kernel<<<grid, kThreads, smem, stream>>>(p, dw, db);
    }
    LAT_LAUNCH_CHECK();
    return grid > 1 && (dw != nullptr || db != nullptr) ? launch_reduce(p, grid, dw, db, stream) : LAT_OK;
}

template <typename T, int V, bool Backward>
int dispatch_split(NormArgs<T> p, bool rms, bool batches, T* dw, T* db, cudaStream_t stream) {
    constexpr int kWidth = Columns<T, V>::kWidth, kMost = kMaxLaneElements / kWidth;
    int k;
    split_row((p.channels + kWidth - 1) / kWidth, kWidth, batches ? 1 : 8, batches ? 8 / kWidth : kMost, p.lanes, k);
#define LAT_NORM_CASE(N)                                                            \
    if constexpr (N <= kMost) {                                                     \
        if (k <= N) {                                                               \
            if constexpr (Backward) {                                               \
                return launch_backward<T, V, N>(p, rms, batches, dw, db, stream);   \
            } else {                                                                \
                return launch_forward<T, V, N>(p, rms, batches, stream);            \
            }                                                                       \
        }                                                                           \
    }
    LAT_NORM_CASE(1)
    LAT_NORM_CASE(2)
    LAT_NORM_CASE(3)
    LAT_NORM_CASE(4)
    LAT_NORM_CASE(6)
    LAT_NORM_CASE(8)
    LAT_NORM_CASE(12)
    LAT_NORM_CASE(16)
#undef LAT_NORM_CASE
    return fail(LAT_INVALID_ARGUMENT, "unsupported channel count.");
}

// Rows of 16-byte vectors; others one behind the other in batches; the rest by elements.
template <typename T, bool Backward>
int dispatch(const NormArgs<T>& p, bool rms, T* dw, T* db, cudaStream_t stream) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const bool aligned = aligned_to(p.x, 16) && aligned_to(p.dy, 16) && aligned_to(p.out, 16);
    if (aligned && p.channels % V == 0 && p.x_stride % V == 0 && p.dy_stride % V == 0 && aligned_to(p.weight, 16) &&
        aligned_to(p.bias, 16)) {
        return dispatch_split<T, V, Backward>(p, rms, false, dw, db, stream);
    }
    if (!aligned || p.x_stride != p.channels || (Backward && p.dy_stride != p.channels)) {
        return dispatch_split<T, 1, Backward>(p, rms, false, dw, db, stream);
    }
    // the widest vectors that rows, weight and bias come in
    const auto fits = [&](int v) {
        return p.channels % v == 0 && aligned_to(p.weight, v * sizeof(T)) && aligned_to(p.bias, v * sizeof(T));
    };
    if constexpr (V == 8) {
        if (fits(4)) {
            return dispatch_split<T, 4, Backward>(p, rms, true, dw, db, stream);
        }
    }
    return fits(2) ? dispatch_split<T, 2, Backward>(p, rms, true, dw, db, stream)
                   : dispatch_split<T, 1, Backward>(p, rms, true, dw, db, stream);
}

template <typename T> int run_forward(const NormArgs<T>& p, bool rms, cudaStream_t stream) {
    if (p.channels > kMaxNarrow) {
        const int grid = static_cast<int>(std::min(p.rows, 148LL * 8));
        if (rms) {
            norm_forward_wide_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
        } else {
            norm_forward_wide_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
        }
        LAT_LAUNCH_CHECK();
        return LAT_OK;
    }
    return dispatch<T, false>(p, rms, nullptr, nullptr, stream);
}

// Partial rows that the backward pass may write.
inline int partial_rows(long long rows) {
    return static_cast<int>(std::max(1LL, std::min<long long>((rows + kWarps - 1) / kWarps, kMaxBackwardBlocks)));
}

template <typename T>
int run_backward(const NormArgs<T>& p, bool rms, T* dw, T* db, cudaStream_t stream) {
    if (p.channels <= kMaxNarrow) {
        return dispatch<T, true>(p, rms, dw, db, stream);
    }
    const int grid = static_cast<int>(std::min(p.rows, 148LL * 8));
    if (rms) {
        norm_backward_wide_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
    } else {
        norm_backward_wide_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
    }
    LAT_LAUNCH_CHECK();
    if (dw == nullptr && db == nullptr) {
        return LAT_OK;
    }
    const long long per_block = (p.rows + partial_rows(p.rows) - 1) / partial_rows(p.rows);
    const int blocks = static_cast<int>((p.rows + per_block - 1) / per_block);
    const dim3 sums_grid(blocks, (p.channels + kThreads - 1) / kThreads);
    if (rms) {
        norm_sums_wide_kernel<T, true><<<sums_grid, kThreads, 0, stream>>>(p, per_block);
    } else {
        norm_sums_wide_kernel<T, false><<<sums_grid, kThreads, 0, stream>>>(p, per_block);
    }
    LAT_LAUNCH_CHECK();
    return launch_reduce(p, blocks, dw, db, stream);
}

template <typename T>
NormArgs<T> norm_args(const void* x, long long x_stride, const void* dy, long long dy_stride, long long rows,
                      int channels, const void* weight, const void* bias, float eps, void* out, void* mean,
                      void* rstd, void* partial) {
    return {static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, rows, channels, 32,
            static_cast<const T*>(weight), static_cast<const T*>(bias), eps, static_cast<T*>(out),
            static_cast<float*>(mean), static_cast<float*>(rstd), static_cast<float*>(partial)};
}

} // namespace

} // namespace lat

using namespace lat;

extern "C" {

int lat_row_norm_forward(
    int32_t dtype, int32_t rms, const void* feats, int64_t rows, int32_t channels, int64_t feat_row_stride,
    const void* weight, const void* bias, float eps, void* out, float* mean, float* rstd, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "normalisation supports float32 and float16 tensors.");
    LAT_REQUIRE(eps > 0.0f, "eps must be positive.");
    LAT_REQUIRE(rows >= 0 && channels > 0 && feat_row_stride >= 0, "feats must have shape (N, C).");
    LAT_REQUIRE(channels <= kMaxChannels, "normalisation supports at most 16776960 channels.");
    LAT_REQUIRE(!rms || bias == nullptr, "rms_norm has no bias.");
    if (rows == 0) {
        return LAT_OK;
    }
    LAT_REQUIRE(feats != nullptr && out != nullptr && rstd != nullptr && (rms || mean != nullptr),
                "the row statistics need a buffer.");
    cudaStream_t stream = as_stream(stream_ptr);
    if (dtype == LAT_F32) {
        return run_forward(norm_args<float>(feats, feat_row_stride, nullptr, 0, rows, channels, weight, bias, eps,
                                            out, mean, rstd, nullptr), rms != 0, stream);
    }
    return run_forward(norm_args<__half>(feats, feat_row_stride, nullptr, 0, rows, channels, weight, bias, eps,
                                         out, mean, rstd, nullptr), rms != 0, stream);
}

size_t lat_row_norm_backward_workspace_bytes(int64_t rows, int32_t channels) {
    if (rows <= 0 || channels <= 0) {
        return 256;
    }
    return align_up(sizeof(float) * 2 * static_cast<size_t>(channels) * partial_rows(rows));
}

int lat_row_norm_backward(
    int32_t dtype, int32_t rms, const void* grad, int64_t grad_row_stride, const void* feats, int64_t rows,
    int32_t channels, int64_t feat_row_stride, const void* weight, const float* mean, const float* rstd,
    void* grad_feats, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "normalisation supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && channels > 0 && feat_row_stride >= 0 && grad_row_stride >= 0,
                "feats must have shape (N, C).");
    LAT_REQUIRE(channels <= kMaxChannels, "normalisation supports at most 16776960 channels.");
    LAT_REQUIRE(!rms || grad_bias == nullptr, "rms_norm has no bias.");
    const bool sums = grad_weight != nullptr || grad_bias != nullptr;
    cudaStream_t stream = as_stream(stream_ptr);
    const size_t element = dtype == LAT_F32 ? 4 : 2;
    if (rows == 0) {
        if (grad_weight != nullptr) {
            LAT_CUDA_CHECK(cudaMemsetAsync(grad_weight, 0, element * channels, stream));
        }
        if (grad_bias != nullptr) {
            LAT_CUDA_CHECK(cudaMemsetAsync(grad_bias, 0, element * channels, stream));
        }
        return LAT_OK;
    }
    LAT_REQUIRE(feats != nullptr && grad != nullptr && grad_feats != nullptr && rstd != nullptr &&
                    (rms || mean != nullptr), "the backward pass needs the statistics of the forward pass.");
    if (sums && (workspace == nullptr || workspace_bytes < lat_row_norm_backward_workspace_bytes(rows, channels))) {
        return fail(LAT_WORKSPACE_TOO_SMALL, "normalisation workspace is too small.");
    }
    void* partial = sums ? workspace : nullptr;
    if (dtype == LAT_F32) {
        return run_backward(norm_args<float>(feats, feat_row_stride, grad, grad_row_stride, rows, channels, weight,
                                             nullptr, 0.0f, grad_feats, const_cast<float*>(mean),
                                             const_cast<float*>(rstd), partial), rms != 0,
                            static_cast<float*>(grad_weight), static_cast<float*>(grad_bias), stream);
    }
    return run_backward(norm_args<__half>(feats, feat_row_stride, grad, grad_row_stride, rows, channels, weight,
                                          nullptr, 0.0f, grad_feats, const_cast<float*>(mean),
                                          const_cast<float*>(rstd), partial), rms != 0,
                        static_cast<__half*>(grad_weight), static_cast<__half*>(grad_bias), stream);
}

} // extern "C"
