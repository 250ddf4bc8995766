// Layer and RMS normalisation of sparse rows for training: the forward pass that also
// leaves the row statistics, and the backward pass with the gradients of x, weight and bias.
//
//   m = mean(x) (0 for RMS), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r
//   y = xh w + b
//   g = dy w:  dx = r (g - mean(g) [layer only] - xh mean(g xh))
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// Both passes are bound by the memory: the forward pass reads x and writes y, the backward
// pass reads x and dy and writes dx. A group of L lanes (a power of two) holds a row in
// registers, so every element is read once and the variance is taken about the mean in a
// second pass over registers. All sums are float32; results are rounded once.
//
// The gradients of weight and bias are sums down the rows. Every lane keeps the sums of the
// channels it owns over all rows it visits, a block adds its lanes' sums up in a fixed order
// and writes one partial row, and a second kernel adds the partial rows in a fixed order: no
// atomics, bitwise repeatable.
#include <algorithm>

#include "common.cuh"
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

// A lane owns the vectors lane, lane + L, ... of its row: K vectors of V elements.
template <typename T, int V, int K, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_forward_kernel(NormArgs<T> p) {
    const int lane = threadIdx.x & 31;
    const int sub = lane & (p.lanes - 1);
    const int rows_per_warp = 32 / p.lanes;
    const float inv_c = static_cast<float>(p.channels);
    const long long warps = static_cast<long long>(gridDim.x) * kWarps;
    const long long warp = blockIdx.x * static_cast<long long>(kWarps) + (threadIdx.x >> 5);
    for (long long row0 = warp * rows_per_warp; row0 < p.rows; row0 += warps * rows_per_warp) {
        const long long row = row0 + lane / p.lanes;
        const bool live = row < p.rows;
        Pack<T, V> x[K];
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (sub + k * p.lanes) * V;
            x[k] = live && c < p.channels ? load_pack<T, V>(p.x + row * p.x_stride + c) : zero_pack<T, V>();
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sum += x[k].get(i);
            }
        }
        const float mean = Rms ? 0.0f : group_sum(sum, p.lanes) / inv_c;
        float squares = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if ((sub + k * p.lanes) * V < p.channels) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = x[k].get(i) - mean;
                    squares = fmaf(d, d, squares);
                }
            }
        }
        const float r = rsqrtf(group_sum(squares, p.lanes) / inv_c + p.eps);
        if (!live) {
            continue;
        }
        if (sub == 0) {
            p.rstd[row] = r;
            if (!Rms) {
                p.mean[row] = mean;
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (sub + k * p.lanes) * V;
            if (c < p.channels) {
                Pack<T, V> w, b, y;
                if (p.weight != nullptr) {
                    w = load_pack<T, V>(p.weight + c);
                }
                if (p.bias != nullptr) {
                    b = load_pack<T, V>(p.bias + c);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float v = (x[k].get(i) - mean) * r;
                    if (p.weight != nullptr) {
                        v *= w.get(i);
                    }
                    if (p.bias != nullptr) {
                        v += b.get(i);
                    }
                    y.set(i, v);
                }
                store_pack<T, V>(p.out + row * p.channels + c, y);
            }
        }
    }
}

template <typename T, int V, int K, bool Rms>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(NormArgs<T> p) {
    extern __shared__ float sums[];  // [2][channels]
    const int lane = threadIdx.x & 31;
    const int sub = lane & (p.lanes - 1);
    const int rows_per_warp = 32 / p.lanes;
    const float count = static_cast<float>(p.channels);
    const long long warps = static_cast<long long>(gridDim.x) * kWarps;
    const long long warp = blockIdx.x * static_cast<long long>(kWarps) + (threadIdx.x >> 5);
    float dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            dw[k][i] = db[k][i] = 0.0f;
        }
    }
    for (long long row0 = warp * rows_per_warp; row0 < p.rows; row0 += warps * rows_per_warp) {
        const long long row = row0 + lane / p.lanes;
        const bool live = row < p.rows;
        Pack<T, V> x[K], dy[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (sub + k * p.lanes) * V;
            const bool in = live && c < p.channels;
            x[k] = in ? load_pack<T, V>(p.x + row * p.x_stride + c) : zero_pack<T, V>();
            dy[k] = in ? load_pack<T, V>(p.dy + row * p.dy_stride + c) : zero_pack<T, V>();
        }
        const float r = live ? p.rstd[row] : 0.0f;
        const float mean = !Rms && live ? p.mean[row] : 0.0f;
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (sub + k * p.lanes) * V;
            if (c < p.channels) {
                Pack<T, V> w;
                if (p.weight != nullptr) {
                    w = load_pack<T, V>(p.weight + c);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = dy[k].get(i);
                    const float xh = (x[k].get(i) - mean) * r;
                    const float g = p.weight != nullptr ? d * w.get(i) : d;
                    c1 += g;
                    c2 = fmaf(g, xh, c2);
                    dw[k][i] = fmaf(d, xh, dw[k][i]);
                    db[k][i] += d;
                }
            }
        }
        c1 = Rms ? 0.0f : group_sum(c1, p.lanes) / count;
        c2 = group_sum(c2, p.lanes) / count;
        if (live) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (sub + k * p.lanes) * V;
                if (c < p.channels) {
                    Pack<T, V> w, dx;
                    if (p.weight != nullptr) {
                        w = load_pack<T, V>(p.weight + c);
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = dy[k].get(i);
                        const float xh = (x[k].get(i) - mean) * r;
                        const float g = p.weight != nullptr ? d * w.get(i) : d;
                        dx.set(i, r * (g - c1 - xh * c2));
                    }
                    store_pack<T, V>(p.out + row * p.channels + c, dx);
                }
            }
        }
    }
    if (p.partial == nullptr) {
        return;
    }
    // lanes of the warp that own the same channels, then the warps one after the other
    for (int d = p.lanes; d < 32; d <<= 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dw[k][i] += __shfl_xor_sync(0xffffffffu, dw[k][i], d);
                db[k][i] += __shfl_xor_sync(0xffffffffu, db[k][i], d);
            }
        }
    }
    for (int w = 0; w < kWarps; ++w) {
        if ((threadIdx.x >> 5) == w && lane < p.lanes) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (sub + k * p.lanes) * V;
                if (c < p.channels) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        sums[c + i] = (w == 0 ? 0.0f : sums[c + i]) + dw[k][i];
                        sums[p.channels + c + i] = (w == 0 ? 0.0f : sums[p.channels + c + i]) + db[k][i];
                    }
                }
            }
        }
        __syncthreads();
    }
    float* partial = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.channels;
    for (int c = threadIdx.x; c < 2 * p.channels; c += kThreads) {
        partial[c] = sums[c];
    }
}

// Rows wider than the registers of a warp: one block per row, three passes over a row that
// stays in L1 / L2.
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

// Sum of the partial rows, 32 channels a block: eight threads of a channel walk every eighth
// partial row, then their sums are added in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_reduce_kernel(
    const float* partial, int blocks, int channels, T* dw, T* db
) {
    __shared__ float tile[kWarps][33];
    const int lane = threadIdx.x & 31;
    const int part = threadIdx.x >> 5;
    const int at = blockIdx.x * 32 + lane;  // over [2][channels]
    float sum = 0.0f;
    if (at < 2 * channels) {
        for (int b = part; b < blocks; b += kWarps) {
            sum += partial[static_cast<size_t>(b) * 2 * channels + at];
        }
    }
    tile[part][lane] = sum;
    __syncthreads();
    if (part == 0 && at < 2 * channels) {
        float total = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            total += tile[w][lane];
        }
        T* out = at < channels ? dw : db;
        if (out != nullptr) {
            out[at < channels ? at : at - channels] = narrow<T>(total);
        }
    }
}

constexpr int kMaxLaneElements = 32;   // values of a row that a lane holds
constexpr int kMaxNarrow = 32 * kMaxLaneElements;

// Lanes per row and vectors per lane: among the splits that leave a lane at most
// kMaxLaneElements values, the one with the fewest idle slots (the wider one on a tie).
inline void split_row(int vectors, int max_per_lane, int& lanes, int& per_lane) {
    long long best = -1;
    lanes = 32;
    per_lane = (vectors + 31) / 32;
    for (int l = 32; l >= 1; l >>= 1) {
        const int k = (vectors + l - 1) / l;
        if (k > max_per_lane) {
            break;
        }
        const long long slots = static_cast<long long>(l) * k;
        if (best < 0 || slots < best) {
            best = slots;
            lanes = l;
            per_lane = k;
        }
    }
}

inline int norm_grid(long long rows, int lanes) {
    const long long per_block = static_cast<long long>(kWarps) * (32 / lanes);
    return static_cast<int>(std::max(1LL, std::min((rows + per_block - 1) / per_block, 148LL * 4)));
}

template <typename T, int V, int K>
int launch_forward(const NormArgs<T>& p, bool rms, cudaStream_t stream) {
    const int grid = norm_grid(p.rows, p.lanes);
    if (rms) {
        norm_forward_kernel<T, V, K, true><<<grid, kThreads, 0, stream>>>(p);
    } else {
        norm_forward_kernel<T, V, K, false><<<grid, kThreads, 0, stream>>>(p);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

template <typename T, int V, int K>
int launch_backward(const NormArgs<T>& p, bool rms, int grid, cudaStream_t stream) {
    const size_t smem = sizeof(float) * 2 * p.channels;
    if (rms) {
        norm_backward_kernel<T, V, K, true><<<grid, kThreads, smem, stream>>>(p);
    } else {
        norm_backward_kernel<T, V, K, false><<<grid, kThreads, smem, stream>>>(p);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

// grid 0: forward
template <typename T, int V>
int dispatch_split(NormArgs<T> p, bool rms, int grid, cudaStream_t stream) {
    constexpr int kMost = kMaxLaneElements / V;
    int k;
    split_row(p.channels / V, kMost, p.lanes, k);
    if (grid > 0) {
        grid = std::min(grid, norm_grid(p.rows, p.lanes));
    }
#define LAT_NORM_CASE(N)                                                            \
    if constexpr (N <= kMost) {                                                     \
        if (k <= N) {                                                               \
            return grid > 0 ? launch_backward<T, V, N>(p, rms, grid, stream)        \
                            : launch_forward<T, V, N>(p, rms, stream);              \
        }                                                                           \
    }
    LAT_NORM_CASE(1)
    LAT_NORM_CASE(2)
    LAT_NORM_CASE(3)
    LAT_NORM_CASE(4)
    LAT_NORM_CASE(6)
    LAT_NORM_CASE(8)
    LAT_NORM_CASE(16)
    LAT_NORM_CASE(32)
#undef LAT_NORM_CASE
    return fail(LAT_INVALID_ARGUMENT, "unsupported channel count.");
}

template <typename T> bool vector_rows(const NormArgs<T>& p) {
    constexpr int V = 16 / sizeof(T);
    return p.channels % V == 0 && p.x_stride % V == 0 && p.dy_stride % V == 0 && aligned_to(p.x, 16) &&
           aligned_to(p.dy, 16) && aligned_to(p.out, 16) && aligned_to(p.weight, 16) && aligned_to(p.bias, 16);
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
    return vector_rows(p) ? dispatch_split<T, 16 / sizeof(T)>(p, rms, 0, stream)
                          : dispatch_split<T, 1>(p, rms, 0, stream);
}

// Blocks of the backward pass, which is also the number of partial rows in the workspace.
inline int backward_blocks(long long rows, int channels) {
    if (channels > kMaxNarrow) {
        return static_cast<int>(std::max(1LL, std::min((rows + 31) / 32, 148LL * 2)));
    }
    return static_cast<int>(std::max(1LL, std::min((rows + kWarps - 1) / kWarps, 148LL * 2)));
}

template <typename T>
int run_backward(NormArgs<T> p, bool rms, T* dw, T* db, cudaStream_t stream) {
    int blocks = backward_blocks(p.rows, p.channels);
    int code;
    if (p.channels > kMaxNarrow) {
        const int grid = static_cast<int>(std::min(p.rows, 148LL * 8));
        if (rms) {
            norm_backward_wide_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
        } else {
            norm_backward_wide_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
        }
        LAT_LAUNCH_CHECK();
        if (p.partial == nullptr) {
            return LAT_OK;
        }
        const long long per_block = (p.rows + blocks - 1) / blocks;
        blocks = static_cast<int>((p.rows + per_block - 1) / per_block);
        const dim3 sums_grid(blocks, (p.channels + kThreads - 1) / kThreads);
        if (rms) {
            norm_sums_wide_kernel<T, true><<<sums_grid, kThreads, 0, stream>>>(p, per_block);
        } else {
            norm_sums_wide_kernel<T, false><<<sums_grid, kThreads, 0, stream>>>(p, per_block);
        }
        LAT_LAUNCH_CHECK();
    } else {
        const bool vec = vector_rows(p);
        int lanes, k;
        split_row(vec ? p.channels * static_cast<int>(sizeof(T)) / 16 : p.channels,
                  vec ? kMaxLaneElements * static_cast<int>(sizeof(T)) / 16 : kMaxLaneElements, lanes, k);
        blocks = std::min(blocks, norm_grid(p.rows, lanes));
        code = vec ? dispatch_split<T, 16 / sizeof(T)>(p, rms, blocks, stream)
                   : dispatch_split<T, 1>(p, rms, blocks, stream);
        if (code != LAT_OK || p.partial == nullptr) {
            return code;
        }
    }
    norm_reduce_kernel<T><<<(2 * p.channels + 31) / 32, kThreads, 0, stream>>>(
        p.partial, blocks, p.channels, dw, db);
    LAT_LAUNCH_CHECK();
    return LAT_OK;
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
    return align_up(sizeof(float) * 2 * static_cast<size_t>(channels) * backward_blocks(rows, channels));
}

int lat_row_norm_backward(
    int32_t dtype, int32_t rms, const void* grad, int64_t grad_row_stride, const void* feats, int64_t rows,
    int32_t channels, int64_t feat_row_stride, const void* weight, const float* mean, const float* rstd,
    void* grad_feats, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "normalisation supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && channels > 0 && feat_row_stride >= 0 && grad_row_stride >= 0,
                "feats must have shape (N, C).");
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
