// Gated linear recurrence along the rows of a sparse tensor, per sequence and channel:
//
//   a_t = sigmoid(z_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h before the first row = initial
//
// forward, or from the last row to the first (`reverse`), with its gradient
//
//   dh_t = dy_t + a_{t+1} dh_{t+1}  (+ dfinal at the last row)
//   dx_t = (1 - a_t) dh_t,  dz_t = a_t (1 - a_t) dh_t (h_{t-1} - x_t),  dinitial = a_1 dh_1
//
// Both a_t and 1 - a_t are computed to full relative precision, so a nearly closed gate lets in what
// it should, and so are A and 1 - A of the maps below, so a long memory does not gather the rounding
// of gates near one.
//
// Both directions are scans over affine maps h -> A h + H, which compose associatively. The
// rows are cut into tiles of 32. Three kernels:
//   maps:   for a group of tiles (a block, 128 rows of 128 bytes) the map (A, H) of the group and,
//           for every tile, of the tiles before it in the group
//   scan:   for every group the map of the groups before it in its window of 64, and the state
//           that reaches every window
//   apply:  those three give the state that reaches a tile; walk the tile from there and write
// Nothing waits for anything inside a kernel, and every sum has a fixed order: results are
// bitwise repeatable.
//
// A row that starts a sequence cuts the chain. Its map ignores the incoming h altogether
// (marked, and selected, not multiplied by zero: a NaN or an infinity of one sequence does not
// reach the next). Within a sequence an infinite h stays infinite. Rows outside all sequences
// give zeros.
//
// The backward pass recomputes h from the state at the start of every eight rows, which the
// forward pass leaves in float32: it reads x, z, dy and writes dx, dz, and its h is not rounded
// to the feature type.
#include <algorithm>

#include "common.cuh"
#include "pairs.cuh"
#include "vector_io.cuh"

namespace lat {

namespace {

constexpr int kTileRows = 32;
constexpr int kPieceRows = 8;                 // of a tile, walked by one thread of the maps kernel
constexpr int kPieces = kTileRows / kPieceRows;
constexpr int kMapThreads = 128;              // of a block of the maps kernel
constexpr int kThreads = 256;                 // of the others
constexpr int kWindow = 64;                   // groups
constexpr int kMapBytes = 16;                 // channels of a thread of the maps and apply kernels
constexpr int kGradientBytes = 8;             // of the gradient kernel, which keeps twice as much of each
constexpr int kScanChannels = 32;             // of a block of the scan kernel
constexpr int kCarryRows = 8;                 // rows from one kept state to the next

// ---- maps ----------------------------------------------------------------------------------
//
// A map h -> A h + H is kept as the pair (m, H). Of A and 1 - A, m holds the one that is at most one
// half: A itself, or -(1 - A), told apart by the sign bit. Both are then known to full relative
// precision. A = 1 - 2^-14 alone would give 1 - A to 2^-11 of itself, and a memory of 2^14 rows h
// no better.
constexpr float kReset = 2.0f;   // m of a map that ignores what comes in

__device__ __forceinline__ bool negative(float v) { return __float_as_int(v) < 0; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __int_as_float(0x7f800000); }

__device__ __forceinline__ float2 make_map(float keep, float rest, float sum, bool cut) {
    const float m = keep <= 0.5f ? keep : -rest;
    return make_float2(cut ? kReset : m, sum);
}
__device__ __forceinline__ float2 identity() { return make_map(1.0f, 0.0f, 0.0f, false); }

// A near one moves h by 1 - A of it, so that a chain of maps does not gather the rounding of A. An
// infinity stays, also where A has become zero.
__device__ __forceinline__ float apply(float2 map, float h) {
    const float moved = __fadd_rn(fmaf(map.x, h, map.y), negative(map.x) ? h : 0.0f);
    const float any = finite(h) ? moved : h + map.y;
    return map.x == kReset ? map.y : any;
}

// Maps, one after the other: A, 1 - A and H of them all. What a later map rounds is relative to the H
// of the ones before it alone. (The products and sums are written as such: a multiply-add that the
// compiler makes of some of them would let results depend on the launch.)
struct Chain {
    float keep = 1.0f, rest = 0.0f, sum = 0.0f;
    bool cut = false;

    __device__ __forceinline__ void add(const Chain& later) {
        rest = fmaf(keep, later.rest, rest);
        keep = __fmul_rn(keep, later.keep);
        const float moved = fmaf(later.keep, sum, later.sum), any = finite(sum) ? moved : __fadd_rn(sum, later.sum);
        sum = later.cut ? later.sum : any;
        cut = cut | later.cut;
    }
    __device__ __forceinline__ void add(float2 later) {
        const bool close = negative(later.x);
        const float plus = __fadd_rn(1.0f, later.x), less = __fsub_rn(1.0f, later.x);
        add(Chain{close ? plus : later.x, close ? -later.x : less, later.y, later.x == kReset});
    }
    __device__ __forceinline__ float2 map() const { return make_map(keep, rest, sum, cut); }
    template <typename Later> __device__ __forceinline__ float2 then(const Later& later) const {
        Chain both = *this;
        both.add(later);
        return both.map();
    }
};

// Rows and sequences in the order of time: row i is row rows - 1 - i of the arrays when the
// recurrence runs backwards, and sequence j is sequence sequences - 1 - j.
struct Order {
    const int32_t* offsets;
    int rows;
    int sequences;
    int reverse;

    __device__ __forceinline__ int begin(int j) const {   // 0 <= j <= sequences
        const int v = min(max(__ldg(offsets + (reverse ? sequences - j : j)), 0), rows);
        return reverse ? rows - v : v;
    }
    __device__ __forceinline__ int row(int i) const { return reverse ? rows - 1 - i : i; }
    __device__ __forceinline__ int sequence(int j) const { return reverse ? sequences - 1 - j : j; }
};

// ---- gates -----------------------------------------------------------------------------

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// one unit in the last place; zero beyond 2^126
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float min_or_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float kMinusLog2E = -1.4426950408889634f;
constexpr float kTiny = 1.1754943508222875e-38f;   // 2^-126

// exp(-z), at most 2^126. The product with log2(e) is rounded once before the exponential, so it is
// off by up to (1.25 |z| + 4) 2^-24 of itself. Zero for z > 87.3.
__device__ __forceinline__ Pair odds_of(Pair z) {
    const Pair t = z * both(kMinusLog2E);
    return {min_or_nan(exp2_fast(t.x), 1.0f / kTiny), min_or_nan(exp2_fast(t.y), 1.0f / kTiny)};
}

// The weights of h and x, each to the relative precision of the odds where it is small and to a few
// 2^-24 where it is not: a = sigmoid(z) = 1 / (1 + exp(-z)), rest = sigmoid(-z) = exp(-z) a. Beyond
// |z| = 87.3 the one is zero and the other one: a state or a value behind such a gate does not count,
// up to the largest float (an infinite one gives a NaN there).
struct Weights {
    Pair a, rest;

    __device__ __forceinline__ explicit Weights(Pair odds) {
        const Pair d = odds + both(1.0f), r = {reciprocal(d.x), reciprocal(d.y)};
        a = r + both(-kTiny);
        rest = odds * r;
    }
    __device__ __forceinline__ Pair blend(Pair h, Pair x) const { return fma(a, h, rest * x); }
};

// What the sequences ask for beside their rows, by the warps of the grid in turn, all threads of a
// block together: one without rows hands on what it was given (`from`, or zeros) to `to`; offsets
// that fall are reported.
__device__ __forceinline__ void visit_sequences(
    const Order& order, const float* from, float* to, int channels, int32_t* status
) {
    const int lane = threadIdx.x & 31;
    const long long threads = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long base = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x - lane; base < order.sequences;
         base += threads) {
        const int j = static_cast<int>(base) + lane;
        bool empty = false;
        if (base + lane < order.sequences) {
            empty = order.begin(j + 1) <= order.begin(j);
            if (__ldg(order.offsets + j + 1) < __ldg(order.offsets + j)) {
                raise_status(status, LAT_STATUS_BAD_INDEX);
            }
        }
        unsigned todo = to != nullptr ? __ballot_sync(0xffffffffu, empty) : 0u;
        for (; todo != 0; todo &= todo - 1) {
            const size_t at = static_cast<size_t>(order.sequence(static_cast<int>(base) + __ffs(todo) - 1)) * channels;
            for (int c = lane; c < channels; c += 32) {
                to[at + c] = from != nullptr ? from[at + c] : 0.0f;
            }
        }
    }
}

// The sequence that holds a row or, for a row outside all of them, the next one; in the order of
// time.
struct Cursor {
    int j, begin, end;

    // Sequences without rows are stepped over one at a time at first, then by bisection of the offsets:
    // a run of a million of them costs twenty dependent loads, not a million.
    static constexpr int kSteps = 4;

    __device__ __forceinline__ void settle(const Order& order) {
        for (int step = 0; j < order.sequences; ++step) {
            begin = order.begin(j);
            end = order.begin(j + 1);
            if (end > begin) {
                return;
            }
            ++j;
            if (step >= kSteps) {   // on to the first sequence that ends behind this place
                int high = order.sequences;
                while (j < high) {
                    const int middle = j + (high - j) / 2;
                    if (order.begin(middle + 1) > begin) {
                        high = middle;
                    } else {
                        j = middle + 1;
                    }
                }
            }
        }
        begin = end = 0x7fffffff;
    }

    // The first sequence that ends behind row `first`. `lanes` threads of a warp (`mask`, this one
    // is number `lane`) ask together, at as many places a step.
    __device__ __forceinline__ void seek(const Order& order, int first, int lane, int lanes, unsigned mask) {
        int low = 0, high = order.sequences;
        while (low < high) {
            const int step = (high - low) / (lanes + 1) + 1, at = low + (lane + 1) * step - 1;
            // the answers rise: the sequence lies behind the last place that says no
            const unsigned no = __ballot_sync(mask, at < high && order.begin(at + 1) <= first) & mask;
            const int count = __popc(no);
            high = count == lanes ? high : min(high, low + (count + 1) * step - 1);
            low += count * step;
        }
        j = low;
        settle(order);
    }

    __device__ __forceinline__ void next(const Order& order) {
        ++j;
        settle(order);
    }

    // the sequence before, where there is one
    __device__ __forceinline__ bool back(const Order& order) {
        int k = j - 1;
        for (int step = 0; k >= 0; ++step) {
            const int b = order.begin(k), e = order.begin(k + 1);
            if (e > b) {
                j = k;
                begin = b;
                end = e;
                return true;
            }
            --k;
            if (step >= kSteps) {   // back to the last sequence that begins before this place
                int low = -1;
                while (low < k) {
                    const int middle = k - (k - low) / 2;
                    if (order.begin(middle) < b) {
                        low = middle;
                    } else {
                        k = middle - 1;
                    }
                }
            }
        }
        return false;
    }

    // no sequence starts or ends among these rows, which all belong to this one
    __device__ __forceinline__ bool covers(int first, int rows) const { return begin < first && end > first + rows; }
};

template <typename T> struct ScanArgs {
    const T* x;
    const T* z;
    const T* dy;
    long long x_stride, z_stride, dy_stride;
    Order order;
    int channels;
    int slabs;              // of the kernel's launch: lanes times a thread's channels
    int lanes;              // threads across a slab
    int per_group;          // tiles of a group
    int tiles;
    int span_tiles;         // that a thread of the gradient kernel walks through
    const float* initial;   // [sequences][channels] or null
    float2* maps;           // [tiles][channels] of the tiles before in the group
    float2* groups;         // [groups][channels] of each group, then of the groups before in the window
    float2* windows;        // [windows][channels] of each window
    float* states;          // [windows][channels] that reach the windows
    int* arrived;           // [scan slabs] blocks of the scan kernel that are done
    float* carries;         // [batches][channels] or null: h before each batch of rows
    T* h;
    float* final;           // [sequences][channels] or null
    const float* dfinal;    // [sequences][channels] or null
    T* dx;
    T* dz;
    float* dinitial;        // [sequences][channels] or null
    int32_t* status;
};

// N channels of a row, as they are stored ...
template <typename T, int N> struct alignas(N * sizeof(T)) Stored {
    T v[N];
};

// ... and as float pairs.
template <int N> struct Row {
    static constexpr int kPairs = N / 2;
    Pair v[kPairs];

    static __device__ __forceinline__ Row filled(float value) {
        Row out;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            out.v[i] = both(value);
        }
        return out;
    }

    template <typename T> static __device__ __forceinline__ Row from(const Stored<T, N>& raw) {
        Row out;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            if constexpr (sizeof(T) == 2) {
                const float2 f = __half22float2(reinterpret_cast<const __half2*>(raw.v)[i]);
                out.v[i] = {f.x, f.y};
            } else {
                out.v[i] = {raw.v[2 * i], raw.v[2 * i + 1]};
            }
        }
        return out;
    }

    __device__ __forceinline__ Row times(const Row& other) const {
        Row out;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            out.v[i] = {__fmul_rn(v[i].x, other.v[i].x), __fmul_rn(v[i].y, other.v[i].y)};
        }
        return out;
    }

    __device__ __forceinline__ float get(int i) const { return i % 2 == 0 ? v[i / 2].x : v[i / 2].y; }
    __device__ __forceinline__ void set(int i, float value) { (i % 2 == 0 ? v[i / 2].x : v[i / 2].y) = value; }
};

// Channels c .. c + count - 1 of a thread, at most N, and how they move. Granule: the bytes that
// move at once, as alignment and channel count allow. Two bytes, float16 rows of an odd width or
// start: no copy is that small, so the four-byte words that hold the channels move, one more than
// the channels fill, and are shifted into place when they are read (960,000 x 63: maps 104 us, apply
// 163, gradient 338; element by element through registers 162, 296, 519).
template <typename T, int N, int Granule> struct Channels {
    static constexpr int kBytes = N * static_cast<int>(sizeof(T));
    static constexpr int kMove = Granule < kBytes ? Granule : kBytes;
    static constexpr bool kShifted = Granule == 2;
    static constexpr int kMoveChannels = kMove / static_cast<int>(sizeof(T));
    int c, count;
    int lane, live;       // this thread and how many of the tile's threads have channels
    long long row_step;   // from a row to the next one, in rows of an array

    __device__ __forceinline__ Channels(const ScanArgs<T>& p, int slab) {
        lane = static_cast<int>(threadIdx.x) % p.lanes;
        c = (slab * p.lanes + lane) * N;
        count = min(max(p.channels - c, 0), N);
        live = min(p.lanes, (p.channels - slab * p.lanes * N + N - 1) / N);
        row_step = p.order.reverse ? -1 : 1;
    }

    // All live threads of the tile, together.
    __device__ __forceinline__ void seek(Cursor& cursor, const Order& order, int first) const {
        const unsigned mask = (live == 32 ? 0xffffffffu : (1u << live) - 1u) << ((threadIdx.x & 31) - lane);
        cursor.seek(order, first, lane, live, mask);
    }

    __device__ __forceinline__ const T* row(const T* from, long long stride, const Order& order, int row) const {
        return from + order.row(row) * stride + c;
    }

    // whether the thread's first channel of a row is the upper half of a word
    __device__ __forceinline__ bool odd(const T* from, long long stride, const Order& order, int row) const {
        return kShifted && (reinterpret_cast<uintptr_t>(this->row(from, stride, order, row)) & 2) != 0;
    }

    // to: the thread's first channel in the row
    __device__ __forceinline__ void store(T* to, const Row<N>& value) const {
        Stored<T, N> raw;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (sizeof(T) == 2) {
                reinterpret_cast<__half2*>(raw.v)[i] = __floats2half2_rn(value.v[i].x, value.v[i].y);
            } else {
                raw.v[2 * i] = value.v[i].x;
                raw.v[2 * i + 1] = value.v[i].y;
            }
        }
        if constexpr (kShifted) {
            // the channels before the first whole word, the words, the channel behind the last
            const int head = (reinterpret_cast<uintptr_t>(to) & 2) != 0;
            if (head) {
                if (count > 0) {
                    to[0] = raw.v[0];
                }
#pragma unroll
                for (int i = 1; i + 1 < N; i += 2) {
                    if (i + 1 < count) {
                        *reinterpret_cast<__half2*>(to + i) = __halves2half2(raw.v[i], raw.v[i + 1]);
                    } else if (i < count) {
                        to[i] = raw.v[i];
                    }
                }
                if (count == N) {
                    to[N - 1] = raw.v[N - 1];
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    if (i + 1 < count) {
                        *reinterpret_cast<__half2*>(to + i) = __halves2half2(raw.v[i], raw.v[i + 1]);
                    } else if (i < count) {
                        to[i] = raw.v[i];
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i += kMoveChannels) {
                if (kMove == kBytes || i < count) {
                    using Part = Stored<T, kMoveChannels>;
                    *reinterpret_cast<Part*>(to + i) = reinterpret_cast<const Part&>(raw.v[i]);
                }
            }
        }
    }

    // Row `row` of a float array [..][channels], or zeros without one.
    __device__ __forceinline__ Row<N> state(const float* from, long long row, int channels) const {
        Row<N> out = Row<N>::filled(0.0f);
        if (from != nullptr) {
            from += row * channels + c;
            if (quads(from, channels)) {
#pragma unroll
                for (int i = 0; i + 3 < N; i += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(from + i);
                    out.set(i, v.x);
                    out.set(i + 1, v.y);
                    out.set(i + 2, v.z);
                    out.set(i + 3, v.w);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i < count) {
                        out.set(i, from[i]);
                    }
                }
            }
        }
        return out;
    }

    // the thread's channels are whole quads of floats there
    static __device__ __forceinline__ bool quads(const float* at, int channels) {
        return kMoveChannels == N && N % 4 == 0 && channels % 4 == 0 && reinterpret_cast<uintptr_t>(at) % 16 == 0;
    }

    __device__ __forceinline__ void store_state(float* to, long long row, int channels, const Row<N>& value) const {
        if (to != nullptr) {
            to += row * channels + c;
            if (quads(to, channels)) {
#pragma unroll
                for (int i = 0; i + 3 < N; i += 4) {
                    *reinterpret_cast<float4*>(to + i) =
                        make_float4(value.get(i), value.get(i + 1), value.get(i + 2), value.get(i + 3));
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i < count) {
                        to[i] = value.get(i);
                    }
                }
            }
        }
    }

    // The state that reaches the tile number `place` of the chain.
    __device__ __forceinline__ Row<N> reaching(const ScanArgs<T>& p, int place) const {
        Row<N> out = Row<N>::filled(0.0f);
        if (p.maps != nullptr) {
            const int group = place / p.per_group, window = group / kWindow;
            const float* state = p.states + static_cast<size_t>(window) * p.channels + c;
            const float2* before = p.groups + static_cast<size_t>(group) * p.channels + c;
            const float2* map = p.maps + static_cast<size_t>(place) * p.channels + c;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (i < count) {
                    out.set(i, apply(map[i], apply(before[i], state[i])));
                }
            }
        }
        return out;
    }
};

// Rows on their way from the arrays to a thread: a ring of stages in shared memory, each with
// Rows rows of every array, filled by asynchronous copies. A thread copies what it reads itself,
// so nothing is synchronised, and the bytes in flight (the memory needs some 50 KB of them per
// SM) cost no registers.
template <typename T, int N, int Granule, int Arrays, int Rows, int Stages, int Threads = kThreads> struct Ring {
    using Lanes = Channels<T, N, Granule>;
    static constexpr int kSlots = Stages * Arrays * Rows * Threads;
    static constexpr int kBytes = kSlots * (Lanes::kBytes + (Lanes::kShifted ? 4 : 0));   // with the words behind

    __device__ __forceinline__ int place(int stage, int array, int row) const {
        return ((stage * Arrays + array) * Rows + row) * Threads + threadIdx.x;
    }
    __device__ __forceinline__ Stored<T, N>* slot(int stage, int array, int row) const {
        extern __shared__ __align__(16) unsigned char ring[];
        return reinterpret_cast<Stored<T, N>*>(ring) + place(stage, array, row);
    }
    __device__ __forceinline__ uint32_t* word_behind(int stage, int array, int row) const {
        extern __shared__ __align__(16) unsigned char ring[];
        return reinterpret_cast<uint32_t*>(ring + kSlots * Lanes::kBytes) + place(stage, array, row);
    }

    // `rows` more rows, at most Rows, from `at` on, which moves on to the row behind them; what
    // lies behind the last row or channel stays undefined.
    __device__ __forceinline__ void fetch(const Lanes& lanes, int stage, int array, const T*& at, long long step, int rows) const {
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(slot(stage, array, 0)));
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            if (rows >= Rows || r < rows) {
                if constexpr (Lanes::kShifted) {
                    // Bytes from the first channel's word on: no byte behind the last channel is read, and
                    // the two before the first one, if any, share its aligned word.
                    const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 2);
                    const int bytes = skip + lanes.count * static_cast<int>(sizeof(T));
                    const unsigned char* words = reinterpret_cast<const unsigned char*>(at) - skip;
                    const uint32_t behind = static_cast<uint32_t>(__cvta_generic_to_shared(word_behind(stage, array, r)));
#pragma unroll
                    for (int i = 0; i <= Lanes::kBytes; i += 4) {
                        if (i < bytes) {
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::
                                             "r"(i < Lanes::kBytes ? to + r * Threads * Lanes::kBytes + i : behind),
                                         "l"(words + i), "r"(min(bytes - i, 4)) : "memory");
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < N; i += Lanes::kMoveChannels) {
                        if (Lanes::kMove == Lanes::kBytes || i < lanes.count) {
                            const uint32_t target = to + r * Threads * Lanes::kBytes + i * static_cast<int>(sizeof(T));
                            if constexpr (Lanes::kMove == 16) {
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(target), "l"(at + i) : "memory");
                            } else {
                                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(target), "l"(at + i),
                                             "n"(Lanes::kMove) : "memory");
                            }
                        }
                    }
                }
            }
            at += step;
        }
    }

    // ends a stage's fetches
    __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // the oldest stage is there; the ones behind it may still be on their way
    __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(Stages - 2) : "memory"); }
    __device__ __forceinline__ void drain() const { asm volatile("cp.async.wait_all;" ::: "memory"); }

    // odd: of that row
    __device__ __forceinline__ Row<N> row(int stage, int array, int r, bool odd) const {
        if constexpr (Lanes::kShifted) {
            constexpr int kWords = Lanes::kBytes / 4;
            union {
                uint32_t words[kWords + 1];
                Stored<T, N> channels;
            } in;
            const uint32_t* from = reinterpret_cast<const uint32_t*>(slot(stage, array, r));
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                in.words[i] = from[i];
            }
            in.words[kWords] = *word_behind(stage, array, r);
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                in.words[i] = odd ? __funnelshift_r(in.words[i], in.words[i + 1], 16) : in.words[i];
            }
            return Row<N>::from(in.channels);
        } else {
            return Row<N>::from(*slot(stage, array, r));
        }
    }
};

// Maps of the pieces of a group -> the maps before each tile in the group, and the group's map.
// Takes the ring's memory. A thread composes N pieces of a channel, a run of them; the runs
// before its own give it the rest.
template <typename T, int N>
__device__ __forceinline__ void share_maps(
    const ScanArgs<T>& p, bool cut, const Row<N>& keep, const Row<N>& rest, const Row<N>& sum
) {
    static_assert(N % kPieces == 0, "a run holds whole tiles");
    extern __shared__ __align__(16) unsigned char ring[];
    float2* maps = reinterpret_cast<float2*>(ring);   // [pieces of the group][N * lanes]
    __shared__ float2 runs[kMapThreads];                 // [runs][N * lanes]
    const int thread = threadIdx.x, width = N * p.lanes;
    const int run = thread / width, lane = thread % width;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        maps[N * thread + i] = make_map(keep.get(i), rest.get(i), sum.get(i), cut);
    }
    __syncthreads();
    Chain before[N / kPieces];   // each tile of the run
    Chain all;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (k % kPieces == 0) {
            before[k / kPieces] = all;
        }
        all.add(maps[(run * N + k) * width + lane]);
    }
    runs[thread] = all.map();
    __syncthreads();
    const int group = blockIdx.x / p.slabs;
    const int channel = (blockIdx.x - group * p.slabs) * width + lane;
    if (channel >= p.channels) {
        return;
    }
    Chain earlier;
    for (int k = 0; k < run; ++k) {
        earlier.add(runs[k * width + lane]);
    }
    const int place = group * p.per_group + run * (N / kPieces);
#pragma unroll
    for (int t = 0; t < N / kPieces; ++t) {
        if (place + t < p.tiles) {
            p.maps[static_cast<size_t>(place + t) * p.channels + channel] = earlier.then(before[t]);
        }
    }
    if (run == kMapThreads / width - 1) {
        p.groups[static_cast<size_t>(group) * p.channels + channel] = earlier.then(all);
    }
}

template <bool Value> struct Flag {
    static constexpr bool value = Value;
};

// One answer for the lanes of a warp that are here: where one of them needs the path with marked
// rows all take it, instead of both paths one after the other.
__device__ __forceinline__ bool all_here(bool value) { return __all_sync(__activemask(), value); }

// A group's rows are fetched at once and lie together, so this kernel streams: a thread walks
// eight of them. 960,000 x 64 float16: 52 us, 4.7 of the 6.55 TB/s that a copy moves, bound by its
// instructions; the two special functions of a gate alone take 27 us. 200,000 x 96 float32 in 5003
// sequences: 46 us, 3.3 TB/s, bound by the searches for a piece's sequence and the rows that start or end one.
//
// Backwards, e_t = a_t dh_t is what a row hands to the row before it: e_t = a_t (e_{t+1} + dy_t), a
// chain of the same kind, from the piece's last row to its first, or from the last row of the first
// sequence in it.
//
// Here and in the gradient kernel dh_t = a_{t+1} dh_{t+1} + dy_t is one multiply-add. A product of pairs
// and a sum behind it become one or not as the compiler likes, and results would depend on the launch.
template <typename T, int Granule, bool Backward>
__global__ void __launch_bounds__(kMapThreads, 6) recurrence_maps_kernel(ScanArgs<T> p) {
    constexpr int N = kMapBytes / static_cast<int>(sizeof(T)), R = kPieceRows;
    const int group = blockIdx.x / p.slabs;
    // pieces in the order of the chain
    const int place = group * p.per_group * kPieces + static_cast<int>(threadIdx.x) / p.lanes;
    const int piece = Backward ? p.tiles * kPieces - 1 - place : place;
    const Channels<T, N, Granule> lanes(p, blockIdx.x - group * p.slabs);
    const Ring<T, N, Granule, 2, R, 1, kMapThreads> ring;
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < (p.channels + kScanChannels - 1) / kScanChannels; i += kMapThreads) {
            p.arrived[i] = 0;
        }
    }
    Row<N> keep = Row<N>::filled(1.0f), rest = Row<N>::filled(0.0f), sum = rest;   // A, 1 - A and H
    Row<N> share = keep;   // backwards: sum is dh of a row, and share of it reaches the next one
    bool cut = false;
    const int first = piece * R, rows = p.order.rows - first;
    if (piece >= 0 && rows > 0 && lanes.count > 0) {
        const T* from = Backward ? lanes.row(p.dy, p.dy_stride, p.order, first) : lanes.row(p.x, p.x_stride, p.order, first);
        const T* gates_from = lanes.row(p.z, p.z_stride, p.order, first);
        ring.fetch(lanes, 0, 0, from, lanes.row_step * (Backward ? p.dy_stride : p.x_stride), rows);
        ring.fetch(lanes, 0, 1, gates_from, lanes.row_step * p.z_stride, rows);
        ring.commit();
        Cursor cursor;   // meanwhile
        lanes.seek(cursor, p.order, first);
        const bool covered = all_here(cursor.covers(first, R));
        ring.drain();
        const auto scan = [&](auto marked) {
            constexpr bool kMarked = decltype(marked)::value;
            const int live = Backward && kMarked ? cursor.end - first : R;   // rows that hand something out
            if (Backward && kMarked && (cursor.begin > first || live <= R)) {
                cut = true;
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = Backward ? R - 1 - i : i;
                if (kMarked && (Backward ? cursor.begin > first || r >= live : first + r < cursor.begin)) {
                    cut = true;   // outside all sequences, or behind the first one's end
                    sum = Row<N>::filled(0.0f);   // backwards no row with anything comes before
                    continue;
                }
                const Row<N> z = ring.row(0, 1, r, lanes.odd(p.z, p.z_stride, p.order, first + r));
                const Row<N> value = ring.row(0, 0, r, Backward ? lanes.odd(p.dy, p.dy_stride, p.order, first + r)
                                                                : lanes.odd(p.x, p.x_stride, p.order, first + r));
                if (Backward && kMarked && r == live - 1) {
                    sum = lanes.state(p.dfinal, p.order.sequence(cursor.j), p.channels);
                }
                if (!Backward && kMarked && first + r == cursor.begin) {
                    cut = true;
                    sum = lanes.state(p.initial, p.order.sequence(cursor.j), p.channels);
                }
#pragma unroll
                for (int c = 0; c < Row<N>::kPairs; ++c) {
                    const Weights w(odds_of(z.v[c]));
                    rest.v[c] = fma(keep.v[c], w.rest, rest.v[c]);
                    keep.v[c] = keep.v[c] * w.a;
                    if constexpr (Backward) {
                        sum.v[c] = fma(share.v[c], sum.v[c], value.v[c]);
                        share.v[c] = w.a;
                    } else {
                        sum.v[c] = w.blend(sum.v[c], value.v[c]);
                    }
                }
                if (!Backward && kMarked && first + r == cursor.end - 1) {
                    cursor.next(p.order);
                }
            }
        };
        if (covered) {
            scan(Flag<false>{});
        } else {
            scan(Flag<true>{});
        }
    }
    if constexpr (Backward) {
        sum = sum.times(share);
    }
    share_maps(p, cut, keep, rest, sum);
}

// 960,000 x 64 float16 with carries: 60 us, 6.6 TB/s, the memory's rate; 200,000 x 96 float32 in 5003
// sequences: 43 us, 5.7 TB/s.
constexpr int kRingRows = 2, kRingStages = 4;

template <typename T, int Granule>
__global__ void __launch_bounds__(kThreads, 3) recurrence_apply_kernel(ScanArgs<T> p) {
    constexpr int N = kMapBytes / static_cast<int>(sizeof(T)), R = kRingRows, S = kRingStages;
    // the last tiles first: the maps kernel read them last
    const int block = gridDim.x - 1 - blockIdx.x;
    const int place = block / p.slabs * (kThreads / p.lanes) + static_cast<int>(threadIdx.x) / p.lanes;
    const Channels<T, N, Granule> lanes(p, block % p.slabs);
    const Ring<T, N, Granule, 2, R, S> ring;
    visit_sequences(p.order, p.initial, p.final, p.channels, p.status);
    if (place >= p.tiles || lanes.count == 0) {
        return;
    }
    const int first = place * kTileRows, end = min(first + kTileRows, p.order.rows);
    const T* from = lanes.row(p.x, p.x_stride, p.order, first);
    const T* gates_from = lanes.row(p.z, p.z_stride, p.order, first);
    const auto fetch = [&](int row, int stage) {
        if (row < end) {
            ring.fetch(lanes, stage, 0, from, lanes.row_step * p.x_stride, end - row);
            ring.fetch(lanes, stage, 1, gates_from, lanes.row_step * p.z_stride, end - row);
        }
        ring.commit();
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        fetch(first + s * R, s);
    }
    Row<N> h = lanes.reaching(p, place);
    Cursor cursor;
    lanes.seek(cursor, p.order, first);
    const long long down = lanes.row_step * p.channels;
    T* out = p.h + static_cast<long long>(p.order.row(first)) * p.channels + lanes.c;
    int stage = 0;
#pragma unroll 1
    for (int row = first; row < end; row += R) {
        ring.wait();
        fetch(row + (S - 1) * R, (stage + S - 1) % S);
        if (row % kCarryRows == 0) {
            lanes.store_state(p.carries, row / kCarryRows, p.channels, h);
        }
        const auto write = [&](auto marked) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (decltype(marked)::value && row + r >= end) {
                    break;
                }
                if (decltype(marked)::value && row + r == cursor.begin) {
                    h = lanes.state(p.initial, p.order.sequence(cursor.j), p.channels);
                }
                const Row<N> z = ring.row(stage, 1, r, lanes.odd(p.z, p.z_stride, p.order, row + r));
                const Row<N> x = ring.row(stage, 0, r, lanes.odd(p.x, p.x_stride, p.order, row + r));
#pragma unroll
                for (int i = 0; i < Row<N>::kPairs; ++i) {
                    h.v[i] = Weights(odds_of(z.v[i])).blend(h.v[i], x.v[i]);
                }
                if (decltype(marked)::value && row + r < cursor.begin) {
                    h = Row<N>::filled(0.0f);
                }
                lanes.store(out, h);
                out += down;
                if (decltype(marked)::value && row + r == cursor.end - 1) {
                    lanes.store_state(p.final, p.order.sequence(cursor.j), p.channels, h);
                    cursor.next(p.order);
                }
            }
        };
        if (all_here(cursor.covers(row, R))) {
            write(Flag<false>{});
        } else {
            write(Flag<true>{});
        }
        stage = (stage + 1) % S;
    }
}

// Batches of rows from the last to the first: h again up to the batch's end, with
// q_t = a_t (h_{t-1} - x_t), then dh_t back from there, and dz_t = dx_t q_t. 960,000 x 64 float16:
// 101 us, 6.3 TB/s, the memory's rate; 200,000 x 96 float32 in 5003 sequences: 84 us, 4.7 TB/s.
template <typename T, int Granule>
__global__ void __launch_bounds__(kThreads, 2) recurrence_gradient_kernel(ScanArgs<T> p) {
    constexpr int N = kGradientBytes / static_cast<int>(sizeof(T)), R = kCarryRows, P = Row<N>::kPairs;
    // time forwards, so the tiles that the maps kernel read last come first
    const int spans = (p.tiles + p.span_tiles - 1) / p.span_tiles, per_block = kThreads / p.lanes;
    const int span = static_cast<int>(blockIdx.x) / p.slabs * per_block + static_cast<int>(threadIdx.x) / p.lanes;
    const Channels<T, N, Granule> lanes(p, blockIdx.x % p.slabs);
    const Ring<T, N, Granule, 3, R, 2> ring;
    // Of each row of a batch that starts or ends a sequence. In local memory, as the loop that writes it is
    // not unrolled: there are no registers left, and shared memory would be the first-level cache's, which
    // the copies come through (102 us become 130).
    int owner[R];
    visit_sequences(p.order, p.dfinal, p.dinitial, p.channels, nullptr);
    if (span >= spans || lanes.count == 0) {
        return;
    }
    const int span_rows = p.span_tiles * kTileRows;
    const int first = span * span_rows, end = min(first + span_rows, p.order.rows);
    const auto fetch = [&](int row, int stage) {
        if (row >= first) {
            const T* x = lanes.row(p.x, p.x_stride, p.order, row);
            const T* z = lanes.row(p.z, p.z_stride, p.order, row);
            const T* dy = lanes.row(p.dy, p.dy_stride, p.order, row);
            ring.fetch(lanes, stage, 0, x, lanes.row_step * p.x_stride, end - row);
            ring.fetch(lanes, stage, 1, z, lanes.row_step * p.z_stride, end - row);
            ring.fetch(lanes, stage, 2, dy, lanes.row_step * p.dy_stride, end - row);
        }
        ring.commit();
    };
    const int last = first + (end - 1 - first) / R * R;
    fetch(last, 0);
    Row<N> e = lanes.reaching(p, p.tiles - 1 - min((span + 1) * p.span_tiles - 1, p.tiles - 1));
    Cursor cursor;
    lanes.seek(cursor, p.order, last);
    const long long down = lanes.row_step * p.channels;
    int stage = 0;
#pragma unroll 1
    for (int row = last; row >= first; row -= R) {
        Row<N> h = lanes.state(p.carries, row / R, p.channels);
        // from the sequence of the batch behind, or the one after it, back to the first that ends
        // behind this batch's first row
        while (cursor.begin > row) {
            Cursor before = cursor;
            if (!before.back(p.order) || before.end <= row) {
                break;
            }
            cursor = before;
        }
        const bool covered = all_here(cursor.covers(row, R));
        // of the batch's rows: start a sequence, end one (whose numbers are kept), lie outside all
        unsigned heads = 0, tails = 0, dead = 0;
        if (!covered) {
            Cursor at = cursor;
#pragma unroll 1
            for (int r = 0; r < R; ++r) {
                dead |= row + r < at.begin ? 1u << r : 0u;
                heads |= row + r == at.begin ? 1u << r : 0u;
                if (row + r == at.begin || row + r == at.end - 1) {
                    owner[r] = p.order.sequence(at.j);
                }
                if (row + r == at.end - 1) {
                    tails |= 1u << r;
                    at.next(p.order);
                }
            }
        }
        ring.wait();
        fetch(row - R, stage ^ 1);
        const long long at0 = static_cast<long long>(p.order.row(row)) * p.channels + lanes.c;
        const auto differentiate = [&](auto marked) {
            Row<N> odds[R], q[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (decltype(marked)::value && (heads >> r & 1u)) {
                    h = lanes.state(p.initial, owner[r], p.channels);
                }
                const Row<N> zr = ring.row(stage, 1, r, lanes.odd(p.z, p.z_stride, p.order, row + r));
                const Row<N> xr = ring.row(stage, 0, r, lanes.odd(p.x, p.x_stride, p.order, row + r));
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    odds[r].v[i] = odds_of(zr.v[i]);
                    const Weights w(odds[r].v[i]);
                    q[r].v[i] = w.a * minus(h.v[i], xr.v[i]);
                    h.v[i] = w.blend(h.v[i], xr.v[i]);
                }
            }
            Row<N> dh = e, share = Row<N>::filled(1.0f);   // share of dh reaches the row before
#pragma unroll
            for (int r = R - 1; r >= 0; --r) {
                if (decltype(marked)::value && (tails >> r & 1u)) {
                    dh = lanes.state(p.dfinal, owner[r], p.channels);
                    share = Row<N>::filled(1.0f);
                }
                const Row<N> up = ring.row(stage, 2, r, lanes.odd(p.dy, p.dy_stride, p.order, row + r));
                Row<N> dx, dz;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const Weights w(odds[r].v[i]);
                    dh.v[i] = fma(share.v[i], dh.v[i], up.v[i]);
                    share.v[i] = w.a;
                    dx.v[i] = w.rest * dh.v[i];
                    dz.v[i] = dx.v[i] * q[r].v[i];
                }
                if (decltype(marked)::value && (dead >> r & 1u)) {
                    dx = dz = dh = share = Row<N>::filled(0.0f);
                }
                if (!decltype(marked)::value || row + r < end) {
                    lanes.store(p.dx + at0 + r * down, dx);
                    lanes.store(p.dz + at0 + r * down, dz);
                }
                if (decltype(marked)::value && (heads >> r & 1u)) {
                    lanes.store_state(p.dinitial, owner[r], p.channels, dh.times(share));
                }
            }
            e = dh.times(share);
        };
        if (covered) {
            differentiate(Flag<false>{});
        } else {
            differentiate(Flag<true>{});
        }
        stage ^= 1;
    }
}

// A run of kRun maps of a channel by every warp of a block, kWindow by the block.
constexpr int kScanWarps = 8, kRun = kWindow / kScanWarps;

// Block: a window of groups for 32 channels. The last block of these channels to be done goes on to
// the states of the windows: which block that is does not change what it computes. 7500 groups of
// 64 channels: 8.4 us, a chain of latencies, among them those of its instructions, which every
// launch fetches anew: with all loops unrolled it takes 10.6 us.
__global__ void __launch_bounds__(32 * kScanWarps) recurrence_scan_kernel(
    float2* groups, int count, int channels, float2* windows, float* states, int* arrived
) {
    __shared__ float2 held[kWindow][32];       // the maps: a thread reads what it wrote itself
    __shared__ float2 shared[kScanWarps][32];   // of the runs
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.y * 32 + lane;
    // maps `first` to `first` + kRun - 1, and the map of all of them in `shared`
    const auto load = [&](const float2* from, int first, int end) {
        float2 maps[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            maps[i] = c < channels && first + i < end ? __ldcg(from + static_cast<size_t>(first + i) * channels + c)
                                                      : identity();
        }
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            held[warp * kRun + i][lane] = maps[i];
        }
        Chain run;
#pragma unroll 1
        for (int i = 0; i < kRun; ++i) {
            run.add(held[warp * kRun + i][lane]);
        }
        shared[warp][lane] = run.map();
        __syncthreads();
    };
    int first = blockIdx.x * kWindow + warp * kRun;
    load(groups, first, count);
    Chain before;
#pragma unroll 1
    for (int w = 0; w < warp; ++w) {
        before.add(shared[w][lane]);
    }
#pragma unroll 1
    for (int i = 0; i < kRun; ++i) {
        if (c < channels && first + i < count) {
            groups[static_cast<size_t>(first + i) * channels + c] = before.map();
        }
        before.add(held[warp * kRun + i][lane]);
    }
    if (warp == kScanWarps - 1 && c < channels) {
        __stcg(windows + static_cast<size_t>(blockIdx.x) * channels + c, before.map());
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(arrived + blockIdx.y, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!last) {
        return;
    }
    __threadfence();
    const int windows_count = gridDim.x;
    float h = 0.0f;
    for (int base = 0; base < windows_count; base += kWindow) {
        first = base + warp * kRun;
        load(windows, first, windows_count);
        float reached = h;   // the state before the warp's run, h the one behind all
#pragma unroll 1
        for (int w = 0; w < kScanWarps; ++w) {
            reached = w == warp ? h : reached;
            h = apply(shared[w][lane], h);
        }
#pragma unroll 1
        for (int i = 0; i < kRun; ++i) {
            if (c < channels && first + i < windows_count) {
                states[static_cast<size_t>(first + i) * channels + c] = reached;
            }
            reached = apply(held[warp * kRun + i][lane], reached);
        }
        __syncthreads();   // the next turn writes what this one reads
    }
}

// One row of every stream: h = a state + (1 - a) x. 16,411 x 192 float32: 8.7 us, 7.3 TB/s, in part from
// the second-level cache; a few rows: 1.5 us, a launch.
template <typename T, int V>
__global__ void __launch_bounds__(256) recurrence_step_kernel(
    const T* x, long long x_stride, const T* z, long long z_stride, const float* state, long long rows,
    int channels, T* h, float* next
) {
    const int vectors = channels / V;
    const long long at = blockIdx.x * 256LL + threadIdx.x;
    const long long row = at / vectors;
    const int c = static_cast<int>(at - row * vectors) * V;
    if (row >= rows) {
        return;
    }
    const Pack<T, V> xs = load_pack<T, V>(x + row * x_stride + c), zs = load_pack<T, V>(z + row * z_stride + c);
    const Pack<float, V> old = load_pack<float, V>(state + row * channels + c);
    Pack<T, V> y;
    Pack<float, V> now;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        now.v[i] = Weights(odds_of(both(zs.get(i)))).blend(both(old.v[i]), both(xs.get(i))).x;
        y.set(i, now.v[i]);
    }
    store_pack<T, V>(h + row * channels + c, y);
    store_pack<float, V>(next + row * channels + c, now);
}

// ---- host -------------------------------------------------------------------------

// Row numbers of the last group, places behind the last sequence that a search tries and their sums
// stay in an int.
constexpr int kMaxRows = 0x7fffffff - kMapThreads * kPieceRows;
constexpr int kMaxSequences = 0x7fffffff - 64;

constexpr int kMaxChannels = 65535 * kScanChannels;   // of the scan kernel's grid

inline int tiles_of(long long rows) { return static_cast<int>((rows + kTileRows - 1) / kTileRows); }

// Threads across a slab for so many threads' worth of channels: `most`, a 128-byte line, or half
// of them where that leaves fewer without a channel; for fewer channels the next power of two.
inline int slab_lanes(int vectors, int most) {
    if (vectors < most) {
        int lanes = 1;
        while (lanes < vectors) {
            lanes <<= 1;
        }
        return lanes;
    }
    const int half = most / 2;
    return (vectors + half - 1) / half * half < (vectors + most - 1) / most * most ? half : most;
}

inline int vectors_of(int channels, int element, int bytes) { return (channels * element + bytes - 1) / bytes; }
inline int map_lanes(int channels, int element) { return slab_lanes(vectors_of(channels, element, kMapBytes), 128 / kMapBytes); }

// tiles of a group: a block of the maps kernel
inline int group_tiles(int lanes) { return kMapThreads / lanes / kPieces; }

struct ScanBytes {
    size_t maps, groups, windows, states, total;
};

inline ScanBytes scan_bytes(long long rows, int channels, int element) {
    ScanBytes b{};
    const long long tiles = tiles_of(rows), per_group = group_tiles(map_lanes(channels, element));
    const long long groups = (tiles + per_group - 1) / per_group, windows = (groups + kWindow - 1) / kWindow;
    b.maps = align_up(sizeof(float2) * channels * tiles);
    b.groups = align_up(sizeof(float2) * channels * groups);
    b.windows = align_up(sizeof(float2) * channels * windows);
    b.states = align_up(sizeof(float) * channels * windows);
    const size_t arrived = align_up(sizeof(int) * ((channels + kScanChannels - 1) / kScanChannels));
    b.total = tiles <= 1 ? 256 : b.maps + b.groups + b.windows + b.states + arrived;
    return b;
}

// Blocks that visit the sequences in one turn, at most so many as are there at a time. More than the
// tiles need where most sequences have no rows: both passes over 64 rows and 1,000,000 such
// sequences of 64 channels took 124 ms with the blocks of the tiles alone, and take 1.0.
inline long long visitors(int sequences) {
    return std::min<long long>((static_cast<long long>(sequences) + kThreads - 1) / kThreads, 2 * 148);
}

template <typename Kernel, typename T>
int launch_walk(Kernel kernel, int threads, int ring_bytes, long long blocks, const ScanArgs<T>& p, cudaStream_t stream) {
    LAT_REQUIRE(blocks <= 0x7fffffffLL, "the recurrence supports at most 2^31 blocks of tiles.");
    LAT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes));
    kernel<<<static_cast<unsigned>(blocks), threads, ring_bytes, stream>>>(p);
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

template <typename T, int Granule, bool Backward>
int launch_scan(ScanArgs<T> p, void* workspace, size_t bytes, cudaStream_t stream) {
    constexpr int kElement = static_cast<int>(sizeof(T)), N = kMapBytes / kElement, M = kGradientBytes / kElement;
    constexpr int kRing = Ring<T, N, Granule, 2, kRingRows, kRingStages>::kBytes;
    constexpr int kMapsRing = Ring<T, N, Granule, 2, kPieceRows, 1, kMapThreads>::kBytes;
    p.tiles = tiles_of(p.order.rows);
    p.lanes = map_lanes(p.channels, kElement);
    p.per_group = group_tiles(p.lanes);
    const int vectors = vectors_of(p.channels, kElement, kMapBytes);
    p.slabs = (vectors + p.lanes - 1) / p.lanes;
    const int groups = (p.tiles + p.per_group - 1) / p.per_group;
    const long long blocks = static_cast<long long>(groups) * p.slabs;
    const ScanBytes b = scan_bytes(p.order.rows, p.channels, kElement);
    if (workspace == nullptr || bytes < b.total) {
        return fail(LAT_WORKSPACE_TOO_SMALL, "recurrence workspace is too small.");
    }
    if (p.tiles > 1) {
        char* base = static_cast<char*>(workspace);
        p.maps = reinterpret_cast<float2*>(base);
        p.groups = reinterpret_cast<float2*>(base + b.maps);
        p.windows = reinterpret_cast<float2*>(base + b.maps + b.groups);
        p.states = reinterpret_cast<float*>(base + b.maps + b.groups + b.windows);
        p.arrived = reinterpret_cast<int*>(base + b.maps + b.groups + b.windows + b.states);
        const int code =
            launch_walk(recurrence_maps_kernel<T, Granule, Backward>, kMapThreads, kMapsRing, blocks, p, stream);
        if (code != LAT_OK) {
            return code;
        }
        const dim3 scan_grid((groups + kWindow - 1) / kWindow, (p.channels + kScanChannels - 1) / kScanChannels);
        recurrence_scan_kernel<<<scan_grid, 32 * kScanWarps, 0, stream>>>(p.groups, groups, p.channels, p.windows,
                                                                          p.states, p.arrived);
        LAT_LAUNCH_CHECK();
    }
    if constexpr (Backward) {
        const int wide = vectors_of(p.channels, kElement, kGradientBytes);
        p.lanes = slab_lanes(wide, 128 / kGradientBytes);
        p.slabs = (wide + p.lanes - 1) / p.lanes;
        const int per_block = kThreads / p.lanes;
        const auto blocks_of = [&](int span_tiles) {
            const long long spans = (p.tiles + span_tiles - 1) / span_tiles;
            return (spans + per_block - 1) / per_block * p.slabs;
        };
        // A walk of two tiles starts less often, a walk of one ends sooner: it is taken where two would
        // leave multiprocessors idle (2168 x 13 float16 in 94 sequences: 45 us, with two tiles 77;
        // 15,191 x 12 float32 in 134: 15 against 24).
        p.span_tiles = blocks_of(2) >= 2 * 148 ? 2 : 1;
        constexpr int kGradientRing = Ring<T, M, Granule, 3, kCarryRows, 2>::kBytes;
        return launch_walk(recurrence_gradient_kernel<T, Granule>, kThreads, kGradientRing,
                           std::max(blocks_of(p.span_tiles), visitors(p.order.sequences)), p, stream);
    } else {
        const int per_block = kThreads / p.lanes;
        const long long walkers = static_cast<long long>((p.tiles + per_block - 1) / per_block) * p.slabs;
        return launch_walk(recurrence_apply_kernel<T, Granule>, kThreads, kRing,
                           std::max(walkers, visitors(p.order.sequences)), p, stream);
    }
}

template <typename T, bool Backward>
int run_scan(const ScanArgs<T>& p, void* workspace, size_t bytes, cudaStream_t stream) {
    const auto fits = [&](int granule) {
        const int n = granule / static_cast<int>(sizeof(T));
        bool ok = p.channels % n == 0 && p.x_stride % n == 0 && p.z_stride % n == 0 && aligned_to(p.x, granule) &&
                  aligned_to(p.z, granule);
        if (Backward) {
            ok = ok && p.dy_stride % n == 0 && aligned_to(p.dy, granule) && aligned_to(p.dx, granule) &&
                 aligned_to(p.dz, granule);
        } else {
            ok = ok && aligned_to(p.h, granule);
        }
        return ok;
    };
    if (fits(16)) {
        return launch_scan<T, 16, Backward>(p, workspace, bytes, stream);
    }
    if (fits(8)) {
        return launch_scan<T, 8, Backward>(p, workspace, bytes, stream);
    }
    if (fits(4)) {
        return launch_scan<T, 4, Backward>(p, workspace, bytes, stream);
    }
    if constexpr (sizeof(T) == 2) {
        return launch_scan<T, 2, Backward>(p, workspace, bytes, stream);
    }
    return fail(LAT_INVALID_ARGUMENT, "float32 features must be aligned to four bytes.");
}

// Without any rows: initial -> final, dfinal -> dinitial.
inline int hand_over(const float* from, float* to, int sequences, int channels, cudaStream_t stream) {
    const size_t bytes = sizeof(float) * static_cast<size_t>(sequences) * channels;
    if (to == nullptr || bytes == 0) {
        return LAT_OK;
    }
    if (from != nullptr) {
        LAT_CUDA_CHECK(cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, stream));
    } else {
        LAT_CUDA_CHECK(cudaMemsetAsync(to, 0, bytes, stream));
    }
    return LAT_OK;
}

template <typename T>
int forward_typed(const void* x, long long x_stride, const void* z, long long z_stride, Order order, int channels,
                  const float* initial, void* h, float* final, float* carries, void* workspace, size_t bytes,
                  int32_t* status, cudaStream_t stream) {
    ScanArgs<T> p{};
    p.x = static_cast<const T*>(x);
    p.z = static_cast<const T*>(z);
    p.x_stride = x_stride;
    p.z_stride = z_stride;
    p.order = order;
    p.channels = channels;
    p.initial = initial;
    p.carries = carries;
    p.h = static_cast<T*>(h);
    p.final = final;
    p.status = status;
    return run_scan<T, false>(p, workspace, bytes, stream);
}

template <typename T>
int backward_typed(const void* dy, long long dy_stride, const float* dfinal, const void* x, long long x_stride,
                   const void* z, long long z_stride, Order order, int channels, const float* initial,
                   const float* carries, void* dx, void* dz, float* dinitial, void* workspace, size_t bytes,
                   int32_t* status, cudaStream_t stream) {
    ScanArgs<T> p{};
    p.x = static_cast<const T*>(x);
    p.z = static_cast<const T*>(z);
    p.dy = static_cast<const T*>(dy);
    p.x_stride = x_stride;
    p.z_stride = z_stride;
    p.dy_stride = dy_stride;
    p.order = order;
    p.channels = channels;
    p.initial = initial;
    p.carries = const_cast<float*>(carries);
    p.dfinal = dfinal;
    p.dx = static_cast<T*>(dx);
    p.dz = static_cast<T*>(dz);
    p.dinitial = dinitial;
    p.status = status;
    return run_scan<T, true>(p, workspace, bytes, stream);
}

} // namespace

} // namespace lat

using namespace lat;

extern "C" {

size_t lat_recurrence_workspace_bytes(int32_t dtype, int32_t rows, int32_t channels) {
    if (rows <= 0 || channels <= 0) {
        return 256;
    }
    return scan_bytes(rows, channels, dtype == LAT_F32 ? 4 : 2).total;
}

int32_t lat_recurrence_carry_rows(int32_t rows) {
    return rows <= 0 ? 0 : (rows - 1) / kCarryRows + 1;
}

int lat_recurrence_forward(
    int32_t dtype, const void* feats, int64_t feat_row_stride, const void* gate, int64_t gate_row_stride,
    int32_t rows, int32_t channels, const int32_t* offsets, int32_t sequences, const float* initial_state,
    int32_t reverse, void* out, float* final_state, float* carries, void* workspace, size_t workspace_bytes,
    int32_t* status, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "the recurrence supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && rows <= kMaxRows && channels > 0 && feat_row_stride >= 0 && gate_row_stride >= 0,
                "feats and gate must have shape (N, C).");
    LAT_REQUIRE(channels <= kMaxChannels, "the recurrence supports at most 2097120 channels.");
    LAT_REQUIRE(sequences >= 0 && (sequences == 0 || offsets != nullptr),
                "offsets must hold one int32 entry per sequence and one more.");
    LAT_REQUIRE(sequences <= kMaxSequences, "the recurrence supports at most 2147483583 sequences.");
    cudaStream_t stream = as_stream(stream_ptr);
    if (rows == 0) {
        return hand_over(initial_state, final_state, sequences, channels, stream);
    }
    LAT_REQUIRE(feats != nullptr && gate != nullptr && out != nullptr, "feats and gate must have shape (N, C).");
    LAT_REQUIRE(offsets != nullptr, "offsets must hold one int32 entry per sequence and one more.");
    const Order order{offsets, rows, sequences, reverse != 0};
    if (dtype == LAT_F32) {
        return forward_typed<float>(feats, feat_row_stride, gate, gate_row_stride, order, channels, initial_state,
                                    out, final_state, carries, workspace, workspace_bytes, status, stream);
    }
    return forward_typed<__half>(feats, feat_row_stride, gate, gate_row_stride, order, channels, initial_state, out,
                                 final_state, carries, workspace, workspace_bytes, status, stream);
}

int lat_recurrence_backward(
    int32_t dtype, const void* grad, int64_t grad_row_stride, const float* grad_final, const void* feats,
    int64_t feat_row_stride, const void* gate, int64_t gate_row_stride, int32_t rows, int32_t channels,
    const int32_t* offsets, int32_t sequences, const float* initial_state, int32_t reverse, const float* carries,
    void* grad_feats, void* grad_gate, float* grad_initial, void* workspace, size_t workspace_bytes,
    int32_t* status, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "the recurrence supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && rows <= kMaxRows && channels > 0 && feat_row_stride >= 0 && gate_row_stride >= 0 &&
                    grad_row_stride >= 0, "feats and gate must have shape (N, C).");
    LAT_REQUIRE(channels <= kMaxChannels, "the recurrence supports at most 2097120 channels.");
    LAT_REQUIRE(sequences >= 0 && (sequences == 0 || offsets != nullptr),
                "offsets must hold one int32 entry per sequence and one more.");
    LAT_REQUIRE(sequences <= kMaxSequences, "the recurrence supports at most 2147483583 sequences.");
    cudaStream_t stream = as_stream(stream_ptr);
    if (rows == 0) {
        return hand_over(grad_final, grad_initial, sequences, channels, stream);
    }
    LAT_REQUIRE(feats != nullptr && gate != nullptr && grad != nullptr && grad_feats != nullptr &&
                    grad_gate != nullptr && carries != nullptr,
                "the backward pass needs the tile states of the forward pass.");
    LAT_REQUIRE(offsets != nullptr, "offsets must hold one int32 entry per sequence and one more.");
    const Order order{offsets, rows, sequences, reverse != 0};
    if (dtype == LAT_F32) {
        return backward_typed<float>(grad, grad_row_stride, grad_final, feats, feat_row_stride, gate,
                                     gate_row_stride, order, channels, initial_state, carries, grad_feats,
                                     grad_gate, grad_initial, workspace, workspace_bytes, status, stream);
    }
    return backward_typed<__half>(grad, grad_row_stride, grad_final, feats, feat_row_stride, gate, gate_row_stride,
                                  order, channels, initial_state, carries, grad_feats, grad_gate, grad_initial,
                                  workspace, workspace_bytes, status, stream);
}

int lat_recurrence_step(
    int32_t dtype, const void* feats, int64_t feat_row_stride, const void* gate, int64_t gate_row_stride,
    const float* state, int64_t rows, int32_t channels, void* out, float* next_state, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "the recurrence supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && channels > 0 && feat_row_stride >= 0 && gate_row_stride >= 0,
                "feats and gate must have shape (N, C).");
    if (rows == 0) {
        return LAT_OK;
    }
    LAT_REQUIRE(feats != nullptr && gate != nullptr && state != nullptr && out != nullptr && next_state != nullptr,
                "feats, gate and state must have shape (N, C).");
    cudaStream_t stream = as_stream(stream_ptr);
    const bool vec = channels % 4 == 0 && feat_row_stride % 4 == 0 && gate_row_stride % 4 == 0 &&
                     aligned_to(feats, 16) && aligned_to(gate, 16) && aligned_to(state, 16) && aligned_to(out, 16) &&
                     aligned_to(next_state, 16);
    const long long threads = rows * (vec ? channels / 4 : channels);
    const long long blocks = (threads + 255) / 256;
    LAT_REQUIRE(blocks <= 0x7fffffffLL, "the recurrence step supports at most 2^39 values.");
    const unsigned grid = static_cast<unsigned>(blocks);
#define LAT_STEP(T, V)                                                                                        \
    recurrence_step_kernel<T, V><<<grid, 256, 0, stream>>>(                                                   \
        static_cast<const T*>(feats), feat_row_stride, static_cast<const T*>(gate), gate_row_stride, state,   \
        rows, channels, static_cast<T*>(out), next_state)
    if (dtype == LAT_F32) {
        if (vec) {
            LAT_STEP(float, 4);
        } else {
            LAT_STEP(float, 1);
        }
    } else if (vec) {
        LAT_STEP(__half, 4);
    } else {
        LAT_STEP(__half, 1);
    }
#undef LAT_STEP
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

} // extern "C"
