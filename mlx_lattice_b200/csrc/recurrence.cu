// Gated linear recurrence along the rows of a sparse tensor, per sequence and channel:
//
//   a_t = sigmoid(z_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h before the first row = initial
//
// forward, or from the last row to the first (`reverse`), with its gradient
//
//   dh_t = dy_t + a_{t+1} dh_{t+1}  (+ dfinal at the last row)
//   dx_t = (1 - a_t) dh_t,  dz_t = a_t (1 - a_t) dh_t (h_{t-1} - x_t),  dinitial = a_1 dh_1
//
// Both directions are scans over affine maps h -> A h + H, which compose associatively. A
// block owns a tile of 128 rows and a slab of channels, holds it in registers, and a thread
// walks 8 rows of a few channels. The maps of the 16 row segments of a tile are composed in
// shared memory; tiles are chained over the rows through the workspace in one pass, so every
// input is read once and every output written once. What bounds it is the memory.
//
// The chain has a fixed shape: a tile composes the maps of the earlier tiles of its group of
// 16, the maps of the earlier groups of its supergroup of 16 groups, and the state at the
// start of the supergroup, always in this order. Results therefore do not depend on which
// block came first, and are bitwise repeatable. Blocks take tiles in ticket order, so a tile
// only waits for tiles that already run; every wait has a clock budget.
//
// A record of the chain is one 64-bit word, (A, H) or (0, h): it is written and read whole,
// so it needs no flag beside it. All ones (no arithmetic result has these bits in its low
// half) means "not yet written".
//
// A row that starts a sequence cuts the chain. Its map ignores the incoming h altogether
// (marked by A = -1, and selected, not multiplied by zero: a NaN or an infinity of one
// sequence does not reach the next). Rows outside all sequences give zeros.
//
// The backward pass recomputes h from the state at the start of each tile, which the forward
// pass leaves in float32 (4 / (128 * element size) of the features): it reads x, z, dy and
// writes dx, dz, and its h is not rounded to the feature type.
#include <algorithm>

#include "common.cuh"
#include "vector_io.cuh"

namespace lat {

namespace {

constexpr int kSegments = 16;
constexpr int kSegmentRows = 8;
constexpr int kTileRows = kSegments * kSegmentRows;
constexpr int kGroup = 16;                    // tiles of a group, groups of a supergroup
constexpr float kReset = -1.0f;

struct Chain {
    unsigned long long* tiles;   // [tiles][channels]    (A, H)
    unsigned long long* groups;  // [groups][channels]   (A, H)
    unsigned long long* states;  // [supergroups][channels]  (0, h at its first tile)
    int* ticket;                 // -1 before the first block
    long long budget;
    int32_t* status;
};

__device__ __forceinline__ unsigned long long record(float low, float high) {
    uint32_t bits = __float_as_uint(low);
    bits = bits == 0xFFFFFFFFu ? 0x7FFFFFFFu : bits;
    return (static_cast<unsigned long long>(__float_as_uint(high)) << 32) | bits;
}

__device__ __forceinline__ unsigned long long read_record(const unsigned long long* p) {
    unsigned long long v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ void write_record(unsigned long long* p, unsigned long long v) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

__device__ __forceinline__ float2 wait_record(const unsigned long long* p, unsigned long long v, const Chain& chain) {
    if (static_cast<uint32_t>(v) == 0xFFFFFFFFu) {
        const long long start = clock64();
        while (static_cast<uint32_t>(v = read_record(p)) == 0xFFFFFFFFu) {
            if (clock64() - start > chain.budget) {
                raise_status(chain.status, LAT_STATUS_WAIT_TIMEOUT);
                v = 0;
                break;
            }
        }
    }
    return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// later after earlier, as maps
__device__ __forceinline__ float2 compose(float2 earlier, float2 later) {
    if (later.x == kReset) {
        return later;
    }
    return make_float2(earlier.x == kReset ? kReset : later.x * earlier.x, fmaf(later.x, earlier.y, later.y));
}

__device__ __forceinline__ float apply(float2 map, float h) {
    return map.x == kReset ? map.y : fmaf(map.x, h, map.y);
}

// Map of `count` consecutive records in order; eight loads in flight.
__device__ __forceinline__ float2 compose_records(
    const unsigned long long* first, int count, int stride, const Chain& chain
) {
    float2 map = make_float2(1.0f, 0.0f);
    for (int base = 0; base < count; base += 8) {
        unsigned long long raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            raw[i] = base + i < count ? read_record(first + static_cast<size_t>(base + i) * stride) : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (base + i < count) {
                map = compose(map, wait_record(first + static_cast<size_t>(base + i) * stride, raw[i], chain));
            }
        }
    }
    return map;
}

// The state that reaches tile `tile` (in chain order) in channel `c`, given the tile's own
// map, which is published for the tiles behind it. `needed` is false when the tile's first
// row cuts the chain.
__device__ __forceinline__ float chain_through(
    const Chain& chain, int tile, int tiles, int channels, int c, float2 own, bool needed
) {
    if (tile + 1 < tiles) {
        write_record(chain.tiles + static_cast<size_t>(tile) * channels + c, record(own.x, own.y));
    }
    const int group = tile / kGroup, member = tile % kGroup;
    const int super = group / kGroup, group_member = group % kGroup;
    const bool last = member == kGroup - 1, last_group = last && group_member == kGroup - 1;
    const bool cut = own.x == kReset;
    float2 near = make_float2(1.0f, 0.0f);
    if (needed || (last && !cut)) {
        near = compose_records(chain.tiles + static_cast<size_t>(group) * kGroup * channels + c, member, channels, chain);
    }
    if (last && tile + 1 < tiles) {
        const float2 map = compose(near, own);
        write_record(chain.groups + static_cast<size_t>(group) * channels + c, record(map.x, map.y));
    }
    float h = 0.0f;
    if (needed || (last_group && !cut)) {
        if (near.x != kReset) {
            const float2 far = compose_records(
                chain.groups + static_cast<size_t>(super) * kGroup * channels + c, group_member, channels, chain);
            if (far.x != kReset && super > 0) {
                const unsigned long long* state = chain.states + static_cast<size_t>(super) * channels + c;
                h = wait_record(state, read_record(state), chain).y;
            }
            h = apply(far, h);
        }
        h = apply(near, h);
    }
    if (last_group && tile + 1 < tiles) {
        write_record(chain.states + static_cast<size_t>(super + 1) * channels + c, record(0.0f, apply(own, h)));
    }
    return h;
}

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

// What the rows of a tile are: `head` the sequence that starts there, -1 a row that follows
// another, -2 a row outside all sequences; `tail` the sequence that ends there or -1.
struct RowTable {
    int head[kTileRows];
    int tail[kTileRows];
};

__device__ __forceinline__ void fill_rows(RowTable& table, const Order& order, int first, int32_t* status) {
    const int begin = order.begin(0), end = order.begin(order.sequences);
    for (int i = threadIdx.x; i < kTileRows; i += blockDim.x) {
        table.head[i] = first + i < begin || first + i >= end ? -2 : -1;
        table.tail[i] = -1;
    }
    // the first sequence that ends behind the tile's first row
    int low = 0, high = order.sequences;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (order.begin(mid + 1) > first) {
            high = mid;
        } else {
            low = mid + 1;
        }
    }
    __syncthreads();
    for (int j = low + static_cast<int>(threadIdx.x); j < order.sequences; j += blockDim.x) {
        const int b = order.begin(j) - first, e = order.begin(j + 1) - first;
        if (e < b) {
            raise_status(status, LAT_STATUS_BAD_INDEX);
        }
        if (b >= kTileRows) {
            break;
        }
        if (e > b) {
            if (b >= 0) {
                table.head[b] = j;
            }
            if (e >= 1 && e <= kTileRows) {
                table.tail[e - 1] = j;
            }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float sigmoid_gate(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// sigmoid(z) and sigmoid(-z), each to full relative precision; z is bounded below so that
// exp(-z) stays finite (a NaN passes)
__device__ __forceinline__ void sigmoid_pair(float z, float& a, float& rest) {
    const float e = __expf(z < -80.0f ? 80.0f : -z);
    a = __fdividef(1.0f, 1.0f + e);
    rest = e * a;
}

template <typename T> struct ScanArgs {
    const T* x;
    const T* z;
    const T* dy;
    long long x_stride, z_stride, dy_stride;
    Order order;
    int channels;
    int slabs;
    int tiles;
    const float* initial;   // [sequences][channels] or null
    float* carries;         // [tiles][channels] or null: h that reaches each tile
    T* h;
    float* final;           // [sequences][channels] or null
    const float* dfinal;    // [sequences][channels] or null
    T* dx;
    T* dz;
    float* dinitial;        // [sequences][channels] or null
    Chain chain;
};

__device__ __forceinline__ int take_ticket(int* ticket) {
    __shared__ int taken;
    if (threadIdx.x == 0) {
        taken = atomicAdd(ticket, 1) + 1;
    }
    __syncthreads();
    return taken;
}

// Block: Q threads across the slab (V channels each) times kSegments down the tile.
template <typename T, int V, int Q>
__global__ void __launch_bounds__(Q * kSegments) recurrence_forward_kernel(ScanArgs<T> p) {
    constexpr int C = Q * V;
    __shared__ RowTable table;
    __shared__ float2 maps[kSegments][C];
    const int id = p.tiles > 1 ? take_ticket(p.chain.ticket) : static_cast<int>(blockIdx.x);
    const int tile = id / p.slabs, slab = id - tile * p.slabs;
    const int first = tile * kTileRows;
    const int segment = threadIdx.x / Q;
    const int in_slab = (threadIdx.x % Q) * V;
    const int c = slab * C + in_slab;
    const bool in = c < p.channels;
    const int begin = first + segment * kSegmentRows;

    Pack<T, V> x[kSegmentRows];
    float a[kSegmentRows][V];
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        const bool live = in && begin + r < p.order.rows;
        const size_t row = live ? p.order.row(begin + r) : 0;
        x[r] = live ? load_pack<T, V>(p.x + row * p.x_stride + c) : zero_pack<T, V>();
        const Pack<T, V> z = live ? load_pack<T, V>(p.z + row * p.z_stride + c) : zero_pack<T, V>();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[r][i] = z.get(i);
        }
    }
    fill_rows(table, p.order, first, p.chain.status);

    float prod[V], h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        prod[i] = 1.0f;
        h[i] = 0.0f;
    }
    bool cut = false;
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        const int head = table.head[segment * kSegmentRows + r];
        if (head != -1) {
            cut = true;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = head >= 0 && in && p.initial != nullptr
                           ? p.initial[static_cast<size_t>(p.order.sequence(head)) * p.channels + c + i]
                           : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[r][i] = sigmoid_gate(a[r][i]);
            prod[i] *= a[r][i];
            h[i] = fmaf(a[r][i], h[i], (1.0f - a[r][i]) * x[r].get(i));
            if (head == -2) {
                h[i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        maps[segment][in_slab + i] = make_float2(cut ? kReset : prod[i], h[i]);
    }
    __syncthreads();
    if (threadIdx.x < C) {
        const int channel = slab * C + threadIdx.x;
        float2 own = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < kSegments; ++s) {
            own = compose(own, maps[s][threadIdx.x]);
        }
        float state = 0.0f;
        if (channel < p.channels) {
            if (p.tiles > 1) {
                state = chain_through(p.chain, tile, p.tiles, p.channels, channel, own, table.head[0] == -1);
            }
            if (p.carries != nullptr) {
                p.carries[static_cast<size_t>(tile) * p.channels + channel] = state;
            }
        }
        for (int s = 0; s < kSegments; ++s) {
            const float2 map = maps[s][threadIdx.x];
            maps[s][threadIdx.x].y = state;
            state = apply(map, state);
        }
    }
    __syncthreads();
    if (!in) {
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = maps[segment][in_slab + i].y;
    }
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        if (begin + r >= p.order.rows) {
            break;
        }
        const int head = table.head[segment * kSegmentRows + r], tail = table.tail[segment * kSegmentRows + r];
        if (head >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = p.initial != nullptr
                           ? p.initial[static_cast<size_t>(p.order.sequence(head)) * p.channels + c + i]
                           : 0.0f;
            }
        }
        Pack<T, V> y;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] = fmaf(a[r][i], h[i], (1.0f - a[r][i]) * x[r].get(i));
            if (head == -2) {
                h[i] = 0.0f;
            }
            y.set(i, h[i]);
        }
        store_pack<T, V>(p.h + static_cast<size_t>(p.order.row(begin + r)) * p.channels + c, y);
        if (tail >= 0 && p.final != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p.final[static_cast<size_t>(p.order.sequence(tail)) * p.channels + c + i] = h[i];
            }
        }
    }
}

// The tiles in falling order. e_t = a_t dh_t is what a row hands to the row before it:
// e_t = a_t e_{t+1} + a_t dy_t, the same kind of map with the same product of gates.
template <typename T, int V, int Q>
__global__ void __launch_bounds__(Q * kSegments) recurrence_backward_kernel(ScanArgs<T> p) {
    constexpr int C = Q * V;
    __shared__ RowTable table;
    __shared__ float2 maps[kSegments][C];    // forward maps, then h at the start of a segment
    __shared__ float2 flows[kSegments][C];   // backward maps, then e at the end of a segment
    const int id = p.tiles > 1 ? take_ticket(p.chain.ticket) : static_cast<int>(blockIdx.x);
    const int place = id / p.slabs, slab = id - place * p.slabs;
    const int tile = p.tiles - 1 - place;
    const int first = tile * kTileRows;
    const int segment = threadIdx.x / Q;
    const int in_slab = (threadIdx.x % Q) * V;
    const int c = slab * C + in_slab;
    const bool in = c < p.channels;
    const int begin = first + segment * kSegmentRows;

    Pack<T, V> x[kSegmentRows], dy[kSegmentRows], z[kSegmentRows];
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        const bool live = in && begin + r < p.order.rows;
        const size_t row = live ? p.order.row(begin + r) : 0;
        x[r] = live ? load_pack<T, V>(p.x + row * p.x_stride + c) : zero_pack<T, V>();
        z[r] = live ? load_pack<T, V>(p.z + row * p.z_stride + c) : zero_pack<T, V>();
        dy[r] = live ? load_pack<T, V>(p.dy + row * p.dy_stride + c) : zero_pack<T, V>();
    }
    fill_rows(table, p.order, first, p.chain.status);

    float a[kSegmentRows][V], prod[V], h[V], e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        prod[i] = 1.0f;
        h[i] = e[i] = 0.0f;
    }
    bool cut = false, flow_cut = false;
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        const int head = table.head[segment * kSegmentRows + r];
        if (head != -1) {
            cut = true;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = head >= 0 && in && p.initial != nullptr
                           ? p.initial[static_cast<size_t>(p.order.sequence(head)) * p.channels + c + i]
                           : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[r][i] = sigmoid_gate(z[r].get(i));
            prod[i] *= a[r][i];
            h[i] = fmaf(a[r][i], h[i], (1.0f - a[r][i]) * x[r].get(i));
            if (head == -2) {
                h[i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int r = kSegmentRows - 1; r >= 0; --r) {
        const int head = table.head[segment * kSegmentRows + r], tail = table.tail[segment * kSegmentRows + r];
        if (tail >= 0 || head == -2) {
            flow_cut = true;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                e[i] = tail >= 0 && in && p.dfinal != nullptr
                           ? p.dfinal[static_cast<size_t>(p.order.sequence(tail)) * p.channels + c + i]
                           : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            e[i] = head == -2 ? 0.0f : a[r][i] * (dy[r].get(i) + e[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        maps[segment][in_slab + i] = make_float2(cut ? kReset : prod[i], h[i]);
        flows[segment][in_slab + i] = make_float2(flow_cut ? kReset : prod[i], e[i]);
    }
    __syncthreads();
    if (threadIdx.x < C) {
        const int channel = slab * C + threadIdx.x;
        float2 own = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int s = kSegments - 1; s >= 0; --s) {
            own = compose(own, flows[s][threadIdx.x]);
        }
        float flow = 0.0f;
        if (channel < p.channels && p.tiles > 1) {
            // the tile's last row decides whether what comes from behind matters
            const bool open = table.tail[kTileRows - 1] < 0 && table.head[kTileRows - 1] != -2;
            flow = chain_through(p.chain, place, p.tiles, p.channels, channel, own, open);
        }
        for (int s = kSegments - 1; s >= 0; --s) {
            const float2 map = flows[s][threadIdx.x];
            flows[s][threadIdx.x].y = flow;
            flow = apply(map, flow);
        }
        float state = channel < p.channels ? p.carries[static_cast<size_t>(tile) * p.channels + channel] : 0.0f;
        for (int s = 0; s < kSegments; ++s) {
            const float2 map = maps[s][threadIdx.x];
            maps[s][threadIdx.x].y = state;
            state = apply(map, state);
        }
    }
    __syncthreads();
    if (!in) {
        return;
    }
    float before[kSegmentRows][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = maps[segment][in_slab + i].y;
        e[i] = flows[segment][in_slab + i].y;
    }
#pragma unroll
    for (int r = 0; r < kSegmentRows; ++r) {
        const int head = table.head[segment * kSegmentRows + r];
        if (head >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = p.initial != nullptr
                           ? p.initial[static_cast<size_t>(p.order.sequence(head)) * p.channels + c + i]
                           : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            before[r][i] = h[i];
            h[i] = fmaf(a[r][i], h[i], (1.0f - a[r][i]) * x[r].get(i));
        }
    }
#pragma unroll
    for (int r = kSegmentRows - 1; r >= 0; --r) {
        if (begin + r >= p.order.rows) {
            continue;
        }
        const int head = table.head[segment * kSegmentRows + r], tail = table.tail[segment * kSegmentRows + r];
        if (tail >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                e[i] = p.dfinal != nullptr
                           ? p.dfinal[static_cast<size_t>(p.order.sequence(tail)) * p.channels + c + i]
                           : 0.0f;
            }
        }
        Pack<T, V> dx, dz;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float gate, rest;
            sigmoid_pair(z[r].get(i), gate, rest);
            const float dh = dy[r].get(i) + e[i];
            const float dxi = rest * dh;
            dx.set(i, head == -2 ? 0.0f : dxi);
            dz.set(i, head == -2 ? 0.0f : a[r][i] * dxi * (before[r][i] - x[r].get(i)));
            e[i] = head == -2 ? 0.0f : a[r][i] * dh;
        }
        const size_t row = p.order.row(begin + r);
        store_pack<T, V>(p.dx + row * p.channels + c, dx);
        store_pack<T, V>(p.dz + row * p.channels + c, dz);
        if (head >= 0 && p.dinitial != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p.dinitial[static_cast<size_t>(p.order.sequence(head)) * p.channels + c + i] = e[i];
            }
        }
    }
}

// One row of every stream: h = a state + (1 - a) x.
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
        const float a = sigmoid_gate(zs.get(i));
        now.v[i] = fmaf(a, old.v[i], (1.0f - a) * xs.get(i));
        y.set(i, now.v[i]);
    }
    store_pack<T, V>(h + row * channels + c, y);
    store_pack<float, V>(next + row * channels + c, now);
}

// ---- host -------------------------------------------------------------------------

constexpr int kMaxRows = 0x7fffffff - kTileRows;   // row numbers of the last tile stay in an int

inline int tiles_of(long long rows) { return static_cast<int>((rows + kTileRows - 1) / kTileRows); }

struct ChainBytes {
    size_t tiles, groups, states, total;
};

inline ChainBytes chain_bytes(long long rows, int channels) {
    ChainBytes b{};
    const long long tiles = tiles_of(rows);
    const long long groups = (tiles + kGroup - 1) / kGroup;
    const size_t line = sizeof(unsigned long long) * channels;
    b.tiles = align_up(line * tiles);
    b.groups = align_up(line * groups);
    b.states = align_up(line * ((groups + kGroup - 1) / kGroup + 1));
    b.total = 256 + b.tiles + b.groups + b.states;
    return b;
}

template <typename T> int prepare_chain(ScanArgs<T>& p, void* workspace, size_t bytes, int32_t* status, cudaStream_t stream) {
    p.tiles = tiles_of(p.order.rows);
    p.chain.budget = wait_budget_cycles();
    p.chain.status = status;
    if (p.tiles <= 1) {
        return LAT_OK;
    }
    const ChainBytes b = chain_bytes(p.order.rows, p.channels);
    if (workspace == nullptr || bytes < b.total) {
        return fail(LAT_WORKSPACE_TOO_SMALL, "recurrence workspace is too small.");
    }
    char* base = static_cast<char*>(workspace);
    p.chain.ticket = reinterpret_cast<int*>(base);
    p.chain.tiles = reinterpret_cast<unsigned long long*>(base + 256);
    p.chain.groups = reinterpret_cast<unsigned long long*>(base + 256 + b.tiles);
    p.chain.states = reinterpret_cast<unsigned long long*>(base + 256 + b.tiles + b.groups);
    // all ones: unwritten records, and a ticket of -1
    LAT_CUDA_CHECK(cudaMemsetAsync(workspace, 0xFF, b.total, stream));
    return LAT_OK;
}

// Threads across a slab: eight vectors (a 128-byte line of the forward pass), fewer where the
// row is shorter or a smaller slab leaves fewer idle threads.
inline int slab_threads(int vectors) {
    int best = 8;
    for (int q = 8; q >= 1; q >>= 1) {
        const int slots = (vectors + q - 1) / q * q, best_slots = (vectors + best - 1) / best * best;
        if (slots < best_slots) {
            best = q;
        }
    }
    return best;
}

template <typename T, int V, int Q, bool Backward> int launch_scan(ScanArgs<T> p, cudaStream_t stream) {
    p.slabs = (p.channels + V * Q - 1) / (V * Q);
    const long long blocks = static_cast<long long>(p.tiles) * p.slabs;
    LAT_REQUIRE(blocks <= 0x7fffffffLL, "the recurrence supports at most 2^31 tiles.");
    if constexpr (Backward) {
        recurrence_backward_kernel<T, V, Q><<<static_cast<unsigned>(blocks), Q * kSegments, 0, stream>>>(p);
    } else {
        recurrence_forward_kernel<T, V, Q><<<static_cast<unsigned>(blocks), Q * kSegments, 0, stream>>>(p);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

template <typename T, bool Backward> int run_scan(const ScanArgs<T>& p, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    bool vec = p.channels % V == 0 && p.x_stride % V == 0 && p.z_stride % V == 0 && aligned_to(p.x, 16) &&
               aligned_to(p.z, 16);
    if (Backward) {
        vec = vec && p.dy_stride % V == 0 && aligned_to(p.dy, 16) && aligned_to(p.dx, 16) && aligned_to(p.dz, 16);
    } else {
        vec = vec && aligned_to(p.h, 16);
    }
    if (!vec) {
        return launch_scan<T, 1, 32, Backward>(p, stream);
    }
    // the backward pass holds twice as many values per element: half as many channels a thread
    constexpr int W = Backward ? V / 2 : V, M = V / W;
    switch (slab_threads(p.channels / V)) {
        case 8: return launch_scan<T, W, 8 * M, Backward>(p, stream);
        case 4: return launch_scan<T, W, 4 * M, Backward>(p, stream);
        case 2: return launch_scan<T, W, 2 * M, Backward>(p, stream);
        default: return launch_scan<T, W, M, Backward>(p, stream);
    }
}

// What a sequence without rows hands on: initial -> final, dfinal -> dinitial.
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
    const int code = prepare_chain(p, workspace, bytes, status, stream);
    return code != LAT_OK ? code : run_scan<T, false>(p, stream);
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
    const int code = prepare_chain(p, workspace, bytes, status, stream);
    return code != LAT_OK ? code : run_scan<T, true>(p, stream);
}

} // namespace

} // namespace lat

using namespace lat;

extern "C" {

size_t lat_recurrence_workspace_bytes(int32_t rows, int32_t channels) {
    if (rows <= kTileRows || channels <= 0) {
        return 256;
    }
    return chain_bytes(rows, channels).total;
}

int32_t lat_recurrence_tiles(int32_t rows) { return rows <= 0 ? 0 : tiles_of(rows); }

int lat_recurrence_forward(
    int32_t dtype, const void* feats, int64_t feat_row_stride, const void* gate, int64_t gate_row_stride,
    int32_t rows, int32_t channels, const int32_t* offsets, int32_t sequences, const float* initial_state,
    int32_t reverse, void* out, float* final_state, float* carries, void* workspace, size_t workspace_bytes,
    int32_t* status, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "the recurrence supports float32 and float16 tensors.");
    LAT_REQUIRE(rows >= 0 && rows <= kMaxRows && channels > 0 && feat_row_stride >= 0 && gate_row_stride >= 0,
                "feats and gate must have shape (N, C).");
    LAT_REQUIRE(sequences >= 0 && (sequences == 0 || offsets != nullptr),
                "offsets must hold one int32 entry per sequence and one more.");
    cudaStream_t stream = as_stream(stream_ptr);
    int code = hand_over(initial_state, final_state, sequences, channels, stream);
    if (code != LAT_OK || rows == 0) {
        return code;
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
    LAT_REQUIRE(sequences >= 0 && (sequences == 0 || offsets != nullptr),
                "offsets must hold one int32 entry per sequence and one more.");
    cudaStream_t stream = as_stream(stream_ptr);
    int code = hand_over(grad_final, grad_initial, sequences, channels, stream);
    if (code != LAT_OK || rows == 0) {
        return code;
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
