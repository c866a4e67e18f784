// RMS norm of queries and keys for each head and the rotation of their pairs by
// position in one pass, its backward pass, and the rotation alone.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (n w)
//   backward: g = R^T dy,  dw = sum over rows of g n,  a = g w,
//             dx = r (a - n mean(a n))
// R turns pair p of a row by the angle position[axis(p)] * inv_freq[p]; pair p is
// dims (2p, 2p + 1) when interleaved, else (p, p + P) with P pairs in all, and
// dims from 2P on are not turned.  Statistics, products and sums are fp32, the
// result is rounded once.
//
// Each kernel reads a row once and writes it once, so HBM bounds it.  A row is
// held by LP = 8, 16 or 32 lanes of 8 dims (4 pairs) each: one 16-byte load and
// store per lane and row of a two-byte type when interleaved, two of 8 bytes
// otherwise, and no exchange between lanes other than the norm's sums.  A
// workgroup takes all heads of a tile of tokens, neighbouring rows in memory
// beside each other (the heads of a token where those are closer together than
// its neighbours, else the tokens of a head), so that what it reads at a time is
// one run of memory.  The cosines and sines of the tile's tokens are formed once,
// into LDS, while its first rows are on their way, and no table is read.  The
// angle in turns is formed in fp64 (position * inv_freq loses its fraction in
// fp32 from a few thousand turns on), its fraction is rounded to fp32.
//
// Measured (a 335 MB copy reaches 5.4 TB/s on the same card): rotation of [1,40,32768,128]
// bf16 134 us, 5.0 TB/s; norm and rotation of q and k [2,16,9216,128] 59 us, 5.1 TB/s, and of
// 56 + 56 heads of 9170 tokens read in place from a fused projection 108 us, 4.9 TB/s; the
// backward pass of [2,16,9216,128] 94 us, 4.8 TB/s.  Calls of a few tokens take 4 us.
// Non-temporal loads and stores measured the same.
#include <stdlib.h>

#include "kernels.hpp"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows in flight per lane
constexpr int kTileTokens = 16;  // most tokens of a tile
constexpr int kMostPairs = 128;

// Vectors of N elements at any element alignment (global loads and stores
// need no more on gfx950).
template <typename T, int N> struct Chunk {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// The dims a lane holds: pairs (a[e], b[e]) of pair index 4 lane + e, at dims
// first + e and second + e (interleaved: 8 lane + 2e and 8 lane + 2e + 1).
struct LaneDims {
    int first, second;
};
template <bool IL> __device__ __forceinline__ LaneDims lane_dims(int lane, int pairs) {
    if (!IL && lane < pairs / 4) return LaneDims{4 * lane, pairs + 4 * lane};
    return LaneDims{8 * lane, 8 * lane + 4};
}

template <typename T, bool IL>
__device__ __forceinline__ void load_row(const T* p, LaneDims d, float (&a)[4], float (&b)[4]) {
    if constexpr (IL) {
        const auto v = *reinterpret_cast<const typename Chunk<T, 8>::type*>(p + d.first);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = to_f32(static_cast<T>(v[2 * e]));
            b[e] = to_f32(static_cast<T>(v[2 * e + 1]));
        }
    } else {
        const auto u = *reinterpret_cast<const typename Chunk<T, 4>::type*>(p + d.first);
        const auto v = *reinterpret_cast<const typename Chunk<T, 4>::type*>(p + d.second);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = to_f32(static_cast<T>(u[e]));
            b[e] = to_f32(static_cast<T>(v[e]));
        }
    }
}

template <typename T, bool IL>
__device__ __forceinline__ void store_row(T* p, LaneDims d, const float (&a)[4], const float (&b)[4]) {
    if constexpr (IL) {
        typename Chunk<T, 8>::type v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = from_f32<T>(a[e]);
            v[2 * e + 1] = from_f32<T>(b[e]);
        }
        *reinterpret_cast<typename Chunk<T, 8>::type*>(p + d.first) = v;
    } else {
        typename Chunk<T, 4>::type u, v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u[e] = from_f32<T>(a[e]);
            v[e] = from_f32<T>(b[e]);
        }
        *reinterpret_cast<typename Chunk<T, 4>::type*>(p + d.first) = u;
        *reinterpret_cast<typename Chunk<T, 4>::type*>(p + d.second) = v;
    }
}

// Norm weights of a lane's dims (1 where there is none).
template <typename T, bool IL>
__device__ __forceinline__ void load_weight(const NormRopeArgs& g, const void* w, bool live, LaneDims d,
                                            float (&a)[4], float (&b)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = b[e] = 1.0f;
    if (!w || !live) return;
    if (g.weight_f32)
        load_row<float, IL>(static_cast<const float*>(w), d, a, b);
    else
        load_row<T, IL>(static_cast<const T*>(w), d, a, b);
}

__device__ __forceinline__ double axis_position(const RopeArgs& r, int b, int t, int axis) {
    if (r.pos_kind == PISA_POSITIONS_GRID) {
        const int row = t / r.grid_w;
        return axis == 2 ? t - row * r.grid_w : axis == 1 ? row % r.grid_h : row / r.grid_h;
    }
    const int64_t o = b * r.pos_sb + t * r.pos_st + axis * r.pos_sa;
    if (r.pos_kind == PISA_POSITIONS_I32) return static_cast<const int32_t*>(r.pos)[o];
    if (r.pos_kind == PISA_POSITIONS_I64) return static_cast<double>(static_cast<const int64_t*>(r.pos)[o]);
    return static_cast<const float*>(r.pos)[o];
}

// Cosines and sines of the tile's tokens, token j's pair p at [j * kMostPairs + p].
struct Angles {
    float c[kTileTokens * kMostPairs], s[kTileTokens * kMostPairs];
};
__device__ __forceinline__ void tile_angles(const RopeArgs& r, int b, int t0, int tokens, Angles& out) {
    constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
    for (int i = threadIdx.x; i < tokens * r.pairs; i += kThreads) {
        const int j = i / r.pairs;
        const int p = i - j * r.pairs;
        const int axis = (p >= r.axis_end[0]) + (p >= r.axis_end[1]) + (p >= r.axis_end[2]);
        double turns = axis_position(r, b, t0 + j, axis) * r.inv_freq[p] * kTurn;
        turns -= __builtin_rint(turns);
        float s, c;
        sincospif(2.0f * static_cast<float>(turns), &s, &c);
        out.c[j * kMostPairs + p] = c;
        out.s[j * kMostPairs + p] = r.inverse ? -s : s;
    }
}
// Those of a lane's four pairs (one and zero past the rotated dims).
__device__ __forceinline__ void lane_angles(const Angles& a, int j, int lane, bool turned, float (&c)[4], float (&s)[4]) {
    f32x4 x = {1.0f, 1.0f, 1.0f, 1.0f}, y = {0.0f, 0.0f, 0.0f, 0.0f};
    if (turned) {
        x = *reinterpret_cast<const f32x4*>(&a.c[j * kMostPairs + 4 * lane]);
        y = *reinterpret_cast<const f32x4*>(&a.s[j * kMostPairs + 4 * lane]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c[e] = x[e];
        s[e] = y[e];
    }
}

template <int LP> __device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, LP);
    return x;
}

// A workgroup's tile: tokens t0 .. t0 + tokens - 1 of batch entry b.
struct Tile {
    int b, t0, tokens;
};
__device__ __forceinline__ Tile tile_of(const NormRopeArgs& g, int64_t tile) {
    Tile w;
    w.b = static_cast<int>(tile / g.tiles_per_batch);
    w.t0 = static_cast<int>(tile - (int64_t)w.b * g.tiles_per_batch) * g.tile_tokens;
    w.tokens = min(g.tile_tokens, g.tokens - w.t0);
    return w;
}
// Row r of a tensor's rows in the tile: its token (of the tile) and head.
struct Row {
    int j, h;
};
__device__ __forceinline__ int tile_rows(const NormRopeArgs& g, const Tile& w, int i) {
    return (g.heads_first[i] ? w.tokens : g.tile_tokens) * g.heads[i];
}
__device__ __forceinline__ Row row_of(const NormRopeArgs& g, int i, int r) {
    if (g.heads_first[i]) {  // g.inv_heads = ceil(2^32 / heads): exact for the few tokens of a tile
        const int j = g.tile_tokens == 1 ? 0 : static_cast<int>(__umulhi(r, g.inv_heads[i]));
        return Row{j, r - j * g.heads[i]};
    }
    return Row{r & (g.tile_tokens - 1), r >> g.tile_shift};
}
template <typename T> __device__ __forceinline__ const T* row_at(const View& v, const Tile& w, Row x) {
    return reinterpret_cast<const T*>(v.data) + w.b * v.sb + x.h * v.sh + (w.t0 + x.j) * v.st;
}
template <typename T> __device__ __forceinline__ T* row_at(const OutView& v, const Tile& w, Row x) {
    return reinterpret_cast<T*>(v.data) + w.b * v.sb + x.h * v.sh + (w.t0 + x.j) * v.st;
}

template <typename T, int LP, bool IL>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs g) {
    constexpr int kSlots = kThreads / LP;
    __shared__ __attribute__((aligned(16))) Angles angles;
    const int lane = threadIdx.x % LP;
    const int slot = threadIdx.x / LP;
    const bool live = 8 * lane < g.head_dim;
    const bool turned = 4 * lane < g.rope.pairs;
    const LaneDims d = live ? lane_dims<IL>(lane, g.rope.pairs) : LaneDims{0, 0};
    const float inv_d = 1.0f / static_cast<float>(g.head_dim);
    const Tile w = tile_of(g, blockIdx.x);
    float a[kUnroll][4], b[kUnroll][4];
    Row x[kUnroll];
    // rows r, r + kSlots, ... of tensor i (past the last one, or on tokens past the tile's, a row that is there)
    auto load = [&](int i, int r) __attribute__((always_inline)) {
        const int rows = tile_rows(g, w, i);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            x[u] = row_of(g, i, min(r + u * kSlots, rows - 1));
            load_row<T, IL>(row_at<T>(g.in[i], w, Row{min(x[u].j, w.tokens - 1), x[u].h}), d, a[u], b[u]);
        }
    };
    load(0, slot);  // on its way while the angles are formed
    if (g.rope.pairs) {
        tile_angles(g.rope, w.b, w.t0, w.tokens, angles);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (g.heads[i] == 0) continue;
        const int rows = tile_rows(g, w, i);
        float wa[4], wb[4];
        load_weight<T, IL>(g, g.weight[i], live, d, wa, wb);
        for (int r = slot; r < rows; r += kSlots * kUnroll) {
            if (i == 1 || r != slot) load(i, r);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float n = 1.0f;
                if (g.norm) {
                    float sq = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) sq = fmaf(a[u][e], a[u][e], fmaf(b[u][e], b[u][e], sq));
                    n = rsqrtf(fmaf(group_sum<LP>(live ? sq : 0.0f), inv_d, g.eps));
                }
                if (!live || r + u * kSlots >= rows || x[u].j >= w.tokens) continue;
                float c[4], s[4], y[4], z[4];
                lane_angles(angles, x[u].j, lane, turned, c, s);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = a[u][e] * n * wa[e], q = b[u][e] * n * wb[e];
                    y[e] = p * c[e] - q * s[e];
                    z[e] = p * s[e] + q * c[e];
                }
                store_row<T, IL>(row_at<T>(g.out[i], w, x[u]), d, y, z);
            }
        }
    }
}

// The backward pass.  Workgroups walk the tiles with the grid's stride and keep
// the weight gradients of their rows in registers; the row slots of a workgroup
// are added through LDS in order and written as one partial per workgroup
// (partial[tensor][dim][workgroup]), which norm_rope_weights_kernel sums: the
// result does not depend on the order in which workgroups run.
template <typename T, int LP, bool IL>
__global__ __launch_bounds__(kThreads) void norm_rope_backward_kernel(NormRopeArgs g) {
    constexpr int kSlots = kThreads / LP;
    constexpr int kRows = 1;  // more in flight bring nothing here, and cost waves
    __shared__ __attribute__((aligned(16))) Angles angles;
    __shared__ float lds[kSlots][LP * 8];
    const int lane = threadIdx.x % LP;
    const int slot = threadIdx.x / LP;
    const bool live = 8 * lane < g.head_dim;
    const bool turned = 4 * lane < g.rope.pairs;
    const LaneDims d = live ? lane_dims<IL>(lane, g.rope.pairs) : LaneDims{0, 0};
    const float inv_d = 1.0f / static_cast<float>(g.head_dim);
    float da[2][4], db[2][4], wa[2][4], wb[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        load_weight<T, IL>(g, g.weight[i], live, d, wa[i], wb[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) da[i][e] = db[i][e] = 0.0f;
    }
    for (int64_t tile = blockIdx.x; tile < g.tiles; tile += gridDim.x) {
        const Tile w = tile_of(g, tile);
        if (g.rope.pairs) {
            if (tile != blockIdx.x) __syncthreads();  // the last tile's angles are read
            tile_angles(g.rope, w.b, w.t0, w.tokens, angles);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (g.heads[i] == 0) continue;
            const int rows = tile_rows(g, w, i);
            for (int r = slot; r < rows; r += kSlots * kRows) {
                float a[kRows][4], b[kRows][4], y[kRows][4], z[kRows][4];
                Row x[kRows];
#pragma unroll
                for (int u = 0; u < kRows; ++u) {
                    x[u] = row_of(g, i, min(r + u * kSlots, rows - 1));
                    const Row there{min(x[u].j, w.tokens - 1), x[u].h};
                    load_row<T, IL>(row_at<T>(g.in[i], w, there), d, a[u], b[u]);
                    load_row<T, IL>(row_at<T>(g.grad[i], w, there), d, y[u], z[u]);
                }
#pragma unroll
                for (int u = 0; u < kRows; ++u) {
                    float c[4], s[4], sq = 0.0f, ax = 0.0f, pa[4], pb[4];
                    lane_angles(angles, min(x[u].j, w.tokens - 1), lane, turned, c, s);  // s is the inverse rotation's
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pa[e] = y[u][e] * c[e] - z[u][e] * s[e];
                        pb[e] = y[u][e] * s[e] + z[u][e] * c[e];
                        sq = fmaf(a[u][e], a[u][e], fmaf(b[u][e], b[u][e], sq));
                        ax = fmaf(pa[e] * wa[i][e], a[u][e], fmaf(pb[e] * wb[i][e], b[u][e], ax));
                    }
                    sq = group_sum<LP>(live ? sq : 0.0f);
                    ax = group_sum<LP>(live ? ax : 0.0f);
                    if (!live || r + u * kSlots >= rows || x[u].j >= w.tokens) continue;
                    const float n = rsqrtf(fmaf(sq, inv_d, g.eps));
                    const float m = ax * n * inv_d;  // mean(a n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float na = a[u][e] * n, nb = b[u][e] * n;
                        da[i][e] = fmaf(pa[e], na, da[i][e]);
                        db[i][e] = fmaf(pb[e], nb, db[i][e]);
                        y[u][e] = n * (pa[e] * wa[i][e] - na * m);
                        z[u][e] = n * (pb[e] * wb[i][e] - nb * m);
                    }
                    store_row<T, IL>(row_at<T>(g.out[i], w, x[u]), d, y[u], z[u]);
                }
            }
        }
    }
    if (!g.partial) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!g.weight_grad[i]) continue;
        if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lds[slot][IL ? d.first + 2 * e : d.first + e] = da[i][e];
                lds[slot][IL ? d.first + 2 * e + 1 : d.second + e] = db[i][e];
            }
        }
        __syncthreads();
        for (int dim = threadIdx.x; dim < g.head_dim; dim += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kSlots; ++j) sum += lds[j][dim];
            g.partial[((int64_t)i * g.head_dim + dim) * gridDim.x + blockIdx.x] = sum;
        }
        __syncthreads();
    }
}

// Weight gradients from the partials: one wave per dim, sums in fp64 in a fixed order.
template <typename T>
__global__ __launch_bounds__(64) void norm_rope_weights_kernel(const float* partial, int parts, int head_dim,
                                                               int weight_f32, void* dq, void* dk) {
    const int i = blockIdx.x / head_dim;
    const int dim = blockIdx.x - i * head_dim;
    void* dst = i == 0 ? dq : dk;
    if (!dst) return;
    const float* src = partial + ((int64_t)i * head_dim + dim) * parts;
    float x[kNormRopeParts / 64];  // all loads at once
#pragma unroll
    for (int j = 0; j < kNormRopeParts / 64; ++j) x[j] = (int)threadIdx.x + 64 * j < parts ? src[threadIdx.x + 64 * j] : 0.0f;
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kNormRopeParts / 64; ++j) sum += x[j];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x != 0) return;
    if (weight_f32)
        static_cast<float*>(dst)[dim] = static_cast<float>(sum);
    else
        static_cast<T*>(dst)[dim] = from_f32<T>(static_cast<float>(sum));
}

template <typename T, int LP>
int launch_lp(const NormRopeArgs& g, bool backward, hipStream_t stream) {
    const int blocks = backward ? norm_rope_parts(g) : static_cast<int>(g.tiles);
    if (backward) {
        if (g.rope.interleaved)
            hipLaunchKernelGGL((norm_rope_backward_kernel<T, LP, true>), dim3(blocks), dim3(kThreads), 0, stream, g);
        else
            hipLaunchKernelGGL((norm_rope_backward_kernel<T, LP, false>), dim3(blocks), dim3(kThreads), 0, stream, g);
        int rc = pisa_host::check_launch("norm_rope_backward_kernel");
        if (rc || !g.partial) return rc;
        hipLaunchKernelGGL((norm_rope_weights_kernel<T>), dim3(2 * g.head_dim), dim3(64), 0, stream, g.partial, blocks,
                           g.head_dim, g.weight_f32, g.weight_grad[0], g.weight_grad[1]);
        return pisa_host::check_launch("norm_rope_weights_kernel");
    }
    if (g.rope.interleaved)
        hipLaunchKernelGGL((norm_rope_kernel<T, LP, true>), dim3(blocks), dim3(kThreads), 0, stream, g);
    else
        hipLaunchKernelGGL((norm_rope_kernel<T, LP, false>), dim3(blocks), dim3(kThreads), 0, stream, g);
    return pisa_host::check_launch("norm_rope_kernel");
}

template <typename T>
int launch_t(const NormRopeArgs& g, bool backward, hipStream_t stream) {
    switch (norm_rope_lanes(g.head_dim)) {
        case 8: return launch_lp<T, 8>(g, backward, stream);
        case 16: return launch_lp<T, 16>(g, backward, stream);
        default: return launch_lp<T, 32>(g, backward, stream);
    }
}

}  // namespace

// Lanes that hold a row.
int norm_rope_lanes(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }

// Tiles of up to 16 tokens (a power of two): a workgroup's slots get eight rows each
// as long as that leaves two workgroups to a CU, and more as long as it leaves
// sixteen.  Tiles of one token, which leave more workgroups, and these, us:
// [2,10,4001,80] fp32 25.4 and 13.0, 8 + 2 heads of [1,4096,128] 16.6 and 9.2; a larger
// tile of [2,16,9216,128], q and k, 56.2 and 59.4.
void norm_rope_split(NormRopeArgs& g) {
    constexpr int64_t kMany = 4096, kFew = 512;
    const int64_t tokens = (int64_t)g.batch * g.tokens;
    const int heads = g.heads[0] + g.heads[1];
    const int rows = 8 * (kThreads / norm_rope_lanes(g.head_dim));
    g.tile_tokens = 1;
    g.tile_shift = 0;
    while (g.tile_tokens < kTileTokens && heads <= 4096 &&
           tokens >= 2 * g.tile_tokens * (heads * g.tile_tokens < rows ? kFew : kMany)) {
        g.tile_tokens *= 2;
        ++g.tile_shift;
    }
    g.tiles_per_batch = (g.tokens + g.tile_tokens - 1) / g.tile_tokens;
    g.tiles = (int64_t)g.batch * g.tiles_per_batch;
    for (int i = 0; i < 2; ++i) {
        // the smaller step in memory first
        g.heads_first[i] = g.heads[i] > 1 && llabs(g.in[i].sh) <= llabs(g.in[i].st);
        g.inv_heads[i] = g.heads[i] > 1 ? static_cast<uint32_t>(((int64_t(1) << 32) + g.heads[i] - 1) / g.heads[i]) : 0;
    }
}

// Workgroups of the backward pass: at most four per CU, which leaves one
// partial weight gradient each.
int norm_rope_parts(const NormRopeArgs& g) { return static_cast<int>(g.tiles < kNormRopeParts ? g.tiles : kNormRopeParts); }

int launch_norm_rope(int dtype, const NormRopeArgs& g, bool backward, hipStream_t stream) {
    if (dtype == PISA_DTYPE_BF16) return launch_t<bf16_t>(g, backward, stream);
    if (dtype == PISA_DTYPE_F16) return launch_t<f16_t>(g, backward, stream);
    return launch_t<float>(g, backward, stream);
}

}  // namespace pisa
