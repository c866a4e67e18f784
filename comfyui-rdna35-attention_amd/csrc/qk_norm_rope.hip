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
// otherwise, and no exchange between lanes other than the norm's sums.  A group of LP lanes takes
// `rows_per_group` heads of one token, so the cosines and sines of a lane's
// four pairs are formed once for all of them and no table is read.  The angle in
// turns is formed in fp64 (position * inv_freq loses its fraction in fp32 from a
// few thousand turns on), its fraction is rounded to fp32.
#include "kernels.hpp"

namespace pisa {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows in flight per lane

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

// Cosine and sine of the lane's four pairs at token (b, t).
__device__ __forceinline__ void lane_angles(const RopeArgs& r, int b, int t, int lane, float (&c)[4], float (&s)[4]) {
    constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int p = 4 * lane + e;
        c[e] = 1.0f;
        s[e] = 0.0f;
        if (p < r.pairs) {
            const int axis = (p >= r.axis_end[0]) + (p >= r.axis_end[1]) + (p >= r.axis_end[2]);
            double turns = axis_position(r, b, t, axis) * r.inv_freq[p] * kTurn;
            turns -= __builtin_rint(turns);
            sincospif(2.0f * static_cast<float>(turns), &s[e], &c[e]);
            if (r.inverse) s[e] = -s[e];
        }
    }
}

template <int LP> __device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, LP);
    return x;
}

// A group's token and its heads [h0, h1) of tensor i (0: queries, 1: keys).
struct GroupWork {
    int b, t, row0, row1;
};
__device__ __forceinline__ GroupWork group_work(const NormRopeArgs& g, int64_t group) {
    const int64_t token = group / g.groups_per_token;
    const int part = static_cast<int>(group - token * g.groups_per_token);
    GroupWork w;
    w.b = static_cast<int>(token / g.tokens);
    w.t = static_cast<int>(token - (int64_t)w.b * g.tokens);
    w.row0 = part * g.rows_per_group;
    w.row1 = min(w.row0 + g.rows_per_group, g.heads[0] + g.heads[1]);
    return w;
}

template <typename T, int LP, bool IL>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs g) {
    const int lane = threadIdx.x % LP;
    const bool live = 8 * lane < g.head_dim;
    const LaneDims d = live ? lane_dims<IL>(lane, g.rope.pairs) : LaneDims{0, 0};
    const float inv_d = 1.0f / static_cast<float>(g.head_dim);
    // whole groups enter and leave the loop: no lane of a group's sums is missing
    for (int64_t group = (int64_t)blockIdx.x * (kThreads / LP) + threadIdx.x / LP; group < g.groups;
         group += (int64_t)gridDim.x * (kThreads / LP)) {
        const GroupWork w = group_work(g, group);
        float c[4], s[4];
        lane_angles(g.rope, w.b, w.t, lane, c, s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int h0 = i == 0 ? w.row0 : max(w.row0 - g.heads[0], 0);
            const int h1 = i == 0 ? min(w.row1, g.heads[0]) : w.row1 - g.heads[0];
            if (h0 >= h1) continue;
            float wa[4], wb[4];
            load_weight<T, IL>(g, g.weight[i], live, d, wa, wb);
            const T* src = reinterpret_cast<const T*>(g.in[i].data) + w.b * g.in[i].sb + w.t * g.in[i].st;
            T* dst = reinterpret_cast<T*>(g.out[i].data) + w.b * g.out[i].sb + w.t * g.out[i].st;
            for (int h = h0; h < h1; h += kUnroll) {
                float a[kUnroll][4], b[kUnroll][4];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)  // rows past the last re-read it
                    load_row<T, IL>(src + min(h + u, h1 - 1) * g.in[i].sh, d, a[u], b[u]);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    float r = 1.0f;
                    if (g.norm) {
                        float sq = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) sq = fmaf(a[u][e], a[u][e], fmaf(b[u][e], b[u][e], sq));
                        r = 1.0f / sqrtf(fmaf(group_sum<LP>(live ? sq : 0.0f), inv_d, g.eps));
                    }
                    if (!live || h + u >= h1) continue;
                    float x[4], y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = a[u][e] * r * wa[e], q = b[u][e] * r * wb[e];
                        x[e] = p * c[e] - q * s[e];
                        y[e] = p * s[e] + q * c[e];
                    }
                    store_row<T, IL>(dst + (h + u) * g.out[i].sh, d, x, y);
                }
            }
        }
    }
}

// The backward pass.  Workgroups walk the groups with the grid's stride and keep
// the weight gradients of their rows in registers; the row slots of a workgroup
// are added through LDS in order and written as one partial per workgroup
// (partial[tensor][dim][workgroup]), which norm_rope_weights_kernel sums: the
// result does not depend on the order in which workgroups run.
template <typename T, int LP, bool IL>
__global__ __launch_bounds__(kThreads) void norm_rope_backward_kernel(NormRopeArgs g) {
    constexpr int kSlots = kThreads / LP;
    constexpr int kRows = 2;  // two tensors to read: as many loads in flight as the forward kernel
    __shared__ float lds[kSlots][LP * 8];
    const int lane = threadIdx.x % LP;
    const int slot = threadIdx.x / LP;
    const bool live = 8 * lane < g.head_dim;
    const LaneDims d = live ? lane_dims<IL>(lane, g.rope.pairs) : LaneDims{0, 0};
    const float inv_d = 1.0f / static_cast<float>(g.head_dim);
    float da[2][4], db[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) da[i][e] = db[i][e] = 0.0f;
    for (int64_t group = (int64_t)blockIdx.x * kSlots + slot; group < g.groups; group += (int64_t)gridDim.x * kSlots) {
        const GroupWork w = group_work(g, group);
        float c[4], s[4];
        lane_angles(g.rope, w.b, w.t, lane, c, s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int h0 = i == 0 ? w.row0 : max(w.row0 - g.heads[0], 0);
            const int h1 = i == 0 ? min(w.row1, g.heads[0]) : w.row1 - g.heads[0];
            if (h0 >= h1) continue;
            float wa[4], wb[4];
            load_weight<T, IL>(g, g.weight[i], live, d, wa, wb);
            const T* src = reinterpret_cast<const T*>(g.in[i].data) + w.b * g.in[i].sb + w.t * g.in[i].st;
            const T* grad = reinterpret_cast<const T*>(g.grad[i].data) + w.b * g.grad[i].sb + w.t * g.grad[i].st;
            T* dst = reinterpret_cast<T*>(g.out[i].data) + w.b * g.out[i].sb + w.t * g.out[i].st;
            for (int h = h0; h < h1; h += kRows) {
                float a[kRows][4], b[kRows][4], x[kRows][4], y[kRows][4];
#pragma unroll
                for (int u = 0; u < kRows; ++u) {
                    const int hu = min(h + u, h1 - 1);
                    load_row<T, IL>(src + hu * g.in[i].sh, d, a[u], b[u]);
                    load_row<T, IL>(grad + hu * g.grad[i].sh, d, x[u], y[u]);
                }
#pragma unroll
                for (int u = 0; u < kRows; ++u) {
                    float sq = 0.0f, ax = 0.0f, pa[4], pb[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pa[e] = x[u][e] * c[e] - y[u][e] * s[e];  // s is the inverse rotation's
                        pb[e] = x[u][e] * s[e] + y[u][e] * c[e];
                        sq = fmaf(a[u][e], a[u][e], fmaf(b[u][e], b[u][e], sq));
                        ax = fmaf(pa[e] * wa[e], a[u][e], fmaf(pb[e] * wb[e], b[u][e], ax));
                    }
                    sq = group_sum<LP>(live ? sq : 0.0f);
                    ax = group_sum<LP>(live ? ax : 0.0f);
                    if (!live || h + u >= h1) continue;
                    const float r = 1.0f / sqrtf(fmaf(sq, inv_d, g.eps));
                    const float m = ax * r * inv_d;  // mean(a n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float na = a[u][e] * r, nb = b[u][e] * r;
                        da[i][e] = fmaf(pa[e], na, da[i][e]);
                        db[i][e] = fmaf(pb[e], nb, db[i][e]);
                        x[u][e] = r * (pa[e] * wa[e] - na * m);
                        y[u][e] = r * (pb[e] * wb[e] - nb * m);
                    }
                    store_row<T, IL>(dst + (h + u) * g.out[i].sh, d, x[u], y[u]);
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
    double sum = 0.0;
    for (int j = threadIdx.x; j < parts; j += 64) sum += partial[((int64_t)i * head_dim + dim) * parts + j];
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
    constexpr int64_t kMostBlocks = int64_t(1) << 20;  // more groups are walked with the grid's stride
    const int64_t need = (g.groups + kThreads / LP - 1) / (kThreads / LP);
    const int blocks = backward ? norm_rope_parts(g) : static_cast<int>(need < kMostBlocks ? need : kMostBlocks);
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

// A group takes as many of a token's rows as leave about eight waves per SIMD:
// the angles of a token cost about as much as two of its rows.
void norm_rope_split(NormRopeArgs& g) {
    constexpr int64_t kWaves = 8 * 1024;
    const int rows = g.heads[0] + g.heads[1];
    const int64_t tokens = (int64_t)g.batch * g.tokens;
    const int64_t want = kWaves * (64 / norm_rope_lanes(g.head_dim));
    int64_t per_token = (want + tokens - 1) / tokens;
    if (per_token > rows) per_token = rows;
    g.rows_per_group = static_cast<int>((rows + per_token - 1) / per_token);
    g.groups_per_token = (rows + g.rows_per_group - 1) / g.rows_per_group;
    g.groups = tokens * g.groups_per_token;
}

// Workgroups of the backward pass: at most four per CU, which leaves one
// partial weight gradient each.
int norm_rope_parts(const NormRopeArgs& g) {
    const int64_t slots = kThreads / norm_rope_lanes(g.head_dim);
    const int64_t blocks = (g.groups + slots - 1) / slots;
    return static_cast<int>(blocks < kNormRopeParts ? blocks : kNormRopeParts);
}

int launch_norm_rope(int dtype, const NormRopeArgs& g, bool backward, hipStream_t stream) {
    if (dtype == PISA_DTYPE_BF16) return launch_t<bf16_t>(g, backward, stream);
    if (dtype == PISA_DTYPE_F16) return launch_t<f16_t>(g, backward, stream);
    return launch_t<float>(g, backward, stream);
}

}  // namespace pisa
