// The backward pass of exact attention: gradients of q, k and v from those of
// the output, with the probabilities formed again from the rows' log sums.
//
//   S = scale q k^T,  P = exp(S - L),  dV = P^T dO,  dP = dO V^T,
//   dS = P (dP - delta),  delta_i = sum_d dO_id O_id,
//   dQ = scale dS K,  dK = scale dS^T Q
//
// Three launches: attention_backward_pack_kernel writes the operands in units of
// 32 rows, attention_backward_kernel forms dK and dV (backward_kv, four products)
// and dQ (backward_q, three), attention_backward_join_kernel adds the fp32 parts of
// tiles whose streamed side was split (none in a large problem).  S and dP are
// formed twice: with all five distinct products in one loop, dQ would be summed
// over key tiles by fp32 atomics, in an order (and with results) that change from
// run to run, or dS (heads x Tq x Tk) written out and read again.
//
// Both parts are one scheme.  A wave owns 32 N columns (keys or query rows)
// whose operands it holds in registers as B operands, and streams the other
// side in units of 32 rows through LDS, shared by the workgroup's four waves:
//     X[row][column] = sum_d A[row][d] B[column][d]          (S and dP)
//     G[dim][column] += sum_row A^T[dim][row] X[row][column]   (dK, dV, dQ)
// The accumulator of the first product is the B operand of the second as it
// stands (32x32x16: a lane holds one column), with the streamed rows in
// swap23 order: no probability passes through LDS.  A unit is one contiguous run
// of memory, copied to LDS without passing through registers, two units ahead;
// rows and columns are both read from it without bank conflicts.  (Packing the
// columns as well, for 16-byte reads of both, took 111 us instead of 67 for
// [2,16,9216,128] against 512 keys, and the main launch 3 to 10 % longer.)  One wave
// per SIMD: the gradients (256 registers at width 128) and own operands fill the
// register file.  The order of products, LDS reads and vector instructions is
// fixed in the source (unrolled, sched_barrier): left to the compiler's scheduler,
// registers spill or reads stand right before their use.  Per 32x32 tile of the
// scores at width 128 the matrix core works 1024 (dK, dV) or 768 (dQ) cycles;
// each fragment read from LDS feeds two tiles.
//
// What bounds it: the matrix cores at the clock that their power leaves.
// [2,16,9216,128] bf16 (seven products, 4.87 TFLOP): 3790 us = 1285 TFLOP/s, on a
// card where an 8192^3 bf16 library product reaches 1214; the matrix cores are busy in 60 %
// of the cycles, at 1.84 GHz.  The pack (115 us there) is memory bound: 690 MB at 6.0 TB/s.
// Small problems are bound by the chain of launches: [1,8,1000,64] 5 (pack) + 19 + 6 (join) us.
//
// A gradient dL of the log sums adds P dL to dS: delta - dL takes delta's place.
// -L (in log2 units) and dL - delta travel with the query rows; the latter is
// the starting value of dP's accumulator.  Packed rows past the end are zero and
// have -L = -infinity, so they add nothing.  Masked keys are packed as zero, get
// probability 0 in the dQ kernel and zero gradients in the other.
//
// Rounding: P and dS are rounded to the input type for the second product (as
// P is in the forward pass); everything else is fp32.  In fp16 both would lose
// their bits to its small range: P is scaled by 2^15, and dS by a power of two
// from the bound |dP - delta + dL| <= 2 max_i |dO_i| max_j |V_j| + max_i |dL_i| of the head, which
// puts its largest possible value just under 2^15; the gradients are scaled back in fp32.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "kernels.hpp"

namespace pisa {

namespace {

constexpr int kWaves = 4;       // waves of a workgroup, sharing the streamed units
constexpr int kUnit = 32;       // streamed rows per step
// Fragments read from LDS ahead of their use, a divisor of those of a unit (4 KT and 3 KT):
// deeper rings measured the same, one of 3 in backward_kv up to 8 % slower.
constexpr int kKvAhead = 4, kQAhead = 6;
constexpr float kShift16 = 15;  // log2 of the factor on P in fp16

template <typename T> constexpr bool kScaled = std::is_same<T, f16_t>::value;

// A unit is two operands of 32 rows (query side Q and dO, key side K and V) as
// D/16 fragments of 1 KB, 16 dims of all rows each: the even ones, 128 bytes, the
// odd ones.  The 128 bytes hold -L (beside Q) and dL - delta (beside dO) of the
// rows, and put fragments 2m and 2m + 1 into different LDS banks.  Both forms of
// an operand are read from it without bank conflicts: rows (A of the first
// product) with one 16-byte read of a lane, columns (A of the second) with two
// transposing 8-byte reads.
template <int D> constexpr int kOperand = D * 64 + 128;  // bytes
template <int D> constexpr int kGap = D * 32;            // of the 128 bytes between the even and the odd fragments
template <int D> constexpr int kUnitFrags = D / 8 + 1;   // 1 KB pieces of a unit
template <int D> constexpr int kUnitBytes = kUnitFrags<D> * 1024;
// Byte in an operand of fragment t's lane 0, and of a lane in its fragment: dims 8 half .. of a row.
template <int D> __host__ __device__ constexpr int frag_at(int t) { return t / 2 * 1024 + (t & 1) * (kGap<D> + 128); }
__host__ __device__ constexpr int lane_at(int half, int row) { return half * 512 + (row ^ (4 * half)) * 16; }
// What lane l points a transposing read at for dims 32 md .. and rows 16 s + 8 u +
// 4 (l / 32) .., less md * 1024 + s * 256 + u * 128.  The 16 lanes of a group read
// 4 rows of 16 dims; lane i of them receives dim i of the 4 rows.
template <int D> __device__ __forceinline__ int transposing_at(int lane) {
    const int j = lane & 15;
    return frag_at<D>((lane >> 4) & 1) + lane_at((j >> 1) & 1, 4 * (lane >> 5) + (j >> 2)) + (j & 1) * 8;
}

// Columns per wave / 32.  Two use a fragment read from LDS twice; above 128 the
// accumulators and own operands of 64 columns do not fit 512 registers.
template <int D> constexpr int columns() { return D <= 128 ? 2 : 1; }
// At width 128 the values of a wave's second 32 keys stay in LDS (read again for
// every unit): with them the kernel would need more than 512 registers.
template <int D> constexpr bool kValuesInLds = D == 128;

// ---------------------------------------------------------------- packing
// One 64-row block of X into an operand of two units, in 16-byte pieces: a wave
// reads whole rows and writes runs of 16 bytes by its number of rows, which the
// next rows' continue.  Rows from `live` on and dims from d_real on are zero.  With
// y, red[0][row][piece] receives the pieces of sum_d X Y; with `squares`,
// red[1][row][piece] those of sum_d X^2.
template <int D> struct PackLds {
    float red[2][kBlock][D / 8 + 1];
};

template <typename T, int D>
__device__ __forceinline__ void pack_block(PackLds<D>& lds, const char* x, int64_t st, const char* y, int64_t yst,
                                           int live, int last, int d_real, char* units, bool squares) {
    typedef typename Elem<T>::vec8 vec8;
    constexpr int kPieces = D / 8;
    constexpr int kGroups = 256 / kPieces;
    constexpr int kBatch = (kBlock + kGroups - 1) / kGroups;
    const int t = threadIdx.x;
    const int pc = t % kPieces;
    const int r0 = t / kPieces;
    const bool live_d = pc * 8 < d_real;
    const int dc = live_d ? pc * 8 : 0;
    if (r0 < kGroups) {
        vec8 xv[kBatch], yv[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {  // rows past the end read the last one
            const int r = min(r0 + i * kGroups, last);
            xv[i] = load8<vec8>(x + (r * st + dc) * (int64_t)sizeof(T));
            if (y) yv[i] = load8<vec8>(y + (r * yst + dc) * (int64_t)sizeof(T));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kGroups;
            if (r >= kBlock) break;
            if (r >= live || !live_d) {
#pragma unroll
                for (int e = 0; e < 8; ++e) xv[i][e] = T(0.0f);
                if (y) yv[i] = xv[i];
            }
            store8(units + (r >> 5) * kUnitBytes<D> + frag_at<D>(pc >> 1) + lane_at(pc & 1, r & 31), xv[i]);
            float dot = 0.0f, sq = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = to_f32(xv[i][e]);
                if (y) dot = fmaf(f, to_f32(yv[i][e]), dot);
                sq = fmaf(f, f, sq);
            }
            if (y) lds.red[0][r][pc] = dot;
            if (squares) lds.red[1][r][pc] = sq;
        }
    }
    __syncthreads();
}

// Largest sqrt of the rows' sums of squares, by the first wave.
template <int D> __device__ __forceinline__ float largest_row(const PackLds<D>& lds) {
    float s = 0.0f;
    for (int j = 0; j < D / 8; ++j) s += lds.red[1][threadIdx.x][j];
    s = sqrtf(s);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = fmaxf(s, __shfl_xor(s, o));
    return s;
}

// One workgroup per 64-row block of one tensor: dO (with O), Q, K, V.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_backward_pack_kernel(BackwardArgs a) {
    __shared__ PackLds<D> lds;
    const int q_blocks = a.q_units / 2, kv_blocks = a.kv_units / 2;
    const int q_work = a.batch * a.heads * q_blocks, kv_work = a.batch * a.k.heads * kv_blocks;
    const int t = threadIdx.x;
    const bool q_side = (int)blockIdx.x < 2 * q_work;
    const int item = q_side ? blockIdx.x : blockIdx.x - 2 * q_work;
    const bool second = item >= (q_side ? q_work : kv_work);
    const int block = second ? item - (q_side ? q_work : kv_work) : item;
    const int bh = block / (q_side ? q_blocks : kv_blocks);
    const int j = block - bh * (q_side ? q_blocks : kv_blocks);
    auto rows = [&](const View& v) { return v.data + v.row(bh, (int64_t)j * kBlock) * (int64_t)sizeof(T); };
    if (q_side) {
        const int live = a.q_tokens - j * kBlock, last = live - 1;
        char* units = a.qx + ((int64_t)bh * a.q_units + 2 * j) * kUnitBytes<D>;
        if (second) {
            pack_block<T, D>(lds, rows(a.q), a.q.st, nullptr, 0, live, last, a.head_dim, units, false);
            return;
        }
        pack_block<T, D>(lds, rows(a.dout), a.dout.st, rows(a.o), a.o.st, live, last, a.head_dim,
                         units + kOperand<D>, kScaled<T>);
        if (t < kBlock) {
            float delta = 0.0f;
            for (int i = 0; i < D / 8; ++i) delta += lds.red[0][t][i];
            const bool valid = t < live;
            const int64_t at = (int64_t)bh * a.q_tokens + (int64_t)j * kBlock + t;
            const float dlse = valid && a.dlse ? a.dlse[at] : 0.0f;
            const float nl = valid ? (kScaled<T> ? kShift16 : 0.0f) - a.lse[at] * kLog2e : -__builtin_inff();
            float* stat = reinterpret_cast<float*>(units + (t >> 5) * kUnitBytes<D> + kGap<D>) + (t & 31);
            *stat = nl;
            stat[kOperand<D> / 4] = dlse - delta;
            if constexpr (kScaled<T>) {
                const float most = largest_row<D>(lds);
                float most_l = fabsf(dlse);
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) most_l = fmaxf(most_l, __shfl_xor(most_l, o));
                if (t == 0) {
                    a.q_most[(int64_t)bh * q_blocks + j] = most;
                    a.l_most[(int64_t)bh * q_blocks + j] = most_l;
                }
            }
        }
    } else {
        const int last = a.kv_tokens - j * kBlock - 1;
        const int live = a.length(bh / a.k.heads) - j * kBlock;
        char* units = a.kx + ((int64_t)bh * a.kv_units + 2 * j) * kUnitBytes<D>;
        if (!second) {
            pack_block<T, D>(lds, rows(a.k), a.k.st, nullptr, 0, live, last, a.head_dim, units, false);
            return;
        }
        pack_block<T, D>(lds, rows(a.v), a.v.st, nullptr, 0, live, last, a.head_dim, units + kOperand<D>, kScaled<T>);
        if constexpr (kScaled<T>) {
            if (t < kBlock) {
                const float most = largest_row<D>(lds);
                if (t == 0) a.v_most[(int64_t)bh * kv_blocks + j] = most;
            }
        }
    }
}

// ---------------------------------------------------------------- streaming
// f(0), f(1), ..., f(N - 1) with the index as a compile-time constant: the steps
// of a unit differ in what they overlap, and loops with bounds that depend on
// an outer unrolled index are not unrolled by the compiler.
template <class F, int... I>
__device__ __forceinline__ void unrolled(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F> __device__ __forceinline__ void unrolled(F&& f) {
    unrolled(f, std::make_integer_sequence<int, N>{});
}

// Waits until this wave's copies and LDS reads have landed, then for the other
// waves.  One asm block, and a compiler barrier: no LDS access moves across it.
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// This wave's share of a unit's copy to LDS (fragments wave, wave + 4, ...; past
// the last fragment the last one again, so that every wave has as many in flight).
// As lds_copy16, with the source address as a scalar base and a lane offset: no
// vector register or instruction per copy.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int FRAGS>
__device__ __forceinline__ void copy_unit(const char* src, uint32_t lds_base, int wave, uint32_t lane_off) {
#pragma unroll
    for (int j = 0; j < (FRAGS + kWaves - 1) / kWaves; ++j) {
        const int f = min(wave + kWaves * j, FRAGS - 1);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :
                     : "v"(lane_off), "s"(src + f * 1024), "s"(lds_base + f * 1024)
                     : "memory", "m0");
    }
}
#pragma clang diagnostic pop

// Pins the own operands to AGPRs (an empty asm with an "a" operand): the matrix
// core reads its B operand there directly, and the architectural registers are
// left to what the vector instructions touch.
template <typename V, int N, int KT> __device__ __forceinline__ void pin_all(V (&frags)[N][KT]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            f32x4 x = __builtin_bit_cast(f32x4, frags[n][t]);
            asm volatile("" : "+a"(x));
            frags[n][t] = __builtin_bit_cast(V, x);
        }
}

template <typename V> __device__ __forceinline__ V lds_frag(const lds_char* p) {
    return __builtin_bit_cast(V, *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(p));
}

// A fragment of columns: rows 16 s + 8 u + 4 half .. (u = 0, 1) of a lane's dim
// (swap23 order), p at transposing_at.
template <typename V> __device__ __forceinline__ V lds_columns(const lds_char* p) {
    typedef short vec4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) vec4 lds_vec4;
    const vec4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec4*)p);
    const vec4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec4*)(p + 128));
    return __builtin_bit_cast(V, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// log2 of the factor on dS in fp16: of the largest power of two that keeps
// `bound` below 2^15 (0 if the bound is zero or not finite).
__device__ __forceinline__ float shift_of(float bound) {
    if (!(bound > 0.0f) || bound == __builtin_inff()) return 0.0f;
    const int exponent = min(max(14 - ilogbf(bound), -60), 60);
    return static_cast<float>(__builtin_amdgcn_readfirstlane(exponent));
}

// The largest of each of three arrays by the whole workgroup, combined into
// dS's bound, the same in every thread.
__device__ __forceinline__ float bound_of(const float* most_o, int n_o, const float* most_v, int n_v, const float* most_l,
                                          float (*scratch)[kWaves]) {
    float m[3] = {0.0f, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < n_o; i += 64 * kWaves) {
        m[0] = fmaxf(m[0], most_o[i]);
        m[2] = fmaxf(m[2], most_l[i]);
    }
    for (int i = threadIdx.x; i < n_v; i += 64 * kWaves) m[1] = fmaxf(m[1], most_v[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < 3; ++j) m[j] = fmaxf(m[j], __shfl_xor(m[j], o));
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int j = 0; j < 3; ++j) scratch[j][threadIdx.x >> 6] = m[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 3; ++j) m[j] = fmaxf(fmaxf(scratch[j][0], scratch[j][1]), fmaxf(scratch[j][2], scratch[j][3]));
    return fmaf(2.0f * m[0], m[1], m[2]);
}

// Stores 32 dims of one row per lane pair: x[v] is dim 8(v/4) + 4half + v%4 of
// the lane's column; a swap of the lane halves makes 16-byte stores.
template <typename T> __device__ __forceinline__ void store_tile(T* row, int d0, int d_real, const f32x16& x, int half) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    u32x2 w[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const vec4 y = {from_f32<T>(x[4 * g]), from_f32<T>(x[4 * g + 1]), from_f32<T>(x[4 * g + 2]), from_f32<T>(x[4 * g + 3])};
        w[g] = __builtin_bit_cast(u32x2, y);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        u32x4 y;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const auto r = __builtin_amdgcn_permlane32_swap(w[2 * p][j], w[2 * p + 1][j], false, false);
            y[j] = r[0];
            y[2 + j] = r[1];
        }
        const int d = d0 + 8 * (2 * p + half);
        if (d < d_real) *reinterpret_cast<u32x4*>(row + d) = y;
    }
}

// The tiles of a launch (kWaves N units of one head each): the first `whole` are
// one workgroup each, the streamed side of the `rest` is split over `parts`
// workgroups.  Consecutive workgroups of an XCD take neighbouring tiles of a
// head, which stream the same units.
struct TileWork {
    int tile, part, parts, slot;  // slot: place among the fp32 parts (-1: whole)
};
__device__ __forceinline__ TileWork tile_work(const BackwardTiles& p, int index) {
    if (index < p.whole) return TileWork{xcd_remap(index, p.whole), 0, 1, -1};
    const int item = xcd_remap(index - p.whole, p.rest * p.parts);
    const int part = item / p.rest, t = item - part * p.rest;
    return TileWork{p.whole + t, part, p.parts, p.parts > 1 ? item : -1};
}

// The gradient of one 32-column unit: to its rows, or, where the streamed side
// is split over several workgroups, in fp32 to this part's slot (summed in order
// by attention_backward_join_kernel).  Element (lane, v) of tile md of a slot is at
// ((md * 4 + v / 4) * 64 + lane) * 4 + v % 4.
template <typename T, int MD>
__device__ __forceinline__ void store_unit(const f32x16 (&g)[MD], float factor, bool live, float* slot, T* row, bool inside,
                                           int d_real, int lane) {
#pragma unroll
    for (int md = 0; md < MD; ++md) {
        f32x16 x;
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = live ? g[md][v] * factor : 0.0f;
        if (slot) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 y = {x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                *reinterpret_cast<f32x4*>(slot + ((md * 4 + q) * 64 + lane) * 4) = y;
            }
        } else if (inside) {  // lanes l and l + 32 (one row) take the same branch
            store_tile<T>(row, md * 32, d_real, x, lane >> 5);
        }
    }
}

// Sums the parts of the split tiles in order and stores their rows; one wave per
// (tensor, tile, unit of the tile, 32 dims): dK, dV, then dQ.
template <typename T, int MD, int UNITS>
__global__ __launch_bounds__(64) void attention_backward_join_kernel(BackwardArgs a) {
    const int lane = threadIdx.x;
    const int md = blockIdx.x % MD;
    int work = blockIdx.x / MD;
    const int u = work % UNITS;
    work /= UNITS;
    const int kv_rest = a.kv_tiles.parts > 1 ? a.kv_tiles.rest : 0;
    const bool q_side = work >= 2 * kv_rest;
    const BackwardTiles& p = q_side ? a.q_tiles : a.kv_tiles;
    work -= q_side ? 2 * kv_rest : 0;
    const int tensor = work / p.rest, t = work - tensor * p.rest;
    const int bh = (p.whole + t) / p.per_head;
    const int unit = ((p.whole + t) - bh * p.per_head) * UNITS + u;
    if (unit >= (q_side ? a.q_units : a.kv_units)) return;
    const int64_t slots = (int64_t)p.rest * UNITS * MD * 1024;  // floats of one part of one tensor
    const float* src = (q_side ? a.q_part : a.kv_part) + tensor * p.parts * slots +
                       (((int64_t)t * UNITS + u) * MD + md) * 1024 + lane * 4;
    f32x16 x;
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = 0.0f;
    constexpr int kBatch = 4;  // parts whose loads go out together
    for (int i0 = 0; i0 < p.parts; i0 += kBatch) {
        f32x4 y[kBatch][4];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                y[i][q] = *reinterpret_cast<const f32x4*>(src + min(i0 + i, p.parts - 1) * slots + q * 256);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (i0 + i < p.parts)
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] += y[i][v / 4][v % 4];
    }
    const OutView& out = q_side ? a.dq : tensor == 0 ? a.dk : a.dv;
    const int token = unit * kUnit + (lane & 31);
    if (token < (q_side ? a.q_tokens : a.kv_tokens))
        store_tile<T>(reinterpret_cast<T*>(out.data) + out.row(bh, token), md * 32, a.head_dim, x, lane >> 5);
}

// LDS of a workgroup: the streamed units, at width 128 a part of the wave's own
// values (kValuesInLds), and a few words to share.
constexpr int kKvStages = 3;  // the unit in use and two on their way
constexpr int kQStages = 4;   // and the unit before, whose columns are read
template <int D> constexpr int kv_lds_bytes() {
    return kKvStages * kUnitBytes<D> + (kValuesInLds<D> ? kWaves * (D / 16) * 1024 : 0);
}
template <int D> constexpr int q_lds_bytes() { return kQStages * kUnitBytes<D>; }

// ---------------------------------------------------------------- dK, dV
template <typename T, int D>
__device__ __forceinline__ void backward_kv(const BackwardArgs& a, int index, lds_char* lds, float (*scratch)[kWaves]) {
    typedef typename Elem<T>::vec8 vec8;
    constexpr int KT = D / 16, MD = D / 32, N = columns<D>(), FRAGS = kUnitFrags<D>, S = kKvStages, R = kKvAhead;
    constexpr int kBytes = kUnitBytes<D>;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const TileWork work = tile_work(a.kv_tiles, index);
    const int bh = work.tile / a.kv_tiles.per_head;
    const int tile = work.tile - bh * a.kv_tiles.per_head;
    const int batch = bh / a.k.heads;
    const int length = a.length(batch);
    const int unit0 = (tile * kWaves + wave) * N;
    const float c = a.scale_log2;

    // steps: the live query units of each of the group's heads, one after the other
    const int q_live = (a.q_tokens + kUnit - 1) / kUnit;
    const int steps = tile * kWaves * N * kUnit < length ? a.kv_group * q_live : 0;
    const int i0 = (int)((int64_t)steps * work.part / work.parts), i1 = (int)((int64_t)steps * (work.part + 1) / work.parts);
    const char* const table = a.qx + (int64_t)bh * a.kv_group * a.q_units * kBytes;  // heads bh * group ..
    auto unit_of = [&](int i) {
        i = min(i, i1 - 1);
        const int h = i / q_live;
        return table + ((int64_t)h * a.q_units + (i - h * q_live)) * kBytes;
    };

    // the first units are on their way to LDS while the own operands are read
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    if (i0 < i1) {
        copy_unit<FRAGS>(unit_of(i0), base, wave, lane * 16);
        copy_unit<FRAGS>(unit_of(i0 + 1), base + kBytes, wave, lane * 16);
    }
    static_assert(4 * KT % R == 0, "the ring goes on into the next unit");
    const int row_lane = lane_at(half, col), column_lane = transposing_at<D>(lane);
    constexpr int NV = kValuesInLds<D> ? N - 1 : N;
    lds_char* const own_v = lds + S * kBytes + wave * KT * 1024 + lane * 16;
    vec8 kf[N][KT], vf[NV][KT];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const char* own = a.kx + ((int64_t)bh * a.kv_units + min(unit0 + n, a.kv_units - 1)) * kBytes + row_lane;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            kf[n][t] = load8<vec8>(own + frag_at<D>(t));
            const vec8 x = load8<vec8>(own + kOperand<D> + frag_at<D>(t));
            if (n < NV)
                vf[n][t] = x;
            else
                *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(own_v + t * 1024) = __builtin_bit_cast(u32x4, x);
        }
    }
    float e = 0.0f;  // log2 of dS's factor
    if constexpr (kScaled<T>) {
        const int q_blocks = a.kv_group * (a.q_units / 2), kv_blocks = a.kv_units / 2;
        e = shift_of(bound_of(a.q_most + (int64_t)bh * q_blocks, q_blocks, a.v_most + (int64_t)bh * kv_blocks, kv_blocks,
                              a.l_most + (int64_t)bh * q_blocks, scratch));
    }
    const float f = __builtin_amdgcn_exp2f(e - kShift16);
    f32x16 dk[N][MD], dv[N][MD];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
            for (int v = 0; v < 16; ++v) dk[n][md][v] = dv[n][md][v] = 0.0f;

    if (i0 < i1) {
        __builtin_amdgcn_s_waitcnt(kWaitVm0);  // the own operands have landed too: only copies are in flight from here on
        wait_copies();
        // fragment used j-th: Q rows, dO rows, dO columns, Q columns
        auto fragment = [&](const lds_char* rows, const lds_char* columns, auto index) __attribute__((always_inline)) {
            constexpr int j = index, phase = j / KT, t = j % KT, at = phase == 1 || phase == 2 ? kOperand<D> : 0;
            if constexpr (phase < 2)
                return lds_frag<vec8>(rows + at + frag_at<D>(t));
            else
                return lds_columns<vec8>(columns + at + t % MD * 1024 + t / MD * 256);
        };
        vec8 ring[R];  // the next fragments, read R steps ahead
        unrolled<R>([&](auto j) __attribute__((always_inline)) { ring[j] = fragment(lds + row_lane, lds, j); });
        int buf = 0;
        for (int i = i0; i < i1; ++i) {
            const int next = buf == S - 1 ? 0 : buf + 1;
            const lds_char* const u = lds + buf * kBytes + row_lane;
            const lds_char* const uc = lds + buf * kBytes + column_lane;
            const lds_char* const un = lds + next * kBytes + row_lane;
            const lds_char* const stat = lds + buf * kBytes + kGap<D> + half * 16;
            pin_all(vf);
            f32x16 s[N], dp[N], nl, nd, zero;
            vec8 p[N][2], ds[N][2], vring[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) zero[v] = 0.0f;
            unrolled<4 * KT>([&](auto index) __attribute__((always_inline)) {
                constexpr int j = index, phase = j / KT, t = j % KT;
                const vec8 x = ring[j % R];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    if constexpr (phase == 0) s[n] = mfma32(x, kf[n][t], t == 0 ? zero : s[n]);
                    if constexpr (phase == 1) dp[n] = mfma32(x, n < NV ? vf[n][t] : vring[t % 2], t == 0 ? nd : dp[n]);
                    if constexpr (phase == 2) dv[n][t % MD] = mfma32(x, p[n][t / MD], dv[n][t % MD]);
                    if constexpr (phase == 3) dk[n][t % MD] = mfma32(x, ds[n][t / MD], dk[n][t % MD]);
                }
                if constexpr (j + R < 4 * KT)
                    ring[j % R] = fragment(u, uc, std::integral_constant<int, j + R>{});
                else
                    ring[j % R] = fragment(un, uc, std::integral_constant<int, j + R - 4 * KT>{});
                if constexpr (kValuesInLds<D> && ((phase == 0 && t >= KT - 2) || (phase == 1 && t < KT - 2)))
                    vring[t % 2] = lds_frag<vec8>(own_v + (phase == 0 ? t - (KT - 2) : t + 2) * 1024);
                if constexpr (phase == 0 && t >= KT - 4) {  // four rows of dL - delta
                    constexpr int q = t - (KT - 4);
                    const f32x4 y = lds_frag<f32x4>(stat + kOperand<D> + q * 32);
#pragma unroll
                    for (int w = 0; w < 4; ++w) nd[4 * q + w] = y[w];
                }
                if constexpr ((phase == 0 && t == KT - 1) || (phase == 1 && t == KT / 2 - 1)) {  // eight rows of -L
#pragma unroll
                    for (int q = 2 * phase; q < 2 * phase + 2; ++q) {
                        const f32x4 y = lds_frag<f32x4>(stat + q * 32);
#pragma unroll
                        for (int w = 0; w < 4; ++w) nl[4 * q + w] = y[w];
                    }
                }
                // probabilities beside the products of dP, dS beside those of dV: pairs of
                // elements in the order (rows 0-15 of each tile, then rows 16-31), from the
                // second step on (the first still waits for the last product)
                if constexpr ((phase == 1 || phase == 2) && t > 0) {
                    constexpr int from = (t - 1) * 8 * N / (KT - 1), to = t * 8 * N / (KT - 1);
                    unrolled<to - from>([&](auto offset) __attribute__((always_inline)) {
                        constexpr int y = from + offset, n = y / 4 % N, ss = y / (4 * N);
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int e = 2 * (y % 4) + w, v = 8 * ss + e;
                            if constexpr (phase == 1) {
                                s[n][v] = __builtin_amdgcn_exp2f(fmaf(s[n][v], c, nl[v]));
                                p[n][ss][e] = from_f32<T>(s[n][v]);
                            } else {
                                ds[n][ss][e] = from_f32<T>(kScaled<T> ? (s[n][v] * f) * dp[n][v] : s[n][v] * dp[n][v]);
                            }
                        }
                    });
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (j == 2 * KT - 1) {
                    // every wave is past unit i - 1, and unit i + 1 has landed: its buffer is the
                    // first one's to fill and the other may be read ahead
                    wait_copies();
                    copy_unit<FRAGS>(unit_of(i + 2), base + (buf == 0 ? S - 1 : buf - 1) * kBytes, wave, lane * 16);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            buf = next;
        }
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no copy outlives the workgroup's LDS
    }
    // at width 128 the lane is not held over the loop (its register is needed there)
    const int lane_out = kValuesInLds<D> ? __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)) : lane;
    const float kfac = a.scale * __builtin_amdgcn_exp2f(-e), vfac = kScaled<T> ? __builtin_amdgcn_exp2f(-kShift16) : 1.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int unit = unit0 + n;
        if (unit >= a.kv_units) continue;
        const int key = unit * kUnit + (lane_out & 31);
        const bool inside = key < a.kv_tokens, live = key < length;
        const int64_t at = inside ? key : 0;
        float* slot = nullptr;
        if (work.slot >= 0) slot = a.kv_part + (((int64_t)work.slot * kWaves + wave) * N + n) * MD * 1024;
        store_unit<T, MD>(dk[n], kfac, live, slot, reinterpret_cast<T*>(a.dk.data) + a.dk.row(bh, at), inside, a.head_dim, lane_out);
        if (slot) slot += (int64_t)a.kv_tiles.parts * a.kv_tiles.rest * kWaves * N * MD * 1024;
        store_unit<T, MD>(dv[n], vfac, live, slot, reinterpret_cast<T*>(a.dv.data) + a.dv.row(bh, at), inside, a.head_dim, lane_out);
    }
}

// ---------------------------------------------------------------- dQ
template <typename T, int D>
__device__ __forceinline__ void backward_q(const BackwardArgs& a, int index, lds_char* lds, float (*scratch)[kWaves]) {
    typedef typename Elem<T>::vec8 vec8;
    constexpr int KT = D / 16, MD = D / 32, N = columns<D>(), FRAGS = kUnitFrags<D>, S = kQStages, R = kQAhead;
    constexpr int kBytes = kUnitBytes<D>;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const TileWork work = tile_work(a.q_tiles, index);
    const int bh = work.tile / a.q_tiles.per_head;
    const int tile = work.tile - bh * a.q_tiles.per_head;
    const int kv_bh = bh / a.kv_group;
    const int length = a.length(bh / a.heads);
    const int unit0 = (tile * kWaves + wave) * N;
    const float c = a.scale_log2;
    const int steps = (length + kUnit - 1) / kUnit;
    const int i0 = (int)((int64_t)steps * work.part / work.parts), i1 = (int)((int64_t)steps * (work.part + 1) / work.parts);
    const char* const table = a.kx + (int64_t)kv_bh * a.kv_units * kBytes;
    auto unit_of = [&](int i) { return table + (int64_t)min(i, i1 - 1) * kBytes; };
    static_assert(3 * KT % R == 0, "the ring goes on into the next step");
    const int row_lane = lane_at(half, col), column_lane = transposing_at<D>(lane);

    const uint32_t base = (uint32_t)(uintptr_t)lds;
    auto copy_step = [&](int i, int b) { copy_unit<FRAGS>(unit_of(i), base + b * kBytes, wave, lane * 16); };
    if (i0 < i1) {
        copy_step(i0, 0);
        copy_step(i0 + 1, 1);
    }
    vec8 qf[N][KT], of[N][KT];
    float nl[N], nd[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const char* own = a.qx + ((int64_t)bh * a.q_units + min(unit0 + n, a.q_units - 1)) * kBytes;
        const float* stat = reinterpret_cast<const float*>(own + kGap<D>) + col;
        nl[n] = *stat;
        nd[n] = stat[kOperand<D> / 4];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            qf[n][t] = load8<vec8>(own + frag_at<D>(t) + row_lane);
            of[n][t] = load8<vec8>(own + kOperand<D> + frag_at<D>(t) + row_lane);
        }
    }
    float e = 0.0f;  // log2 of dS's factor
    if constexpr (kScaled<T>) {
        const int q_blocks = a.q_units / 2, kv_blocks = a.kv_units / 2;
        e = shift_of(bound_of(a.q_most + (int64_t)bh * q_blocks, q_blocks, a.v_most + (int64_t)kv_bh * kv_blocks, kv_blocks,
                              a.l_most + (int64_t)bh * q_blocks, scratch));
#pragma unroll
        for (int n = 0; n < N; ++n) nl[n] += e - kShift16;
    }
    f32x16 dq[N][MD];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
            for (int v = 0; v < 16; ++v) dq[n][md][v] = 0.0f;

    // Step i forms S and dP of unit i and adds unit i - 1 to dQ: dS of i - 1 is formed
    // beside the products of S, the probabilities of i beside those of dQ.
    if (i0 < i1) {
        __builtin_amdgcn_s_waitcnt(kWaitVm0);
        wait_copies();
        // fragment used j-th: K rows of unit i, K columns of i - 1, V rows of i
        auto fragment = [&](const lds_char* rows, const lds_char* columns, auto index) __attribute__((always_inline)) {
            constexpr int j = index, phase = j / KT, t = j % KT;
            if constexpr (phase == 1)
                return lds_columns<vec8>(columns + t % MD * 1024 + t / MD * 256);
            else
                return lds_frag<vec8>(rows + (phase == 2 ? kOperand<D> : 0) + frag_at<D>(t));
        };
        vec8 ring[R];
        unrolled<R>([&](auto j) __attribute__((always_inline)) {
            ring[j] = fragment(lds + row_lane, lds + (S - 1) * kBytes + column_lane, j);
        });
        f32x16 s[N], dp[N];
        int buf = 0;
        // first: there is no unit i - 1; last: no unit i
        auto step = [&](int i, auto is_first, auto is_last) __attribute__((always_inline)) {
            constexpr bool first = is_first, last = is_last;
            const int next = buf == S - 1 ? 0 : buf + 1;
            const lds_char* const u = lds + buf * kBytes + row_lane;
            const lds_char* const uc = lds + (buf == 0 ? S - 1 : buf - 1) * kBytes + column_lane;  // of unit i - 1
            const lds_char* const un = lds + next * kBytes + row_lane;
            const lds_char* const unc = lds + buf * kBytes + column_lane;
            pin_all(qf);
            pin_all(of);
            f32x16 sn[N], zero, start[N];
            vec8 ds[N][2];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                zero[v] = 0.0f;
#pragma unroll
                for (int n = 0; n < N; ++n) start[n][v] = nd[n];
            }
            unrolled<3 * KT>([&](auto index) __attribute__((always_inline)) {
                constexpr int j = index, phase = j / KT, t = j % KT;
                const vec8 x = ring[j % R];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    if constexpr (phase == 0 && !last) sn[n] = mfma32(x, qf[n][t], t == 0 ? zero : sn[n]);
                    if constexpr (phase == 1 && !first) dq[n][t % MD] = mfma32(x, ds[n][t / MD], dq[n][t % MD]);
                    if constexpr (phase == 2 && !last) dp[n] = mfma32(x, of[n][t], t == 0 ? start[n] : dp[n]);
                }
                if constexpr (j + R < 3 * KT)
                    ring[j % R] = fragment(u, uc, std::integral_constant<int, j + R>{});
                else if constexpr (!last)
                    ring[j % R] = fragment(un, unc, std::integral_constant<int, j + R - 3 * KT>{});
                if constexpr (phase == 0 ? !first : phase == 1 && !last && t > 0) {
                    constexpr int part = phase == 0 ? t : t - 1, parts = phase == 0 ? KT : KT - 1;
                    constexpr int from = part * 8 * N / parts, to = (part + 1) * 8 * N / parts;
                    unrolled<to - from>([&](auto offset) __attribute__((always_inline)) {
                        constexpr int y = from + offset, n = y / 4 % N, ss = y / (4 * N);
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int e = 2 * (y % 4) + w, v = 8 * ss + e;
                            if constexpr (phase == 0)
                                ds[n][ss][e] = from_f32<T>(s[n][v] * dp[n][v]);
                            else
                                sn[n][v] = __builtin_amdgcn_exp2f(fmaf(sn[n][v], c, nl[n]));
                        }
                    });
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (j == KT - 1) {
                    if (!last && (i + 1) * kUnit > length) {  // the last unit's masked keys: probability 0
                        asm volatile("");  // a branch, not selects in every step
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (i * kUnit + 8 * (v >> 2) + 4 * half + (v & 3) >= length)
#pragma unroll
                                for (int n = 0; n < N; ++n) sn[n][v] = -__builtin_inff();
                    }
                    // every wave is past step i - 1 (and unit i - 2), and unit i + 1 has landed
                    wait_copies();
                    if constexpr (!last) copy_step(i + 2, buf ^ 2);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
#pragma unroll
            for (int n = 0; n < N; ++n) s[n] = sn[n];
            buf = next;
        };
        step(i0, std::true_type{}, std::false_type{});
        for (int i = i0 + 1; i < i1; ++i) step(i, std::false_type{}, std::false_type{});
        step(i1, std::false_type{}, std::true_type{});
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    }
    const float fac = a.scale * __builtin_amdgcn_exp2f(-e);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int unit = unit0 + n;
        if (unit >= a.q_units) continue;
        const int row = unit * kUnit + col;
        const bool inside = row < a.q_tokens;
        float* slot = nullptr;
        if (work.slot >= 0) slot = a.q_part + (((int64_t)work.slot * kWaves + wave) * N + n) * MD * 1024;
        store_unit<T, MD>(dq[n], fac, true, slot, reinterpret_cast<T*>(a.dq.data) + a.dq.row(bh, inside ? row : 0), inside,
                          a.head_dim, lane);
    }
}

// Workgroups [0, kv): tiles of dK and dV; the rest: tiles of dQ.  One launch, so
// that CUs that have no tile of the first left go on with the second.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
void attention_backward_kernel(BackwardArgs a) {
    constexpr int kBytes = kv_lds_bytes<D>() > q_lds_bytes<D>() ? kv_lds_bytes<D>() : q_lds_bytes<D>();
    __shared__ __attribute__((aligned(1024))) char lds[kBytes];
    __shared__ float scratch[3][kWaves];
    const int kv = a.kv_tiles.whole + a.kv_tiles.rest * a.kv_tiles.parts;
    if ((int)blockIdx.x < kv)
        backward_kv<T, D>(a, blockIdx.x, (lds_char*)lds, scratch);
    else
        backward_q<T, D>(a, blockIdx.x - kv, (lds_char*)lds, scratch);
}

template <typename T, int D>
int launch_t(const BackwardArgs& a, hipStream_t stream) {
    constexpr int MD = D / 32, kTile = kWaves * columns<D>();
    const int bh = a.batch * a.heads, kv_bh = a.batch * a.k.heads;
    int rc;
    hipLaunchKernelGGL((attention_backward_pack_kernel<T, D>), dim3(bh * a.q_units + kv_bh * a.kv_units), dim3(256),
                       0, stream, a);
    if ((rc = pisa_host::check_launch("attention_backward_pack_kernel"))) return rc;
    auto workgroups = [](const BackwardTiles& p) { return p.whole + p.rest * p.parts; };
    hipLaunchKernelGGL((attention_backward_kernel<T, D>), dim3(workgroups(a.kv_tiles) + workgroups(a.q_tiles)),
                       dim3(64 * kWaves), 0, stream, a);
    if ((rc = pisa_host::check_launch("attention_backward_kernel"))) return rc;
    const int joined = (a.kv_tiles.parts > 1 ? 2 * a.kv_tiles.rest : 0) + (a.q_tiles.parts > 1 ? a.q_tiles.rest : 0);
    if (joined == 0) return PISA_OK;
    hipLaunchKernelGGL((attention_backward_join_kernel<T, MD, kTile>), dim3(joined * kTile * MD), dim3(64), 0, stream, a);
    return pisa_host::check_launch("attention_backward_join_kernel");
}

template <typename T>
int launch_d(int padded, const BackwardArgs& a, hipStream_t stream) {
    switch (padded) {
        case 64: return launch_t<T, 64>(a, stream);
        case 96: return launch_t<T, 96>(a, stream);
        case 128: return launch_t<T, 128>(a, stream);
        case 160: return launch_t<T, 160>(a, stream);
        case 192: return launch_t<T, 192>(a, stream);
        case 256: return launch_t<T, 256>(a, stream);
        default: return pisa_host::fail(PISA_ERR_UNSUPPORTED, "attention backward: padded head dim %d", padded);
    }
}

}  // namespace

// ---- how the tiles are split
// A tile's workgroup has a CU to itself.  The tiles of dK and dV are dispatched
// first, those of dQ as CUs become free.  Splitting the streamed side of every
// tile of a kind over several workgroups shortens the end of a launch and fills
// CUs that a small problem leaves idle; it costs a start-up and an fp32 write for
// each part and the launch that joins them.  plan_tiles takes the numbers of
// parts with the smallest estimate of the launch's end.  Costs are in quarters
// of the time of a dK, dV step at width 128 (about 0.45 us).  Unsplit and split, us, the
// joining launch included: [1,8,1000,64] 35.5 and 25, [2,16,9216,128] against 512 keys 422
// and 274, [1,16 over 4,4001,128] 736 and 421.
struct TileKind {
    int64_t tiles;  // 0: not formed
    int64_t steps;
    double step_cost, tile_bytes;
};

constexpr int kSlots = 256;        // workgroups at once
constexpr double kStart = 16.0;    // start-up and end of a workgroup
constexpr double kJoin = 18.0;     // the joining launch
constexpr double kByteCost = 1.0 / 2.25e6;

// End of a launch of m0 workgroups of cost c0 followed by m1 of cost c1, each
// taken by the slot that is free first.
static double end_of(int64_t m0, double c0, int64_t m1, double c1) {
    const int64_t rounds = m0 / kSlots, late = m0 % kSlots;  // `late` slots are free a c0 after the others
    const double t0 = rounds * c0, t1 = t0 + (late ? c0 : 0.0);
    if (m1 == 0) return t1;
    const int64_t early = kSlots - late;
    auto done = [&](double t) {  // of the second kind by time t
        return early * static_cast<int64_t>((t - t0) / c1 + 1e-9) +
               (t > t1 ? late * static_cast<int64_t>((t - t1) / c1 + 1e-9) : 0);
    };
    // the end is a multiple of c1 after t0 or t1: just below and above the even share
    const double even = (m1 * c1 + early * t0 + late * t1) / kSlots;
    double best = 1e300;
    for (int g = 0; g < 2; ++g) {
        const double from = g == 0 ? t0 : t1;
        int64_t k = static_cast<int64_t>((even - from) / c1);
        if (k < 0) k = 0;
        for (int64_t i = k; i < k + 3; ++i)
            if (done(from + i * c1) >= m1) {
                if (from + i * c1 < best) best = from + i * c1;
                break;
            }
    }
    return best > t1 ? best : t1;
}

static void plan_tiles(const TileKind& kv, const TileKind& q, int& kv_parts, int& q_parts) {
    constexpr int kMostParts = 32;
    auto most = [](const TileKind& x) {
        if (x.tiles == 0 || x.tiles >= 4 * kSlots) return 1;
        // eight steps to a part at least, and hardly more parts than fill the CUs
        const int64_t n = std::min(x.steps / 8, (kSlots + x.tiles - 1) / x.tiles + 1);
        return static_cast<int>(n < 1 ? 1 : n > kMostParts ? kMostParts : n);
    };
    double best = 1e300;
    kv_parts = q_parts = 1;
    const int kv_most = most(kv), q_most = most(q);
    for (int i = 1; i <= kv_most; ++i)
        for (int j = 1; j <= q_most; ++j) {
            const double kv_cost = (kv.steps + i - 1) / i * kv.step_cost + kStart;
            const double q_cost = (q.steps + j - 1) / j * q.step_cost + kStart;
            double cost = end_of(kv.tiles * i, kv_cost, q.tiles * j, q_cost);
            if ((kv.tiles && i > 1) || (q.tiles && j > 1)) cost += kJoin;
            // parts are written and read again
            if (i > 1) cost += 2.0 * kv.tiles * i * kv.tile_bytes * kByteCost;
            if (j > 1) cost += 2.0 * q.tiles * j * q.tile_bytes * kByteCost;
            if (cost < best) {
                best = cost;
                kv_parts = i;
                q_parts = j;
            }
        }
}

static BackwardTiles tiles_of(const TileKind& x, int per_head, int parts) {
    BackwardTiles p;
    p.per_head = per_head;
    p.whole = parts > 1 ? 0 : static_cast<int>(x.tiles);
    p.rest = parts > 1 ? static_cast<int>(x.tiles) : 0;
    p.parts = parts;
    return p;
}

BackwardPlan plan_backward(int batch, int heads, int kv_heads, int q_tokens, int kv_tokens, int padded, bool scaled,
                           bool with_q, bool with_kv) {
    BackwardPlan p;
    const int tile = kWaves * (padded <= 128 ? 2 : 1);
    p.q_units = (q_tokens + kBlock - 1) / kBlock * 2;
    p.kv_units = (kv_tokens + kBlock - 1) / kBlock * 2;
    const int64_t bh = (int64_t)batch * heads, kv_bh = (int64_t)batch * kv_heads;
    const int q_per_head = (p.q_units + tile - 1) / tile, kv_per_head = (p.kv_units + tile - 1) / tile;
    const double tile_bytes = (double)tile * padded * kUnit * sizeof(float), width = padded / 128.0 * (padded <= 128 ? 1 : 0.6);
    const TileKind kv{with_kv ? kv_bh * kv_per_head : 0, (int64_t)p.q_units * (heads / kv_heads), 4 * width, 2 * tile_bytes};
    const TileKind q{with_q ? bh * q_per_head : 0, p.kv_units, 3 * width, tile_bytes};
    int kv_parts, q_parts;
    plan_tiles(kv, q, kv_parts, q_parts);
    p.kv_tiles = tiles_of(kv, kv_per_head, kv_parts);
    p.q_tiles = tiles_of(q, q_per_head, q_parts);
    p.qx_bytes = bh * p.q_units * (padded / 8 + 1) * 1024;
    p.kx_bytes = kv_bh * p.kv_units * (padded / 8 + 1) * 1024;
    p.q_most_bytes = scaled ? bh * (p.q_units / 2) * (int64_t)sizeof(float) : 0;
    p.l_most_bytes = p.q_most_bytes;
    p.v_most_bytes = scaled ? kv_bh * (p.kv_units / 2) * (int64_t)sizeof(float) : 0;
    const int64_t part_bytes = (int64_t)tile * padded * kUnit * sizeof(float);
    p.q_part_bytes = q_parts > 1 ? q_parts * q.tiles * part_bytes : 0;
    p.kv_part_bytes = kv_parts > 1 ? 2 * kv_parts * kv.tiles * part_bytes : 0;
    return p;
}

int launch_attention_backward(int dtype, int padded, const BackwardArgs& a, hipStream_t stream) {
    if (dtype == PISA_DTYPE_BF16) return launch_d<bf16_t>(padded, a, stream);
    return launch_d<f16_t>(padded, a, stream);
}

}  // namespace pisa
