// Projection + softmax cross entropy for small problems (a policy head on a mini-batch: 512 positions, hundreds of classes),
// where launches and not arithmetic take the time: three launches, everything in float32 on the f32 matrix cores.
//
//   small_logits_kernel  l = X W^T + b to the workspace (16 MB at most), and the number of rows that count
//   small_rows_kernel    a row's statistics, loss, entropy, and D in place of its logits
//   small_grads_kernel   dX = D W, dW = D^T X, db, and the totals
//
// A workgroup makes a 32 x 32 tile of a product; its eight waves take an eighth of the sum each (blocks of 16 in turn) and
// join through LDS.  Operands come straight from memory (L2) into the fragments of v_mfma_f32_16x16x4_f32: a lane of group
// g = lane / 16 holds k = 4 g + j for the j-th of four instructions, so that where k is contiguous the four are one load.
// Bound by latency, of launches and of loads from the L2: 512 positions on 8 x 8 (256 features, 64 classes) take 5 + 4 + 8 us, on
// 15 x 15 (900, 225) 11 + 5 + 17 us; the tiled path takes 33 us and 58 us for them.
#pragma once
#include "azg_linear_ce.hpp"

namespace azgops {

constexpr int kSmallTile = 32;

struct SmallArgs {
    const void *x, *w, *bias;
    long long xs, ws;                         // row strides
    int n, H, V;
    const long long *target; long long ignore;
    const float *probs; long long ldp;
    float *logits;                            // [n][ldl]: logits, then D
    int ldl;
    float4 *stats;                            // [n]
    float *ent;                               // [n] or null
    int reduction;
    float *loss, *ent_out;                    // [n] or [1], null: not asked for
    const float *dloss; float grad_scale;
    int *count;                               // rows that count
    bool backward;
    void *dx, *dw, *db;                       // null: not asked for
    long long dxs, dws;
    int tiles_x, tiles_w;                     // workgroups of the products, then db's, then one for the totals
};

// sum over a workgroup of W waves in a fixed order, for every thread
template <int W, typename T>
__device__ inline T block_sum(T v, T *red)
{
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = red[0];
#pragma unroll
    for (int w = 1; w < W; w++) r += red[w];
    return r;
}

// Four k of one m (the caller keeps m inside): k contiguous (KC) or across rows.  WHOLE: all four exist; else zero past K.
// `skip`: null, or the targets whose rows (k) read as zero where they are `ignore`.
template <bool WHOLE, typename T, bool KC>
__device__ inline fx4 small_frag(const T *p, long long ld, int m, int k, int K, const long long *skip, long long ignore)
{
    fx4 f = {0.f, 0.f, 0.f, 0.f};
    if constexpr (KC && WHOLE) {
        const Pack<T, 4> v = *reinterpret_cast<const Pack<T, 4> *>(p + (long long)m * ld + k);
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = (float)v.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (WHOLE || k + j < K) {
                const float v = (float)(KC ? p[(long long)m * ld + k + j] : p[(long long)(k + j) * ld + m]);
                f[j] = skip && skip[k + j] == ignore ? 0.f : v;
            }
    }
    return f;
}

// A 32 x 32 tile at (m0, n0), the eight waves' parts of the sum joined through LDS; out: rows 4 wave + lane / 32 + 2 i, column
// lane & 31.  Four of a wave's blocks are on their way while four are multiplied: the loads' latency is what bounds these tiles.
constexpr int kSmallWaves = 8;
typedef float SmallLds[kSmallWaves][kSmallTile][kSmallTile + 1];
template <typename TA, bool KA, typename TB, bool KB>
__device__ inline void small_product(const TA *A, long long lda, int m0, int M, const TB *B, long long ldb, int n0, int N, int K,
                                     const long long *skip, long long ignore, SmallLds &lds, float (&out)[2])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    fx4 acc[2][2] = {{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
    constexpr int kAhead = 4, kStep = kSmallWaves * 16;
    fx4 a[kAhead][2], b[kAhead][2];
    // (rows past the end repeat the last one: they reach only results that are not stored)
    int ma[2], nb[2];
#pragma unroll
    for (int t = 0; t < 2; t++) { ma[t] = min(m0 + 16 * t + c, M - 1); nb[t] = min(n0 + 16 * t + c, N - 1); }
    auto load = [&](auto whole, int u, int k) {
        constexpr bool W = whole.value;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            a[u][t] = small_frag<W, TA, KA>(A, lda, ma[t], k + 4 * g, K, nullptr, 0);
            b[u][t] = small_frag<W, TB, KB>(B, ldb, nb[t], k + 4 * g, K, skip, ignore);
        }
    };
    auto multiply = [&](int u) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int t = 0; t < 2; t++) acc[s][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][s][j], b[u][t][j], acc[s][t], 0, 0, 0);
    };
    for (int k = wave * 16; k < K; k += kAhead * kStep) {
        // whole blocks of this turn; a block cut short by the end of K can only be its wave's last one
        const int whole = max(0, min(kAhead, (K - 16 - k) / kStep + (K - 16 >= k)));
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (u < whole) load(std::true_type{}, u, k + u * kStep);
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (u < whole) multiply(u);
        if (whole < kAhead && k + whole * kStep < K) {
            load(std::false_type{}, 0, k + whole * kStep);
            multiply(0);
        }
    }
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) lds[wave][16 * s + 4 * g + i][16 * t + c] = acc[s][t][i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = wave * 4 + (lane >> 5) + 2 * i, q = lane & 31;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kSmallWaves; w++) s += lds[w][r][q];
        out[i] = s;
    }
}

// The same for 16-bit rows of k on both sides, on the 16-bit matrix cores: blocks of 32, a lane of group g holds k = 8 g .. 8 g + 7,
// 16 bytes of any alignment.  TWO: A has more than sixteen rows.
template <typename T, bool TWO>
__device__ inline void few_product(const T *A, long long lda, int M, const T *B, long long ldb, int n0, int N, int K, SmallLds &lds, float (&out)[2])
{
    using V = typename Frag<T>::V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    constexpr int MT = TWO ? 2 : 1, kAhead = 4, kStep = kSmallWaves * 32;
    fx4 acc[2][2] = {{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
    V a[kAhead][MT], b[kAhead][2];
    const T *pa[MT], *pb[2];
#pragma unroll
    for (int t = 0; t < MT; t++) pa[t] = A + (long long)min(16 * t + c, M - 1) * lda + 8 * g;
#pragma unroll
    for (int t = 0; t < 2; t++) pb[t] = B + (long long)min(n0 + 16 * t + c, N - 1) * ldb + 8 * g;
    auto take = [&](auto whole, const T *p, int k) {
        union { Pack<T, 8> q; V v; } u;
        if constexpr (whole.value) {
            u.q = *reinterpret_cast<const Pack<T, 8> *>(p + k);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) u.q.v[j] = k + 8 * g + j < K ? p[k + j] : (T)0.f;
        }
        return u.v;
    };
    auto load = [&](auto whole, int u, int k) {
#pragma unroll
        for (int t = 0; t < MT; t++) a[u][t] = take(whole, pa[t], k);
#pragma unroll
        for (int t = 0; t < 2; t++) b[u][t] = take(whole, pb[t], k);
    };
    auto multiply = [&](int u) {
#pragma unroll
        for (int s = 0; s < MT; s++)
#pragma unroll
            for (int t = 0; t < 2; t++) acc[s][t] = Frag<T>::mfma(a[u][s], b[u][t], acc[s][t]);
    };
    for (int k = wave * 32; k < K; k += kAhead * kStep) {
        const int whole = max(0, min(kAhead, (K - 32 - k) / kStep + (K - 32 >= k)));
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (u < whole) load(std::true_type{}, u, k + u * kStep);
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (u < whole) multiply(u);
        if (whole < kAhead && k + whole * kStep < K) {
            load(std::false_type{}, 0, k + whole * kStep);
            multiply(0);
        }
    }
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) lds[wave][16 * s + 4 * g + i][16 * t + c] = acc[s][t][i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = wave * 4 + (lane >> 5) + 2 * i, q = lane & 31;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kSmallWaves; w++) s += lds[w][r][q];
        out[i] = s;
    }
}

// l[n][v]: rows of the tile are rows of X, columns are classes
template <typename T>
__global__ __launch_bounds__(kSmallWaves * 64) void small_logits_kernel(SmallArgs a)
{
    __shared__ SmallLds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tv = (a.V + kSmallTile - 1) / kSmallTile, tn = (a.n + kSmallTile - 1) / kSmallTile;
    if ((int)blockIdx.x == tv * tn) {                         // the last workgroup: how many rows count
        int s = 0;
        for (int i = tid; i < a.n; i += kSmallWaves * 64) s += a.target && a.target[i] == a.ignore ? 0 : 1;
        s = block_sum<kSmallWaves>(s, reinterpret_cast<int *>(lds));
        if (tid == 0) *a.count = s;
        return;
    }
    const int n0 = (int)blockIdx.x / tv * kSmallTile, v0 = (int)blockIdx.x % tv * kSmallTile;
    float out[2];
    small_product<T, true, T, true>(static_cast<const T *>(a.x), a.xs, n0, a.n, static_cast<const T *>(a.w), a.ws, v0, a.V, a.H, nullptr, 0, lds, out);
    const int v = v0 + (lane & 31);
    const float b = a.bias && v < a.V ? (float)static_cast<const T *>(a.bias)[v] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = n0 + wave * 4 + (lane >> 5) + 2 * i;
        if (r < a.n && v < a.V) a.logits[(long long)r * a.ldl + v] = out[i] + b;
    }
}

// The loss alone of at most 32 rows over many classes, for operands that the tiled path would have to copy first (float32, rows
// that do not start at 16 bytes): the weights are read once, as they lie, and a tile's logits leave it as the statistics of a span
// of 32 classes (rows_kernel joins them).  4 x 1892 x 50047 half precision: 50 us, 112 with a copy; 27 x 711 x 26667 float32:
// 40 us, 81 with a copy in parts.
struct FewArgs {
    const void *x, *w, *bias;
    long long xs, ws;
    int n, H, V;
    const long long *target;
    const float *probs; long long ldp;
    float2 *part; float *part_e; float2 *part_t; float *tlogit;                  // as the tiled path's
};
template <typename T>
__global__ __launch_bounds__(kSmallWaves * 64) void few_rows_kernel(FewArgs a)
{
    __shared__ SmallLds lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v0 = (int)blockIdx.x * kSmallTile, v = v0 + (lane & 31);
    float out[2];
    const T *x = static_cast<const T *>(a.x), *w = static_cast<const T *>(a.w);
    if constexpr (sizeof(T) == 4) small_product<T, true, T, true>(x, a.xs, 0, a.n, w, a.ws, v0, a.V, a.H, nullptr, 0, lds, out);
    else if (a.n > 16) few_product<T, true>(x, a.xs, a.n, w, a.ws, v0, a.V, a.H, lds, out);
    else few_product<T, false>(x, a.xs, a.n, w, a.ws, v0, a.V, a.H, lds, out);
    const float b = a.bias && v < a.V ? (float)static_cast<const T *>(a.bias)[v] : 0.f;
    auto sum32 = [](float q) {
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) q += __shfl_xor(q, s, 64);
        return q;
    };
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = wave * 4 + (lane >> 5) + 2 * i;
        const bool live = row < a.n;
        const float l = v < a.V ? out[i] + b : -INFINITY;
        float mx = l;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
        const float d = l - (mx == -INFINITY ? 0.f : mx), x = __builtin_amdgcn_exp2f(d * kLog2e);
        const float s = sum32(x), e = a.part_e ? sum32(x != 0.f ? x * d : 0.f) : 0.f;
        const float p = a.probs && live && v < a.V ? a.probs[row * a.ldp + v] : 0.f;
        const float tl = a.probs ? sum32(p != 0.f ? p * d : 0.f) : 0.f, ts = a.probs ? sum32(p) : 0.f;
        if (!live) continue;
        if (a.target && v < a.V && a.target[row] == v) a.tlogit[row] = l;
        if ((lane & 31) == 0) {
            const long long at = (long long)blockIdx.x * a.n + row;
            a.part[at] = make_float2(mx, s);
            if (a.part_e) a.part_e[at] = e;
            if (a.probs) a.part_t[at] = make_float2(tl, ts);
        }
    }
}

// one workgroup a row
__global__ __launch_bounds__(256) void small_rows_kernel(SmallArgs a)
{
    __shared__ float red[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    float *l = a.logits + (long long)row * a.ldl;
    const float *pr = a.probs ? a.probs + (long long)row * a.ldp : nullptr;
    float mx = -INFINITY;
    for (int v = tid; v < a.V; v += 256) mx = fmaxf(mx, l[v]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    const float base = mx == -INFINITY ? 0.f : mx;
    float s = 0.f, e = 0.f, tl = 0.f, ts = 0.f;
    for (int v = tid; v < a.V; v += 256) {
        const float x = l[v] - base, p = __builtin_amdgcn_exp2f(x * kLog2e);
        s += p;
        e += p != 0.f ? p * x : 0.f;
        if (pr) { const float q = pr[v]; ts += q; tl += q != 0.f ? q * x : 0.f; }
    }
    s = block_sum<4>(s, red);
    if (a.ent) e = block_sum<4>(e, red);
    if (pr) { tl = block_sum<4>(tl, red); ts = block_sum<4>(ts, red); }
    const float ls = logf(s);                                 // (everything relative to the maximum: loss and entropy need no large difference)
    const long long t = a.target ? a.target[row] : -1;
    bool used = true;
    float loss, ent = ls - e / s;
    if (a.target) {
        ts = 1.f;
        if (t == a.ignore) { used = false; loss = ent = ts = 0.f; }
        else if (t < 0 || t >= a.V) loss = ent = ts = NAN;
        else loss = ls - (l[t] - base);
    } else {
        loss = ls * ts - tl;
    }
    __syncthreads();                                          // (l[t] is read before it becomes D)
    if (tid == 0) {
        a.stats[row] = make_float4(mx, ts / s, 0.f, loss);
        if (a.ent) a.ent[row] = ent;
        if (a.reduction == 0) {
            if (a.loss) a.loss[row] = loss;
            if (a.ent_out) a.ent_out[row] = ent;
        }
    }
    if (!a.backward) return;
    float g = (a.dloss ? a.dloss[a.reduction == 0 ? row : 0] : 1.f) * a.grad_scale;
    if (a.reduction == 2) { const int c = *a.count; g = c > 0 ? g / (float)c : 0.f; }
    const float f = ts / s;
    for (int v = tid; v < a.V; v += 256) {
        float q = __builtin_amdgcn_exp2f((l[v] - base) * kLog2e) * f;
        if (pr) q -= pr[v];
        else if (v == t) q -= 1.f;
        l[v] = used ? q * g : 0.f;                            // a row that counts for nothing: zero whatever it holds
    }
}

// sum or mean of the rows' losses and entropies, in double and in a fixed order
template <int W>
__device__ inline void small_totals(const SmallArgs &a)
{
    __shared__ double red[W];
    double l = 0.0, e = 0.0;
    for (int i = threadIdx.x; i < a.n; i += W * 64) {
        l += a.stats[i].w;
        if (a.ent) e += a.ent[i];
    }
    l = block_sum<W>(l, red);
    if (a.ent) e = block_sum<W>(e, red);
    if (threadIdx.x) return;
    const int c = *a.count;
    const double by = a.reduction == 2 ? (c > 0 ? 1.0 / c : 0.0) : 1.0;
    if (a.loss) a.loss[0] = (float)(l * by);
    if (a.ent_out) a.ent_out[0] = (float)(e * by);
}

// Workgroups: tiles of dX, tiles of dW, columns of db, totals.  Output tiles have the contiguous dimension (features) as columns.
template <typename T>
__global__ __launch_bounds__(kSmallWaves * 64) void small_grads_kernel(SmallArgs a)
{
    __shared__ SmallLds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, th = (a.H + kSmallTile - 1) / kSmallTile;
    int b = blockIdx.x;
    float out[2];
    if (b < a.tiles_x) {
        const int n0 = b / th * kSmallTile, h0 = b % th * kSmallTile;
        small_product<float, true, T, false>(a.logits, a.ldl, n0, a.n, static_cast<const T *>(a.w), a.ws, h0, a.H, a.V, nullptr, 0, lds, out);
        const int h = h0 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = n0 + wave * 4 + (lane >> 5) + 2 * i;
            if (r < a.n && h < a.H) static_cast<T *>(a.dx)[(long long)r * a.dxs + h] = (T)out[i];
        }
        return;
    }
    b -= a.tiles_x;
    if (b < a.tiles_w) {
        // (X's rows that count for nothing read as zero, whatever they hold)
        const int v0 = b / th * kSmallTile, h0 = b % th * kSmallTile;
        small_product<float, false, T, false>(a.logits, a.ldl, v0, a.V, static_cast<const T *>(a.x), a.xs, h0, a.H, a.n, a.target, a.ignore, lds, out);
        const int h = h0 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int v = v0 + wave * 4 + (lane >> 5) + 2 * i;
            if (v < a.V && h < a.H) static_cast<T *>(a.dw)[(long long)v * a.dws + h] = (T)out[i];
        }
        return;
    }
    b -= a.tiles_w;
    const int tb = a.db ? (a.V + 63) / 64 : 0;
    if (b < tb) {                                             // 64 classes, an eighth of the rows a wave
        const int v = b * 64 + lane;
        float s = 0.f;
        if (v < a.V)
#pragma unroll 8
            for (int r = wave; r < a.n; r += kSmallWaves) s += a.logits[(long long)r * a.ldl + v];
        float *red = &lds[0][0][0];
        red[wave * 64 + lane] = s;
        __syncthreads();
        if (wave == 0 && v < a.V) {
            s = red[lane];
#pragma unroll
            for (int w = 1; w < kSmallWaves; w++) s += red[w * 64 + lane];
            static_cast<T *>(a.db)[v] = (T)s;
        }
        return;
    }
    small_totals<kSmallWaves>(a);
}

// forward alone: the totals
__global__ __launch_bounds__(256) void small_totals_kernel(SmallArgs a) { small_totals<4>(a); }

}  // namespace azgops
