// C entry points of the training-head operators (include/azgomoku.h): argument checks, plans, launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <hip/hip_runtime.h>

#include "../../include/azgomoku.h"
#include "azg_dropout.hpp"
#include "azg_linear_ce.hpp"
#include "azg_linear_ce_small.hpp"

using namespace azgops;

extern "C" void azg_set_error_text(const char *text);        // azgomoku.hip: what azg_last_error(NULL) returns

namespace {

int fail(int code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    azg_set_error_text(buf);
    return code;
}

#define OPS_HIP(call)                                                                                   \
    do {                                                                                                \
        hipError_t e_ = (call);                                                                         \
        if (e_ != hipSuccess) return fail(AZG_EHIP, "%s failed: %s (%s:%d)", #call, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)
#define OPS_TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

// makes a device current for the time of a call
struct DeviceScope {
    int before = -1;
    bool changed = false;
    int enter(int device)
    {
        OPS_HIP(hipGetDevice(&before));
        if (before != device) { OPS_HIP(hipSetDevice(device)); changed = true; }
        return AZG_OK;
    }
    ~DeviceScope() { if (changed) (void)hipSetDevice(before); }
};

long long up_to(long long v, long long m) { return (v + m - 1) / m * m; }
// Row stride of an image of `cols` columns in `parts`: an odd number of 128-byte lines, so that the lines that the rows of a
// tile have in one stage lie in different channels of the L2 and of memory.
long long image_stride(long long cols, int parts) { const long long l = up_to(cols, 64) / 64 * parts; return (l | 1) * 64; }

bool bad_matrix(long long rows, long long cols, long long stride) { return rows > 1 && stride < cols; }

}  // namespace

// ---------------------------------------------------------------- dropout
extern "C" int azg_dropout(const azg_dropout_args *a)
{
    if (!a) return fail(AZG_EINVAL, "null argument");
    if (a->dtype != AZG_F32 && a->dtype != AZG_BF16 && a->dtype != AZG_F16) return fail(AZG_EINVAL, "azg_dropout: unknown dtype %d", a->dtype);
    if (!(a->p >= 0.0 && a->p <= 1.0)) return fail(AZG_EINVAL, "azg_dropout: p must lie in [0, 1]");
    if (a->rows < 0 || a->cols < 0) return fail(AZG_EINVAL, "azg_dropout: negative size");
    if (a->rows == 0 || a->cols == 0) return AZG_OK;
    if (a->rows > (1LL << 46) / a->cols) return fail(AZG_EINVAL, "azg_dropout: too many elements");
    if (!a->x || !a->out) return fail(AZG_EINVAL, "null argument");
    if (bad_matrix(a->rows, a->cols, a->x_stride) || bad_matrix(a->rows, a->cols, a->out_stride) || (a->residual && bad_matrix(a->rows, a->cols, a->residual_stride)))
        return fail(AZG_EINVAL, "azg_dropout: a row stride is smaller than a row");
    DeviceScope scope;
    OPS_TRY(scope.enter(a->device));
    DropoutArgs d{};
    d.x = a->x; d.res = a->residual; d.out = a->out;
    d.rows = a->rows; d.cols = a->cols; d.xs = a->x_stride; d.rs = a->residual_stride; d.os = a->out_stride;
    d.seed = a->seed; d.offset = a->offset;
    d.first = (unsigned long long)a->first_row * (unsigned long long)a->cols;
    d.step = (unsigned long long)a->row_step * (unsigned long long)a->cols;
    d.offset_dev = reinterpret_cast<const long long *>(a->offset_dev);
    const long T = std::lround(a->p * 65536.0);
    d.threshold = (unsigned)T;
    d.scale = T < 65536 ? (float)(65536.0 / (double)(65536 - T)) : 0.f;
    if (a->row_step == 1 && a->x_stride == a->cols && a->out_stride == a->cols && (!a->residual || a->residual_stride == a->cols)) {
        d.cols = a->rows * a->cols;                           // one long row: element numbers run on from row to row
        d.rows = 1;
    }
    const long long blocks_per_row = d.cols / 8 + 2;          // a row that starts inside a block touches one more
    const long long grid = std::min<long long>((d.rows * blocks_per_row + 255) / 256, 1 << 20);
    hipStream_t s = static_cast<hipStream_t>(a->stream);
    if (a->dtype == AZG_F32) hipLaunchKernelGGL((dropout_kernel<float>), dim3(grid), dim3(256), 0, s, d, blocks_per_row);
    else if (a->dtype == AZG_F16) hipLaunchKernelGGL((dropout_kernel<_Float16>), dim3(grid), dim3(256), 0, s, d, blocks_per_row);
    else hipLaunchKernelGGL((dropout_kernel<__bf16>), dim3(grid), dim3(256), 0, s, d, blocks_per_row);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}

// ---------------------------------------------------------------- projection + softmax cross entropy
namespace {

// Which problems the three-launch float32 path takes.  Measured, the tiled path against it, microseconds of GPU time:
//   float32, loss and gradients: 512 x 256 x 64 (rows, features, classes) 33 / 17, 512 x 900 x 225 58 / 31, 256 x 1024 x 1024
//     67 / 49, then 2048 x 1024 x 256 80 / 96; with long sums or few tiles it falls behind: 32 x 1024 x 4096 67 / 70,
//     4096 x 64 x 64 34 / 79;
//   float32, the loss alone: 512 x 1024 x 256 41 / 17, 512 x 2048 x 512 68 / 29, 4096 x 64 x 64 20 / 16, then 16384 x 64 x 64
//     29 / 45, 40 x 64 x 32768 28 / 63;
//   16 bits, whose matrix instructions are sixteen times as fast as float32's (bfloat16; half precision is a little slower
//     tiled): 128 x 256 x 1024 26 / 21, 512 x 256 x 64 26 / 18, then 512 x 1024 x 256 28 / 33, 16 x 512 x 4096 25 / 47
//     (the loss alone 13 / 11, 13 / 10, 16 / 17, 13 / 17).
constexpr long long kSmallLogits = 1LL << 22;                 // 16 MB of float32
bool takes_small(bool f32, bool backward, long long n, long long h, long long v)
{
    const long long side = f32 && !backward ? 4096 : 1024;
    const double work = (double)n * (double)h * (double)v;
    return n <= side && v <= side && n * v <= kSmallLogits && work <= (f32 ? backward ? 1LL << 28 : 1LL << 29 : 1LL << 25);
}
constexpr double kMaxThreads = 4294967295.0;                  // of a launch

// Room that the images of D, of W and of its transpose may take together before the classes are cut into pieces.
constexpr long long kPieceBytes = 1LL << 30;

struct Take {                                                 // offsets into the caller's workspace
    size_t off = 0;
    size_t operator()(size_t bytes) { const size_t at = off; off += (bytes + 255) / 256 * 256; return at; }
};

enum Shape { T256, T128, T64, T64FEW, TROW };
struct ShapeDim { int tm, tn, wm, threads; };
constexpr ShapeDim kDims[5] = {{256, 256, 2, 512}, {128, 128, 2, 256}, {64, 64, 2, 256}, {64, 64, 1, 256}, {128, 32, 4, 256}};
constexpr long long kFewTiles = 512;                          // T64FEW: two workgroups a CU, longer rings

long long tiles_of(Shape s, long long m, long long n) { return ((m + kDims[s].tm - 1) / kDims[s].tm) * ((n + kDims[s].tn - 1) / kDims[s].tn); }

// Tile of the logits.  Measured in bfloat16, microseconds of the loss alone: few rows 128 x 32 against larger tiles, 1 x 4096 x
// 65536 122 / 156, 32 x 4096 x 32000 52 / 53; 256 x 256 against 128 x 128, 1024 x 1024 x 8192 (128 tiles of 256) 35 / 29, 2048 x
// 1024 x 5000 (160) 36 / 39; 128 x 128 against 64 x 64, 1024 x 2048 x 2048 (128 tiles of 128) 30 / 24.  No tile is wider than the
// classes need.
Shape pick_logits(long long m, long long n, bool grad, long long stride)
{
    if (!grad && n <= 32) return TROW;
    // (a tile's rows lie within 2^32 bytes: 128 rows of 2^22 float32 features do)
    if (m > 128 && tiles_of(T256, m, n) >= 150 && 256 * 2 * stride < 1LL << 32) return T256;
    if (m > 64 && tiles_of(T128, m, n) >= 200) return T128;
    return tiles_of(T64, m, n) <= kFewTiles ? T64FEW : T64;
}
// Tile of the gradients' products, which share a launch, and the splits of their sums, by an estimate in microseconds: the
// launch takes its stages at the rate of the whole card or as long as its longest workgroup, whichever is more, and splits
// cost a join.  Per stage and tile (measured): 256 x 256 1.0 with a CU to itself,
// 128 x 128 0.30 a CU's share and 0.6 from start to end, 64 x 64 0.16 and 0.45, with longer rings 0.35.
struct GradPick { Shape shape; int splits_x, kper_x, splits_w, kper_w; };
GradPick pick_grads(long long n, long long h, long long v, long long kx, long long kw, bool want_x, bool want_w)
{
    static constexpr double share[4] = {1.0, 0.30, 0.16, 0.16}, alone[4] = {1.0, 0.6, 0.45, 0.35};
    GradPick best{};
    double least = 1e30;
    for (Shape s : {T256, T128, T64, T64FEW}) {
        const long long tx = want_x ? tiles_of(s, h, n) : 0, tw = want_w ? tiles_of(s, h, v) : 0;
        if ((double)(tx + tw) * 32 * kDims[s].threads > kMaxThreads && s != T256) continue;
        for (long long per = 4; per == 4 || per < 2 * std::max(kx, kw); per *= 2) {          // stages of a workgroup at most
            GradPick g{};
            auto split = [&](long long k, int *splits, int *kper) {
                const long long parts = std::min<long long>(32, (k + per - 1) / per);
                *kper = (int)((k + parts - 1) / parts);
                *splits = (int)((k + *kper - 1) / *kper);
            };
            g.shape = s;
            split(kx, &g.splits_x, &g.kper_x);
            split(kw, &g.splits_w, &g.kper_w);
            if (s == T64FEW && tx * g.splits_x + tw * g.splits_w > kFewTiles) continue;
            double joined = 0;                                                  // bytes of the splits, written and read
            if (tx && g.splits_x > 1) joined += 8.0 * g.splits_x * n * h;
            if (tw && g.splits_w > 1) joined += 8.0 * g.splits_w * v * h;
            const double work = (double)(tx * kx + tw * kw) * share[s] / 256.0;
            const double longest = std::max(tx ? g.kper_x : 0, tw ? g.kper_w : 0) * alone[s];
            // (dX's workgroups start first; of the others half a one on average is lost at the end)
            const double last = (tw ? g.kper_w : g.kper_x) * alone[s];
            const double t = std::max(work + 0.5 * last, longest) + joined / 4e6 + (joined > 0 ? 3.0 : 0.0);
            if (t < least) { least = t; best = g; }
        }
    }
    return best;
}

struct Plan {
    bool small, few, forward, backward, keep;                 // keep: the forward pass leaves exponentials for the backward pass
    bool pack_w, pack_x, grad_w, grad_x;                      // images of W and X for the logits; of their own for the gradients
    long long n, H, V, vp, pieces;
    long long kimg, ldl, ldg, ldd;                            // columns of the images of W and X; row strides of these and of D's
    int lparts, gparts;                                       // parts of an element in the logits' and the gradients' products
    Shape lshape;
    int large_m, behind_m;                                    // the loss alone: tiles of 256 and, behind them, of 128 classes (0: none)
    long long spans;                                          // of a piece
    GradPick g;
    int fix_rows;
    size_t ximg, wimg, gximg, gwimg, part, part_e, part_t, tlogit, stats, ent, rowg, sums, factor, d, dbpart, dxacc, dwacc, logits, count, total;
};

bool aligned16(const void *p, long long stride, long long cols, long long rows)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && cols % 8 == 0 && (rows <= 1 || stride % 8 == 0);
}

int make_plan(const azg_linear_ce_args *a, Plan *p)
{
    const bool f32 = a->dtype == AZG_F32;
    p->lparts = f32 ? OpF32::Logits::parts : 1;
    p->gparts = f32 ? OpF32::Grad::parts : a->dtype == AZG_F16 ? OpF16::Grad::parts : OpBF16::Grad::parts;
    p->forward = a->loss != nullptr;
    p->backward = a->dx || a->dw || a->db;
    p->n = a->n; p->H = a->hidden; p->V = a->classes;
    // A forward pass whose stats are kept takes the path of the backward pass to come: the logits that are made again there have to
    // be the same bits (every tile adds up k in one order), or a large logit's exponential leaves [0, 1].
    const bool differentiable = p->backward || a->stats;
    p->small = takes_small(f32, differentiable, p->n, p->H, p->V);
    if (p->small) {
        Take t;
        p->logits = t((size_t)p->n * p->V * 4);
        p->stats = t((size_t)p->n * 16);
        p->ent = t((size_t)p->n * 4);
        p->count = t(4);
        p->total = t.off;
        return AZG_OK;
    }
    p->kimg = up_to(p->H, 64);
    p->ldl = image_stride(p->H, p->lparts);
    p->ldg = image_stride(p->H, p->gparts);
    // (dW multiplies the rows that count for nothing by zero: they are copied as zeros, whatever they hold)
    const bool shared = p->lparts == p->gparts;               // the gradients' products take the same images
    p->pack_x = p->lparts > 1 || !aligned16(a->x, a->x_stride, a->hidden, a->n) || (shared && a->dw && a->target);
    p->pack_w = p->lparts > 1 || !aligned16(a->w, a->w_stride, a->hidden, a->classes);
    p->grad_x = !shared && a->dw;
    p->grad_w = !shared && a->dx;
    p->few = !differentiable && p->n <= 32 && p->pack_w;
    if (p->few) p->pack_x = p->pack_w = false;
    // bytes a class of a piece costs
    long long cost = (p->pack_w ? p->ldl * 2 : 0) + (p->grad_w ? p->ldg * 2 : 0);
    if (p->backward) cost += p->n * p->gparts * 2;
    p->vp = p->V;
    if (cost) p->vp = std::min<long long>(p->V, std::max<long long>(1024, kPieceBytes / cost / 256 * 256));
    p->pieces = (p->V + p->vp - 1) / p->vp;
    if (p->pieces > 1) {                                      // even pieces
        p->vp = std::min<long long>(p->V, up_to((p->V + p->pieces - 1) / p->pieces, 256));
        p->pieces = (p->V + p->vp - 1) / p->vp;
    }
    // (against probabilities D is the difference of two numbers that training brings together: exponentials of 16 bits would leave
    // little of it, and the logits are made again)
    p->keep = p->forward && p->backward && p->pieces == 1 && !(a->probs && p->gparts == 1);
    p->ldd = image_stride(p->vp, p->gparts);
    p->lshape = pick_logits(p->vp, p->n, p->backward || f32, p->lparts > 1 ? p->ldl : 0);   // (float32 has no tile for few rows)
    const int pairs = p->gparts * (p->gparts + 1) / 2;
    p->g = pick_grads(p->n, p->H, p->vp, (p->vp + 63) / 64 * pairs, (p->n + 63) / 64 * pairs, a->dx != nullptr, a->dw != nullptr);
    // rows a workgroup turns into D: up to 64, fewer while they would not give four workgroups a CU
    // (more for very many rows: db is joined from one sum a run of rows, one after the other)
    p->fix_rows = 64;
    while ((p->n + p->fix_rows - 1) / p->fix_rows > 1024) p->fix_rows *= 2;
    while (p->fix_rows > 8 && (p->n + p->fix_rows - 1) / p->fix_rows * ((p->vp + kFixCols - 1) / kFixCols) < 1024) p->fix_rows /= 2;
    const ShapeDim dim = kDims[p->lshape];
    p->large_m = p->behind_m = 0;
    const long long lm = (p->vp + dim.tm - 1) / dim.tm, ln = (p->n + dim.tn - 1) / dim.tn;
    const double grad_tiles = (a->dx ? (double)tiles_of(p->g.shape, p->H, p->n) * p->g.splits_x : 0.0) + (a->dw ? (double)tiles_of(p->g.shape, p->H, p->vp) * p->g.splits_w : 0.0);
    if ((double)lm * ln * dim.threads > kMaxThreads || grad_tiles * kDims[p->g.shape].threads > kMaxThreads)
        return fail(AZG_EINVAL, "azg_linear_ce: the problem is too large");
    p->spans = lm * dim.wm;
    if (!p->backward && p->pieces == 1 && p->lshape == T256) {           // (never with few rows)
        // the tiles that do not fill a round of the 256 CUs, cut into quarters, if one round takes those
        const long long whole = lm * ln / 256 * 256 / ln, behind = (p->V - whole * 256 + 127) / 128;
        if (whole > 0 && whole < lm && behind * ((p->n + 127) / 128) <= 256) {
            p->large_m = (int)whole;
            p->behind_m = (int)behind;
            p->spans = (whole + behind) * 2;
        }
    }
    if (p->few) p->spans = (p->V + kSmallTile - 1) / kSmallTile;
    Take t;
    p->ximg = t(p->pack_x ? (size_t)p->n * p->ldl * 2 : 0);
    p->wimg = t(p->pack_w ? (size_t)p->vp * p->ldl * 2 : 0);
    p->gximg = t(p->grad_x ? (size_t)p->n * p->ldg * 2 : 0);
    p->gwimg = t(p->grad_w ? (size_t)p->vp * p->ldg * 2 : 0);
    const size_t entries = (size_t)p->pieces * p->spans * p->n;
    p->part = t(p->forward ? entries * 8 : 0);
    p->part_e = t(p->forward && a->entropy ? entries * 4 : 0);
    p->part_t = t(p->forward && a->probs ? entries * 8 : 0);
    p->tlogit = t((size_t)p->n * 4);
    p->stats = t((size_t)p->n * 16);
    p->ent = t((size_t)p->n * 4);
    p->rowg = t((size_t)p->n * 4);
    p->sums = t(p->n > kOneTotal ? kMaxSums * sizeof(RowSums) : 0);
    p->factor = t(4);
    p->d = t(p->backward ? (size_t)p->n * p->ldd * 2 : 0);
    p->dbpart = t(a->db ? (size_t)std::max(ln, (p->n + p->fix_rows - 1) / p->fix_rows) * p->vp * 4 : 0);
    p->dxacc = t(a->dx && (p->g.splits_x > 1 || p->pieces > 1) ? (size_t)p->g.splits_x * p->n * p->H * 4 : 0);
    p->dwacc = t(a->dw && p->g.splits_w > 1 ? (size_t)p->g.splits_w * p->vp * p->H * 4 : 0);
    p->total = t.off;
    return AZG_OK;
}

int check(const azg_linear_ce_args *a)
{
    if (!a) return fail(AZG_EINVAL, "null argument");
    if (a->dtype != AZG_F32 && a->dtype != AZG_BF16 && a->dtype != AZG_F16) return fail(AZG_EINVAL, "azg_linear_ce: unknown dtype %d", a->dtype);
    if (a->n < 0 || a->hidden < 1 || a->classes < 1) return fail(AZG_EINVAL, "azg_linear_ce: sizes must be n >= 0, hidden >= 1, classes >= 1");
    if (a->n >= 1 << 26 || a->classes >= 1 << 27 || a->hidden > (1 << 22)) return fail(AZG_EINVAL, "azg_linear_ce: a size is too large");
    if (a->reduction < AZG_REDUCE_NONE || a->reduction > AZG_REDUCE_MEAN) return fail(AZG_EINVAL, "azg_linear_ce: unknown reduction %d", a->reduction);
    if (bad_matrix(a->n, a->hidden, a->x_stride) || bad_matrix(a->classes, a->hidden, a->w_stride)) return fail(AZG_EINVAL, "azg_linear_ce: a row stride is smaller than a row");
    if ((a->n > 1 && a->x_stride > (1LL << 22)) || (a->classes > 1 && a->w_stride > (1LL << 22))) return fail(AZG_EINVAL, "azg_linear_ce: a row stride is too large");
    return AZG_OK;
}

template <typename K> int allow_lds(K kernel, int bytes)
{
    if (bytes > 65536) OPS_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return AZG_OK;
}

template <typename Op, int TM, int TN, int WM, int WN, bool GRAD>
int launch_logits_shape(CeArgs c, hipStream_t s)
{
    using S = TileShape<TM, TN, WM, WN>;
    c.mtiles = (int)((c.classes + TM - 1) / TM);
    c.ntiles = (int)((c.n + TN - 1) / TN);
    const int lds = S::lds_bytes;
    OPS_TRY(allow_lds(logits_kernel<Op, TM, TN, WM, WN, GRAD>, lds));
    hipLaunchKernelGGL((logits_kernel<Op, TM, TN, WM, WN, GRAD>), dim3((unsigned)c.mtiles * c.ntiles), dim3(S::threads), lds, s, c);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}
template <typename Op, bool GRAD>
int launch_logits(Shape shape, const CeArgs &c, hipStream_t s)
{
    switch (shape) {
    case T256: return launch_logits_shape<Op, 256, 256, 2, 4, GRAD>(c, s);
    case T128: return launch_logits_shape<Op, 128, 128, 2, 2, GRAD>(c, s);
    case T64: return launch_logits_shape<Op, 64, 64, 2, 2, GRAD>(c, s);
    case T64FEW: return launch_logits_shape<Op, 64, 64, 1, 4, GRAD>(c, s);
    default:
        if constexpr (!GRAD && Op::Logits::parts == 1) return launch_logits_shape<Op, 128, 32, 4, 1, false>(c, s);
        return fail(AZG_EINVAL, "azg_linear_ce: internal: no such tile");
    }
}

template <typename Op>
int launch_logits_mixed(const CeArgs &c, hipStream_t s)
{
    using S = TileShape<256, 256, 2, 4>;
    OPS_TRY(allow_lds(logits_mixed_kernel<Op>, S::lds_bytes));
    hipLaunchKernelGGL((logits_mixed_kernel<Op>), dim3((unsigned)(c.mtiles * c.ntiles + c.mtiles_behind * ((c.n + 127) / 128))), dim3(S::threads), S::lds_bytes, s, c);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}

template <typename Op, int TM, int TN, int WM, int WN>
int launch_grads_shape(GradArgs x, GradArgs w, hipStream_t s)
{
    using S = TileShape<TM, TN, WM, WN>;
    unsigned wgs[2];
    int i = 0;
    for (GradArgs *g : {&x, &w}) {
        g->mtiles = (int)((g->m + TM - 1) / TM);
        g->ntiles = (int)((g->n + TN - 1) / TN);
        wgs[i++] = g->out ? (unsigned)g->mtiles * g->ntiles * g->splits : 0;
    }
    OPS_TRY(allow_lds(grads_kernel<Op, TM, TN, WM, WN>, S::lds_bytes));
    hipLaunchKernelGGL((grads_kernel<Op, TM, TN, WM, WN>), dim3(wgs[0] + wgs[1]), dim3(S::threads), S::lds_bytes, s, x, w, wgs[0]);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}
template <typename Op>
int launch_grads(Shape shape, const GradArgs &x, const GradArgs &w, hipStream_t s)
{
    switch (shape) {
    case T256: return launch_grads_shape<Op, 256, 256, 2, 4>(x, w, s);
    case T128: return launch_grads_shape<Op, 128, 128, 2, 2>(x, w, s);
    case T64: return launch_grads_shape<Op, 64, 64, 2, 2>(x, w, s);
    default: return launch_grads_shape<Op, 64, 64, 1, 4>(x, w, s);
    }
}
// up to three joins in one launch
template <typename Op>
int launch_joins(JoinList l, int count, hipStream_t s)
{
    unsigned grid = 0;
    for (int i = 0; i < count; i++) {
        const int outputs = l.j[i].splits > kFewSplits ? kJoinCols : 256;           // of a workgroup
        l.j[i].wgs = (unsigned)std::min<long long>((l.j[i].n * l.j[i].m + outputs - 1) / outputs, 1 << 16);
        grid += l.j[i].wgs;
    }
    if (!grid) return AZG_OK;
    hipLaunchKernelGGL((join_kernel<Op>), dim3(grid), dim3(256), 0, s, l);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}
// the images of a list, `count` of them
template <typename In>
int launch_packs(PackList l, int count, hipStream_t s)
{
    unsigned grid = 0;
    for (int i = 0; i < count; i++) {
        l.p[i].wgs = (unsigned)std::min<long long>((l.p[i].rows * (l.p[i].icols / 8) + 255) / 256, 1 << 16);
        grid += l.p[i].wgs;
    }
    if (!grid) return AZG_OK;
    hipLaunchKernelGGL((pack_kernel<In>), dim3(grid), dim3(256), 0, s, l);
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}

template <typename Op>
int run_ce(const azg_linear_ce_args *a, const Plan &p)
{
    using In = typename Op::In;
    hipStream_t s = static_cast<hipStream_t>(a->stream);
    char *ws = static_cast<char *>(a->workspace);
    auto f32 = [&](size_t o) { return reinterpret_cast<float *>(ws + o); };
    const long long *target = reinterpret_cast<const long long *>(a->target);
    float4 *stats = a->stats ? static_cast<float4 *>(a->stats) : reinterpret_cast<float4 *>(ws + p.stats);
    const In *W = static_cast<const In *>(a->w);
    const ShapeDim dim = kDims[p.lshape];

    bool x_packed = false;
    CeArgs c{};
    const int lblock = p.lparts * 64, gblock = p.gparts * 64;
    c.x = p.pack_x ? Operand{ws + p.ximg, p.ldl, a->n, p.kimg, lblock} : Operand{a->x, a->x_stride, a->n, a->hidden, lblock};
    const Operand grad_x_op = p.grad_x ? Operand{ws + p.gximg, p.ldg, a->n, p.kimg, gblock} : c.x;
    Operand grad_w_op{};
    c.ktiles = (int)((p.H + 63) / 64) * Op::Logits::pairs;
    c.n = a->n; c.target = target; c.ignore = a->ignore_index; c.ldp = a->probs_stride;

    // a piece of the classes, its images, and before the first piece X's; `grads`: the gradients' products are going to follow
    auto piece = [&](long long i, bool grads) -> int {
        const long long v0 = i * p.vp, vn = std::min(p.vp, a->classes - v0);
        c.v0 = v0; c.classes = vn;
        c.bias = a->bias ? static_cast<const In *>(a->bias) + v0 : nullptr;
        c.probs = a->probs ? a->probs + v0 : nullptr;
        c.ldd = p.ldd;
        c.dcols = up_to(vn, 64);
        const In *w = W + v0 * a->w_stride;
        PackList list{};
        int count = 0;
        auto image = [&](const void *src, long long ld, long long rows, size_t at, long long ldi, int parts, const long long *rows_of) {
            PackArgs &q = list.p[count++];
            q.src = src; q.ld = ld; q.rows = rows; q.cols = a->hidden; q.img = ws + at; q.ldi = ldi; q.icols = p.kimg; q.parts = parts;
            q.target = rows_of; q.ignore = a->ignore_index;
        };
        if (!x_packed && p.pack_x) image(a->x, a->x_stride, a->n, p.ximg, p.ldl, p.lparts, target);
        if (!x_packed && p.grad_x) image(a->x, a->x_stride, a->n, p.gximg, p.ldg, p.gparts, target);
        if (p.pack_w) image(w, a->w_stride, vn, p.wimg, p.ldl, p.lparts, nullptr);
        if (p.grad_w && grads) image(w, a->w_stride, vn, p.gwimg, p.ldg, p.gparts, nullptr);
        OPS_TRY(launch_packs<In>(list, count, s));
        x_packed = true;
        c.w = p.pack_w ? Operand{ws + p.wimg, p.ldl, vn, p.kimg, lblock} : Operand{w, a->w_stride, vn, a->hidden, lblock};
        grad_w_op = p.grad_w ? Operand{ws + p.gwimg, p.ldg, vn, p.kimg, gblock} : c.w;
        return AZG_OK;
    };

    if (p.forward) {
        const long long full = p.spans;                       // of a whole piece
        long long spans = 0;
        if (p.few) {
            FewArgs f{};
            f.x = a->x; f.w = a->w; f.bias = a->bias; f.xs = a->x_stride; f.ws = a->w_stride;
            f.n = (int)a->n; f.H = (int)a->hidden; f.V = (int)a->classes; f.target = target; f.probs = a->probs; f.ldp = a->probs_stride;
            f.part = reinterpret_cast<float2 *>(ws + p.part); f.part_e = a->entropy ? f32(p.part_e) : nullptr;
            f.part_t = a->probs ? reinterpret_cast<float2 *>(ws + p.part_t) : nullptr; f.tlogit = f32(p.tlogit);
            hipLaunchKernelGGL((few_rows_kernel<In>), dim3((unsigned)full), dim3(kSmallWaves * 64), 0, s, f);
            spans = full;
        } else for (long long i = 0; i < p.pieces; i++) {
            OPS_TRY(piece(i, p.backward && p.pieces == 1));
            c.part = reinterpret_cast<float2 *>(ws + p.part) + i * full * a->n;
            c.part_e = a->entropy ? f32(p.part_e) + i * full * a->n : nullptr;
            c.part_t = a->probs ? reinterpret_cast<float2 *>(ws + p.part_t) + i * full * a->n : nullptr;
            c.tlogit = f32(p.tlogit);
            c.d = p.keep ? ws + p.d : nullptr;
            if (p.behind_m) {
                c.mtiles = p.large_m; c.mtiles_behind = p.behind_m; c.ntiles = (int)((a->n + 255) / 256);
                OPS_TRY(launch_logits_mixed<Op>(c, s));
                spans = full;
            } else {
                OPS_TRY((launch_logits<Op, false>(p.lshape, c, s)));
                spans += (c.classes + dim.tm - 1) / dim.tm * dim.wm;
            }
        }
        RowArgs r{};
        r.n = a->n; r.classes = a->classes; r.spans = (int)spans;
        r.part = reinterpret_cast<float2 *>(ws + p.part); r.part_e = a->entropy ? f32(p.part_e) : nullptr;
        r.part_t = a->probs ? reinterpret_cast<float2 *>(ws + p.part_t) : nullptr; r.tlogit = f32(p.tlogit);
        r.target = target; r.ignore = a->ignore_index; r.stats = stats; r.ent = a->entropy ? f32(p.ent) : nullptr;
        if (a->reduction == AZG_REDUCE_NONE) { r.loss_out = a->loss; r.ent_out = a->entropy; }
        hipLaunchKernelGGL(rows_kernel, dim3((unsigned)((a->n + 3) / 4)), dim3(256), 0, s, r);
    }
    TotalArgs t{};
    t.n = a->n; t.reduction = a->reduction; t.stats = stats; t.ent = p.forward && a->entropy ? f32(p.ent) : nullptr;
    t.target = target; t.ignore = a->ignore_index;
    if (p.forward && a->reduction != AZG_REDUCE_NONE) { t.loss = a->loss; t.ent_out = a->entropy; }
    t.dloss = a->dloss; t.grad_scale = (float)a->grad_scale;
    t.rowg = p.backward ? f32(p.rowg) : nullptr; t.factor = p.backward ? f32(p.factor) : nullptr;
    // class numbers and a common g: the rows' factors are 1 or 0, and the totals can ride on the next launch (with many classes
    // its other workgroups take longer than the one that does the totals, however many rows there are)
    const bool ride = p.keep && target && a->reduction != AZG_REDUCE_NONE && (a->n <= kOneTotal || p.V >= 4096);
    if (ride) t.rowg = nullptr;
    else if (p.backward || a->reduction != AZG_REDUCE_NONE) {
        const bool many = a->n > kOneTotal;
        if (many && a->reduction != AZG_REDUCE_NONE) {
            t.sums = reinterpret_cast<RowSums *>(ws + p.sums);
            hipLaunchKernelGGL(sums_kernel, dim3(kMaxSums), dim3(256), 0, s, t);
        }
        hipLaunchKernelGGL(totals_kernel, dim3(many ? 64 : 1), dim3(1024), 0, s, t);
    }
    OPS_HIP(hipGetLastError());
    if (!p.backward) return AZG_OK;

    for (long long i = 0; i < p.pieces; i++) {
        if (!p.forward || p.pieces > 1) OPS_TRY(piece(i, true));            // (else its images are there)
        const long long vn = c.classes;
        int dbparts;
        if (p.keep) {
            FixArgs f{};
            f.n = a->n; f.classes = vn; f.rows = p.fix_rows; f.span = dim.tm / dim.wm; f.d = ws + p.d; f.ldd = c.ldd; f.dcols = c.dcols;
            f.part = reinterpret_cast<float2 *>(ws + p.part); f.stats = stats; f.rowg = t.rowg;
            f.target = target; f.ignore = a->ignore_index; f.probs = a->probs; f.ldp = a->probs_stride; f.dbpart = a->db ? f32(p.dbpart) : nullptr;
            f.totals = t;
            if (!ride) f.totals.n = -1;
            dbparts = (int)((a->n + p.fix_rows - 1) / p.fix_rows);
            hipLaunchKernelGGL((fix_kernel<Op>), dim3((unsigned)((c.dcols + kFixCols - 1) / kFixCols), dbparts + (ride ? 1 : 0)), dim3(256), 0, s, f);
            OPS_HIP(hipGetLastError());
        } else {
            c.stats = stats; c.rowg = f32(p.rowg);
            c.d = a->dx || a->dw ? ws + p.d : nullptr;
            c.dbpart = a->db ? f32(p.dbpart) : nullptr;
            dbparts = (int)((a->n + dim.tn - 1) / dim.tn);
            OPS_TRY((launch_logits<Op, true>(p.lshape, c, s)));
        }
        GradArgs gx{}, gw{};
        JoinList joins{};
        int count = 0;
        const Operand d{ws + p.d, c.ldd, a->n, c.dcols, gblock};
        if (a->dx) {
            gx.a = grad_w_op; gx.b = d;
            gx.ktiles = (int)((vn + 63) / 64) * Op::Grad::pairs; gx.kper = p.g.kper_x; gx.splits = p.g.splits_x; gx.m = a->hidden; gx.n = a->n;
            gx.factor = f32(p.factor);
            const bool acc = p.g.splits_x > 1 || p.pieces > 1;
            gx.acc = acc ? f32(p.dxacc) : nullptr; gx.add = i > 0;
            gx.out = a->dx; gx.ldo = a->dx_stride;
            if (acc && i == p.pieces - 1) joins.j[count++] = {gx.acc, gx.splits, gx.n, gx.m, gx.out, gx.ldo, gx.factor, 0};
        }
        if (a->dw) {
            gw.a = grad_x_op; gw.b = d;
            gw.ktiles = (int)((a->n + 63) / 64) * Op::Grad::pairs; gw.kper = p.g.kper_w; gw.splits = p.g.splits_w; gw.m = a->hidden; gw.n = vn;
            gw.factor = f32(p.factor);
            gw.acc = p.g.splits_w > 1 ? f32(p.dwacc) : nullptr; gw.add = false;
            gw.out = static_cast<In *>(a->dw) + i * p.vp * a->dw_stride; gw.ldo = a->dw_stride;
            if (gw.acc) joins.j[count++] = {gw.acc, gw.splits, gw.n, gw.m, gw.out, gw.ldo, gw.factor, 0};
        }
        if (a->dx || a->dw) OPS_TRY(launch_grads<Op>(p.g.shape, gx, gw, s));
        if (a->db) joins.j[count++] = {f32(p.dbpart), dbparts, 1, vn, static_cast<In *>(a->db) + i * p.vp, vn, f32(p.factor), 0};
        OPS_TRY(launch_joins<Op>(joins, count, s));
    }
    return AZG_OK;
}

template <typename In>
int run_small(const azg_linear_ce_args *a, const Plan &p)
{
    hipStream_t s = static_cast<hipStream_t>(a->stream);
    char *ws = static_cast<char *>(a->workspace);
    SmallArgs g{};
    g.x = a->x; g.w = a->w; g.bias = a->bias; g.xs = a->x_stride; g.ws = a->w_stride;
    g.n = (int)a->n; g.H = (int)a->hidden; g.V = (int)a->classes;
    g.target = reinterpret_cast<const long long *>(a->target); g.ignore = a->ignore_index; g.probs = a->probs; g.ldp = a->probs_stride;
    g.logits = reinterpret_cast<float *>(ws + p.logits); g.ldl = g.V;
    // (a backward pass by itself repeats the rows' statistics; the caller's are left alone)
    g.stats = a->stats && p.forward ? static_cast<float4 *>(a->stats) : reinterpret_cast<float4 *>(ws + p.stats);
    g.ent = a->entropy ? reinterpret_cast<float *>(ws + p.ent) : nullptr;
    g.reduction = a->reduction; g.loss = a->loss; g.ent_out = a->entropy;
    g.dloss = a->dloss; g.grad_scale = (float)a->grad_scale;
    g.count = reinterpret_cast<int *>(ws + p.count);
    g.backward = p.backward; g.dx = a->dx; g.dw = a->dw; g.db = a->db; g.dxs = a->dx_stride; g.dws = a->dw_stride;
    auto tiles = [](int v) { return (v + kSmallTile - 1) / kSmallTile; };
    hipLaunchKernelGGL((small_logits_kernel<In>), dim3(tiles(g.n) * tiles(g.V) + 1), dim3(kSmallWaves * 64), 0, s, g);
    hipLaunchKernelGGL(small_rows_kernel, dim3(g.n), dim3(256), 0, s, g);
    const bool totals = p.forward && g.reduction != AZG_REDUCE_NONE;
    if (p.backward) {
        g.tiles_x = g.dx ? tiles(g.n) * tiles(g.H) : 0;
        g.tiles_w = g.dw ? tiles(g.V) * tiles(g.H) : 0;
        const int grid = g.tiles_x + g.tiles_w + (g.db ? (g.V + 63) / 64 : 0) + (totals ? 1 : 0);
        hipLaunchKernelGGL((small_grads_kernel<In>), dim3(grid), dim3(kSmallWaves * 64), 0, s, g);
    } else if (totals) {
        hipLaunchKernelGGL(small_totals_kernel, dim3(1), dim3(256), 0, s, g);
    }
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}

template <typename In>
int empty_batch(const azg_linear_ce_args *a)
{
    hipStream_t s = static_cast<hipStream_t>(a->stream);
    if (a->dw) hipLaunchKernelGGL((zero_rows_kernel<In>), dim3(1024), dim3(256), 0, s, static_cast<In *>(a->dw), (long long)a->classes, (long long)a->hidden, (long long)a->dw_stride);
    if (a->db) hipLaunchKernelGGL((zero_rows_kernel<In>), dim3(64), dim3(256), 0, s, static_cast<In *>(a->db), 1LL, (long long)a->classes, (long long)a->classes);
    if (a->reduction != AZG_REDUCE_NONE) {
        if (a->loss) hipLaunchKernelGGL((zero_rows_kernel<float>), dim3(1), dim3(64), 0, s, a->loss, 1LL, 1LL, 1LL);
        if (a->entropy) hipLaunchKernelGGL((zero_rows_kernel<float>), dim3(1), dim3(64), 0, s, a->entropy, 1LL, 1LL, 1LL);
    }
    OPS_HIP(hipGetLastError());
    return AZG_OK;
}

}  // namespace

extern "C" int64_t azg_linear_ce_workspace(const azg_linear_ce_args *a)
{
    const int rc = check(a);
    if (rc) return rc;
    if (a->n == 0) return 0;
    Plan p{};
    const int rc2 = make_plan(a, &p);
    return rc2 ? rc2 : (int64_t)p.total;
}

extern "C" int azg_linear_ce(const azg_linear_ce_args *a)
{
    OPS_TRY(check(a));
    const bool backward = a->dx || a->dw || a->db;
    if (!a->loss && !backward) return fail(AZG_EINVAL, "azg_linear_ce: neither a loss nor a gradient is asked for");
    if (a->n > 0 && !a->loss && !a->stats) return fail(AZG_EINVAL, "azg_linear_ce: a backward pass by itself needs the forward pass's stats");
    if (reinterpret_cast<uintptr_t>(a->stats) & 15) return fail(AZG_EINVAL, "azg_linear_ce: stats must be 16-byte aligned");
    if (a->entropy && !a->loss) return fail(AZG_EINVAL, "azg_linear_ce: the entropy comes with the loss");
    if ((a->dx && bad_matrix(a->n, a->hidden, a->dx_stride)) || (a->dw && bad_matrix(a->classes, a->hidden, a->dw_stride)))
        return fail(AZG_EINVAL, "azg_linear_ce: a row stride is smaller than a row");
    if (a->n > 0) {
        if (!a->x || !a->w) return fail(AZG_EINVAL, "null argument");
        if ((a->target != nullptr) == (a->probs != nullptr)) return fail(AZG_EINVAL, "azg_linear_ce: either target or probs");
        if (a->probs && bad_matrix(a->n, a->classes, a->probs_stride)) return fail(AZG_EINVAL, "azg_linear_ce: a row stride is smaller than a row");
    }
    DeviceScope scope;
    OPS_TRY(scope.enter(a->device));
    if (a->n == 0) return a->dtype == AZG_F32 ? empty_batch<float>(a) : a->dtype == AZG_F16 ? empty_batch<_Float16>(a) : empty_batch<__bf16>(a);
    Plan p{};
    OPS_TRY(make_plan(a, &p));
    if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255) || a->workspace_bytes < (int64_t)p.total)
        return fail(AZG_EINVAL, "azg_linear_ce: the workspace must be 256-byte aligned and hold %lld bytes", (long long)p.total);
    if (p.small) return a->dtype == AZG_F32 ? run_small<float>(a, p) : a->dtype == AZG_F16 ? run_small<_Float16>(a, p) : run_small<__bf16>(a, p);
    if (a->dtype == AZG_F32) return run_ce<OpF32>(a, p);
    if (a->dtype == AZG_F16) return run_ce<OpF16>(a, p);
    return run_ce<OpBF16>(a, p);
}
