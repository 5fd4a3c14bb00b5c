// Softmax cross entropy of a projection, l = X W^T + b, with its gradient, in pieces of the classes: the logits
// live in the accumulators of a matrix-core tile and leave it as softmax statistics, and where a gradient is asked
// for as what it is made of, one piece of the classes at a time.
//
//   lse_i  = log sum_v exp l_iv, from (maximum, sum) pairs of runs of classes ("spans": a wave's part of a tile)
//   loss_i = lse_i - l_{i,t}   or   lse_i sum_v pi_iv - sum_v pi_iv l_iv
//   D_iv   = g_i (p_iv sum_v pi_iv - pi_iv);   dX = D W;   dW = D^T X;   db = sum_i D_i
//
// Loss and gradients in one call, one piece: the logits' kernel also stores exp(l - the span's maximum), 16 bits an element
// (float32: 4 bytes), and a pass in place turns that into the image of D once the rows' sums are known.  That costs two
// passes over the image and saves a product: 4096 rows of 2048 features against 32000 classes (bfloat16) take 1.40 ms so, 1.72 ms
// with the logits made a second time.  A backward pass by itself, or of more than one piece, makes the logits again and
// stores D at once; so does bfloat16 against probabilities, whose D is a difference that 16 bits of the one number would not carry.
//
// All three products are one kernel core: C[m][n] = sum_k A[m][k] B[n][k], each operand stored with either index
// contiguous: what runs against the sum is transposed on its way from LDS to the registers.  Operands that the loads
// cannot take (float32, odd sizes or alignments) and rows that must read as zero are copied once into an "image".
//
// float32 runs on the 16-bit matrix cores too: an element is the sum of three bfloat16 numbers, x = x0 + x1 + x2, each the
// rounding of what the ones before it leave.  Eight bits a part and its sign hold all 24 bits of x, and every part has
// float32's range of exponents, so nothing is scaled and what the other elements are does not matter.  A product of two
// elements is the six products of parts i, j with i + j < 3; what is left out is at most 2^-24 of it (|x1| <= 2^-8 |x|,
// |x2| <= 2^-17 |x|).  That is twice the matrix work of two half-precision parts, which have neither the range nor, below 2^-17 of
// their tensor's largest element, the bits (2048 x 1024 x 32000 with gradients: 2.1 ms, 1.15 so).  Gradients of half precision take two parts -- all of an operand's 11 bits; the gradient at the logits is
// off by 2^-17 of itself -- and three products, which leave out 2^-16: half precision itself has not the range for
// probabilities (2048 x 1024 x 32000: 1.0 ms, 0.44 with one half-precision number, which loses classes below 2^-39).  bfloat16
// is one part: its gradient at the logits has the type's own 8 bits, half a step of which the results are rounded by anyway, and
// float32's range; a second part would make three products of each of the gradients' two.  An image row holds blocks of 64 columns, 64 elements of part 0, then of part 1, ...; a
// product walks over the pairs of parts of one block of k and then over the blocks, every pair a stage of its own.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace azgops {

typedef float fx4 __attribute__((ext_vector_type(4)));
typedef _Float16 hx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bx8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;

// What a product runs on: parts of an element and their type.
template <typename T, int N> struct Parts {
    using Img = T;
    static constexpr int parts = N, pairs = N * (N + 1) / 2, block = 64 * N;
    // part of either side in the q-th pair, largest products first: (0,0) (0,1) (1,0) (0,2) (1,1) (2,0)
    static __device__ inline int of_a(int q) { return N == 1 ? 0 : 0x910 >> (2 * q) & 3; }
    static __device__ inline int of_b(int q) { return N == 1 ? 0 : 0x184 >> (2 * q) & 3; }
};
// Operand element types, and what the logits' and the gradients' products run on.
struct OpF32 { using In = float; using Logits = Parts<__bf16, 3>; using Grad = Parts<__bf16, 3>; };
struct OpF16 { using In = _Float16; using Logits = Parts<_Float16, 1>; using Grad = Parts<__bf16, 2>; };
struct OpBF16 { using In = __bf16; using Logits = Parts<__bf16, 1>; using Grad = Parts<__bf16, 1>; };

__device__ __align__(256) unsigned char g_zero_page[256];

template <typename Img> struct Frag;
template <> struct Frag<_Float16> {
    using V = hx8;
    static __device__ inline fx4 mfma(V a, V b, fx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<__bf16> {
    using V = bx8;
    static __device__ inline fx4 mfma(V a, V b, fx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// ---------------------------------------------------------------- the tile product
// Bound by the matrix cores and, behind them, by the latency of loads: at 8192 x 4096 x 65536 in bfloat16 the two gradients run
// at 1.35 PFLOP/s and the logits, with their epilogue, at 1.22 (a library's plain product of this size: 1.45); counters at
// 4096 x 2048 x 32000: matrix cores busy 68 % and 61 % of the time, no bank conflict in LDS.  In float32, 2048 x 1024 x 32000, the
// products of parts run at 1.25 and 1.39 PFLOP/s, busy 68 % and 71 %.  Measured and not taken: 128 x 128
// tiles for the logits, two workgroups a CU (the whole call 5 % slower there, scores of 2048 x 1024 x 50001 14 %), four waves with 128 x 128 each (the accumulators
// spill into copies), stages of 32 k with longer rings, workgroups that keep their CU and walk over tiles (no overlap gained:
// all waves reach their epilogue together).
// TM x TN output tile, WM x WN waves, 16x16x32 matrix instructions, stages of 64 k of a pair of parts.  Each operand has a ring
// of stages in LDS, filled by loads that go from global memory straight there, 16 bytes a lane.
//   k contiguous in memory: LDS rows are 128 bytes of one m, eight 16-byte chunks, chunk c of row r at c ^ (r & 7), so the
//     sixteen rows of a fragment read (16 bytes a lane) spread over all banks;
//   k across the rows: LDS rows are one k, TM columns of the image; a fragment is read by the transposing load
//     (ds_read_b64_tr_b16: a group of sixteen lanes reads four k of sixteen columns, 8 bytes a lane, and lane i gets
//     column i's four k), 32-byte unit j of row k at j ^ unit_swizzle(k), so that the eight rows that half a wave reads
//     lie in different banks.
struct Operand {
    const void *p;       // image, or the caller's 16-bit tensor
    long long ld;        // row stride, elements
    long long rows;      // rows that exist; past them: k contiguous - any row, the result is not stored; k across - zero
    long long cols;      // columns that exist (a multiple of 8); past them zero
    int block;           // elements that 64 columns of all parts take
};

template <int TM, int TN, int WM, int WN>
struct TileShape {
    static constexpr int waves = WM * WN, threads = waves * 64;
    static constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
    // stages of A and of B in LDS: the 256 x 256 tile takes all of a CU's 160 KB, 128 x 128 leaves room for a second
    // workgroup; the tile for few rows, and 64 x 64 where there are few of them (one wave across m), do little but wait for
    // memory and keep more in flight (550 x 3717 x 488 with gradients, float32 190 -> 159 us, bfloat16 65 -> 55; where three workgroups fit a CU
    // they hide each other's waits, and longer rings cost 8 %: 974 x 2924 x 2167)
    static constexpr int ring_a = TN <= 32 ? 5 : TN == 64 && WM == 1 ? 4 : 3, ring_b = TN <= 32 ? 5 : TN == 64 && WM == 1 ? 4 : 2;
    static constexpr int bytes_a = TM * 128, bytes_b = TN * 128, lds_bytes = ring_a * bytes_a + ring_b * bytes_b;
};

typedef __attribute__((address_space(3))) void *lds_ptr;
typedef short sx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) sx4 *lds_sx4;

// One operand of a tile: T rows of m, k contiguous (TR false) or across the rows (TR true).  `groups` of 1024 LDS bytes, one
// load instruction of a wave each.
template <typename P, int T, bool TR>
struct Side {
    using V = typename Frag<typename P::Img>::V;
    static constexpr int groups = T / 8;
    static constexpr int row_bytes = TR ? T * 2 : 128, row_chunks = row_bytes / 16;
    static_assert(!TR || T % 64 == 0, "columns of an image come in blocks of 64");

    static __device__ inline int unit_swizzle(int k)
    {
        return row_bytes >= 256 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
    }
    // where block kb of k begins in memory, part 0, for a tile that starts at m0, how far a block is, and a part
    static __device__ inline const char *base(const Operand &O, long long m0, int kb)
    {
        return static_cast<const char *>(O.p) + (TR ? (long long)kb * 64 * O.ld + (m0 >> 6) * O.block : m0 * O.ld + (long long)kb * O.block) * 2;
    }
    static __device__ inline long long step(const Operand &O) { return TR ? O.ld * 128 : O.block * 2; }
    static constexpr int part_bytes = 128;
    // this lane's 16 bytes of group g: offset from the base and its k.  What lies past the last m repeats the last one: it
    // reaches only results that are not stored.
    static __device__ inline unsigned offset(const Operand &O, long long m0, int g, int lane, int *at)
    {
        const int c = g * 64 + lane, row = c / row_chunks, pos = c % row_chunks;
        if constexpr (TR) {
            long long col = m0 + (pos ^ (unit_swizzle(row) << 1)) * 8;
            if (col >= O.cols) col = O.cols - 8;
            *at = row;
            return (unsigned)((row * O.ld + ((col >> 6) - (m0 >> 6)) * O.block + (col & 63)) * 2);
        } else {
            const long long last = O.rows - 1 - m0;
            *at = (pos ^ (row & 7)) * 8;
            return (unsigned)(((row < last ? row : last) * O.ld + *at) * 2);
        }
    }
    static __device__ inline long long kcount(const Operand &O) { return TR ? O.rows : O.cols; }

    // fragment t (sixteen m), half h of the stage: k 32 h .. 32 h + 31
    static __device__ inline V read(const char *base, int lane, int t, int h)
    {
        if constexpr (TR) {
            const int g = lane >> 4, s = lane & 15, k = g * 8 + (s >> 2);
            const char *p = base + (32 * h + k) * row_bytes + ((t ^ unit_swizzle(k)) * 32) + (s & 3) * 8;
            union { sx4 q[2]; V v; } u;
            u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_sx4)p);
            u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_sx4)(p + 4 * row_bytes));
            return u.v;
        } else {
            return *reinterpret_cast<const V *>(base + (t * 16 + (lane & 15)) * 128 + (((h * 4 + (lane >> 4)) ^ (lane & 7)) * 16));
        }
    }
};

template <typename P, int TM, int TN, int WM, int WN, bool TA, bool TB>
struct TileProduct {
    using S = TileShape<TM, TN, WM, WN>;
    using F = Frag<typename P::Img>;
    using A_ = Side<P, TM, TA>;
    using B_ = Side<P, TN, TB>;
    static constexpr int kLoadsA = A_::groups / S::waves, kLoadsB = B_::groups / S::waves, kLoads = kLoadsA + kLoadsB;
    static constexpr int MH = S::MT / 2, RA = TA ? 2 : 1, RB = TB ? 2 : 1;       // LDS reads a fragment
    static_assert(A_::groups % S::waves == 0 && B_::groups % S::waves == 0, "every wave issues the same loads");

    // The end of a phase: everything read from LDS during it is there.
    static __device__ inline void phase_end()
    {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);                  // lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
    }
    // Spreads `reads` LDS reads over the first half of `products` matrix instructions.
    template <int products, int reads>
    static __device__ inline void interleave()
    {
        constexpr int each = products / reads / 2 > 0 ? products / reads / 2 : 1;
#pragma unroll
        for (int i = 0; i < reads; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, each, 0);
        }
    }
    // 16 bytes a lane from base + off to LDS at `to` + 16 lane.  Written out because the compiler, which cannot tell the
    // ring's places apart, would wait for all of these loads in front of every transposing read; what is read has arrived is
    // seen to by meet().  (No other instruction of these kernels uses m0.)  Buffer addressing: a scalar base that moves and a
    // 32-bit offset that stays, in range by construction.
    static __device__ inline void load_lds(const char *base, unsigned off, unsigned to)
    {
        typedef unsigned ux4 __attribute__((ext_vector_type(4)));
        const uint64_t at = reinterpret_cast<uint64_t>(base);
        const ux4 rsrc = {(unsigned)at, (unsigned)(at >> 32) & 0xFFFFu, 0xFFFFFFFFu, 0x00020000u};
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(rsrc) : "memory");
    }
    static __device__ inline void load_lds(const char *from, unsigned to)        // from an address of the lane's own
    {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
    }
    // Own reads done and all but the newest `left` of the own loads arrived; then everyone's.  (A barrier by itself does not
    // wait for loads that write LDS.)
    template <int left>
    static __device__ inline void meet()
    {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(left) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    // acc[mt][nt][i]: row wm*(TM/WM) + 16 mt + 4 (lane >> 4) + i of A, row wn*(TN/WN) + 16 nt + (lane & 15) of B.
    // Stages k0 .. k1 - 1 of ktotal, P::pairs of them a block of 64 k.  A stage has four phases, each with half of A's fragments
    // of half of its k; a phase reads the next one's fragments from LDS behind its own matrix instructions.  In front of
    // the fourth phase the waves meet: all hold the rest of the stage in registers, the next stage has arrived, and the
    // places of this one are free.  They are refilled a few loads at a time -- B's during the fourth and the next stage's
    // first phase, A's, whose ring is longer, during the two phases after that -- because a burst of loads holds up the
    // wave's matrix instructions behind it.
    static __device__ inline void run(fx4 (&acc)[S::MT][S::NT], const Operand &A, long long m0, const Operand &B, long long n0,
                                      int k0, int k1, int ktotal, char *lds)
    {
        if (k0 >= k1) return;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        unsigned off_a[kLoadsA], off_b[kLoadsB];
        int at_a[kLoadsA], at_b[kLoadsB];
#pragma unroll
        for (int i = 0; i < kLoadsA; i++) off_a[i] = A_::offset(A, m0, i * S::waves + wave, lane, &at_a[i]);
#pragma unroll
        for (int i = 0; i < kLoadsB; i++) off_b[i] = B_::offset(B, n0, i * S::waves + wave, lane, &at_b[i]);
        // next stage to load of either side: its block, its pair of parts, its place in memory and in the ring
        const char *block_a = A_::base(A, m0, k0 / P::pairs), *block_b = B_::base(B, n0, k0 / P::pairs);
        const long long step_a = A_::step(A), step_b = B_::step(B);
        int la = k0, lb = k0, qa = k0 % P::pairs, qb = qa, slot_a = 0, slot_b = 0;
        const char *base_a = block_a + P::of_a(qa) * A_::part_bytes, *base_b = block_b + P::of_b(qb) * B_::part_bytes;
        char *lds_b = lds + S::ring_a * S::bytes_a;
        const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)lds + wave * 1024;
        // load i of the next stage
        auto load = [&](auto side_a, int i) {
            if constexpr (side_a.value) load_lds(base_a, off_a[i], lds0 + slot_a * S::bytes_a + i * S::waves * 1024);
            else load_lds(base_b, off_b[i], lds0 + S::ring_a * S::bytes_a + slot_b * S::bytes_b + i * S::waves * 1024);
        };
        // a whole stage; the stages of the last block have zeros past the end of k
        const int last_block = (ktotal / P::pairs - 1) * 64;
        auto load_stage = [&](auto side_a, bool last) {
            constexpr bool a_side = side_a.value;
            constexpr int loads = a_side ? kLoadsA : kLoadsB;
            if (!last) {
#pragma unroll
                for (int i = 0; i < loads; i++) load(side_a, i);
            } else {
                const char *base = a_side ? base_a : base_b;
                const unsigned to = lds0 + (a_side ? slot_a * S::bytes_a : S::ring_a * S::bytes_a + slot_b * S::bytes_b);
                const long long left = (a_side ? A_::kcount(A) : B_::kcount(B)) - last_block;
#pragma unroll
                for (int i = 0; i < loads; i++) {
                    const char *p = base + (a_side ? off_a[i] : off_b[i]);
                    if ((a_side ? at_a[i] : at_b[i]) >= left) p = reinterpret_cast<const char *>(g_zero_page);
                    load_lds(p, to + i * S::waves * 1024);
                }
            }
        };
        constexpr std::true_type side_a{};
        constexpr std::false_type side_b{};
        auto next_a = [&]() {
            la++;
            if (++qa == P::pairs) { qa = 0; block_a += step_a; }
            base_a = block_a + P::of_a(qa) * A_::part_bytes;
            slot_a = slot_a + 1 == S::ring_a ? 0 : slot_a + 1;
        };
        auto next_b = [&]() {
            lb++;
            if (++qb == P::pairs) { qb = 0; block_b += step_b; }
            base_b = block_b + P::of_b(qb) * B_::part_bytes;
            slot_b = slot_b + 1 == S::ring_b ? 0 : slot_b + 1;
        };
        auto whole_a = [&](int before) { if (la < min(k1, before)) { load_stage(side_a, la + P::pairs >= ktotal); next_a(); } };
        auto whole_b = [&](int before) { if (lb < min(k1, before)) { load_stage(side_b, lb + P::pairs >= ktotal); next_b(); } };
        // a wave's part of a side begins a whole number of rows or 32-byte units into it
        const int oa = TA ? 0 : wm * (TM / WM) * 128, ob = TB ? 0 : wn * (TN / WN) * 128;
        const int ta = TA ? wm * S::MT : 0, tb = TB ? wn * S::NT : 0;
        typename F::V a[2][MH], b[2][S::NT];
        int ra = 0, rb = 0;                                   // ring places that are being read
        // fragments of phase p of a stage
        auto read_a = [&](int slot, int p) {
            const char *pa = lds + slot * S::bytes_a + oa;
#pragma unroll
            for (int t = 0; t < MH; t++) a[p & 1][t] = A_::read(pa, lane, ta + (p & 1) * MH + t, p >> 1);
        };
        auto read_b = [&](typename F::V (&to)[S::NT], int slot, int h) {
            const char *pb = lds_b + slot * S::bytes_b + ob;
#pragma unroll
            for (int t = 0; t < S::NT; t++) to[t] = B_::read(pb, lane, tb + t, h);
        };
        constexpr int PP = MH * S::NT;
        // matrix instructions i0 .. i1 - 1 of phase p
        auto products = [&](int p, int i0, int i1) {
            const int half = p & 1, h = p >> 1;
#pragma unroll
            for (int mt = 0; mt < MH; mt++)
#pragma unroll
                for (int nt = 0; nt < S::NT; nt++)
                    if (mt * S::NT + nt >= i0 && mt * S::NT + nt < i1)
                        acc[half * MH + mt][nt] = F::mfma(a[p & 1][mt], b[h][nt], acc[half * MH + mt][nt]);
        };
        // phase p's matrix instructions behind its `reads` LDS reads, with loads l0 .. l1 - 1 of the next stage of a side near their end
        auto phase = [&](int p, auto reads, auto side, auto l0, auto l1) {
            constexpr int loads = l1.value - l0.value, per = loads ? loads : 1, tail = PP - 2 * loads > 0 ? PP - 2 * loads : 0;
            products(p, 0, tail);
            interleave<tail, reads.value>();
#pragma unroll
            for (int i = 0; i < loads; i++) {
                __builtin_amdgcn_sched_barrier(0);
                load(side, l0.value + i);
                __builtin_amdgcn_sched_barrier(0);
                products(p, tail + (PP - tail) * i / per, tail + (PP - tail) * (i + 1) / per);
            }
            phase_end();
        };
        // fill the rings in the order of the loop's loads and wait for the first stage
        whole_a(k1);
        if (S::ring_b == S::ring_a) whole_b(k1);
#pragma unroll
        for (int i = 1; i < S::ring_a; i++) {
            if (S::ring_b == S::ring_a || i > S::ring_a - 1 - S::ring_b) whole_b(k1);
            whole_a(k1);
        }
        if (k1 - k0 >= S::ring_a) meet<(S::ring_a - 1) * kLoadsA + (S::ring_b - 1) * kLoadsB>();
        else meet<0>();
        read_b(b[0], 0, 0);
        read_a(0, 0);
        int kt = k0;
        constexpr int B1 = kLoadsB / 2, A1 = kLoadsA / 2;
        // loads issued after the later of the two that the next stage needs
        constexpr int newer = S::ring_a > S::ring_b ? kLoadsA + (S::ring_b - 2) * kLoads : (S::ring_a - 2) * kLoads;
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
#define AZG_INT(v) std::integral_constant<int, v>{}
        auto stage = [&](auto fast_, auto full_) {            // fast: with the loads of a steady state; full: the rings are
            constexpr bool fast = fast_.value, full = full_.value;
            const int sa = ra + 1 == S::ring_a ? 0 : ra + 1, sb = rb + 1 == S::ring_b ? 0 : rb + 1;
            read_a(ra, 1);
            phase(0, AZG_INT(MH * RA), side_b, AZG_INT(B1), AZG_INT(fast ? kLoadsB : B1));
            if (fast) next_b();
            read_a(ra, 2);
            read_b(b[1], rb, 1);
            phase(1, AZG_INT(MH * RA + S::NT * RB), side_a, AZG_INT(0), AZG_INT(fast ? A1 : 0));
            read_a(ra, 3);
            phase(2, AZG_INT(MH * RA), side_a, AZG_INT(A1), AZG_INT(fast ? kLoadsA : A1));
            if (fast) next_a();
            meet<full ? newer : 0>();
            // (after the last stage what is read is stale and not used)
            read_a(sa, 0);
            read_b(b[0], sb, 0);
            phase(3, AZG_INT(MH * RA + S::NT * RB), side_b, AZG_INT(0), AZG_INT(fast ? B1 : 0));
            ra = sa; rb = sb;
            kt++;
        };
        // The fast loop's stage kt issues the rest of B's stage kt - 1 + ring_b, all of A's kt - 1 + ring_a and the first part of
        // B's kt + ring_b; around it: the first stage's loads in one go, whole stages, and the rest of a begun one.
        const bool tail = A_::kcount(A) % 64 != 0 || B_::kcount(B) % 64 != 0;
        const int end = tail ? min(k1, ktotal - P::pairs) : k1, fast_end = min(end - S::ring_a + 1, end - S::ring_b);
        if (kt + 1 < fast_end) {
            stage(no, yes);
#pragma unroll
            for (int i = 0; i < B1; i++) load(side_b, i);
            while (kt < fast_end) stage(yes, yes);
#pragma unroll
            for (int i = B1; i < kLoadsB; i++) load(side_b, i);
            next_b();
        }
        while (kt < k1) {
            whole_b(kt + S::ring_b);
            whole_a(kt + S::ring_a);
            stage(no, no);
        }
#undef AZG_INT
        __syncthreads();
    }
};

// Workgroup number -> place in a list of `total`.  Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its
// own: an XCD gets a contiguous run of the list.
__device__ inline unsigned xcd_run(unsigned wg, unsigned total)
{
    const unsigned per = total / 8, rest = total % 8, x = wg % 8;
    return x * per + (x < rest ? x : rest) + wg / 8;
}
// The list of a product's tiles walks in strips of STRIP tiles of m, so that the tiles in flight on an XCD (32, or 16 where two
// products share a launch) share rows of both operands: 8 for the logits (4: 2 % slower at 2048 x 1024 x 50001), 4 for the
// gradients (8: 1 % slower at 8192 x 4096 x 65536).
template <int STRIP>
__device__ inline void tile_at(unsigned t, int mt, int nt, int *m, int *n)
{
    const unsigned strip = t / (unsigned)(STRIP * nt), first = strip * STRIP;
    const unsigned h = min((unsigned)STRIP, (unsigned)mt - first), in = t - strip * STRIP * nt;
    *m = (int)(first + in % h);
    *n = (int)(in / h);
}

// ---------------------------------------------------------------- images
template <typename T, int N> struct __attribute__((packed)) Pack { T v[N]; };      // N elements of any alignment

struct PackArgs {
    const void *src;              // [rows][cols], stride ld
    long long ld, rows, cols;
    void *img;                    // [rows][ldi]
    long long ldi, icols;         // row stride (image elements), padded columns
    int parts;                    // 1: elements as they are; else bfloat16 parts
    const long long *target;      // not null: rows whose target is ignore_index are read as zero
    long long ignore;
    unsigned wgs;                 // workgroups of this one
};
struct PackList { PackArgs p[4]; };

// N bfloat16 parts of x: part[i] is the rounding of x - part[0] - ... - part[i - 1], exact in float32.  What would round to
// infinity takes the largest finite number; infinities and NaN are part 0.
template <int N>
__device__ inline void split_parts(float x, __bf16 (&part)[N])
{
    constexpr float top = 3.3895313892515355e38f;             // (2 - 2^-7) 2^127
#pragma unroll
    for (int i = 0; i < N; i++) {
        __bf16 h = (__bf16)x;
        if (i == 0 && fabsf(x) < INFINITY && fabsf((float)h) == INFINITY) h = (__bf16)copysignf(top, x);
        part[i] = h;
        x = fabsf(x) < INFINITY ? x - (float)h : 0.f;
    }
}

// Images of up to four matrices, zeros in the padding: a thread eight columns of a row.  Bound by memory: 139 MB of float32
// read and 209 MB of parts written in 53 us, 6.5 TB/s.
template <typename In>
__global__ __launch_bounds__(256) void pack_kernel(PackList list)
{
    unsigned wg = blockIdx.x;
    int which = 0;
    while (wg >= list.p[which].wgs) wg -= list.p[which++].wgs;
    const PackArgs a = list.p[which];
    const long long row_chunks = a.icols / 8, total = a.rows * row_chunks;
    for (long long i = (long long)wg * 256 + threadIdx.x; i < total; i += (long long)a.wgs * 256) {
        const long long r = i / row_chunks, c = (i - r * row_chunks) * 8;
        const In *p = static_cast<const In *>(a.src) + r * a.ld + c;
        const bool skip = a.target && a.target[r] == a.ignore;
        In v[8];
        if (!skip && c + 8 <= a.cols) {
            *reinterpret_cast<Pack<In, 8> *>(v) = *reinterpret_cast<const Pack<In, 8> *>(p);
        } else {
#pragma unroll
            for (int q = 0; q < 8; q++) {
                v[q] = (In)0.f;
                if (!skip && c + q < a.cols) v[q] = p[q];
            }
        }
        auto in_parts = [&](auto n) {
            constexpr int N = decltype(n)::value;
            __bf16 *o = static_cast<__bf16 *>(a.img) + r * a.ldi + (c >> 6) * (64 * N) + (c & 63);
            bx8 h[N];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                __bf16 part[N];
                split_parts<N>((float)v[q], part);
#pragma unroll
                for (int k = 0; k < N; k++) h[k][q] = part[k];
            }
#pragma unroll
            for (int k = 0; k < N; k++) *reinterpret_cast<bx8 *>(o + k * 64) = h[k];
        };
        if constexpr (sizeof(In) == 4) in_parts(std::integral_constant<int, 3>{});
        else if (std::is_same_v<In, _Float16> && a.parts == 2) in_parts(std::integral_constant<int, 2>{});
        else *reinterpret_cast<Pack<In, 8> *>(static_cast<In *>(a.img) + r * a.ldi + c) = *reinterpret_cast<const Pack<In, 8> *>(v);
    }
}

// ---------------------------------------------------------------- logits: statistics or gradient
struct CeArgs {
    Operand w, x;                 // classes (of this piece) x k, rows x k
    int ktiles, mtiles, ntiles, mtiles_behind;
    long long n, classes, v0;     // classes of this piece; v0 = first class of the piece
    const void *bias;             // this piece's, operand type, or null
    const long long *target;
    long long ignore;
    const float *probs;           // [n][ldp], already offset to the piece's first class
    long long ldp;
    // statistics, one entry a row and a wave's run of TM / WM classes ("span")
    float2 *part;                 // [spans][n]: maximum m, sum of exp(l - m)
    float *part_e;                // [spans][n]: sum of exp(l - m) (l - m), or null
    float2 *part_t;               // probabilities: sum pi (l - m), sum pi
    float *tlogit;                // index: [n]
    // gradient
    const float4 *stats;          // [n]: m, sum pi / s, ... (RowArgs)
    const float *rowg;            // [n]
    void *d;                      // image [n][ldd] of D; statistics: of exp(l - the span's maximum), or null
    long long ldd, dcols;         // row stride in image elements; padded classes
    float *dbpart;                // [ntiles][classes] or null
};

// four probabilities of a row from class v, zeros past the last class
__device__ inline Pack<float, 4> four_of(const float *row, long long v, long long classes, bool whole)
{
    if (whole) return *reinterpret_cast<const Pack<float, 4> *>(row + v);
    Pack<float, 4> p;
#pragma unroll
    for (int i = 0; i < 4; i++) p.v[i] = row[min(v + i, classes - 1)];
#pragma unroll
    for (int i = 0; i < 4; i++) p.v[i] = v + i < classes ? p.v[i] : 0.f;
    return p;
}

// exp(l - the span's maximum) on its way to becoming D in the same place: float32 where D will be parts.  Where D will be 16
// bits it is a code of 16 bits, which D's own rounding to 8 bits lets it be, with float32's range: a number from 2^-39 to 1
// keeps ten bits after its first (off by 2^-11 of itself at most), one below keeps eight (2^-9); the codes of both run on from
// each other.  (Half precision, which this was, has nothing below 2^-24.)
template <typename Op> using Expo = std::conditional_t<Op::Grad::parts == 1, uint16_t, float>;
constexpr uint32_t kFine = 88u << 23, kFineCodes = (kFine >> 13) - (kFine >> 15);        // 2^-39
template <typename E>
__device__ inline E expo(float x)                             // 0 <= x <= 1; a NaN: any code (the row's factor is NaN)
{
    if constexpr (sizeof(E) == 4) return x;
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return (E)(b >= kFine ? ((b + (1u << 12)) >> 13) - kFineCodes : (b + (1u << 14)) >> 15);
}
__device__ inline float expo_of(float e) { return e; }
__device__ inline float expo_of(uint16_t e)
{
    return __builtin_bit_cast(float, e >= kFine >> 15 ? ((uint32_t)e + kFineCodes) << 13 : (uint32_t)e << 15);
}
// where the image of D (the exponentials on their way there: counted in their own size) holds column c
template <typename Op, typename T>
__device__ inline T *place(void *d, long long row, long long ldd, long long c)
{
    return reinterpret_cast<T *>(static_cast<uint16_t *>(d) + row * ldd + (c >> 6) * Op::Grad::block) + (c & 63);
}

// A tile of logits; a lane holds four classes of a row next to each other (classes are the tile's m), sixteen rows a fragment.
// Forward (GRAD false): span statistics and, where asked for, the exponentials; GRAD: D from the rows' statistics.  A 256 x 256
// tile takes 10 us around one stage of 64 features (2048 x 64 x 49152: 60 us, six rounds; with a bias 10.7): filling the
// rings and this epilogue, an exponential an element on top of the maximum, the sum and the stores; and 1.1 us a stage more.
template <typename Op, int TM, int TN, int WM, int WN, bool GRAD>
__device__ inline void logits_tile(const CeArgs &a, long long m_first, int span_first, int mtiles, int ntiles, unsigned wg, char *lds)
{
    using S = TileShape<TM, TN, WM, WN>;
    int tm, tn;
    tile_at<8>(xcd_run(wg, (unsigned)mtiles * ntiles), mtiles, ntiles, &tm, &tn);
    const long long m0 = m_first + (long long)tm * TM, n0 = (long long)tn * TN;
    fx4 acc[S::MT][S::NT];
#pragma unroll
    for (int i = 0; i < S::MT; i++)
#pragma unroll
        for (int j = 0; j < S::NT; j++) acc[i][j] = fx4{0.f, 0.f, 0.f, 0.f};
    TileProduct<typename Op::Logits, TM, TN, WM, WN, false, false>::run(acc, a.w, m0, a.x, n0, 0, a.ktiles, a.ktiles, lds);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const typename Op::In *bias = static_cast<const typename Op::In *>(a.bias);
    const long long vw = m0 + wm * (TM / WM) + 4 * (lane >> 4);                  // this lane's first class of the piece
    // (what the rows and classes bring along is loaded in one go: each load by itself would cost its latency)
    const bool whole = m0 + TM <= a.classes;
    if (bias || !whole) {
        typename Op::In bv[S::MT][4];
        if (bias && whole) {
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++) *reinterpret_cast<Pack<typename Op::In, 4> *>(bv[mt]) = *reinterpret_cast<const Pack<typename Op::In, 4> *>(bias + vw + mt * 16);
        } else if (bias) {
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) bv[mt][i] = bias[min(vw + mt * 16 + i, a.classes - 1)];
        }
#pragma unroll
        for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float b = bias ? (float)bv[mt][i] : 0.f;
#pragma unroll
                for (int nt = 0; nt < S::NT; nt++) acc[mt][nt][i] += b;
            }
        if (!whole)
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (vw + mt * 16 + i >= a.classes)
#pragma unroll
                        for (int nt = 0; nt < S::NT; nt++) acc[mt][nt][i] = -INFINITY;
    }
    const long long nw = n0 + wn * (TN / WN) + (lane & 15);
    const long long dpad = a.dcols;
    int tt[S::NT];                                            // the rows' targets, counted from vw; -1: none of this span's classes
#pragma unroll
    for (int nt = 0; nt < S::NT; nt++) tt[nt] = -1;
    if (a.target) {
        const long long left = min(a.classes - vw, (long long)(TM / WM));
#pragma unroll
        for (int nt = 0; nt < S::NT; nt++) {
            const long long t = a.target[min(nw + nt * 16, a.n - 1)] - a.v0 - vw;
            tt[nt] = t >= 0 && t < left ? (int)t : -1;
        }
    }
    if constexpr (!GRAD) {
        // per row: maximum and sum over the span; lanes 16 and 32 apart share a row
        using E = Expo<Op>;
#pragma unroll
        for (int nt = 0; nt < S::NT; nt++) {
            const long long row = nw + nt * 16;
            const bool live = row < a.n;
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, acc[mt][nt][i]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            // Everything is summed relative to the maximum, which enters unrounded: exp(l - m) is 1 at the maximum, so a sum is at
            // least 1, a loss and an entropy at least 0, and neither loses bits to an offset that all logits share.
            // (A NaN is passed over by fmaxf: it comes back through the sum; a maximum of -inf leaves every term 2^-inf.)
            const float base = mx == -INFINITY ? 0.f : mx;
            float s = 0.f, e = 0.f, tl = 0.f, ts = 0.f;
            if (a.part_e)
#pragma unroll
                for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float d = acc[mt][nt][i] - base, x = __builtin_amdgcn_exp2f(d * kLog2e);
                        e += x != 0.f ? x * d : 0.f;
                    }
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = __builtin_amdgcn_exp2f((acc[mt][nt][i] - base) * kLog2e);
                    s += x[i];
                }
                if (a.d && live && vw + mt * 16 < dpad) {
                    Pack<E, 4> keep;
#pragma unroll
                    for (int i = 0; i < 4; i++) keep.v[i] = expo<E>(x[i]);
                    *reinterpret_cast<Pack<E, 4> *>(place<Op, E>(a.d, row, a.ldd, vw + mt * 16)) = keep;
                }
            }
            if (a.probs) {
                const float *pr = a.probs + min(row, a.n - 1) * a.ldp;
                Pack<float, 4> pv[S::MT];
#pragma unroll
                for (int mt = 0; mt < S::MT; mt++) pv[mt] = four_of(pr, vw + mt * 16, a.classes, whole);
#pragma unroll
                for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = pv[mt].v[i];
                        ts += p;
                        tl += p != 0.f ? p * (acc[mt][nt][i] - base) : 0.f;
                    }
            }
            if (tt[nt] >= 0 && live) {
                float l = 0.f;
#pragma unroll
                for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) l = tt[nt] == mt * 16 + i ? acc[mt][nt][i] : l;
                // (a lane has four classes of every sixteen)
                if ((tt[nt] & 15) < 4) a.tlogit[row] = l;
            }
#define AZG_PAIR(v) v += __shfl_xor(v, 16, 64); v += __shfl_xor(v, 32, 64)
            AZG_PAIR(s);
            if (a.part_e) { AZG_PAIR(e); }
            if (a.probs) { AZG_PAIR(tl); AZG_PAIR(ts); }
#undef AZG_PAIR
            if (lane < 16 && live) {
                const long long at = (span_first + (long long)tm * WM + wm) * a.n + row;
                a.part[at] = make_float2(mx, s);
                if (a.part_e) a.part_e[at] = e;
                if (a.probs) a.part_t[at] = make_float2(tl, ts);
            }
        }
    } else {
        using Img = typename Op::Grad::Img;
        float db[S::MT][4], gs[S::NT];
        float2 sts[S::NT];
#pragma unroll
        for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) db[mt][i] = 0.f;
#pragma unroll
        for (int nt = 0; nt < S::NT; nt++) {
            const long long row = min(nw + nt * 16, a.n - 1);
            sts[nt] = *reinterpret_cast<const float2 *>(a.stats + row);
            gs[nt] = a.rowg[row];
        }
#pragma unroll
        for (int nt = 0; nt < S::NT; nt++) {
            const long long row = nw + nt * 16;
            const bool live = row < a.n;
            const float2 st = sts[nt];
            const float g = live ? gs[nt] : 0.f;
            const int t = tt[nt];
            const float *pr = a.probs ? a.probs + min(row, a.n - 1) * a.ldp : nullptr;
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++) {
                constexpr int N = Op::Grad::parts;
                Pack<Img, 4> h[N];
                const long long cls = vw + mt * 16;
                Pack<float, 4> pv;
                if (pr) pv = four_of(pr, cls, a.classes, whole);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float q = __builtin_amdgcn_exp2f((acc[mt][nt][i] - st.x) * kLog2e) * st.y;
                    if (pr) q -= pv.v[i];
                    else if (t == mt * 16 + i) q -= 1.f;
                    q = g == 0.f || cls + i >= a.classes ? 0.f : q * g;         // a row that counts for nothing: zero whatever it holds
                    db[mt][i] += q;
#pragma unroll
                    for (int k = 0; k < N; k++) { h[k].v[i] = (Img)q; q -= (float)h[k].v[i]; }
                }
                if (a.d && live && cls < dpad) {
                    Img *o = place<Op, Img>(a.d, row, a.ldd, cls);
#pragma unroll
                    for (int k = 0; k < N; k++) *reinterpret_cast<Pack<Img, 4> *>(o + k * 64) = h[k];
                }
            }
        }
        if (a.dbpart) {
            float *sm = reinterpret_cast<float *>(lds);                         // [WN][TM]; the stages are done with
#pragma unroll
            for (int mt = 0; mt < S::MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float s = db[mt][i];
                    s += __shfl_xor(s, 1, 64); s += __shfl_xor(s, 2, 64); s += __shfl_xor(s, 4, 64); s += __shfl_xor(s, 8, 64);
                    if ((lane & 15) == 0) sm[wn * TM + wm * (TM / WM) + mt * 16 + 4 * (lane >> 4) + i] = s;
                }
            __syncthreads();
            for (int v = tid; v < TM; v += S::threads)
                if (m0 + v < a.classes) {
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < WN; w++) s += sm[w * TM + v];
                    a.dbpart[(long long)tn * a.classes + m0 + v] = s;
                }
        }
    }
}

template <typename Op, int TM, int TN, int WM, int WN, bool GRAD>
__global__ __launch_bounds__(WM * WN * 64) void logits_kernel(CeArgs a)
{
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    logits_tile<Op, TM, TN, WM, WN, GRAD>(a, 0, 0, a.mtiles, a.ntiles, blockIdx.x, lds);
}
// The loss alone, where 256 x 256 tiles of all classes would leave the last round of the CUs mostly empty: whole rounds of them,
// and 128 x 128 tiles of the classes behind.  2048 x 1024 x 50001: 1536 and 112 tiles, 206 us instead of 218.
template <typename Op>
__global__ __launch_bounds__(512) void logits_mixed_kernel(CeArgs a)
{
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const unsigned large = (unsigned)a.mtiles * a.ntiles;
    if (blockIdx.x < large) logits_tile<Op, 256, 256, 2, 4, false>(a, 0, 0, a.mtiles, a.ntiles, blockIdx.x, lds);
    else logits_tile<Op, 128, 128, 2, 4, false>(a, a.mtiles * 256LL, a.mtiles * 2, a.mtiles_behind, (int)((a.n + 127) / 128), blockIdx.x - large, lds);
}

// ---------------------------------------------------------------- rows and totals
struct RowArgs {
    long long n, classes;
    int spans;
    const float2 *part; const float *part_e; const float2 *part_t; const float *tlogit;
    const long long *target; long long ignore;
    float *loss_out, *ent_out;    // [n], or null: rows' results that nothing else has to be added to
    float4 *stats;                // [n]: m, sum pi / s, 0, loss with lse = m + log s (so that p takes no rounding of lse)
    float *ent;                   // [n] or null
};
// One wave per row: join the spans' sums, each relative to its span's maximum m_j, in a fixed order; relative to m they are
// s_j f, (e_j + (m_j - m) s_j) f and t_j + (m_j - m) sum pi, f = exp(m_j - m).  Latency: 9 us for 2048 rows of 392 spans, 8 us for
// one row of 2048.
__device__ inline void shift(float m, float base, float &s, float &e, float &tl, float ts)
{
    const float from = m == -INFINITY ? 0.f : m, d = from - base, f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(d * kLog2e);
    e = f != 0.f ? (e + d * s) * f : 0.f;                     // (d may be as low as the type's lowest value)
    s *= f;
    tl += ts != 0.f ? d * ts : 0.f;
}
__global__ __launch_bounds__(256) void rows_kernel(RowArgs a)
{
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.n) return;
    float mx = -INFINITY, s = 0.f, e = 0.f, tl = 0.f, ts = 0.f;
    // four spans a lane at a time: their maximum first, so that the loads do not wait for the sums
    for (int t0 = lane; t0 < a.spans; t0 += 256) {
        float2 p[4];
        float q[4];
        float2 u[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool in = t0 + 64 * j < a.spans;
            const long long at = (long long)(in ? t0 + 64 * j : t0) * a.n + row;
            p[j] = a.part[at];
            q[j] = a.part_e ? a.part_e[at] : 0.f;
            u[j] = a.part_t ? a.part_t[at] : make_float2(0.f, 0.f);
            if (!in) { p[j] = make_float2(-INFINITY, 0.f); q[j] = 0.f; u[j] = make_float2(0.f, 0.f); }
        }
        const float m = fmaxf(fmaxf(mx, fmaxf(p[0].x, p[1].x)), fmaxf(p[2].x, p[3].x)), base = m == -INFINITY ? 0.f : m;
        // (a span without a class counts from 0 and adds nothing; a NaN sum stays NaN)
        shift(mx, base, s, e, tl, ts);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            shift(p[j].x, base, p[j].y, q[j], u[j].x, u[j].y);
            s += p[j].y; e += q[j]; tl += u[j].x; ts += u[j].y;
        }
        mx = m;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float om = __shfl_xor(mx, d, 64);
        float os = __shfl_xor(s, d, 64), oe = __shfl_xor(e, d, 64), ot = 0.f, op = 0.f;
        if (a.part_t) { ot = __shfl_xor(tl, d, 64); op = __shfl_xor(ts, d, 64); }
        const float m = fmaxf(mx, om), base = m == -INFINITY ? 0.f : m;
        shift(mx, base, s, e, tl, ts);
        shift(om, base, os, oe, ot, op);
        s += os; e += oe; tl += ot; ts += op; mx = m;
    }
    if (lane) return;
    const float ls = logf(s), m = mx == -INFINITY ? 0.f : mx;
    float loss, ent = ls - e / s;
    if (a.target) {
        const long long t = a.target[row];
        ts = 1.f;
        if (t == a.ignore) loss = ent = ts = 0.f;
        else if (t < 0 || t >= a.classes) loss = ent = ts = NAN;
        else loss = (m - a.tlogit[row]) + ls;
    } else {
        loss = ls * ts - tl;
    }
    a.stats[row] = make_float4(mx, ts / s, 0.f, loss);
    if (a.ent) a.ent[row] = ent;
    if (a.loss_out) a.loss_out[row] = loss;
    if (a.ent_out) a.ent_out[row] = ent;
}

struct RowSums { double loss, ent, count; };
constexpr int kMaxSums = 256;                 // a multiple of 64, at most 1024
constexpr long long kOneTotal = 8192;         // rows that one workgroup adds up in no more time than another launch takes

// sum over a workgroup of W waves in a fixed order, for every thread
template <int W>
__device__ inline RowSums join_sums(RowSums v, RowSums *red)
{
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        v.loss += __shfl_xor(v.loss, s, 64); v.ent += __shfl_xor(v.ent, s, 64); v.count += __shfl_xor(v.count, s, 64);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < W; w++) { v.loss += red[w].loss; v.ent += red[w].ent; v.count += red[w].count; }
    return v;
}

struct TotalArgs {
    long long n;
    RowSums *sums;                // null, or kMaxSums sums over the rows to take instead of the rows
    int reduction;                // 0 none, 1 sum, 2 mean
    const float4 *stats; const float *ent;
    const long long *target; long long ignore;
    float *loss, *ent_out;        // [1]; null: not asked for
    const float *dloss;           // [n], [1] or null
    float grad_scale;
    float *rowg;                  // [n]: g_i, 0 for rows that count for nothing; null: they are 1 and 0 (class numbers and a common
                                  // g, which is `factor`) or no gradient is asked for
    float *factor;                // [1]: the common g, or 1; null without a backward pass
};
// What the rows add up to, W waves: losses, entropies, rows that count.  A fixed order, in double.
template <int W>
__device__ inline RowSums row_sums(const TotalArgs &a, long long first, long long step)
{
    __shared__ RowSums red[W];
    RowSums s{0.0, 0.0, 0.0};
#pragma unroll 4
    for (long long i = first; i < a.n; i += step) {
        const float4 st = a.stats[i];
        const bool used = !(a.target && a.target[i] == a.ignore);
        s.loss += st.w; s.count += used ? 1.0 : 0.0;
        if (a.ent) s.ent += a.ent[i];
    }
    return join_sums<W>(s, red);
}
// for many rows (more than kOneTotal): the sums of a workgroup's share of them
__global__ __launch_bounds__(256) void sums_kernel(TotalArgs a)
{
    const RowSums s = row_sums<4>(a, (long long)blockIdx.x * 256 + threadIdx.x, (long long)kMaxSums * 256);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = s;
}
// The totals, and the rows' gradient factors; the first of `wgs` workgroups writes the totals.
template <int THREADS>
__device__ inline void totals(const TotalArgs &a, unsigned wg, unsigned wgs)
{
    constexpr int W = THREADS / 64;
    const int tid = threadIdx.x;
    float common = 1.f;
    if (a.reduction) {
        RowSums s;
        if (a.sums) {
            __shared__ RowSums red[W];
            s = tid < kMaxSums ? a.sums[tid] : RowSums{0.0, 0.0, 0.0};
            s = join_sums<W>(s, red);
        } else {
            s = row_sums<W>(a, tid, THREADS);
        }
        const double by = a.reduction == 2 ? (s.count > 0.0 ? 1.0 / s.count : 0.0) : 1.0;
        if (wg == 0 && tid == 0) {
            if (a.loss) a.loss[0] = (float)(s.loss * by);
            if (a.ent_out) a.ent_out[0] = (float)(s.ent * by);
        }
        common = (a.dloss ? a.dloss[0] : 1.f) * a.grad_scale * (float)by;
    }
    if (!a.factor) return;
    if (a.rowg)
        for (long long i = (long long)wg * THREADS + tid; i < a.n; i += (long long)wgs * THREADS) {
            const bool used = !(a.target && a.target[i] == a.ignore);
            const float g = a.reduction ? 1.f : (a.dloss ? a.dloss[i] : 1.f) * a.grad_scale;
            a.rowg[i] = used ? g : 0.f;
        }
    if (wg == 0 && tid == 0) a.factor[0] = common;
}
__global__ __launch_bounds__(1024) void totals_kernel(TotalArgs a) { totals<1024>(a, blockIdx.x, gridDim.x); }

// ---------------------------------------------------------------- exponentials -> D, in place
constexpr int kFixCols = 512;
struct FixArgs {
    long long n, classes;
    int rows;                     // a workgroup's, a multiple of 4
    TotalArgs totals;             // the last row of workgroups does these instead (rowg null), or has n < 0
    int span;                     // classes an entry of part stands for
    void *d; long long ldd, dcols;
    const float2 *part; const float4 *stats; const float *rowg;
    const long long *target; long long ignore;
    const float *probs; long long ldp;
    float *dbpart;                // [runs of `rows`][classes] or null
};
// `rows` rows x 512 classes per workgroup; a wave takes a row at a time, a lane eight classes of it.  Bound by memory: 2 bytes
// (float32: 4) read and written an element, 4096 x 32000 in 111 us, 4.7 TB/s.
template <typename Op>
__global__ __launch_bounds__(256) void fix_kernel(FixArgs a)
{
    using Img = typename Op::Grad::Img;
    using E = Expo<Op>;
    constexpr int N = Op::Grad::parts;
    typedef E ex8 __attribute__((ext_vector_type(8)));
    __shared__ float red[4][kFixCols];
    if (a.totals.n >= 0 && blockIdx.y == gridDim.y - 1) {
        if (blockIdx.x == 0) totals<256>(a.totals, 0, 1);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const long long c0 = (long long)blockIdx.x * kFixCols, c = c0 + lane * 8;
    const long long r0 = (long long)blockIdx.y * a.rows;
    const float2 *part = a.part + (c < a.classes ? c : 0) / a.span * a.n;
    float db[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int j = 0; j < a.rows / 4; j++) {
        const long long row = r0 + j * 4 + wave;
        if (row >= a.n) break;
        const float4 st = a.stats[row];
        const long long cls = a.target ? a.target[row] : -1, t = a.target ? cls - c : -1;
        const float g = a.rowg ? a.rowg[row] : (a.target && cls == a.ignore ? 0.f : 1.f);
        if (c >= a.dcols) continue;
        // (a span with every class blocked: zeros, but NaN where the row has no other span or no finite loss)
        const float mp = part[row].x, f = (mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mp - st.x) * kLog2e)) * st.y;
        const ex8 v = *reinterpret_cast<const ex8 *>(place<Op, E>(a.d, row, a.ldd, c));
        // (parts land on exponentials of the same 64 columns that other lanes of this wave read: no store moves in front of the loads)
        if constexpr (N > 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        Pack<float, 8> pv;
        if (a.probs) {
            const float *pr = a.probs + row * a.ldp + c;
            if (c + 8 <= a.classes) pv = *reinterpret_cast<const Pack<float, 8> *>(pr);
            else
#pragma unroll
                for (int i = 0; i < 8; i++) pv.v[i] = c + i < a.classes ? pr[i] : 0.f;
        }
        typename Frag<Img>::V h[N];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool out = c + i >= a.classes;
            float q = expo_of((E)v[i]) * f;
            if (a.probs) q -= pv.v[i];
            else if (t == i) q -= 1.f;
            q = g == 0.f || out ? 0.f : q * g;                                  // a row that counts for nothing: zero whatever it holds
            db[i] += q;
#pragma unroll
            for (int k = 0; k < N; k++) { h[k][i] = (Img)q; q -= (float)h[k][i]; }
        }
        Img *o = place<Op, Img>(a.d, row, a.ldd, c);
#pragma unroll
        for (int k = 0; k < N; k++) *reinterpret_cast<typename Frag<Img>::V *>(o + k * 64) = h[k];
    }
    if (!a.dbpart) return;
#pragma unroll
    for (int i = 0; i < 8; i++) red[wave][lane * 8 + i] = db[i];
    __syncthreads();
    for (int i = tid; i < kFixCols; i += 256)
        if (c0 + i < a.classes) a.dbpart[(long long)blockIdx.y * a.classes + c0 + i] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
}

// ---------------------------------------------------------------- the gradients' products
struct GradArgs {
    Operand a, b;                 // a: the output's contiguous dimension, b: its rows
    int ktiles, mtiles, ntiles, kper, splits;   // kper: stages per split
    long long m, n;
    void *out; long long ldo;     // [n][ldo], operand type (one split), or
    float *acc;                   // float32 [splits][n][m]
    bool add;                     // add to acc instead of starting it
    const float *factor;
};

template <typename Op, int TM, int TN, int WM, int WN, bool TB>
__device__ inline void grad_tile(const GradArgs &a, unsigned wg, char *lds)
{
    using S = TileShape<TM, TN, WM, WN>;
    const unsigned tiles = (unsigned)a.mtiles * a.ntiles, t = xcd_run(wg, tiles * a.splits), split = t / tiles;
    int tm, tn;
    tile_at<4>(t - split * tiles, a.mtiles, a.ntiles, &tm, &tn);
    const long long m0 = (long long)tm * TM, n0 = (long long)tn * TN;
    const int k0 = (int)split * a.kper, k1 = min(a.ktiles, k0 + a.kper);
    fx4 acc[S::MT][S::NT];
#pragma unroll
    for (int i = 0; i < S::MT; i++)
#pragma unroll
        for (int j = 0; j < S::NT; j++) acc[i][j] = fx4{0.f, 0.f, 0.f, 0.f};
    TileProduct<typename Op::Grad, TM, TN, WM, WN, true, TB>::run(acc, a.a, m0, a.b, n0, k0, k1, a.ktiles, lds);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const float f = *a.factor;
    const long long mw = m0 + wm * (TM / WM) + 4 * (lane >> 4), nw = n0 + wn * (TN / WN) + (lane & 15);
#pragma unroll
    for (int nt = 0; nt < S::NT; nt++) {
        const long long n = nw + nt * 16;
        if (n >= a.n) continue;
#pragma unroll
        for (int mt = 0; mt < S::MT; mt++) {
            const long long m = mw + mt * 16;
            if (m >= a.m) continue;
            fx4 v = acc[mt][nt];
            if (a.acc) {
                float *o = a.acc + ((long long)split * a.n + n) * a.m + m;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (m + i < a.m) o[i] = a.add ? o[i] + v[i] : v[i];
            } else {
                typename Op::In *o = static_cast<typename Op::In *>(a.out) + n * a.ldo + m;
                if (m + 4 <= a.m) {
                    Pack<typename Op::In, 4> q;
#pragma unroll
                    for (int i = 0; i < 4; i++) q.v[i] = (typename Op::In)(v[i] * f);
                    *reinterpret_cast<Pack<typename Op::In, 4> *>(o) = q;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (m + i < a.m) o[i] = (typename Op::In)(v[i] * f);
                }
            }
        }
    }
}

// dX = D W (D as it lies) by the first wgs_x workgroups, dW = D^T X (D transposed) by the others; the other factor, W or X,
// is transposed in both.  One launch, so that the workgroups of the one fill the CUs that the other leaves at its end: 4096 rows,
// 2048 features, 32000 classes 0.82 ms, 1.31 PFLOP/s (1128 workgroups, four and a half rounds of the CUs).
template <typename Op, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void grads_kernel(GradArgs x, GradArgs w, unsigned wgs_x)
{
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    if (blockIdx.x < wgs_x) grad_tile<Op, TM, TN, WM, WN, false>(x, blockIdx.x, lds);
    else grad_tile<Op, TM, TN, WM, WN, true>(w, blockIdx.x - wgs_x, lds);
}

struct JoinArgs {
    const float *acc;             // [splits][n][m]
    int splits;
    long long n, m;
    void *out; long long ldo;
    const float *factor;
    unsigned wgs;                 // workgroups of this one
};
struct JoinList { JoinArgs j[3]; };
// Of a sum of more splits than this (db's, a run of rows each) 32 threads take an output; 7699 rows x 280 classes: 963 splits,
// 44 us with a thread an output, 7 us so.
constexpr int kFewSplits = 32, kJoinCols = 8;
// out[n][m] = factor * sum over splits, in a fixed order
template <typename Op>
__global__ __launch_bounds__(256) void join_kernel(JoinList l)
{
    __shared__ float red[256];
    unsigned wg = blockIdx.x;
    int q = 0;
    while (wg >= l.j[q].wgs) wg -= l.j[q++].wgs;
    const JoinArgs a = l.j[q];
    const float f = *a.factor;
    const long long total = a.n * a.m;
    auto store = [&](long long i, float s) {
        const long long r = i / a.m, c = i - r * a.m;
        static_cast<typename Op::In *>(a.out)[r * a.ldo + c] = (typename Op::In)(s * f);
    };
    if (a.splits > kFewSplits) {
        const int c = threadIdx.x % kJoinCols, g = threadIdx.x / kJoinCols;
        for (long long i0 = (long long)wg * kJoinCols; i0 < total; i0 += (long long)a.wgs * kJoinCols) {
            float s = 0.f;
            if (i0 + c < total)
#pragma unroll 8
                for (int z = g; z < a.splits; z += 256 / kJoinCols) s += a.acc[(long long)z * total + i0 + c];
            red[threadIdx.x] = s;
            __syncthreads();
            if (g == 0 && i0 + c < total) {
                for (int z = 1; z < 256 / kJoinCols; z++) s += red[z * kJoinCols + c];
                store(i0 + c, s);
            }
            __syncthreads();
        }
        return;
    }
    for (long long i = (long long)wg * 256 + threadIdx.x; i < total; i += (long long)a.wgs * 256) {
        float s = 0.f;
#pragma unroll 8
        for (int z = 0; z < a.splits; z++) s += a.acc[(long long)z * total + i];
        store(i, s);
    }
}

// zeros for gradients of an empty batch
template <typename T>
__global__ __launch_bounds__(256) void zero_rows_kernel(T *out, long long rows, long long cols, long long ld)
{
    const long long total = rows * cols;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256)
        out[i / cols * ld + i % cols] = (T)0.f;
}

}  // namespace azgops
