// Softmax cross entropy behind a linear layer over a large vocabulary, in pieces of the vocabulary, without keeping the logits.
//
//   z = H W^T + b      lse_r = log sum_v exp z_rv      nll_r = lse_r - z[r][t_r]          (t_r outside [0, V): row left out)
//   G_rv = w_r (exp(z_rv - lse_r) - [v = t_r])         dH = G W      dW = G^T H      db_v = sum_r G_rv
//
// Loss: one product over all tiles of z; each tile leaves the maximum and the sum of exponentials of its 256 columns per row and
// the target's logit.  Gradient: for one piece of the vocabulary after the other, the tiles of z are made again and G of the
// piece is written to the workspace, then two products take it up.
// Bound by, and measured (the same commit is up to 7 % apart on different cards):
//   wide rows, many of them: the matrix units, 6 R V D flops for loss and gradient and 2 R V D for making z again.  8192 x 131072 x 1024
//     bf16 7.2 ms, 1.22e15 a second of these 8.8e12 (a library's products of these shapes alone 1.10 .. 1.24e15).
//   many rows, width up to 256: G, which is written once and read twice.  21800 x 20000 x 200 bf16 1.03 ms; the launches of its
//     gradients move 4.4 TB/s with the matrix units busy a third of the time.  fp32 has three parts of G: 2049 x 17770 x 150 0.345 ms,
//     where its six bf16 products take 0.19.
//   65 to some hundred rows against a large W: its copy in blocks, written once and read three times.  146 x 157269 x 1024 bf16 0.63 ms.
//   loss alone, up to 512 rows of 16 bits: exponentials and pieces of 64 bytes of W's rows.  256 x 1000000 x 256 fp16 0.21 ms.
//
// All products run on one core: 256 x BN outputs a workgroup, steps of 32 along the contraction, three stages of LDS filled by
// LDS-DMA (the stages are LDS variables of their own, so that the compiler can tell reads of one from writes to the other and
// does not wait for the prefetch), v_mfma_f32_16x16x32, a wave makes 128 x 64.
//   H, W and G are kept as blocks of 16 rows x 32 columns, 1 KiB: LDS-DMA fetches whole blocks (of W's own rows it would fetch
//     64-byte pieces, at half the rate), and a block can be the operand of a contraction along its columns as it stands or of one
//     over its rows with transposing LDS reads, without bank conflicts either way.
//   z^T tile: A = W, B = H, both along the columns.  C has the row of H in the lane and four vocabulary entries in registers, so
//     a row's maximum and sum are mostly in-lane work, and the eight values of G that a lane makes are two pieces of a block.
//   G W: A = W over its rows, B = G along its columns.  G^T H: A = H, B = G, both over their rows.
// Up to 512 rows of 16 bits and no gradient: W is read once, as it lies, if its address and rows are multiples of 16 bytes (PLAIN).
// Up to 32 rows, or 64, with or without gradients: the kernels of xent_few.h, which take W as it lies at any address.
//
// Types: bf16 and fp16 go to the matrix units as they are; G is rounded to the inputs' type (relative 2^-8 / 2^-11 of each
// term, as the inputs themselves are) after scaling by the largest row weight: the matrix units take 16-bit operands, and a second
// part of G would make both products twice as long.  Relative error of bf16 gradients 0.0022 (0.0017 is the results' own rounding).
// In fp16 steps of G end at 2^-38 of the largest weight: a row 2^20 lighter than it loses probabilities below 2^-19.  db is the sum of
// the rounded G, so that it is the gradient that dW is.  fp32 is carried as three bf16 parts (24 bits) and every product by its six
// leading terms.
#include "elem.h"

namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int BM = 256;                   // outputs of a workgroup along A
constexpr int BK = 32;                    // contraction of a step
constexpr int STAGES = 3;
constexpr int WAVES = 4;
constexpr int AHEAD = 4;                  // fragments of A that are read in front of their products
constexpr unsigned BUF_FLAGS = 0x00020000u;
constexpr unsigned NOWHERE = 0xFFFFFFF0u; // past every buffer's end: such a lane loads zeros
constexpr float LOG2E = 1.4426950408889634f;

template <typename E>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma<__bf16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma<_Float16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0, 0);
}

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, char* lds, unsigned off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ s16x4 tr16(const char* p) {
    return __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// the six leading products of two numbers in three parts each, smallest first: part of A, part of B
__device__ __forceinline__ constexpr int part_a(int s) { return (0x001102 >> (4 * s)) & 15; }
__device__ __forceinline__ constexpr int part_b(int s) { return (0x010120 >> (4 * s)) & 15; }

// ------------------------------------------------------------------------------------------------
// The core: acc[t][n] (16 x 16 each; A side t, B side n) += A B over `steps` steps of 32.
//   PLAIN   rows as they lie, contraction along them; LDS image [rows][32], 16-byte chunk c of row r at c ^ (-(r / 4) % 4)
//   ALONG   blocks, contraction along their columns      ACROSS   blocks, contraction over their rows
// An 8-byte LDS read serves 32 lanes in a row in a cycle; the images keep those on different banks (a wave's read takes 2 cycles).
// PARTS 3: every step runs over the six pairs of parts; the parts of an operand lie `part` bytes apart.
// ------------------------------------------------------------------------------------------------
enum { PLAIN, ALONG, ACROSS };

// A block of 16 rows x 32 columns: two halves of 16 columns, 512 bytes each; row r at 32 r, its four entries from column 4 q of
// the half on at chunk q ^ 2 (r / 8) of 8 bytes.
__device__ __forceinline__ unsigned in_block(int r, int q) { return (unsigned)(r * 32 + (q ^ ((r >> 3) << 1)) * 8); }

struct Operand {
    const char* p;        // step 0 of the tile
    long long step;       // bytes from one step to the next
    long long part;       // bytes from one part to the next
    unsigned bytes;       // what a step may read, from its p on (PLAIN: from step 0's p on)
    unsigned ld;          // bytes between rows (PLAIN) or between the blocks of one and the next 16 rows
    int kmax;             // PLAIN: length of a row in elements; chunks behind it are loaded as zeros
};

template <int BN>
struct Lay {
    static constexpr int WN = BN / 64;                  // waves along B, 64 outputs each
    static constexpr int WM = WAVES / WN;               // waves along A
    static constexpr int MT = BM / WM / 16;             // 16-wide tiles of a wave along A, at most; tile t of wave w is number WM t + w
    static constexpr int NA = BM * BK * 2 / 1024 / WAVES, NB = BN * BK * 2 / 1024 / WAVES;     // LDS-DMA instructions of a wave and step
};

// lane offset of LDS-DMA instruction `inst` (it fills 1 KiB: 16 rows of 4 chunks, or one block) of a tile of W rows or columns
template <int KIND, int W>
__device__ __forceinline__ unsigned dma_offset(unsigned inst, int lane, unsigned ld) {
    if (KIND == PLAIN) return (inst * 16u + (unsigned)(lane >> 2)) * ld + (unsigned)((lane & 3) ^ (-(lane >> 4) & 3)) * 16u;
    if (KIND == ALONG) return inst * ld + (unsigned)lane * 16u;
    return inst / (W / 32) * ld + inst % (W / 32) * 1024u + (unsigned)lane * 16u;
}
// Fragments of a stage: number `first` + EVERY j (16 rows or columns each; EVERY: 1, 2 or 4)
struct Frag {
    unsigned lo, hi;
};
template <int KIND, int W>
__device__ __forceinline__ Frag frag_offset(int first, int lane) {
    const int i16 = lane & 15, q = lane >> 4;
    Frag f;
    if (KIND == PLAIN) {
        const unsigned row = (unsigned)(first * 16 + i16) * 64u, sw = (unsigned)(-(i16 >> 2) & 3), at = (unsigned)(q & 1) * 8u;
        f.lo = row + ((unsigned)(q >> 1) ^ sw) * 16u + at;
        f.hi = row + ((unsigned)(2 + (q >> 1)) ^ sw) * 16u + at;
    } else if (KIND == ALONG) {
        f.lo = (unsigned)first * 1024u + in_block(i16, q);
        f.hi = f.lo + 512u;
    } else {
        f.lo = (unsigned)first * 512u + in_block(4 * q + (i16 >> 2), i16 & 3);      // (a block has two of them)
        f.hi = f.lo + (W / 32) * 1024u;
    }
    return f;
}
// entries 4 q ... and 16 + 4 q ... of the contraction's 32, whatever the kind
template <int KIND, int EVERY>
__device__ __forceinline__ s16x8 read_frag(const char* stage, const Frag& f, int j) {
    if (KIND == ACROSS) return join(tr16(stage + f.lo + j * EVERY * 512), tr16(stage + f.hi + j * EVERY * 512));
    // (volatile: else the compiler makes one ds_read2_b64 of two reads, which takes 12 cycles instead of 2 x 2)
    typedef const volatile __attribute__((address_space(3))) s16x4* P;
    const s16x4 lo = *(P)(stage + f.lo + j * EVERY * 1024), hi = *(P)(stage + f.hi + j * EVERY * 1024);
    return join(lo, hi);
}

template <typename E, int BN, int MT, int AKIND, int BKIND, int PARTS, bool COLSUM>
__device__ __forceinline__ void core(const Operand& A, const Operand& B, int steps, char* const (&sa)[STAGES], char* const (&sb)[STAGES],
                                     f32x4 (&acc)[MT][4], f32x4 (&cs)[4]) {
    typedef Lay<BN> L;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned oa[L::NA], ob[L::NB];
#pragma unroll
    for (int j = 0; j < L::NA; ++j) {
        const unsigned inst = (unsigned)(wave * L::NA + j);
        oa[j] = dma_offset<AKIND, BM>(inst, lane, A.ld);
        if (AKIND == ACROSS && inst % (BM / 32) * 32u >= 16u * L::WM * MT) oa[j] = NOWHERE;          // columns of no tile
    }
#pragma unroll
    for (int j = 0; j < L::NB; ++j) ob[j] = dma_offset<BKIND, BN>((unsigned)(wave * L::NB + j), lane, B.ld);
    const Frag fa = frag_offset<AKIND, BM>(wave / L::WN, lane), fb = frag_offset<BKIND, BN>((wave % L::WN) * 4, lane);
    const int chunk = ((lane & 3) ^ (-(lane >> 4) & 3)) * 8;         // PLAIN: first element of the lane's chunk

    const char *pa = A.p, *pb = B.p;                     // of the next step to be fetched
    unsigned na = A.bytes, nb = B.bytes;
    int kf = 0;
    auto fetch = [&](int s, char* da, char* db) {        // pair of parts s (PARTS 3; a constant where it is called)
        const char* qa = PARTS == 1 || part_a(s) == 0 ? pa : pa + part_a(s) * A.part;
        const char* qb = PARTS == 1 || part_b(s) == 0 ? pb : pb + part_b(s) * B.part;
        // (uniform as they are; readfirstlane keeps the selects on the scalar side)
        const unsigned ra = (unsigned)__builtin_amdgcn_readfirstlane((int)(kf >= steps ? 0u : na));
        const unsigned rb = (unsigned)__builtin_amdgcn_readfirstlane((int)(kf >= steps ? 0u : nb));
        const __amdgpu_buffer_rsrc_t va = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(qa), 0, ra, BUF_FLAGS);
        const __amdgpu_buffer_rsrc_t vb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(qb), 0, rb, BUF_FLAGS);
        const bool in = AKIND != PLAIN || chunk < A.kmax - kf * BK;
#pragma unroll
        for (int j = 0; j < L::NA; ++j) dma16(va, da + (wave * L::NA + j) * 1024, in ? oa[j] : NOWHERE);
#pragma unroll
        for (int j = 0; j < L::NB; ++j) dma16(vb, db + (wave * L::NB + j) * 1024, ob[j]);
        if (PARTS == 1 || s == 5) {
            ++kf;
            pa += A.step;
            pb += B.step;
            if (AKIND == PLAIN) na -= BK * 2;
            if (BKIND == PLAIN) nb -= BK * 2;
        }
    };
    auto multiply = [&](int s, const char* da, const char* db) {
        s16x8 a[MT], b[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) b[n] = read_frag<BKIND, 1>(db, fb, n);
#pragma unroll
        for (int t = 0; t < AHEAD && t < MT; ++t) a[t] = read_frag<AKIND, L::WM>(da, fa, t);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            __builtin_amdgcn_sched_barrier(0);           // reads stay AHEAD tiles in front of the products
            if (t + AHEAD < MT) a[t + AHEAD] = read_frag<AKIND, L::WM>(da, fa, t + AHEAD);
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[t][n] = mfma<E>(a[t], b[n], acc[t][n]);
        }
        if (COLSUM && (PARTS == 1 || part_a(s) == 0)) {
            const short one = __builtin_bit_cast(short, (E)1.0f);
            const s16x8 ones = {one, one, one, one, one, one, one, one};
#pragma unroll
            for (int n = 0; n < 4; ++n) cs[n] = mfma<E>(ones, b[n], cs[n]);
        }
    };
    // A step: its stage has landed for every wave (own loads but the next step's, then the barrier), every wave has read the
    // stage of the step before (reads done before the barrier): that one is filled again.  Loads behind the last step are issued
    // like the others, from an empty buffer, so that waits are counted the same everywhere.
    auto step = [&](int s, int stage) {                  // s: pair of parts
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (L::NA + L::NB));      // vmcnt(the next step's), lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch((s + 2) % 6, sa[(stage + 2) % STAGES], sb[(stage + 2) % STAGES]);
        multiply(s, sa[stage], sb[stage]);
        __builtin_amdgcn_sched_barrier(0);
    };
    static_assert(STAGES == 3 && L::NA + L::NB < 16, "waits are counted for three stages");
    if (steps <= 0) return;
    fetch(0, sa[0], sb[0]);
    fetch(1, sa[1], sb[1]);
    if (PARTS == 1) {
        for (int it = 0;;) {
            step(0, 0);
            if (++it >= steps) break;
            step(0, 1);
            if (++it >= steps) break;
            step(0, 2);
            if (++it >= steps) break;
        }
    } else {
        for (int it = 0; it < steps; ++it) {
            step(0, 0);
            step(1, 1);
            step(2, 2);
            step(3, 0);
            step(4, 1);
            step(5, 2);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);                  // no load may be on its way into LDS that the workgroup gives back
    asm volatile("" ::: "memory");
}

// position in the launch -> tile: consecutive workgroups go to the 8 XCDs in turn; each gets a run of consecutive tiles, so
// that what they share is fetched into one L2
__device__ __forceinline__ int tile_of(unsigned block, int total) {
    const int per = (total + 7) / 8;
    const int t = (int)(block & 7) * per + (int)(block >> 3);
    return (int)(block >> 3) < per && t < total ? t : -1;
}
inline unsigned blocks_for(long long tiles) { return (unsigned)((tiles + 7) / 8 * 8); }
// launches of more than 2^24 workgroups of 256 threads need a second dimension (threads are counted in 32 bits); workgroups behind
// the last one asked for have to find nothing to do
constexpr long long MOST_BLOCKS = 1ll << 23;
inline dim3 grid_of(long long blocks) {
    return blocks <= MOST_BLOCKS ? dim3((unsigned)blocks) : dim3((unsigned)MOST_BLOCKS, (unsigned)((blocks + MOST_BLOCKS - 1) / MOST_BLOCKS));
}
__device__ __forceinline__ long long block_of() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// exp(z - x) as exp2(z LOG2E - x LOG2E), one operation in front of the exponential, has the rounding of x LOG2E in its exponent: 2^-24
// |x|, up to 2^-17 here.  Farther from 0 (logits masked by large finite numbers: 1e10 would be off by hundreds, 3e38 infinite) the
// difference comes first.  Waves choose: two operations for every logit cost 1.6 % at 21800 x 20000 x 200, bf16, the choice 0.7 %
// (nothing at 8192 x 131072 x 1024).
constexpr float FAR_FROM_0 = 128.f;
__device__ __forceinline__ bool far_from_0(float x) { return fabsf(x) > FAR_FROM_0 && x != -INFINITY; }

// (maximum, sum of exponentials above it) of two sets of logits
__device__ __forceinline__ void join_sums(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    s = s * __builtin_amdgcn_exp2f((m - base) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - base) * LOG2E);
    m = top;
}

// ------------------------------------------------------------------------------------------------
// z^T tiles: loss statistics (GRAD = false) or blocks of G (GRAD = true)
// ------------------------------------------------------------------------------------------------
struct LogitArgs {
    const char* w;            // W: its rows, ldw bytes apart (PLAIN), or blocks
    const char* h;            // copy of H: rows of Dp elements (PLAIN) or blocks
    const float* bias;        // [Vp], -inf behind V
    const int* tgt;           // [Rp], -1: left out
    float2* part;             // loss: [vocabulary tiles][Rp] (maximum, sum of exponentials)
    float* zt;                // loss: [Rp] the target's logit
    const float* lse;         // gradient: [Rp]
    const float* wrow;        // gradient: [Rp], 0 for rows without a part in it
    const float* scale;       // gradient: the scale of G
    char* g;                  // gradient: blocks of G, [Rp / 16][vocabulary tiles * 8], parts g_part bytes apart
    long long w_part, h_part, g_part;
    unsigned ldw;
    int V, D, Dp, Rp, v_begin, nvt, nrt;      // vocabulary of this launch: tiles v_begin / 256 ..., nvt of them
};

// red: [waves along A][BN], for the loss
template <typename E, int BN, int KIND, int PARTS, bool GRAD>
__device__ __forceinline__ void logit_tile(const LogitArgs& a, int tile, char* const (&sa)[STAGES], char* const (&sb)[STAGES], float2 (*red)[BN]) {
    typedef Lay<BN> L;
    // bands of 8 row tiles, vocabulary tiles outside: the workgroups of an XCD share a few vocabulary and 8 row tiles
    const int band = tile / (8 * a.nvt), in = tile - band * 8 * a.nvt;
    const int wide = a.nrt - band * 8 < 8 ? a.nrt - band * 8 : 8;
    const int vt = in / wide, rt = band * 8 + in % wide;
    const long long v0 = (long long)a.v_begin + (long long)vt * BM;
    const long long r0 = (long long)rt * BN;

    Operand A, B;
    if (KIND == PLAIN) {
        A.p = a.w + v0 * a.ldw;
        A.bytes = (unsigned)(((a.V - v0 < BM ? a.V - v0 : BM) - 1) * a.ldw + a.D * 2ll);
        A.step = B.step = BK * 2;
        A.ld = a.ldw;
        A.kmax = a.D;
        B.p = a.h + r0 * a.Dp * 2;
        B.bytes = (unsigned)BN * a.Dp * 2u;
        B.ld = (unsigned)a.Dp * 2u;
    } else {
        A.ld = B.ld = (unsigned)(a.Dp / 32) * 1024u;
        A.p = a.w + (v0 >> 4) * A.ld;
        B.p = a.h + (r0 >> 4) * B.ld;
        A.bytes = (BM / 16 - 1) * A.ld + 1024u;
        B.bytes = (BN / 16 - 1) * B.ld + 1024u;
        A.step = B.step = 1024;
        A.kmax = 0;
    }
    A.part = a.w_part; B.part = a.h_part; B.kmax = 0;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w0 = 16 * (wave / L::WN), wn = (wave % L::WN) * 64;        // tile t: vocabulary entries from w0 + 16 WM t on
    const int i16 = lane & 15, q = lane >> 4;
    constexpr int EVERY = 16 * L::WM;
    const float* bias = a.bias + v0 + w0 + 4 * q;
    // the sums start from the bias; loss and gradient make the same bits of z, so that errors of z cancel against those of lse
    f32x4 acc[L::MT][4], none[4];
#pragma unroll
    for (int t = 0; t < L::MT; ++t) {
        const f32x4 bv = *reinterpret_cast<const f32x4*>(bias + EVERY * t);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[t][n] = bv;
    }
    core<E, BN, L::MT, KIND, KIND, PARTS, false>(A, B, a.Dp / BK, sa, sb, acc, none);

    // where a lane has the logit of a row's target: most tiles have none of a wave's 16 rows' targets
    auto mine = [&](int n) { return a.tgt[r0 + wn + 16 * n + i16] - ((int)v0 + w0 + 4 * q); };
    auto has = [&](int rel) { return rel >= 0 && rel < EVERY * L::MT && rel % EVERY < 4; };
    auto some = [&](int rel) { return __any(has(rel)); };
    auto subtract = [&](int n, float x) {
#pragma unroll
        for (int t = 0; t < L::MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][n][i] -= x;
    };
    if (!GRAD) {
        float top[4], sum[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int rel = mine(n);
            if (some(rel)) {
                float z = 0.f;
#pragma unroll
                for (int t = 0; t < L::MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z = rel == EVERY * t + i ? acc[t][n][i] : z;
                if (has(rel)) a.zt[r0 + wn + 16 * n + i16] = z;
            }
            float m = -INFINITY;
#pragma unroll
            for (int t = 0; t < L::MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) m = fmaxf(m, acc[t][n][i]);
            top[n] = m;
            // fmaxf leaves NaN out; the sum brings it back (exp(NaN - top))
            float base = m == -INFINITY ? 0.f : m * -LOG2E;
            if (__any(far_from_0(m))) {
                subtract(n, m == -INFINITY ? 0.f : m);
                base = 0.f;
            }
            float s = 0.f;
#pragma unroll
            for (int t = 0; t < L::MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f(fmaf(acc[t][n][i], LOG2E, base));
            sum[n] = s;
        }
        // lanes 16 apart hold other vocabulary entries of the same row
#pragma unroll
        for (int o = 16; o < 64; o <<= 1)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float m2 = __shfl_xor(top[n], o, 64), s2 = __shfl_xor(sum[n], o, 64);
                join_sums(top[n], sum[n], m2, s2);
            }
        if (q == 0) {
#pragma unroll
            for (int n = 0; n < 4; ++n) red[wave / L::WN][wn + 16 * n + i16] = make_float2(top[n], sum[n]);
        }
        __syncthreads();
        if ((int)threadIdx.x < BN) {
            float m = red[0][threadIdx.x].x, s = red[0][threadIdx.x].y;
#pragma unroll
            for (int w = 1; w < L::WM; ++w) join_sums(m, s, red[w][threadIdx.x].x, red[w][threadIdx.x].y);
            a.part[(long long)vt * a.Rp + r0 + threadIdx.x] = make_float2(m, s);
        }
    } else {
        const float up = a.scale[0];
        const long long nv32 = (long long)a.nvt * (BM / 32);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const long long r = r0 + wn + 16 * n + i16;
            const float w = a.wrow[r] * up, lse = a.lse[r];
            float low = -lse * LOG2E;
            if (PARTS > 1 || __any(far_from_0(lse))) {
                subtract(n, lse);
                low = 0.f;
            }
#pragma unroll
            for (int t = 0; t < L::MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][n][i] = __builtin_amdgcn_exp2f(fmaf(acc[t][n][i], LOG2E, low));
            const int rel = mine(n);
            if (some(rel)) {
#pragma unroll
                for (int t = 0; t < L::MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][n][i] -= rel == EVERY * t + i ? 1.f : 0.f;
            }
            if (__any(w == 0.f)) {                       // no part in the gradient, whatever W makes of such a row's zeros
#pragma unroll
                for (int t = 0; t < L::MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][n][i] = w == 0.f ? 0.f : acc[t][n][i];
            }
            char* dst = a.g + ((r >> 4) * nv32 + (long long)vt * (BM / 32)) * 1024 + in_block(i16, q);
#pragma unroll
            for (int t = 0; t < L::MT; ++t) {
                const int half = L::WM * t + (w0 >> 4);  // 16 columns: half a block
                float g[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) g[i] = acc[t][n][i] * w;
#pragma unroll
                for (int s = 0; s < PARTS; ++s) {
                    s16x4 out;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const E e = (E)g[i];
                        out[i] = __builtin_bit_cast(short, e);
                        g[i] -= (float)e;
                    }
                    *reinterpret_cast<s16x4*>(dst + s * a.g_part + half * 512) = out;
                }
            }
        }
    }
}

template <typename E, int BN, int KIND, int PARTS>
__global__ __launch_bounds__(64 * WAVES, 2) void xent_loss_kernel(LogitArgs a) {
    __shared__ __attribute__((aligned(1024))) char a0[BM * BK * 2], a1[BM * BK * 2], a2[BM * BK * 2], b0[BN * BK * 2], b1[BN * BK * 2], b2[BN * BK * 2];
    char* const sa[STAGES] = {a0, a1, a2};
    char* const sb[STAGES] = {b0, b1, b2};
    __shared__ float2 red[Lay<BN>::WM][BN];
    const int tile = tile_of(blockIdx.x, a.nvt * a.nrt);
    if (tile >= 0) logit_tile<E, BN, KIND, PARTS, false>(a, tile, sa, sb, red);
}

// ------------------------------------------------------------------------------------------------
// The two gradient products.  A = W or H, up to 256 columns of it a tile (in steps of 32, so that the tiles of a width are alike
// and nearly full); B = G.
//   OVER_V true:  out[r][d] = sum over v of G[r][v] W[v][d]       rows of out: rows of H
//   OVER_V false: out[v][d] = sum over r of G[r][v] H[r][d]       rows of out: the piece's vocabulary; bias gradient too
// The contraction is cut into `splits` parts when there are too few tiles for the chip; each leaves fp32 sums in a slab.
// ------------------------------------------------------------------------------------------------
struct ProductArgs {
    const char* x;            // blocks of W (from the piece's first row on) or of H
    const char* g;            // blocks of G
    float* slab;              // [splits][...][Dp], added to when add != 0; NULL: out is written
    float* bslab;             // [splits][...] bias gradient, or NULL
    void* out;                // [rows][ld_out] of the caller's type
    void* bout;
    const float* scale;       // scale[1] takes the scale of G out again (with the final result)
    long long x_part, g_part, ld_out, slab_stride, bslab_stride;
    int D, Dp, rows, ndt, nnt, splits, steps, nv32, add;
};

template <typename E, typename T, int BN, int MT, int PARTS, bool OVER_V>
__device__ __forceinline__ void product_tile(const ProductArgs& a, int tile, char* const (&sa)[STAGES], char* const (&sb)[STAGES]) {
    typedef Lay<BN> L;
    const int dt = tile % a.ndt, nt = tile / a.ndt % a.nnt, split = tile / (a.ndt * a.nnt);
    const int k0 = (int)((long long)a.steps * split / a.splits), k1 = (int)((long long)a.steps * (split + 1) / a.splits);

    Operand A, B;
    A.ld = (unsigned)(a.Dp / 32) * 1024u;
    A.part = a.x_part; A.step = 2ll * A.ld; A.kmax = 0;
    constexpr int WIDE = 16 * L::WM * MT;                // columns of x that this workgroup makes
    A.p = a.x + k0 * A.step + (long long)dt * (WIDE / 32) * 1024;
    A.bytes = 2 * A.ld - (unsigned)dt * (WIDE / 32) * 1024u;        // columns behind Dp: blocks of the next rows, or nothing
    B.kmax = 0; B.part = a.g_part; B.ld = (unsigned)a.nv32 * 1024u;
    if (OVER_V) {
        B.step = 1024;
        B.p = a.g + (long long)nt * (BN / 16) * B.ld + k0 * B.step;
        B.bytes = (unsigned)(BN / 16 - 1) * B.ld + 1024u;
    } else {
        B.step = 2ll * B.ld;
        B.p = a.g + (long long)nt * (BN / 32) * 1024 + k0 * B.step;
        B.bytes = B.ld + (BN / 32) * 1024u;
    }
    f32x4 acc[MT][4], cs[4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[t][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 4; ++n) cs[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    core<E, BN, MT, ACROSS, OVER_V ? ALONG : ACROSS, PARTS, !OVER_V>(A, B, k1 - k0, sa, sb, acc, cs);

    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));                       // (addresses of the results are not made, and kept, in front of the products)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w0 = 16 * (wave / L::WN), wn = (wave % L::WN) * 64;
    const int i16 = lane & 15, q = lane >> 4;
    const float down = a.scale[1];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int r = nt * BN + wn + 16 * n + i16;
        if (r >= a.rows) continue;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int d = dt * WIDE + w0 + 16 * L::WM * t + 4 * q;
            if (a.slab != nullptr) {
                if (d < a.Dp) {
                    f32x4* s = reinterpret_cast<f32x4*>(a.slab + split * a.slab_stride + (long long)r * a.Dp + d);
                    *s = a.add ? *s + acc[t][n] : acc[t][n];
                }
            } else {
                T* o = reinterpret_cast<T*>(a.out) + (long long)r * a.ld_out + d;
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = acc[t][n][i] * down;
                if (d + 3 < a.D) sv_store<4>(o, v);
                else {
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        if (d + i < a.D) o[i] = (T)v[i];
                }
            }
        }
        if (!OVER_V && dt == 0 && w0 == 0 && q == 0) {
            if (a.bslab != nullptr) a.bslab[split * a.bslab_stride + r] = cs[n][0];
            else if (a.bout != nullptr) reinterpret_cast<T*>(a.bout)[r] = (T)(cs[n][0] * down);
        }
    }
}

// out[r][d] = sum of the slabs, in order
struct SumArgs {
    const float* slab;
    void* out;
    const float* scale;
    long long slab_stride, ld_out;
    int splits, rows, D, Dp;              // (the bias gradient: one column, Dp = 1)
    long long blocks;
};
template <typename T>
__device__ __forceinline__ void sum_slabs(const SumArgs& a, long long block) {
    if (block >= a.blocks) return;
    const float down = a.scale[1];
    const long long i = block * 256 + threadIdx.x;
    if (a.Dp == 1) {
        if (i >= a.rows) return;
        float s = 0.f;
        for (int k = 0; k < a.splits; ++k) s += a.slab[k * a.slab_stride + i];
        reinterpret_cast<T*>(a.out)[i] = (T)(s * down);
        return;
    }
    const int per = a.Dp / 4;
    const long long r = i / per;
    const int d = (int)(i - r * per) * 4;
    if (r >= a.rows || d >= a.D) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) s += *reinterpret_cast<const f32x4*>(a.slab + k * a.slab_stride + r * a.Dp + d);
    T* o = reinterpret_cast<T*>(a.out) + r * a.ld_out + d;
    const float v[4] = {s[0] * down, s[1] * down, s[2] * down, s[3] * down};
    if (d + 3 < a.D) sv_store<4>(o, v);
    else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (d + j < a.D) o[j] = (T)v[j];
    }
}

// One launch of the gradient: G of one piece of the vocabulary, the products of the piece before (its G is in the other of two
// buffers), and the sums of the slabs that dW and db have of the piece before that (in the other of two again, so that slabs take the
// memory of two pieces, whatever the vocabulary).  The long workgroups come first, the short tiles of G fill what they leave; the sums
// in between (21800 x 20000 x 200 bf16 1073 us, behind them 1097).
struct PieceArgs {
    LogitArgs z;
    ProductArgs h, w;
    SumArgs sw, sb;
    unsigned nh, nw;          // workgroups of dH and of dW, multiples of 8; then those of the sums; the rest make G
};

template <typename E, typename T, int BN, int MT, int PARTS>
__global__ __launch_bounds__(64 * WAVES, 2) void xent_piece_kernel(PieceArgs a) {
    __shared__ __attribute__((aligned(1024))) char a0[BM * BK * 2], a1[BM * BK * 2], a2[BM * BK * 2], b0[128 * BK * 2], b1[128 * BK * 2], b2[128 * BK * 2];
    char* const sa[STAGES] = {a0, a1, a2};
    char* const sb[STAGES] = {b0, b1, b2};
    const unsigned ns = (unsigned)(a.sw.blocks + a.sb.blocks);
    if (blockIdx.x < a.nw) {
        const int tile = tile_of(blockIdx.x, a.w.ndt * a.w.nnt * a.w.splits);
        if (tile >= 0) product_tile<E, T, 128, MT, PARTS, false>(a.w, tile, sa, sb);
    } else if (blockIdx.x < a.nw + a.nh) {
        const int tile = tile_of(blockIdx.x - a.nw, a.h.ndt * a.h.nnt * a.h.splits);
        if (tile >= 0) product_tile<E, T, BN, BN == 64 ? MT / 2 : MT, PARTS, true>(a.h, tile, sa, sb);
    } else if (blockIdx.x < a.nw + a.nh + ns) {
        const long long block = blockIdx.x - a.nw - a.nh;
        if (block < a.sw.blocks) sum_slabs<T>(a.sw, block);
        else sum_slabs<T>(a.sb, block - a.sw.blocks);
    } else {
        const int tile = tile_of(blockIdx.x - a.nw - a.nh - ns, a.z.nvt * a.z.nrt);
        if (tile >= 0) logit_tile<E, BN, ALONG, PARTS, true>(a.z, tile, sa, sb, (float2(*)[BN])nullptr);
    }
}

// the slabs of dH, and those of dW and of the bias gradient that the last piece has, in one launch
template <typename T>
__global__ __launch_bounds__(256) void xent_slab_sum_kernel(SumArgs h, SumArgs w, SumArgs b) {
    const long long block = block_of();
    if (block < h.blocks) sum_slabs<T>(h, block);
    else if (block < h.blocks + w.blocks) sum_slabs<T>(w, block - h.blocks);
    else sum_slabs<T>(b, block - h.blocks - w.blocks);
}

// ------------------------------------------------------------------------------------------------
// Copies: rows of H that take part, as blocks (or as rows), padded with zeros to [Rp][Dp] (a row that does not take part is zeros,
// whatever it holds); targets, weights and lse of the rows; the bias in fp32, -inf behind the vocabulary; W as
// blocks, zeros behind the vocabulary.  fp32 in three bf16 parts.  One launch, workgroup ranges.
// ------------------------------------------------------------------------------------------------
struct PrepArgs {
    const void *h, *w, *bias, *tok;
    const float *row_weight, *lse;        // NULL: loss only
    char *hc, *hg, *wc;                   // hg (or NULL): without the rows of weight 0; wc NULL: W is not copied, and hc has rows
    float *biasf, *wrow, *lsec;           // lsec: a copy of lse, where it is given
    int* tgt;
    long long ldh, ldw, h_part, w_part, nh, nb;       // nh, nb: workgroups of H and of the bias; the others copy W
    int tok64, R, Rp, V, Vp, D, Dp;
};

// eight columns of one row: from T to E, in PARTS parts
template <typename T, typename E, int PARTS>
__device__ __forceinline__ void copy8(const T* __restrict__ src, int left, bool live, char* dst, long long part) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (live && left >= 8) sv_load<8>(src, v);
    else if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) v[j] = (float)src[j];
    }
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        s16x8 out;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const E e = (E)v[j];
            out[j] = __builtin_bit_cast(short, e);
            v[j] -= (float)e;
        }
        *reinterpret_cast<s16x8*>(dst + s * part) = out;
    }
}
// where eight columns from c on of row r are in blocks of a matrix of Dp columns
__device__ __forceinline__ long long block_at(long long r, int c, int Dp) {
    return ((r >> 4) * (Dp >> 5) + (c >> 5)) * 1024 + ((c >> 4) & 1) * 512 + in_block((int)(r & 15), (c & 15) >> 2);
}

template <typename T, typename E, int PARTS>
__global__ __launch_bounds__(256) void xent_prep_kernel(PrepArgs a) {
    const int per = a.Dp / 8;
    const long long block = block_of(), i = block * 256 + threadIdx.x;
    if (block < a.nh) {
        const long long r = i / per;
        const int c = (int)(i - r * per) * 8;
        if (r >= a.Rp) return;
        int tg = -1;
        float w = 0.f;
        if (r < a.R) {
            const long long t = a.tok64 ? reinterpret_cast<const long long*>(a.tok)[r] : (long long)reinterpret_cast<const int*>(a.tok)[r];
            if (t >= 0 && t < a.V) tg = (int)t;
            if (tg >= 0 && a.row_weight != nullptr) w = a.row_weight[r];
        }
        if (c == 0) {
            a.tgt[r] = tg;
            if (a.row_weight != nullptr) a.wrow[r] = w;
            if (a.lse != nullptr) a.lsec[r] = r < a.R ? a.lse[r] : 0.f;
        }
        const T* src = reinterpret_cast<const T*>(a.h) + (tg >= 0 ? r : 0) * a.ldh + c;
        const long long to = a.wc != nullptr ? block_at(r, c, a.Dp) : (r * a.Dp + c) * 2;
        if (a.hc != nullptr) copy8<T, E, PARTS>(src, a.D - c, tg >= 0, a.hc + to, a.h_part);
        if (a.hg != nullptr) copy8<T, E, PARTS>(src, a.D - c, w != 0.f, a.hg + to, a.h_part);
    } else if (block < a.nh + a.nb) {
        const long long v = i - a.nh * 256;
        if (v < a.Vp) a.biasf[v] = v >= a.V ? -INFINITY : a.bias != nullptr ? (float)reinterpret_cast<const T*>(a.bias)[v] : 0.f;
    } else {
        const long long j = i - (a.nh + a.nb) * 256, r = j / per;
        const int c = (int)(j - r * per) * 8;
        if (r >= a.Vp) return;
        copy8<T, E, PARTS>(reinterpret_cast<const T*>(a.w) + (r < a.V ? r : 0) * a.ldw + c, a.D - c, r < a.V, a.wc + block_at(r, c, a.Dp), a.w_part);
    }
}

// What G is multiplied with: its largest weight becomes 2^14 (fp16) or 1, so that heavy rows, and all rows where weights are
// equal, lose least to G's rounding (with equal weights a target of small probability loses nothing), and small entries stay
// above the subnormals of fp16, or of bf16 in the third part of fp32.  scale[1] takes it out of the results.
__device__ __forceinline__ void find_scale(const float* __restrict__ wrow, int Rp, float top, float* __restrict__ scale) {
    __shared__ float red[4];
    float m = 0.f;
#pragma unroll 4
    for (int r = threadIdx.x; r < Rp / 4; r += 256) {
        const f32x4 w = reinterpret_cast<const f32x4*>(wrow)[r];
        m = fmaxf(m, fmaxf(fmaxf(fabsf(w[0]), fabsf(w[1])), fmaxf(fabsf(w[2]), fabsf(w[3]))));
    }
    m = sv_wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    m = m < INFINITY ? fmaxf(m, 0x1p-100f) : top;
    scale[0] = top / m;
    scale[1] = m / top;
}
__global__ __launch_bounds__(256) void xent_scale_kernel(const float* __restrict__ wrow, int Rp, float top, float* __restrict__ scale) {
    find_scale(wrow, Rp, top, scale);
}

// lse and loss from the tiles' statistics; one workgroup more for the scale, where it is wanted.  FEW: a workgroup for a row, its
// threads share the tiles; else 32 rows a workgroup, eight threads for each.  run: the statistics of the launches before, where the
// vocabulary is taken in several (begun: there are any), to which this launch adds; the last one (lse) has the results.
template <bool FEW>
__global__ __launch_bounds__(256) void xent_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
                                                        const int* __restrict__ tgt, int R, int Rp, int nvt, float2* __restrict__ run, int begun,
                                                        float* __restrict__ nll, float* __restrict__ lse, float* __restrict__ lsec,
                                                        const float* __restrict__ wrow, float top, float* __restrict__ scale) {
    if (scale != nullptr && blockIdx.x == gridDim.x - 1) {
        find_scale(wrow, Rp, top, scale);
        return;
    }
    constexpr int SLICES = FEW ? 256 : 8, ROWS = 256 / SLICES;
    __shared__ float2 red[8][33];
    const int i = threadIdx.x % ROWS, s = threadIdx.x / ROWS;
    const long long r = (long long)blockIdx.x * ROWS + i;
    float m = -INFINITY, sum = 0.f;
    if (begun && s == 0) {
        m = run[r].x;
        sum = run[r].y;
    }
    for (int v = s; v < nvt; v += 4 * SLICES) {          // four tiles at a time: their loads do not wait for each other
        float2 p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            p[k] = v + k * SLICES < nvt ? part[(long long)(v + k * SLICES) * Rp + r] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) join_sums(m, sum, p[k].x, p[k].y);
    }
    if (FEW) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(sum, o, 64);
            join_sums(m, sum, m2, s2);
        }
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = make_float2(m, sum);
    } else red[s][i] = make_float2(m, sum);
    __syncthreads();
    if ((int)threadIdx.x >= ROWS) return;
    if (FEW) {
        m = red[0][0].x;
        sum = red[0][0].y;
    }
    for (int k = 1; k < (FEW ? 4 : 8); ++k) join_sums(m, sum, red[k][i].x, red[k][i].y);
    if (lse == nullptr) {
        run[r] = make_float2(m, sum);
        return;
    }
    const bool here = tgt[r] >= 0;
    const float l = m + logf(sum);
    if (lsec != nullptr) lsec[r] = here ? l : 0.f;
    if (r >= R) return;
    lse[r] = here ? l : 0.f;
    nll[r] = here ? l - zt[r] : 0.f;
}

// sum of the losses and number of rows with a target; in a fixed order, in 64 bits (a mean over no rows is 0).  One workgroup: 21 800
// rows 7 us, 131 072 31 us; of more its share of the loss and gradients is smaller (2^20 rows 0.6 ms, 2^24 9.5 ms: bound by latency)
__global__ __launch_bounds__(1024) void xent_reduce_kernel(const float* __restrict__ nll, const void* __restrict__ tok, int tok64,
                                                           int R, int V, int mean, float* __restrict__ out) {
    __shared__ double red[1024];
    __shared__ int cnt[1024];
    double s = 0.0;
    int n = 0;
    for (int r = threadIdx.x; r < R; r += 1024) {
        const long long t = tok64 ? reinterpret_cast<const long long*>(tok)[r] : (long long)reinterpret_cast<const int*>(tok)[r];
        s += (double)nll[r];
        n += t >= 0 && t < V;
    }
    red[threadIdx.x] = s;
    cnt[threadIdx.x] = n;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) {
            red[threadIdx.x] += red[threadIdx.x + o];
            cnt[threadIdx.x] += cnt[threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const int c = cnt[0] > 0 ? cnt[0] : 1;
        out[0] = (float)(mean ? red[0] / c : red[0]);
        out[1] = (float)(mean ? 1.0 / c : 1.0);
    }
}

#include "xent_few.h"

// ------------------------------------------------------------------------------------------------
// Host side: shapes, workspace, launches
// ------------------------------------------------------------------------------------------------
// Up to here: the kernels for few rows.  More than 32 rows of 16 bits only for a W of 2^23 numbers or more, whose copy costs more than
// those kernels' slower start (64 rows, loss and gradients in us, few | many: 5000 x 64 41 | 35, 32768 x 256 (2^23: about even) 55 | 51,
// 32768 x 1024 93 | 99, 65536 x 256 64 | 90; fp32 39 | 41, 83 | 114, 221 | 344, 113 | 285).
constexpr int FEW_ROWS = 64, FEW_ROWS_16 = 32;
constexpr long long FEW_WEIGHT_16 = 1ll << 23;
// vocabulary tiles up to which logits of one tile of rows take H as it lies: without the launch for the copy, which however is
// read faster (bf16, loss of one row: 5000 x 64 17 us | 20 with a copy, 411353 x 96 (1607 tiles) 27 | 28, 1000000 x 256 (3907) 114 | 105)
constexpr int FEW_OWN_TILES = 2048;
constexpr int DIRECT_ROWS = 512;                           // up to here a loss takes W as it lies
constexpr long long PIECE_LEAST = 128ll << 20, PIECE_MOST = 512ll << 20;     // what G of a piece may take; there are two
constexpr long long STATISTICS_MOST = 512ll << 20;         // what the loss's tiles may leave before their rows are joined
constexpr int SLOTS = 512;                                 // workgroups at a time: two on each of 256 CUs

struct Shape {
    int parts, Rp, Vp, Dp, BN, nrt, nvt, direct, pieces, piece_tiles, h_splits, w_splits, ndt, dblocks;
    int few, R4, wd, chunks;  // few: the kernels for few rows, with this many tiles of 16
    int slice;                // vocabulary tiles of a launch of the loss, at most
    long long h, hg, h_part, w, w_part, ldw, bias, tgt, wrow, lse, zt, part, scale, run, g[2], g_part, h_slab, w_slab[2], b_slab[2], z, total;
};

// parts of a product's contraction: no workgroup should work longer than a slot's share of the launch
inline int splits_for(double unit, double whole) {
    const double s = unit * SLOTS / whole;
    return s <= 1.0 ? 1 : s >= 32.0 ? 32 : (int)(s + 0.999);
}

enum { LOSS = 0, GRADIENT = 1 };

inline int shape_of(const void* weight, long long ld_w, int type, long long R, long long V, long long D, int grad, Shape* s) {
    SV_CHECK_ARG(type >= 0 && type <= 2, "svae_xent: type %d", type);
    SV_CHECK_ARG(R > 0 && R <= 1 << 24 && V > 0 && V <= 1 << 28 && D > 0 && D <= 1 << 16 && ld_w >= D && ld_w <= 1 << 20,
                 "svae_xent: sizes R %lld, V %lld, D %lld, ld %lld", R, V, D, ld_w);
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long p = at;
        at += (bytes + 1023) / 1024 * 1024;
        return p;
    };
    if (R <= FEW_ROWS_16 || (R <= FEW_ROWS && (type == SV_F32 || V * D >= FEW_WEIGHT_16))) {
        s->few = R <= 16 ? 1 : R <= 32 ? 2 : 4;
        s->Rp = 16 * s->few;
        s->R4 = (int)(R + 3) / 4 * 4;
        s->nvt = (int)((V + 255) / 256);
        s->Dp = (int)((D + 63) / 64 * 64);
        s->wd = D <= 64 ? 1 : D <= 128 ? 2 : 4;
        s->ndt = (s->Dp / 64 + s->wd - 1) / s->wd;
        const int step = type == SV_F32 || s->few == 1 ? few_step(s->wd) : few_step16(s->wd);
        const int steps = (int)((V + step - 1) / step), most = (s->few == 1 ? 768 : 512) / s->ndt;      // as many as run at a time: three or two on a CU
        s->chunks = most < 1 ? 1 : most < steps ? most : steps;
        s->h = take((long long)s->Rp * s->Dp * sv_elem_size(type));
        s->tgt = take(4ll * s->Rp);
        s->zt = take(4ll * s->Rp);
        s->part = take(8ll * s->nvt * s->Rp);
        if (grad != LOSS) {
            s->z = take(4ll * V * s->R4);
            s->h_slab = take(4ll * s->chunks * (4 / s->wd) * R * s->Dp);
        }
        s->total = at;
        return 0;
    }
    s->parts = type == SV_F32 ? 3 : 1;
    s->direct = grad == LOSS && type != SV_F32 && R <= DIRECT_ROWS && D % 8 == 0 && ld_w % 8 == 0 && (unsigned long long)weight % 16 == 0;
    // 128 rows a tile, but 64 where that leaves less than a workgroup for each CU (loss and gradients in us, 64 | 128 rows: fp32
    // 184 x 6038 x 1024, 48 tiles of 128 rows, 159 | 240; bf16 300 x 20000 x 512, 237 tiles, 67 | 71; 200 x 50000 x 512, 392, 119 | 112)
    s->BN = (R + 127) / 128 * ((V + 255) / 256) < SLOTS / 2 ? 64 : 128;
    s->Rp = (int)((R + s->BN - 1) / s->BN * s->BN);
    s->Vp = (int)((V + BM - 1) / BM * BM);
    s->Dp = (int)((D + BK - 1) / BK * BK);
    s->nrt = s->Rp / s->BN;
    s->nvt = s->Vp / BM;
    // tiles of the width: as few as 256 columns a tile allow, of equal numbers of 32-column blocks
    s->ndt = (s->Dp + BM - 1) / BM;
    s->dblocks = (s->Dp / 32 + s->ndt - 1) / s->ndt;
    s->dblocks = s->BN == 64 ? 8 : s->dblocks <= 2 ? 2 : s->dblocks <= 4 ? 4 : s->dblocks;
    s->h_part = (long long)s->Rp * s->Dp * 2;
    s->h = take(s->h_part * s->parts);
    s->hg = grad == LOSS ? 0 : take(s->h_part * s->parts);
    s->w_part = s->direct ? 0 : (long long)s->Vp * s->Dp * 2;
    s->ldw = ld_w * 2;
    s->w = take(s->w_part * s->parts);
    s->bias = take(4ll * s->Vp);
    s->tgt = take(4ll * s->Rp);
    s->wrow = take(4ll * s->Rp);
    s->lse = take(4ll * s->Rp);
    s->zt = take(4ll * s->Rp);
    s->scale = take(8);
    long long slice = STATISTICS_MOST / (8ll * s->Rp);
    slice = slice < MOST_BLOCKS / s->nrt ? slice : MOST_BLOCKS / s->nrt;
    s->slice = (int)(slice < s->nvt ? slice : s->nvt);     // (at least four: Rp is at most 2^24)
    s->run = take(s->slice < s->nvt ? 8ll * s->Rp : 0);
    s->part = s->g[0] = at;                                // the loss's statistics are done with when G is made
    const long long end = at + 8ll * s->slice * s->Rp;
    if (grad != LOSS) {
        // A piece's G is written and read twice, and every piece adds to all of dH's sums (4 Rp Dp bytes, read and written): at
        // least four times those, and 128 MiB for large launches (8192 x 131072 x 1024: 7.2 ms with pieces of 128 MiB, 7.4 with 512)
        long long bytes = 16ll * s->Rp * s->Dp;
        bytes = bytes < PIECE_LEAST ? PIECE_LEAST : bytes > PIECE_MOST ? PIECE_MOST : bytes;
        long long tiles = bytes / (2ll * s->parts * s->Rp * BM);
        tiles = tiles < 1 ? 1 : tiles > s->nvt ? s->nvt : tiles;
        s->pieces = (int)((s->nvt + tiles - 1) / tiles);
        s->piece_tiles = (s->nvt + s->pieces - 1) / s->pieces;
        s->pieces = (s->nvt + s->piece_tiles - 1) / s->piece_tiles;
        s->g_part = 2ll * s->Rp * s->piece_tiles * BM;
        s->g[0] = take(s->g_part * s->parts);
        s->g[1] = s->pieces > 1 ? take(s->g_part * s->parts) : s->g[0];
        // steps of 32 in a launch (a tile of G: as many as its epilogue takes, about ten, beside its own)
        const double k = s->parts == 1 ? 1 : 6, h_unit = k * s->piece_tiles * (BM / BK), w_unit = k * (s->Rp / BK);
        const double h_all = h_unit * s->ndt * s->nrt, w_all = w_unit * s->ndt * s->piece_tiles * (BM / 128);
        const double z_all = s->pieces > 1 ? (k * (s->Dp / BK) + 10) * s->piece_tiles * s->nrt : 0;
        s->h_splits = splits_for(h_unit, h_all + w_all + z_all);
        s->w_splits = splits_for(w_unit, h_all + w_all + z_all);
        if (s->h_splits > s->piece_tiles * (BM / BK) / 4) s->h_splits = s->piece_tiles * (BM / BK) / 4;
        if (s->w_splits > s->Rp / BK / 2) s->w_splits = s->Rp / BK / 2;
        s->h_slab = take(4ll * s->Rp * s->Dp * s->h_splits);
        // (more than one slab only of fewer than 512 tiles: 128 MiB at most, of dH's as of a piece of dW's)
        for (int k = 0; k < 2; ++k) {
            const long long rows = s->w_splits > 1 && k < s->pieces ? (long long)s->piece_tiles * BM * s->w_splits : 0;
            s->w_slab[k] = take(4 * rows * s->Dp);
            s->b_slab[k] = take(4 * rows);
        }
    }
    s->total = at > end ? at : end;
    return 0;
}

// what the largest row weight becomes in G
inline float top_of(int type) { return type == SV_F16 ? 16384.f : 1.f; }

struct Call {
    const void *hidden, *weight, *bias, *targets;
    long long ld_h, ld_w;
    int tok64, type, R, V, D;
    char* work;
    hipStream_t stream;
};

// calls f(T{}, E{}, parts) with the caller's and the matrix units' element types
template <typename F>
inline void by_type(int type, F f) {
    if (type == SV_F32) f(float{}, __bf16{}, std::integral_constant<int, 3>{});
    else if (type == SV_BF16) f(__bf16{}, __bf16{}, std::integral_constant<int, 1>{});
    else f(_Float16{}, _Float16{}, std::integral_constant<int, 1>{});
}

// loss: whether the rows with a target are wanted; row_weight: the rows of the gradient are; lse: fwd's, where it is not to be made
inline int prepare(const Call& c, const Shape& s, bool loss, const float* row_weight, const float* lse) {
    PrepArgs p;
    p.h = c.hidden; p.w = c.weight; p.bias = c.bias; p.tok = c.targets; p.row_weight = row_weight; p.lse = lse;
    p.hc = loss ? c.work + s.h : nullptr;
    p.hg = row_weight != nullptr ? c.work + s.hg : nullptr;
    p.wc = s.direct ? nullptr : c.work + s.w;
    p.biasf = (float*)(c.work + s.bias); p.wrow = (float*)(c.work + s.wrow); p.tgt = (int*)(c.work + s.tgt); p.lsec = (float*)(c.work + s.lse);
    p.ldh = c.ld_h; p.ldw = c.ld_w; p.h_part = s.h_part; p.w_part = s.w_part;
    p.tok64 = c.tok64; p.R = c.R; p.Rp = s.Rp; p.V = c.V; p.Vp = s.Vp; p.D = c.D; p.Dp = s.Dp;
    const long long nh = ((long long)s.Rp * (s.Dp / 8) + 255) / 256, nb = (s.Vp + 255) / 256,
                    nw = s.direct ? 0 : ((long long)s.Vp * (s.Dp / 8) + 255) / 256;
    p.nh = nh; p.nb = nb;
    by_type(c.type, [&](auto t, auto e, auto parts) {
        hipLaunchKernelGGL((xent_prep_kernel<decltype(t), decltype(e), decltype(parts)::value>), grid_of(nh + nb + nw), dim3(256), 0, c.stream, p);
    });
    SV_LAUNCH_CHECK();
    return 0;
}

inline LogitArgs logit_args(const Call& c, const Shape& s) {
    LogitArgs a{};
    a.w = s.direct ? (const char*)c.weight : c.work + s.w;
    a.h = c.work + s.h;
    a.bias = (const float*)(c.work + s.bias); a.tgt = (const int*)(c.work + s.tgt);
    a.w_part = s.w_part; a.h_part = s.h_part; a.g_part = s.g_part;
    a.ldw = (unsigned)s.ldw;
    a.V = c.V; a.D = c.D; a.Dp = s.Dp; a.Rp = s.Rp; a.nrt = s.nrt;
    return a;
}

// grad: gradients follow, which read lse and the scale from the workspace
inline int loss(const Call& c, const Shape& s, float* nll, float* lse, bool grad) {
    LogitArgs a = logit_args(c, s);
    a.zt = (float*)(c.work + s.zt);
    a.part = (float2*)(c.work + s.part);
    const bool few_rows = c.R <= 1024 && s.nvt > 64;
    for (int v = 0; v < s.nvt; v += s.slice) {
        const bool last = v + s.slice >= s.nvt;
        a.v_begin = v * BM;
        a.nvt = last ? s.nvt - v : s.slice;
        by_type(c.type, [&](auto, auto e, auto parts) {
            typedef decltype(e) E;
            constexpr int P = decltype(parts)::value;
            const dim3 grid(blocks_for((long long)a.nvt * a.nrt));
            auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * WAVES), 0, c.stream, a); };
            if constexpr (P == 1) {
                if (s.direct) {
                    if (s.BN == 64) go(xent_loss_kernel<E, 64, PLAIN, P>);
                    else go(xent_loss_kernel<E, 128, PLAIN, P>);
                    return;
                }
            }
            if (s.BN == 64) go(xent_loss_kernel<E, 64, ALONG, P>);
            else go(xent_loss_kernel<E, 128, ALONG, P>);
        });
        SV_LAUNCH_CHECK();
        // (rows behind R: their statistics are kept, their lse is for the gradients)
        float* const scale = grad && last ? (float*)(c.work + s.scale) : nullptr;
        const unsigned blocks = (unsigned)(!few_rows ? s.Rp / 32 : grad || !last ? s.Rp : c.R) + (scale ? 1 : 0);
        hipLaunchKernelGGL(few_rows ? xent_rows_kernel<true> : xent_rows_kernel<false>, dim3(blocks), dim3(256), 0, c.stream, (const float2*)a.part, a.zt,
                           a.tgt, c.R, s.Rp, a.nvt, (float2*)(c.work + s.run), v > 0, nll, last ? lse : nullptr, grad ? (float*)(c.work + s.lse) : nullptr,
                           (const float*)(c.work + s.wrow), top_of(c.type), scale);
        SV_LAUNCH_CHECK();
    }
    return 0;
}

inline void piece(const Call& c, const Shape& s, const PieceArgs& a, unsigned blocks) {
    by_type(c.type, [&](auto t, auto e, auto parts) {
        typedef decltype(t) T;
        typedef decltype(e) E;
        constexpr int P = decltype(parts)::value;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * WAVES), 0, c.stream, a); };
        if (s.BN == 64) go(xent_piece_kernel<E, T, 64, 8, P>);
        else if (s.dblocks == 2) go(xent_piece_kernel<E, T, 128, 2, P>);
        else if (s.dblocks == 4) go(xent_piece_kernel<E, T, 128, 4, P>);
        else if (s.dblocks == 5) go(xent_piece_kernel<E, T, 128, 5, P>);
        else if (s.dblocks == 6) go(xent_piece_kernel<E, T, 128, 6, P>);
        else if (s.dblocks == 7) go(xent_piece_kernel<E, T, 128, 7, P>);
        else go(xent_piece_kernel<E, T, 128, 8, P>);
    });
}

// the kernels for few rows: loss (nll and lse are written), gradients (row_weight; dh or dw is written; given: fwd's lse, where no
// loss is wanted)
inline int few(const Call& c, const Shape& s, float* nll, float* lse, const float* given, const float* row_weight, void* dh, long long ld_dh,
               void* dw, long long ld_dw, void* db) {
    FewArgs a{};
    a.w = c.weight; a.hidden = a.h = c.hidden; a.bias = c.bias; a.tok = c.targets; a.tgt = (int*)(c.work + s.tgt);
    a.lse = given ? given : lse; a.row_weight = row_weight;
    a.part = nll ? (float2*)(c.work + s.part) : nullptr; a.zt = (float*)(c.work + s.zt);
    a.z = row_weight ? (float*)(c.work + s.z) : nullptr; a.slab = dh ? (float*)(c.work + s.h_slab) : nullptr;
    a.dw = dw; a.db = db; a.ldw = c.ld_w; a.ld_dw = ld_dw; a.ldh = c.ld_h; a.tok64 = c.tok64;
    a.V = c.V; a.D = c.D; a.Dp = s.Dp; a.R = c.R; a.R4 = s.R4; a.Rp = s.Rp; a.ndt = s.ndt; a.chunks = s.chunks;
    int rc = 0;
    sv_by_type(c.type, [&](auto type) {
        typedef decltype(type) T;
        auto go = [&](auto kernel, long long blocks, auto... args) {
            if (rc == 0) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, c.stream, args...);
                rc = [&]() -> int {
                    SV_LAUNCH_CHECK();
                    return 0;
                }();
            }
        };
        if (s.few == 1 && s.nvt <= FEW_OWN_TILES) go(few_logit_kernel<T, 1, true>, s.nvt, a);
        else {
            FewPrepArgs p;
            p.h = c.hidden; p.tok = c.targets; p.hc = c.work + s.h; p.tgt = a.tgt;
            p.ldh = c.ld_h; p.tok64 = c.tok64; p.R = c.R; p.Rp = s.Rp; p.V = c.V; p.D = c.D; p.Dp = s.Dp;
            go(few_prep_kernel<T>, ((long long)s.Rp * s.Dp + 255) / 256, p);
            a.h = p.hc;
            if (s.few == 1) go(few_logit_kernel<T, 1, false>, s.nvt, a);
            else if (s.few == 2) go(few_logit_kernel<T, 2, false>, s.nvt, a);
            else go(few_logit_kernel<T, 4, false>, s.nvt, a);
        }
        if (nll)
            go(xent_rows_kernel<true>, c.R, (const float2*)a.part, (const float*)a.zt, (const int*)a.tgt, c.R, s.Rp, s.nvt, (float2*)nullptr, 0,
               nll, lse, (float*)nullptr, (const float*)nullptr, 0.f, (float*)nullptr);
        if (!dh && !dw) return;
        const long long blocks = (long long)s.chunks * s.ndt;
        auto grad = [&](auto wide) {
            constexpr int WD = decltype(wide)::value;
            if (s.few == 1) go(few_grad_kernel<T, 1, WD>, blocks, a);
            else if constexpr (sizeof(T) == 2) {
                if (s.few == 2) go(few_grad16_kernel<T, 2, WD>, blocks, a, top_of(c.type));
                else go(few_grad16_kernel<T, 4, WD>, blocks, a, top_of(c.type));
            } else {
                if (s.few == 2) go(few_grad_kernel<T, 2, WD>, blocks, a);
                else go(few_grad_kernel<T, 4, WD>, blocks, a);
            }
        };
        if (s.wd == 1) grad(std::integral_constant<int, 1>{});
        else if (s.wd == 2) grad(std::integral_constant<int, 2>{});
        else grad(std::integral_constant<int, 4>{});
        if (dh) go(few_sum_kernel<T>, (long long)c.R * (s.Dp / 4) / 8, (const float*)a.slab, s.chunks * (4 / s.wd), c.R, c.D, s.Dp, (T*)dh, ld_dh);
    });
    return rc;
}

// h: the rows of H that tiles of z are made from (the loss's or the gradient's copy; rows of weight 0 come to nothing either way)
inline int gradients(const Call& c, const Shape& s, long long h, void* dh, long long ld_dh, void* dw, long long ld_dw, void* db) {
    const float* const scale = (const float*)(c.work + s.scale);
    const int es = sv_elem_size(c.type);
    LogitArgs z = logit_args(c, s);
    z.h = c.work + h;
    z.lse = (const float*)(c.work + s.lse); z.wrow = (const float*)(c.work + s.wrow); z.scale = scale;
    ProductArgs d{};
    d.scale = scale; d.g_part = s.g_part; d.D = c.D; d.Dp = s.Dp; d.ndt = s.ndt;
    const bool slabs = s.w_splits > 1;
    const long long piece_rows = (long long)s.piece_tiles * BM;
    // the sums of the slabs of dW and db that piece p has
    auto sums = [&](int p, SumArgs& w, SumArgs& b) {
        if (!dw || !slabs) return;
        const long long v0 = p * piece_rows;
        w.slab = (float*)(c.work + s.w_slab[p & 1]); w.slab_stride = piece_rows * s.Dp; w.out = (char*)dw + v0 * ld_dw * es; w.ld_out = ld_dw;
        w.scale = scale; w.splits = s.w_splits; w.rows = (int)(c.V - v0 < piece_rows ? c.V - v0 : piece_rows); w.D = c.D; w.Dp = s.Dp;
        w.blocks = ((long long)w.rows * (s.Dp / 4) + 255) / 256;
        if (!db) return;
        b = w;
        b.slab = (float*)(c.work + s.b_slab[p & 1]); b.slab_stride = piece_rows; b.out = (char*)db + v0 * es; b.D = b.Dp = 1;
        b.blocks = (w.rows + 255) / 256;
    };
    for (int p = 0; p <= s.pieces; ++p) {                  // launch p: G of piece p, products of piece p - 1, sums of piece p - 2
        PieceArgs a{};
        unsigned nz = 0;
        if (p < s.pieces) {
            const int t0 = p * s.piece_tiles;
            a.z = z;
            a.z.v_begin = t0 * BM;
            a.z.nvt = s.nvt - t0 < s.piece_tiles ? s.nvt - t0 : s.piece_tiles;
            a.z.g = c.work + s.g[p & 1];
            nz = blocks_for((long long)a.z.nvt * a.z.nrt);
        }
        if (p > 0) {
            const int t0 = (p - 1) * s.piece_tiles, nt = s.nvt - t0 < s.piece_tiles ? s.nvt - t0 : s.piece_tiles;
            const long long v0 = (long long)t0 * BM;
            d.g = c.work + s.g[(p - 1) & 1];
            d.nv32 = nt * (BM / 32);
            if (dh) {
                a.h = d;
                a.h.x = c.work + s.w + v0 * s.Dp * 2; a.h.x_part = s.w_part;
                a.h.slab = (float*)(c.work + s.h_slab); a.h.slab_stride = (long long)s.Rp * s.Dp;
                a.h.rows = s.Rp; a.h.nnt = s.nrt; a.h.splits = s.h_splits; a.h.steps = nt * (BM / BK); a.h.add = p > 1;
                a.nh = blocks_for((long long)a.h.ndt * a.h.nnt * a.h.splits);
            }
            if (dw) {
                a.w = d;
                a.w.x = c.work + s.hg; a.w.x_part = s.h_part;
                a.w.rows = (int)(c.V - v0 < (long long)nt * BM ? c.V - v0 : (long long)nt * BM);
                a.w.nnt = nt * (BM / 128); a.w.splits = s.w_splits; a.w.steps = s.Rp / BK; a.w.add = 0;
                a.w.out = (char*)dw + v0 * ld_dw * es; a.w.ld_out = ld_dw;
                a.w.bout = db ? (char*)db + v0 * es : nullptr;
                a.w.slab = slabs ? (float*)(c.work + s.w_slab[(p - 1) & 1]) : nullptr; a.w.slab_stride = piece_rows * s.Dp;
                a.w.bslab = slabs && db ? (float*)(c.work + s.b_slab[(p - 1) & 1]) : nullptr; a.w.bslab_stride = piece_rows;
                a.nw = blocks_for((long long)a.w.ndt * a.w.nnt * a.w.splits);
            }
        }
        if (p > 1) sums(p - 2, a.sw, a.sb);
        const long long blocks = (long long)nz + a.nh + a.nw + a.sw.blocks + a.sb.blocks;
        SV_CHECK_ARG(blocks < 1ll << 24, "svae_xent: R %d, V %d, D %d need too many workgroups", c.R, c.V, c.D);
        piece(c, s, a, (unsigned)blocks);
        SV_LAUNCH_CHECK();
    }
    SumArgs h1{}, w1{}, b1{};
    if (dh) {
        h1.slab = (const float*)(c.work + s.h_slab); h1.slab_stride = (long long)s.Rp * s.Dp; h1.out = dh; h1.ld_out = ld_dh;
        h1.scale = scale; h1.splits = s.h_splits; h1.rows = c.R; h1.D = c.D; h1.Dp = s.Dp;
        h1.blocks = ((long long)c.R * (s.Dp / 4) + 255) / 256;
    }
    sums(s.pieces - 1, w1, b1);
    if (h1.blocks + w1.blocks + b1.blocks > 0) {
        by_type(c.type, [&](auto t, auto, auto) {
            hipLaunchKernelGGL(xent_slab_sum_kernel<decltype(t)>, grid_of(h1.blocks + w1.blocks + b1.blocks), dim3(256), 0, c.stream, h1, w1, b1);
        });
        SV_LAUNCH_CHECK();
    }
    return 0;
}

inline int check_call(const char* name, const Call& c, const void* work, long long work_bytes, int grad, Shape* s) {
    SV_CHECK_ARG(c.hidden && c.weight && c.targets && work, "%s: null pointer", name);
    SV_CHECK_ARG(c.ld_h >= c.D, "%s: ld %lld of the hidden rows is below D %d", name, c.ld_h, c.D);
    SV_CHECK_ARG((unsigned long long)work % 256 == 0, "%s: the workspace must be aligned to 256 bytes", name);
    const int rc = shape_of(c.weight, c.ld_w, c.type, c.R, c.V, c.D, grad, s);
    if (rc != 0) return rc;
    SV_CHECK_ARG(work_bytes >= s->total, "%s: workspace of %lld bytes, %lld needed", name, work_bytes, s->total);
    return 0;
}
inline int check_gradients(const char* name, int D, const float* row_weight, void* dh, long long ld_dh, void* dw, long long ld_dw, void* db) {
    SV_CHECK_ARG(row_weight, "%s: null pointer", name);
    SV_CHECK_ARG((!dh || ld_dh >= D) && (!dw || ld_dw >= D), "%s: ld %lld, %lld below D %d", name, ld_dh, ld_dw, D);
    SV_CHECK_ARG(!db || dw, "%s: the bias gradient comes with the weight gradient", name);
    return 0;
}

}  // namespace

extern "C" int svae_xent_bytes(int weight_align, long long ld_w, int type, int R, int V, int D, int grad, long long* bytes) {
    SV_CHECK_ARG(bytes != nullptr, "svae_xent_bytes: null pointer");
    Shape s{};
    const int rc = shape_of((const void*)(size_t)(weight_align & 15), ld_w, type, R, V, D, grad ? GRADIENT : LOSS, &s);
    if (rc != 0) return rc;
    *bytes = s.total;
    return 0;
}

extern "C" int svae_xent_fwd(const void* hidden, long long ld_h, const void* weight, long long ld_w, const void* bias,
                             const void* targets, int tok64, int type, int R, int V, int D, float* nll, float* lse, void* work,
                             long long work_bytes, void* stream) {
    Call c{hidden, weight, bias, targets, ld_h, ld_w, tok64, type, R, V, D, (char*)work, (hipStream_t)stream};
    Shape s{};
    int rc = check_call("svae_xent_fwd", c, work, work_bytes, LOSS, &s);
    if (rc != 0) return rc;
    SV_CHECK_ARG(nll && lse, "svae_xent_fwd: null pointer");
    if (s.few) return few(c, s, nll, lse, nullptr, nullptr, nullptr, 0, nullptr, 0, nullptr);
    rc = prepare(c, s, true, nullptr, nullptr);
    if (rc != 0) return rc;
    return loss(c, s, nll, lse, false);
}

extern "C" int svae_xent_reduce(const float* nll, const void* targets, int tok64, int R, int V, int mean, float* out, void* stream) {
    SV_CHECK_ARG(nll && targets && out && R > 0 && R <= 1 << 24 && V > 0, "svae_xent_reduce: bad arguments");
    hipLaunchKernelGGL(xent_reduce_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, nll, targets, tok64, R, V, mean, out);
    SV_LAUNCH_CHECK();
    return 0;
}

extern "C" int svae_xent_bwd(const void* hidden, long long ld_h, const void* weight, long long ld_w, const void* bias,
                             const void* targets, int tok64, int type, int R, int V, int D, const float* lse,
                             const float* row_weight, void* dh, long long ld_dh, void* dw, long long ld_dw, void* db, void* work,
                             long long work_bytes, void* stream) {
    Call c{hidden, weight, bias, targets, ld_h, ld_w, tok64, type, R, V, D, (char*)work, (hipStream_t)stream};
    Shape s{};
    int rc = check_call("svae_xent_bwd", c, work, work_bytes, GRADIENT, &s);
    if (rc == 0) rc = check_gradients("svae_xent_bwd", D, row_weight, dh, ld_dh, dw, ld_dw, db);
    if (rc != 0) return rc;
    SV_CHECK_ARG(lse, "svae_xent_bwd: null pointer");
    if (!dh && !dw) return 0;
    if (s.few) return few(c, s, nullptr, nullptr, lse, row_weight, dh, ld_dh, dw, ld_dw, db);
    rc = prepare(c, s, false, row_weight, lse);
    if (rc != 0) return rc;
    hipLaunchKernelGGL(xent_scale_kernel, dim3(1), dim3(256), 0, c.stream, (const float*)(c.work + s.wrow), s.Rp, top_of(type), (float*)(c.work + s.scale));
    SV_LAUNCH_CHECK();
    return gradients(c, s, s.hg, dh, ld_dh, dw, ld_dw, db);
}

extern "C" int svae_xent_fwd_bwd(const void* hidden, long long ld_h, const void* weight, long long ld_w, const void* bias,
                                 const void* targets, int tok64, int type, int R, int V, int D, const float* row_weight, float* nll,
                                 float* lse, void* dh, long long ld_dh, void* dw, long long ld_dw, void* db, void* work,
                                 long long work_bytes, void* stream) {
    Call c{hidden, weight, bias, targets, ld_h, ld_w, tok64, type, R, V, D, (char*)work, (hipStream_t)stream};
    Shape s{};
    int rc = check_call("svae_xent_fwd_bwd", c, work, work_bytes, GRADIENT, &s);
    if (rc == 0) rc = check_gradients("svae_xent_fwd_bwd", D, row_weight, dh, ld_dh, dw, ld_dw, db);
    if (rc != 0) return rc;
    SV_CHECK_ARG(nll && lse, "svae_xent_fwd_bwd: null pointer");
    if (s.few) return few(c, s, nll, lse, nullptr, row_weight, dh, ld_dh, dw, ld_dw, db);
    rc = prepare(c, s, true, row_weight, nullptr);
    if (rc == 0) rc = loss(c, s, nll, lse, true);
    if (rc != 0 || (!dh && !dw)) return rc;
    return gradients(c, s, s.h, dh, ld_dh, dw, ld_dw, db);
}
