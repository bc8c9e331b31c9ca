// Classifier over many classes fused with its loss (gfx950): softmax cross
// entropy and distillation from a teacher's top logits on
//     z = H W^T + b        H [n x D] rows of hidden, W [V x D] classes,
// without ever keeping z, and their gradients.
//
// Mathematics.  With y = z log2(e) / T and L_i = log2 sum_v 2^y_iv:
//   cross entropy (T = 1)   loss_i = ln2 (L_i - y_i,label)
//   distillation            loss_i = T^2 (sum_k q_ik ln q_ik
//                                         + ln2 (L_i - sum_k q_ik y_i,k)),
//                           q_i = softmax of the teacher's listed logits / T
//   gradient                dz_iv = s_i T (2^(y_iv - L_i) - q_iv),
//                           dH = dz W, dW = dz^T H, db = column sums of dz,
// where q of cross entropy is 1 at the label.
//
// Forward: one product whose epilogue reduces each 16 TP classes of a row to
// (m, sum of 2^(y - m)) in registers; a second kernel joins them.
// Backward: pieces of the classes.  For each piece the product is made again
// and its epilogue writes G = p - q, p = 2^(y - L), in 16 bits to a scratch
// matrix (a small kernel puts a teacher's entries in place), and two products
// read G: dW's rows of the piece (complete), and dH (added up over the pieces
// in fp32).  Few rows have a kernel of their own for the logits.  Many rows go
// through in blocks, so that neither the strips' (m, sum) nor G grow with rows
// x classes.
//
// G is rounded to the operands' 16-bit type because the matrix cores take no
// wider one; p - q is formed in fp32 and rounded once.  Its factor s_i T is
// applied to the fp32 sums instead (f16: G carries 2^15, so that
// probabilities down to 2^-29 stay normal numbers).  That rounding shows at
// any number of classes: against 64 bits a bf16 gradient is off by 0.0018 to
// 0.0024 of its norm, where rounding the gradient alone is 0.0017 (f16:
// 0.00025-0.0003 against 0.0002; 4,096 rows of 47 to 65,536 classes).  Up to
// kFewClasses classes G keeps a second plane, what the rounding left over, and
// only the gradient's own rounding remains.  It costs nothing for 1,024 rows
// and, for 16,384 rows of width 256, 11% of a call at 172 classes and 25% at
// 1,024; at 2,048 it would be 40%, which is where it stops.
//
// F32 operands: x = a + b + c with three bf16 (the top, middle and low 8 of
// 24 significant bits, truncated, so the split is exact and never
// overflows), and the product is the sum of the six plane products
// ac, ca, bb, ba, ab, aa; the three left out are below 2^-23 of |x||y|, a
// rounding of the fp32 sum.  Six bf16 MFMAs take less time than one f32 MFMA
// of the same products (2,500 / 6 against 157 TFLOP/s).
//
// The product (gemm_core).  Out[q][p] = sum_k P[p,k] Q[q,k]; work-groups own
// BP x BQ tiles, waves TP x TQ tiles of v_mfma_f32_16x16x32.  Both operands
// go straight to LDS (16-byte buffer loads with range checks, so ragged
// edges read zeros), two stages of 64 k.  An operand is either contiguous
// along k (rows of 128 B a stage, 16-byte chunks XORed with the row so that
// a b128 read of 16 rows spreads over all banks) or strided along k (rows of
// BP or BQ columns, 32-byte chunks XORed with the row, read by gfx950's
// transposing LDS read, two per 32 k).
#include "grws_internal.h"

namespace grws {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 tr_v4bf16_t;
typedef __attribute__((address_space(3))) tr_v4bf16_t lds_v4bf16_t;
typedef __attribute__((address_space(3))) short8_t lds_short8_t;
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) char lds_char_t;

constexpr int kK = 64;               // k of a stage; the operands' k is padded to whole stages
constexpr int64_t kIgnoreLabel = -100;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kPastEnd = 0x80000000u;  // past every resource: the load returns zeros

// An operand in memory.  Contiguous along k: `rows` rows of `k` elements.
// Strided along k: `k` rows (the sum's index) of `rows` columns.
struct Opnd {
    const char* p;
    int64_t ld;     // bytes between rows
    int64_t plane;  // bytes between the planes of a split f32 operand
    int64_t rows;
    int64_t k;
};

struct Gemm {
    Opnd P, Q;
    int32_t nseg;    // plane products: 1, 6 for split f32 operands, or 2 (Q, which is G, in two planes)
    int32_t ksteps;  // stages per plane product
    int32_t tp, tq;  // tiles along p and q
    int32_t splits;  // work-groups per tile along k
};

// The planes of product `seg`: the last nseg of these six, small products
// first (plane 0 by plane 0 is the only one of 16-bit operands, plane 0 by Q's
// plane 1 the one before).
__device__ __forceinline__ int plane_p(int seg) { return (0x001102 >> (4 * seg)) & 15; }
__device__ __forceinline__ int plane_q(int seg) { return (0x010120 >> (4 * seg)) & 15; }

template <int DT>
__device__ __forceinline__ float4_t mma(short8_t a, short8_t b, float4_t c) {
    if constexpr (DT == GRWS_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b),
                                                      c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// One operand's tile of B rows (or columns) of a stage: its direct loads and
// its fragment reads.  PAIRED (P contiguous along k only): fragments 2 i and
// 2 i + 1 share 32 rows so that a lane's outputs of both are 8 consecutive
// ones: row r of fragment f is row 8 (r / 4) + 4 (f % 2) + r % 4.
template <bool STRIDED, int B, int NW, bool PAIRED = false>
struct Tile {
    static constexpr int BYTES = B * kK * 2;
    static constexpr int NL = BYTES / 1024 / NW;  // 1 KiB loads per wave and stage
    static_assert(NL == 4 && NL * NW * 1024 == BYTES, "four loads a wave");
    static constexpr int CH = STRIDED ? B / 8 : kK / 8;  // 16-byte chunks per row
    static constexpr int ROWS = 64 / CH;                 // rows of a load
    const char* base;
    int64_t ld, plane, left;  // left: strided: k rows; contiguous: k
    int64_t edge;             // bytes: strided: of the last row; contiguous: up to the last row
    uint32_t off[2];          // of the loads' two patterns
    int kfirst[2];            // contiguous: first k of the lane's chunk
    const char* cur;          // of the next load
    int64_t rec, some;        // bytes and k from there on

    // what a row's chunks (strided: pairs of them) are XORed with, so that
    // the rows that one LDS read takes lie in different banks
    static __device__ __forceinline__ int key(int row) {
        if constexpr (STRIDED) return ((row & 3) | (((row >> 3) & 3) << 2)) & (CH / 2 - 1);
        else return PAIRED ? (row & 3) | ((row >> 1) & 4) : row & 7;
    }
    // loads 0..3 have the keys of loads 0 1 0 1 (ROWS < 4 or 8) or 0 0 2 2
    static constexpr int pattern(int i) { return STRIDED && ROWS == 4 ? i >> 1 : i & 1; }
    static constexpr int first_of(int pat) { return STRIDED && ROWS == 4 ? 2 * pat : pat; }

    __device__ __forceinline__ void init(const Opnd& o, int64_t t0, int wave, int lane) {
        ld = o.ld;
        plane = o.plane;
        left = o.k;
        if constexpr (!STRIDED) {
            base = o.p + t0 * ld;
            const int64_t rows = o.rows - t0 < B ? o.rows - t0 : B;
            edge = (rows - 1) * ld;
        } else {
            base = o.p + t0 * 2;
            edge = (o.rows - t0) * 2;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int row = (wave * NL + first_of(v)) * ROWS + lane / CH;
            const int chunk = (lane % CH) ^ (STRIDED ? key(row) << 1 : key(row));
            off[v] = (uint32_t)(row * ld) + (uint32_t)(chunk * 16);
            kfirst[v] = chunk * 8;
        }
    }
    // the next load() reads plane `pl` from k0 on
    __device__ __forceinline__ void start(int pl, int64_t k0) {
        if constexpr (!STRIDED) {
            cur = base + pl * plane + k0 * 2;
            rec = edge + (left - k0) * 2;
        } else {
            cur = base + pl * plane + k0 * ld;
            rec = (left - k0 - 1) * ld + edge;
        }
        some = left - k0;
    }
    __device__ __forceinline__ void load(char* lds, int wave) {
        int records = rec > 0x7fffffff ? 0x7fffffff : (int)rec;
        if constexpr (STRIDED) records = rec < 0 ? 0 : records;
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)cur, (short)0, records, 0x00020000);
#pragma unroll
        for (int v = 0; v < 2; ++v) asm volatile("" : "+v"(off[v]));  // the four sums are made here, not kept
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int v = pattern(i);
            uint32_t o = off[v] + (uint32_t)((i - first_of(v)) * ROWS * ld);
            if constexpr (!STRIDED) o = kfirst[v] < some ? o : kPastEnd;  // past the row's k: not the next row's
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)((lds_char_t*)lds + (wave * NL + i) * 1024), 16,
                                                     (int)o, 0, 0, 0);
        }
        const int64_t step = STRIDED ? kK * ld : kK * 2;
        cur += step;
        rec -= step;
        some -= kK;
    }
    // rows (columns) of fragment f from `first` and k = 32 half + 8 (lane / 16)
    // + 0..7 as an MFMA operand: lane l holds row l % 16.
    static __device__ __forceinline__ short8_t frag(const char* lds, int first, int f, int half, int lane) {
        if constexpr (!STRIDED) {
            const int r = lane & 15;
            const int in = PAIRED ? 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3) : 16 * f + r;
            const char* p = lds + (first + in) * (kK * 2) + (((half * 4 + (lane >> 4)) ^ key(in)) * 16);
            return *(const lds_short8_t*)(lds_char_t*)p;
        } else {
            const int g = lane >> 4, a = (lane >> 2) & 3;
            const char* p = lds + (32 * half + 8 * g + a) * (B * 2) + ((first / 16 + f) ^ key(8 * g + a)) * 32 +
                            (lane & 3) * 8;
            const short4_t lo = __builtin_bit_cast(short4_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                                                 (lds_v4bf16_t*)(lds_char_t*)p));
            const short4_t hi = __builtin_bit_cast(short4_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                                                 (lds_v4bf16_t*)(lds_char_t*)(p + 4 * B * 2)));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// Work-group -> tile.  Work-group b runs on XCD b % 8; each XCD takes a
// contiguous run of tiles, ordered in columns of 8 q tiles, so that the
// tiles in flight on an XCD share operand rows in its L2.
__device__ __forceinline__ void tile_of(const Gemm& g, int& tp, int& tq) {
    const int n = g.tp * g.tq;
    const int b = blockIdx.x;
    const int per = n >> 3, rem = n & 7;
    const int x = b & 7;
    const int t = x * per + (x < rem ? x : rem) + (b >> 3);
    const int col = 8 * g.tp;
    const int c = t / col;
    const int w = g.tq - 8 * c < 8 ? g.tq - 8 * c : 8;
    const int r = t - c * col;
    tq = 8 * c + r % w;
    tp = r / w;
}

template <int DT, bool PS, bool QS, int BP, int BQ, int WP, int WQ>
struct Core {
    static constexpr int NW = WP * WQ;
    static constexpr int TP = BP / WP / 16, TQ = BQ / WQ / 16;
    static constexpr bool PAIRED = !PS;
    using TileP = Tile<PS, BP, NW, PAIRED>;
    using TileQ = Tile<QS, BQ, NW>;
    // p of element e of accumulator i, of the wave's block
    static __device__ __forceinline__ int p_of(int i, int lane) {
        return PAIRED ? 32 * (i >> 1) + 8 * (lane >> 4) + 4 * (i & 1) : 16 * i + 4 * (lane >> 4);
    }

    static __device__ __forceinline__ void zero(float4_t (&acc)[TP][TQ]) {
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TQ; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Adds to acc[i][j] (lane l, element e: p = p_of(i, l) + e, q = 16 j +
    // l % 16 of the wave's block) stages kb..ke of every plane product.
    static __device__ __forceinline__ void run(const Gemm& g, int tp, int tq, int kb, int ke, char* p0, char* q0,
                                               char* p1, char* q1, float4_t (&acc)[TP][TQ]) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wp = (wave % WP) * (TP * 16), wq = (wave / WP) * (TQ * 16);
        TileP P;
        TileQ Q;
        P.init(g.P, (int64_t)tp * BP, wave, lane);
        Q.init(g.Q, (int64_t)tq * BQ, wave, lane);
        const int per = ke - kb;
        if (per <= 0) return;  // uniform over the work-group
        const int total = g.nseg * per;
        int seg = 6 - g.nseg, ks = kb;
        P.start(plane_p(seg), (int64_t)kb * kK);
        Q.start(plane_q(seg), (int64_t)kb * kK);
        int left = total;  // stages to fetch
        auto fetch = [&](char* sp, char* sq) {
            if (left-- <= 0) return;  // uniform
            P.load(sp, wave);
            Q.load(sq, wave);
            if (++ks == ke) {
                ks = kb;
                ++seg;
                P.start(plane_p(seg), (int64_t)kb * kK);
                Q.start(plane_q(seg), (int64_t)kb * kK);
            }
        };
        // This wave's loads into this stage have landed before the barrier, which
        // does not wait for loads into LDS; after it every wave's have, and
        // every wave is done reading the other stage.  The buffers are named
        // arrays, one an operand and stage: the compiler otherwise waits for
        // the loads into the next stage before it reads this one (dW at 8,192
        // x 131,072 x 4,096 took 1.12 ms a piece instead of 0.90).  The next
        // stage's loads go out behind the first reads, whose latency covers
        // their address arithmetic.
        auto step = [&](char* cp, char* cq, char* np, char* nq) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < kK / 32; ++h) {
                short8_t a[TP], b[TQ];
#pragma unroll
                for (int j = 0; j < TQ; ++j) b[j] = TileQ::frag(cq, wq, j, h, lane);
#pragma unroll
                for (int i = 0; i < TP; ++i) a[i] = TileP::frag(cp, wp, i, h, lane);
                if (h == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(np, nq);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < TP; ++i)
#pragma unroll
                    for (int j = 0; j < TQ; ++j) acc[i][j] = mma<DT>(a[i], b[j], acc[i][j]);
                // no reads of the next half among these: 256 registers hold
                // the accumulators and one half's operands
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        fetch(p0, q0);
        int t = 0;
        for (; t + 1 < total; t += 2) {
            step(p0, q0, p1, q1);
            step(p1, q1, p0, q0);
        }
        if (t < total) step(p0, q0, p1, q1);
    }
};

#define GRWS_HEAD_LDS(C)                                               \
    __shared__ __attribute__((aligned(1024))) char p0[C::TileP::BYTES]; \
    __shared__ __attribute__((aligned(1024))) char q0[C::TileQ::BYTES]; \
    __shared__ __attribute__((aligned(1024))) char p1[C::TileP::BYTES]; \
    __shared__ __attribute__((aligned(1024))) char q1[C::TileQ::BYTES];

// ---------------------------------------------------------------------------
// the product's epilogues
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float4_t load_bias4(const void* bias, int64_t v, int left) {
    float4_t b{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) b[e] = to_float(static_cast<const T*>(bias)[v + e]);
    return b;
}

__device__ __forceinline__ float4_t bias4(const void* bias, int32_t dt, int64_t v, int left) {
    if (dt == GRWS_F32) return load_bias4<float>(bias, v, left);
    if (dt == GRWS_F16) return load_bias4<_Float16>(bias, v, left);
    return load_bias4<__hip_bfloat16>(bias, v, left);
}

// The sums of a wave's classes begin with their bias, or -inf past the last
// class (whose weights read as zeros).
template <typename C, int TP, int TQ>
__device__ __forceinline__ void begin_logits(float4_t (&acc)[TP][TQ], int64_t vfirst, int64_t classes,
                                             const void* bias, int32_t bias_dt, int lane) {
    C::zero(acc);
    if (!bias && vfirst + 16 * TP <= classes) return;  // uniform
    const int left = (int)(classes - vfirst < 16 * TP ? classes - vfirst : 16 * TP);
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        const int p = C::p_of(i, lane);
        float4_t b{0.f, 0.f, 0.f, 0.f};
        if (bias) b = bias4(bias, bias_dt, vfirst + p, left - p);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (p + e >= left) b[e] = -INFINITY;
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = b;
    }
}

// The maxima stay logits: two of them can be one float when multiplied by c1,
// and a hit is a matter of which is larger.  The exponentials of a row are
// 2^(z c - ref), ref the rounded m c, of a largest logit m.  c is c1, but a
// half where m c1 overflows (m a mask of the type's lowest value): floats of
// that size lie so far apart that any c leaves zero of a z other than m, and
// with a power of two m c is exact and leaves one of m.
__device__ __forceinline__ float base2(float m, float c1) {
    return fabsf(m * c1) == INFINITY && fabsf(m) != INFINITY ? 0.5f : c1;
}
// what makes a strip's sum one against m c1 itself
__device__ __forceinline__ float past_rounding(float m, float c1) {
    const float ref = m * c1;
    return fabsf(ref) == INFINITY ? 1.f : __builtin_amdgcn_exp2f(-fmaf(m, c1, -ref));
}

struct StatsArgs {
    Gemm g;
    int64_t v0, classes;  // first class of the piece, all classes
    int64_t n, np;        // rows, padded rows
    float c1;
    const void* bias;
    int32_t bias_dt;
    const int64_t* labels;  // NULL: none to look for
    float2* part;           // [strips][np]: largest logit m, sum of 2^(z c1 - the rounded m c1)
    float* ylabel;          // [n]: the label's logit
    int32_t* earlier;       // [n]: an earlier class of the label's strip has the label's logit
};

// Bound by the matrix cores for wide D (8,192 x 131,072 x 4,096 bf16: 6.6 ms,
// 1,330 TFLOP/s, MFMA busy 65% of the time; the library's plain product of
// 8,192^3 reaches 1,295) and by the exponentials, a quarter of the vector rate,
// for narrow D (16,384 x 100,003 x 256: 1.03-1.08 ms, 800 TFLOP/s; a tile's
// 8,200 MFMA cycles and about 9,000 VALU cycles follow one another).  p are
// classes and q rows, so a lane holds 4 TP classes of TQ rows and the
// reduction over classes takes two cross-lane steps a row.
template <int DT, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(WP * WQ * 64) void head_stats_kernel(StatsArgs a) {
    using C = Core<DT, false, false, BP, BQ, WP, WQ>;
    constexpr int TP = C::TP, TQ = C::TQ;
    GRWS_HEAD_LDS(C)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tp, tq;
    tile_of(a.g, tp, tq);
    float4_t acc[TP][TQ];
    const int64_t vfirst = a.v0 + (int64_t)tp * BP + (wave % WP) * (TP * 16);
    begin_logits<C>(acc, vfirst, a.classes, a.bias, a.bias_dt, lane);
    C::run(a.g, tp, tq, 0, a.g.ksteps, p0, q0, p1, q1, acc);
    const int64_t strip = vfirst / (TP * 16);
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int64_t row = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15);
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[i][j][e]);
        m = fmaxf(m, __shfl_xor(m, 16, kWave));
        m = fmaxf(m, __shfl_xor(m, 32, kWave));
        const float c1 = base2(m, a.c1), ref = m == -INFINITY ? 0.f : m * c1;  // nothing but -inf: a sum of zeros
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c1, -ref));
        s += __shfl_xor(s, 16, kWave);
        s += __shfl_xor(s, 32, kWave);
        if (lane < 16) a.part[strip * a.np + row] = make_float2(m, s);
        if (a.labels) {
            const int64_t lab = row < a.n ? a.labels[row] - vfirst : -1;
            const bool here = lab >= 0 && lab < TP * 16 && lab + vfirst < a.classes;
            if (__any(here)) {
                const int l = here ? (int)lab : 0;
                float y = 0.f;
#pragma unroll
                for (int i = 0; i < TP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y = C::p_of(i, lane) + e == l ? acc[i][j][e] : y;
                y = __shfl(y, (((l >> 3) & 3) << 4) | (lane & 15), kWave);  // its lane: p_of's
                int tie = 0;
#pragma unroll
                for (int i = 0; i < TP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        tie |= acc[i][j][e] == y && C::p_of(i, lane) + e < l;
                tie |= __shfl_xor(tie, 16, kWave);
                tie |= __shfl_xor(tie, 32, kWave);
                if (here && lane < 16) {
                    a.ylabel[row] = y;
                    a.earlier[row] = tie;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // one q at a time: the registers are full
    }
}

// What the forward leaves of a row for the gradients, p = 2^(z c - ref) factor:
//   lse = m c1 + log2 s rounded (m the largest logit, s the sum against it),
//     +inf for a row that does not count; -inf where m c1 overflows, as for
//     logits that are all masks of the type's lowest value;
//   factor: 2^(lse - m c1) / s, what the rounding took (up to 4% of p beside
//     an m of 10^6); 1 / s where lse is -inf.  Of a row that does not count 0,
//     or NaN where its zeros met a weight that is not finite.
// factor lies `stride` apart: in the place of a label's logit, or of a list's
// first probability, which nothing needs after the forward.
struct RowStats {
    const float* lse;
    const float* factor;
    int64_t stride;
    __device__ __forceinline__ float2 of(int64_t i) const { return make_float2(lse[i], factor[i * stride]); }
    RowStats from(int64_t r0) const { return RowStats{lse + r0, factor + r0 * stride, stride}; }
};

// c and ref of a row.  (Where lse is -inf every logit that is not -inf itself
// is of the largest one's size: a c of 2^-149 makes one of it.)
__device__ __forceinline__ float2 base_of(float lse, float c1) {
    return lse == -INFINITY ? make_float2(__uint_as_float(1), 0.f) : make_float2(c1, lse);
}

struct GradArgs {
    Gemm g;
    int64_t v0, classes, n;
    float c1;
    const void* bias;
    int32_t bias_dt;
    RowStats stats;
    const int64_t* labels;   // NULL: the targets are subtracted by head_subtract_kernel
    const float* row_scale;  // [n] or NULL
    float gscale;
    uint16_t* G;  // [planes][np][ldg]
    int64_t ldg, plane;
    float* bias_part;  // [np / kBiasRows][vt]: column sums, or NULL
    int64_t vt;
};

__device__ __forceinline__ uint16_t top16(float x) { return (uint16_t)(__float_as_uint(x) >> 16); }
__device__ __forceinline__ float from_top16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }

// x = a + b + c exactly: three truncated bf16.  A NaN goes into a (with a bit
// in its upper half).  An infinity goes into c, which meets only the other
// operand's a in the six plane products, so that its products have the sign
// they should (in a it would meet zero planes: NaN); a is then one of its
// sign, for the other operand's infinities to meet.
__device__ __forceinline__ void split3(float x, uint16_t* a, uint16_t* b, uint16_t* c) {
    *a = top16(x);
    if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) {
        *b = *c = 0;
        if (x != x) {
            *a |= 0x40;
        } else {
            *c = *a;
            *a = (*a & 0x8000) | 0x3f80;
        }
        return;
    }
    const float r = x - from_top16(*a);
    *b = top16(r);
    *c = top16(r - from_top16(*b));
}

template <int DT>
__device__ __forceinline__ uint16_t round16(float x) {
    if constexpr (DT == GRWS_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
    else return __builtin_bit_cast(uint16_t, __float2bfloat16(x));
}

template <int DT>
__device__ __forceinline__ float from16(uint16_t h) {
    if constexpr (DT == GRWS_F16) return (float)__builtin_bit_cast(_Float16, h);
    else return from_top16(h);
}

// an entry of G in its planes
template <int DT, int PLANES>
__device__ __forceinline__ void planes_of(float x, uint16_t (&h)[PLANES]) {
    if constexpr (PLANES == 3) {
        split3(x, &h[0], &h[1], &h[2]);
    } else {
        h[0] = round16<DT>(x);
        if constexpr (PLANES == 2) h[1] = round16<DT>(x - from16<DT>(h[0]));
    }
}

// x of the lane N further in its row of 16
template <int N>
__device__ __forceinline__ float rotate(float x) {
    return __builtin_bit_cast(float,
                              __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, true));
}

constexpr int kBiasRows = 64;  // rows of a part of the bias gradient's sums

// The same product, leaving G.  8,192 x 65,536 of 4,096: 3.52 ms (1,250
// TFLOP/s); 16,384 x 20,224 of 256: 304 us (558), where 660 MB of G go out
// beside the exponentials.
template <int DT, int PLANES, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(WP * WQ * 64) void head_grad_kernel(GradArgs a) {
    using C = Core<DT, false, false, BP, BQ, WP, WQ>;
    constexpr int TP = C::TP, TQ = C::TQ;
    GRWS_HEAD_LDS(C)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tp, tq;
    tile_of(a.g, tp, tq);
    float4_t acc[TP][TQ];
    const int64_t pfirst = (int64_t)tp * BP + (wave % WP) * (TP * 16);
    // the rows' statistics are here when the product is (asked for behind it,
    // 16,384 x 20,224 of 256 takes 322 us, not 300); run() has barriers
    __shared__ float2 row_stats[BQ];
    if (threadIdx.x < BQ) {
        const int64_t row = (int64_t)tq * BQ + threadIdx.x;
        row_stats[threadIdx.x] = row < a.n ? a.stats.of(row) : make_float2(INFINITY, 0.f);
    }
    begin_logits<C>(acc, a.v0 + pfirst, a.classes, a.bias, a.bias_dt, lane);
    C::run(a.g, tp, tq, 0, a.g.ksteps, p0, q0, p1, q1, acc);
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int64_t row = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15);
        // of a row that does not count, whose lse is +inf, all are 2^-inf
        // (its hidden row is zeros, so a logit is its bias)
        const float2 st = row_stats[row - (int64_t)tq * BQ];
        const float lse = st.x, c1 = base_of(lse, a.c1).x, ref = base_of(lse, a.c1).y;
        const float s = a.row_scale && row < a.n ? a.row_scale[row] * a.gscale : a.gscale;
        const bool stray = row >= a.n || (lse == INFINITY && st.y != 0.f);
        const float f = stray ? 0.f : st.y * s;
        if (__any(stray)) {
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = stray ? -INFINITY : acc[i][j][e];
        }
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c1, -ref));
#pragma unroll
        for (int i = 0; i < TP; ++i) acc[i][j] *= f;
        if (a.labels) {
            const int64_t lab = lse != INFINITY ? a.labels[row] - a.v0 - pfirst : -1;
            const bool here = lab >= 0 && lab < TP * 16;
            if (__any(here)) {
                const int at = here ? (int)lab : -1;
#pragma unroll
                for (int i = 0; i < TP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] -= at == C::p_of(i, lane) + e ? s : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < TP; i += 2) {  // 8 consecutive classes of accumulators i and i + 1
            const int64_t at = row * a.ldg + pfirst + C::p_of(i, lane);
            uint16_t h[8][PLANES];
#pragma unroll
            for (int e = 0; e < 8; ++e) planes_of<DT, PLANES>(acc[i + (e >> 2)][j][e & 3], h[e]);
#pragma unroll
            for (int z = 0; z < PLANES; ++z) {
                u32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (uint32_t)h[2 * e][z] | ((uint32_t)h[2 * e + 1][z] << 16);
                *reinterpret_cast<u32x4_t*>(a.G + z * a.plane + at) = w;
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // one q at a time: the registers are full
    }
    if (a.bias_part) {
        // the wave's 64 rows: TQ of a lane, then the 16 lanes that share the
        // classes (rotations within a row of 16 lanes)
        static_assert(TQ * 16 == kBiasRows, "rows of a part");
        const int64_t at = ((int64_t)tq * WQ + wave / WP) * a.vt + pfirst;
#pragma unroll
        for (int i = 0; i < TP; ++i) {
            float4_t x = acc[i][0];
#pragma unroll
            for (int j = 1; j < TQ; ++j) x += acc[i][j];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] += rotate<8>(x[e]);
                x[e] += rotate<4>(x[e]);
                x[e] += rotate<2>(x[e]);
                x[e] += rotate<1>(x[e]);
            }
            if ((lane & 15) == 0) *reinterpret_cast<float4_t*>(a.bias_part + at + C::p_of(i, lane)) = x;
        }
    }
}

// four consecutive elements of a row with `left` of them to go
template <int OT>
__device__ __forceinline__ void store4(void* out, int64_t at, float4_t v, int64_t left, int32_t vec) {
    if constexpr (OT == GRWS_F32) {
        float* o = static_cast<float*>(out) + at;
        if (vec && left >= 4) {
            *reinterpret_cast<float4_t*>(o) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) o[e] = v[e];
        }
    } else {
        uint16_t* o = static_cast<uint16_t*>(out) + at;
        uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = round16<OT>(v[e]);
        if (vec && left >= 4) {
            *reinterpret_cast<u32x2_t*>(o) =
                u32x2_t{(uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) o[e] = h[e];
        }
    }
}

// dW rows of a piece: p are columns of H, q the piece's classes, k the rows,
// cut into `splits` runs when the tiles alone leave CUs idle (their fp32 sums
// are added in order by head_weight_out_kernel).  65,536 x 4,096 over 8,192
// rows: 3.63 ms (1,212 TFLOP/s; both operands take two 8-byte LDS reads where
// the others take one of 16 bytes).
struct WeightArgs {
    Gemm g;
    const float* alpha;
    void* out;  // first class of the piece
    int64_t ldo, classes, width;  // classes of the piece
    int32_t vec;  // rows of the output take 4-element stores
    float* part;  // [splits][vp][dp], or NULL: this one run is all of the sum
    int64_t vp, dp;
    int32_t first;  // the first block of rows stores, the others add
};

template <int DT, int OT, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(WP * WQ * 64) void head_dweight_kernel(WeightArgs a) {
    using C = Core<DT, true, true, BP, BQ, WP, WQ>;
    constexpr int TP = C::TP, TQ = C::TQ;
    GRWS_HEAD_LDS(C)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tp, tq;
    tile_of(a.g, tp, tq);
    const int sp = blockIdx.y;
    const int kb = (int)((int64_t)a.g.ksteps * sp / a.g.splits), ke = (int)((int64_t)a.g.ksteps * (sp + 1) / a.g.splits);
    float4_t acc[TP][TQ];
    C::zero(acc);
    C::run(a.g, tp, tq, kb, ke, p0, q0, p1, q1, acc);
    if (a.part) {
        float* out = a.part + sp * a.vp * a.dp;
#pragma unroll
        for (int j = 0; j < TQ; ++j) {
            const int64_t v = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15);
#pragma unroll
            for (int i = 0; i < TP; ++i) {
                const int64_t d = (int64_t)tp * BP + (wave % WP) * (TP * 16) + C::p_of(i, lane);
                if (d >= a.dp || v >= a.classes) continue;
                float4_t* o = reinterpret_cast<float4_t*>(out + v * a.dp + d);
                *o = a.first ? acc[i][j] : *o + acc[i][j];
            }
        }
        return;
    }
    const float alpha = *a.alpha;
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int64_t v = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15);
        if (v >= a.classes) continue;
#pragma unroll
        for (int i = 0; i < TP; ++i) {
            const int64_t d = (int64_t)tp * BP + (wave % WP) * (TP * 16) + C::p_of(i, lane);
            if (d >= a.width) continue;
            store4<OT>(a.out, v * a.ldo + d, acc[i][j] * alpha, a.width - d, a.vec);
        }
    }
}

// dH of a piece: p are columns of W, q the rows, k the piece's classes, cut
// into `splits` runs; each run adds to its own fp32 sums (piece after piece,
// so the order is fixed).  8,192 x 4,096 over 65,536 classes: 3.33 ms (1,320
// TFLOP/s).

struct HiddenArgs {
    Gemm g;
    float* part;  // [splits][np][dp]
    int64_t np, dp;
    int32_t first;  // the first piece stores
    // the last piece of a single run writes dH itself
    int32_t last;
    int32_t vec;  // rows of the output take 4-element stores
    const float* alpha;
    void* out;
    int64_t ldo, n, width, hidden_rows;
    const int64_t* rows;
    RowStats stats;  // a row that does not count gets zeros, whatever alpha and W hold
};

template <int DT, int OT, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(WP * WQ * 64) void head_dhidden_kernel(HiddenArgs a) {
    using C = Core<DT, true, false, BP, BQ, WP, WQ>;
    constexpr int TP = C::TP, TQ = C::TQ;
    GRWS_HEAD_LDS(C)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tp, tq;
    tile_of(a.g, tp, tq);
    const int sp = blockIdx.y;
    const int kb = (int)((int64_t)a.g.ksteps * sp / a.g.splits), ke = (int)((int64_t)a.g.ksteps * (sp + 1) / a.g.splits);
    float4_t acc[TP][TQ];
    C::zero(acc);
    C::run(a.g, tp, tq, kb, ke, p0, q0, p1, q1, acc);
    float* out = a.part + sp * a.np * a.dp;
    // the rows' places and factors (0: does not count), all asked for at once
    int64_t place[TQ];
    float factor[TQ];
    const float alpha = a.last ? *a.alpha : 0.f;
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int64_t row = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15);
        const bool live = a.last && row < a.n;
        place[j] = !live ? -1 : a.rows ? a.rows[row] : row;
        if (place[j] >= a.hidden_rows) place[j] = -1;
        factor[j] = live && a.stats.lse[row] != INFINITY ? alpha : 0.f;
    }
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int64_t row = (int64_t)tq * BQ + (wave / WP) * (TQ * 16) + 16 * j + (lane & 15), to = place[j];
#pragma unroll
        for (int i = 0; i < TP; ++i) {
            const int64_t d = (int64_t)tp * BP + (wave % WP) * (TP * 16) + C::p_of(i, lane);
            if (d >= a.dp) continue;
            float4_t* o = reinterpret_cast<float4_t*>(out + row * a.dp + d);
            const float4_t v = a.first ? acc[i][j] : *o + acc[i][j];
            if (!a.last) *o = v;
            else if (to >= 0 && d < a.width)
                store4<OT>(a.out, to * a.ldo + d, factor[j] != 0.f ? v * factor[j] : float4_t{0.f, 0.f, 0.f, 0.f},
                           a.width - d, a.vec);
        }
    }
}

// ---------------------------------------------------------------------------
// small kernels
// ---------------------------------------------------------------------------
// A row counts when it has a target: a label in range, or a listed teacher
// entry.  0: does not count, 1: counts, 2: bad input (counts as none).
struct Targets {
    const int64_t* labels;
    const void* tindex;
    const float* tlogit;
    const int64_t* rows;
    int64_t hidden_rows, classes;
    int32_t k, i64;
};

__device__ __forceinline__ int64_t teacher_at(const Targets& t, int64_t i, int k) {
    return t.i64 ? static_cast<const int64_t*>(t.tindex)[i * t.k + k]
                 : (int64_t) static_cast<const int32_t*>(t.tindex)[i * t.k + k];
}

// an entry of weight zero (a logit of -inf) is not listed
__device__ __forceinline__ bool teacher_listed(const Targets& t, int64_t i, int k, int64_t idx) {
    return idx >= 0 && idx < t.classes && t.tlogit[i * t.k + k] != -INFINITY;
}

// `lanes` lanes of a wave, of which this is `sub`, ask together (all of them
// with the same i); the answer is the same in each.
template <int LANES>
__device__ __forceinline__ int row_state(const Targets& t, int64_t i, int sub) {
    const int64_t row = t.rows ? t.rows[i] : i;
    if (row < 0 || row >= t.hidden_rows) return 2;
    if (t.labels) {
        const int64_t l = t.labels[i];
        if (l == kIgnoreLabel) return 0;
        return l >= 0 && l < t.classes ? 1 : 2;
    }
    int st = 0;
    for (int k = sub; k < t.k; k += LANES) {
        const int64_t idx = teacher_at(t, i, k);
        if (idx < -1 || idx >= t.classes) st |= 2;
        else if (teacher_listed(t, i, k, idx)) st |= 1;
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) st |= __shfl_xor(st, d, kWave);
    return st & 2 ? 2 : st;
}

// The factor of the gradient sums: dloss T / (counted gscale), or for a
// gradient per row the largest finite |dloss| in place of dloss / counted, with
// the rows' shares of it in row_scale (so that G stays within 16 bits' range)
struct Alpha {
    float* out;  // NULL: none
    const float* dloss;
    const int64_t* counts;
    const uint32_t* most;  // NULL: of the mean
    float factor;
};

// (8,192 rows of 4,096 bf16 packed: 24 us, 5.6 TB/s read and written.)
// Copies a row of `width` elements to dp 16-bit elements (three planes of
// f32), zeros past the width; a wave, 8 elements a lane.
template <typename T, bool SPLIT>
__device__ __forceinline__ void pack_row(const T* __restrict__ x, bool live, int64_t width, int64_t dp, bool vec,
                                         uint16_t* __restrict__ out, int64_t plane, int lane) {
    for (int64_t c = lane * 8; c < dp; c += 512) {
        T v[8] = {};
        if (live && c < width) {
            if (vec && c + 8 <= width) {
                __builtin_memcpy(v, __builtin_assume_aligned(x + c, 16), sizeof(v));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < width) v[e] = x[c + e];
            }
        }
        uint16_t h[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (SPLIT) split3(v[e], &h[0][e], &h[1][e], &h[2][e]);
            else h[0][e] = v[e];
        }
#pragma unroll
        for (int z = 0; z < (SPLIT ? 3 : 1); ++z) {
            u32x4_t w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)h[z][2 * e] | ((uint32_t)h[z][2 * e + 1] << 16);
            *reinterpret_cast<u32x4_t*>(out + z * plane + c) = w;
        }
    }
}

// hidden[rows] in the layout the products read: np rows of dp elements (one
// plane, or three for f32), zeros past n and the width and in rows that do
// not count (what such a row holds, NaN too, stays out of every sum).
// One wave per row; the first also makes alpha (see Alpha) or clears `done`.
// owner (or NULL): owner[rows[i]] = i, of a row listed again any of its i.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void head_pack_hidden_kernel(Targets t, const T* __restrict__ hidden, int64_t ld,
                                                               int64_t n, int64_t np, int64_t width, int64_t dp,
                                                               int32_t vec, uint16_t* __restrict__ out, Alpha al,
                                                               int32_t* __restrict__ done, int32_t* owner) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= np) return;
    if (owner && lane == 0 && i < n && t.rows[i] >= 0 && t.rows[i] < t.hidden_rows)
        __hip_atomic_store(owner + t.rows[i], (int32_t)i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (i == 0 && lane == 0) {
        if (done) *done = 0;
        if (al.out) {
            if (al.most) *al.out = __uint_as_float(*al.most) * al.factor;
            else *al.out = al.counts[1] > 0 ? al.dloss[0] / (float)al.counts[1] * al.factor : 0.f;
        }
    }
    const bool live = i < n && row_state<64>(t, i, lane) == 1;
    const T* x = hidden + (live ? (t.rows ? t.rows[i] : i) * ld : 0);
    pack_row<T, SPLIT>(x, live, width, dp, vec, out + i * dp, np * dp, lane);
}

// weight rows v0.. of the piece likewise (`vp` rows)
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void head_pack_weight_kernel(const T* __restrict__ w, int64_t ld, int64_t rows,
                                                               int64_t vp, int64_t width, int64_t dp, int32_t vec,
                                                               uint16_t* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= rows) return;
    pack_row<T, SPLIT>(w + i * ld, true, width, dp, vec, out + i * dp, vp * dp, threadIdx.x & 63);
}

// 8 elements from c (zeros past the width) as floats
template <typename T>
__device__ __forceinline__ void load8(const T* x, int64_t c, int64_t width, bool vec, float (&f)[8]) {
    T v[8] = {};
    if (vec && c + 8 <= width) {
        __builtin_memcpy(v, __builtin_assume_aligned(x + c, 16), sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < width) v[e] = x[c + e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_float(v[e]);
}

// The student's logits at the teacher's entries, a wave per 4 entries of a
// row (16 lanes share a dot product): n k rows of W are read, from beyond the
// L2 (8,192 x 64 rows of 2 KB: 225 us, 4.8 TB/s).  The row's first wave also makes the teacher's probabilities: prob
// [n k] (0 where an entry is not listed) and coef [n k], what the
// gradient subtracts at the entry's class: the sum over the entries that list
// the class, at the first of them; -1 at every other entry.
template <typename T>
__global__ __launch_bounds__(256) void head_targets_kernel(Targets t, const T* __restrict__ hidden, int64_t ldh,
                                                           const T* __restrict__ w, int64_t ldw, const T* bias,
                                                           int64_t n, int64_t width, int32_t vec, float inv_t,
                                                           float* __restrict__ prob, float* __restrict__ coef,
                                                           float* __restrict__ y, int32_t* __restrict__ state) {
    const int lane = threadIdx.x & 63;
    const int groups = (t.k + 3) / 4;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= n * groups) return;
    const int64_t i = at / groups;
    const int k0 = (int)(at - i * groups) * 4;
    const int st = row_state<64>(t, i, lane);
    const bool live = st == 1;  // uniform over the wave
    {
        const T* h = hidden + (live ? (t.rows ? t.rows[i] : i) * ldh : 0);
        const int k = k0 + (lane >> 4);
        int64_t idx = -1;
        if (live && k < t.k) {
            idx = teacher_at(t, i, k);
            if (!teacher_listed(t, i, k, idx)) idx = -1;
        }
        const T* x = w + (idx >= 0 ? idx * ldw : 0);
        float d = 0.f;
        if (idx >= 0) {
            for (int64_t c = (lane & 15) * 8; c < width; c += 128) {
                float a[8], b[8];
                load8(h, c, width, vec, a);
                load8(x, c, width, vec, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) d += a[e] * b[e];
            }
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) d += __shfl_xor(d, x, kWave);
        if ((lane & 15) == 0 && k < t.k)
            y[i * t.k + k] = idx >= 0 ? d + (bias ? to_float(bias[idx]) : 0.f) : 0.f;
    }
    if (k0 != 0) return;
    if (lane == 0) state[i] = st;
    float m = -INFINITY;
    for (int k = lane; k < t.k && live; k += 64)
        if (teacher_listed(t, i, k, teacher_at(t, i, k))) m = fmaxf(m, t.tlogit[i * t.k + k] * inv_t);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    float s = 0.f;
    for (int k = lane; k < t.k && live; k += 64)
        if (teacher_listed(t, i, k, teacher_at(t, i, k))) s += expf(t.tlogit[i * t.k + k] * inv_t - m);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, kWave);
    auto entry = [&](int k, int64_t* idx) {
        *idx = live && k < t.k ? teacher_at(t, i, k) : -1;
        if (*idx >= 0 && !teacher_listed(t, i, k, *idx)) *idx = -1;
        return *idx >= 0 ? expf(t.tlogit[i * t.k + k] * inv_t - m) / s : 0.f;
    };
    for (int kb = 0; kb < t.k; kb += 64) {
        const int k = kb + lane;
        int64_t idx;
        const float q = entry(k, &idx);
        float sum = q;
        bool first = true;
        for (int ob = 0; ob < t.k; ob += 64) {
            int64_t oidx;
            const float oq = entry(ob + lane, &oidx);
            const int most = t.k - ob < 64 ? t.k - ob : 64;
            for (int o = 0; o < most; ++o) {
                const int other = __shfl((int)oidx, o, kWave);
                const float p = __shfl(oq, o, kWave);
                if (ob + o != k && other == (int)idx) {
                    sum += p;
                    first = first && ob + o > k;
                }
            }
        }
        if (k < t.k) {
            prob[i * t.k + k] = q;
            coef[i * t.k + k] = idx >= 0 && first ? sum : -1.f;
        }
    }
}

// Logits of few rows (16 NQ a work-group, 64 at most): W is read once, as it lies, straight
// into the MFMA's operands; nothing of it is packed or staged.  A wave owns 32
// classes; f32 operands go to the f32 MFMA.  Forward: the strips' statistics
// (strips of 32 classes); backward (GRAD): G.  Bound by W's stream.
struct FewArgs {
    Targets t;
    const void *hidden, *weight, *bias;
    int64_t ldh, ldw, n, np, width, v0, vend, classes;  // classes v0..vend of a piece
    float c1;
    // forward
    const int32_t* states;  // of a teacher's lists
    float2* part;
    float* ylabel;
    int32_t* earlier;
    int32_t* done;
    // backward
    RowStats stats;
    const float* row_scale;
    float gscale;
    uint16_t* G;
    int64_t ldg, plane;
    float* bias_part;
    int64_t vt;
};

template <typename T, int NQ, int PLANES, bool VEC>
__global__ __launch_bounds__(256) void head_few_kernel(FewArgs a) {
    constexpr bool GRAD = PLANES > 0;
    constexpr int DT = std::is_same_v<T, _Float16> ? GRWS_F16 : GRWS_BF16;
    constexpr int E = 16 / sizeof(T);  // elements of a 16-byte load
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int64_t first = (int64_t)blockIdx.y * (16 * NQ);  // row
    if (!GRAD && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.done = 0;
    const int64_t vfirst = a.v0 + ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 32;
    const T* w[2];
    const T* h[NQ];
    bool live[NQ];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t v = vfirst + 16 * i + r;
        w[i] = static_cast<const T*>(a.weight) + (v < a.classes ? v : 0) * a.ldw;
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int64_t row = first + 16 * j + r;
        if constexpr (GRAD) live[j] = row < a.n && a.stats.lse[row] != INFINITY;
        else live[j] = row < a.n && (a.t.labels ? row_state<1>(a.t, row, 0) : a.states[row]) == 1;
        h[j] = static_cast<const T*>(a.hidden) + (live[j] ? (a.t.rows ? a.t.rows[row] : row) * a.ldh : 0);
    }
    float4_t acc[2][NQ];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
    struct Frag {
        T x[E];
    };
    auto read = [&](const T* p, int64_t c, bool whole) {
        Frag f;
        if (VEC && whole) {
            __builtin_memcpy(&f, __builtin_assume_aligned(p + c, 16), 16);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) f.x[e] = whole || c + e < a.width ? p[c + e] : from_float<T>(0.f);
        }
        return f;
    };
    constexpr int STEP = 4 * E;                       // k of a step: the four lane groups
    constexpr int U = NQ == 1 ? 4 : NQ == 2 ? 3 : 2;  // steps whose loads are in flight
    auto multiply = [&](int64_t c, int steps, bool whole) {
        Frag x[U][2], y[U][NQ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= steps) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) x[u][i] = read(w[i], c + u * STEP, whole);
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                y[u][j] = read(h[j], c + u * STEP, whole);
                if (!live[j]) y[u][j] = Frag{};  // what such a row holds stays out
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= steps) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[u][i].x[e], y[u][j].x[e], acc[i][j], 0,
                                                                             0, 0);
                    } else {
                        acc[i][j] = mma<DT>(__builtin_bit_cast(short8_t, x[u][i]),
                                            __builtin_bit_cast(short8_t, y[u][j]), acc[i][j]);
                    }
                }
        }
    };
    int64_t c = g * E;
    for (; c - g * E + U * STEP <= a.width; c += U * STEP) multiply(c, U, true);
    for (; c - g * E + STEP <= a.width; c += STEP) multiply(c, 1, true);
    if (c - g * E < a.width) multiply(c, 1, false);
    // class vfirst + 16 i + 4 g + e
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t v = vfirst + 16 * i + 4 * g + e;
            const bool in = v < a.vend;
            const float b = a.bias && in ? to_float(static_cast<const T*>(a.bias)[v]) : 0.f;
#pragma unroll
            for (int j = 0; j < NQ; ++j) acc[i][j][e] = in ? acc[i][j][e] + b : -INFINITY;
        }
    float4_t sums[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int64_t row = first + 16 * j + r;
        const int64_t lab = live[j] && a.t.labels ? a.t.labels[row] - vfirst : -1;
        const bool here = lab >= 0 && lab < 32;
        const int l = here ? (int)lab : -1;
        if constexpr (!GRAD) {
            float m = -INFINITY, y = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m = fmaxf(m, acc[i][j][e]);
                    y = 16 * i + 4 * g + e == l ? acc[i][j][e] : y;
                }
            m = fmaxf(m, __shfl_xor(m, 16, kWave));
            m = fmaxf(m, __shfl_xor(m, 32, kWave));
            y = __shfl(y, (((l >> 2) & 3) << 4) | r, kWave);
            const float c1 = base2(m, a.c1), ref = m == -INFINITY ? 0.f : m * c1;
            float s = 0.f;
            int tie = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c1, -ref));
                    tie |= acc[i][j][e] == y && 16 * i + 4 * g + e < l;
                }
            s += __shfl_xor(s, 16, kWave);
            s += __shfl_xor(s, 32, kWave);
            tie |= __shfl_xor(tie, 16, kWave);
            tie |= __shfl_xor(tie, 32, kWave);
            if (g == 0) {
                a.part[vfirst / 32 * a.np + row] = make_float2(m, s);
                if (here) {
                    a.ylabel[row] = y;
                    a.earlier[row] = tie;
                }
            }
        } else {
            const float2 st = live[j] ? a.stats.of(row) : make_float2(INFINITY, 0.f);
            const float c1 = base_of(st.x, a.c1).x, ref = base_of(st.x, a.c1).y;
            const float sc = a.row_scale && live[j] ? a.row_scale[row] * a.gscale : a.gscale;
            const float f = st.y * sc;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint16_t x[4][PLANES > 0 ? PLANES : 1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p = live[j] ? __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c1, -ref)) * f : 0.f;
                    p = 16 * i + 4 * g + e == l ? p - sc : p;
                    sums[i][e] += p;
                    planes_of<DT, PLANES>(p, x[e]);
                }
#pragma unroll
                for (int z = 0; z < PLANES; ++z)
                    *reinterpret_cast<u32x2_t*>(a.G + z * a.plane + row * a.ldg + (vfirst - a.v0) + 16 * i + 4 * g) =
                        u32x2_t{(uint32_t)x[0][z] | ((uint32_t)x[1][z] << 16),
                                (uint32_t)x[2][z] | ((uint32_t)x[3][z] << 16)};
            }
        }
    }
    if constexpr (GRAD) {
        // the padding rows, which dW's product reads: the last rows' work-group
        const bool last = blockIdx.y + 1 == gridDim.y;
        for (int64_t row = first + 16 * NQ + r; last && row < a.np; row += 16)
#pragma unroll
            for (int z = 0; z < PLANES; ++z)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *reinterpret_cast<u32x2_t*>(a.G + z * a.plane + row * a.ldg + (vfirst - a.v0) + 16 * i + 4 * g) =
                        u32x2_t{0u, 0u};
        if (a.bias_part) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sums[i][e] += rotate<8>(sums[i][e]);
                    sums[i][e] += rotate<4>(sums[i][e]);
                    sums[i][e] += rotate<2>(sums[i][e]);
                    sums[i][e] += rotate<1>(sums[i][e]);
                }
                // 16 NQ rows are a part, or (up to 64 rows) the only one with rows
                for (int64_t b = blockIdx.y; b < (last ? a.np / kBiasRows : blockIdx.y + 1); ++b)
                    if (r == 0)
                        *reinterpret_cast<float4_t*>(a.bias_part + b * a.vt + (vfirst - a.v0) + 16 * i + 4 * g) =
                            b == blockIdx.y ? sums[i] : float4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
}

// dH of few f32 rows: W is read once, as it lies, on the f32 MFMA; a wave owns
// 64 columns of 16 NQ rows over a run of classes, 16 at a time: lane (g, r)
// reads columns 4 r .. + 3 of classes 4 g .. + 3 (256 bytes a class), which are
// the operands of four tiles with columns 4 r + c.  1 row x 32,000 x 2,048 with
// gradients: 702 -> 463 us against dH from packed planes of W, 64 rows 791 ->
// 667, 128 rows 895 -> 865.
struct FewHiddenArgs {
    const float* weight;  // first class of the piece
    int64_t ldw, width, dp, n, np, vc;
    const uint16_t* G;
    int64_t ldg, plane;
    float* part;  // [splits][np][dp]
    int32_t splits, first;
};

template <int NQ, bool VEC>
__global__ __launch_bounds__(256) void head_few_dhidden_kernel(FewHiddenArgs a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int64_t sp = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
    if (sp >= a.splits) return;  // uniform over the wave
    const int64_t d0 = (int64_t)blockIdx.x * 64, first = (int64_t)blockIdx.z * (16 * NQ);
    const int64_t blocks = (a.vc + 15) / 16, kb = blocks * sp / a.splits, ke = blocks * (sp + 1) / a.splits;
    const int64_t d = d0 + 4 * r;
    const bool whole = VEC && d + 4 <= a.width;
    float4_t acc[4][NQ];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[c][j] = float4_t{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 2;  // blocks whose loads are in flight
    auto multiply = [&](int64_t b, int some) {
        float4_t w[U][4], x[U][NQ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= some) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t v = (b + u) * 16 + 4 * g + k;
                w[u][k] = float4_t{0.f, 0.f, 0.f, 0.f};
                if (v < a.vc) {
                    const float* p = a.weight + v * a.ldw + d;
                    if (whole) {
                        w[u][k] = *reinterpret_cast<const float4_t*>(p);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (d + c < a.width) w[u][k][c] = p[c];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                const uint16_t* q = a.G + (first + 16 * j + r) * a.ldg + (b + u) * 16 + 4 * g;
                uint16_t h[3][4];
#pragma unroll
                for (int z = 0; z < 3; ++z) __builtin_memcpy(h[z], __builtin_assume_aligned(q + z * a.plane, 8), 8);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    x[u][j][k] = from_top16(h[0][k]) + (from_top16(h[1][k]) + from_top16(h[2][k]));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= some) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < NQ; ++j)
                        acc[c][j] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(w[u][k][c], x[u][j][k], acc[c][j], 0, 0, 0);
        }
    };
    int64_t b = kb;
    for (; b + U <= ke; b += U) multiply(b, U);
    for (; b < ke; ++b) multiply(b, 1);
    // acc[c][j][e]: column 4 (4 g + e) + c, row 16 j + r
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int64_t row = first + 16 * j + r;
        if (row >= a.n) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float4_t* o =
                reinterpret_cast<float4_t*>(a.part + (sp * a.np + row) * a.dp + d0 + 16 * g + 4 * e);
            const float4_t x{acc[0][j][e], acc[1][j][e], acc[2][j][e], acc[3][j][e]};
            *o = a.first ? x : *o + x;
        }
    }
}

__device__ __forceinline__ void join(float c1, float& m, float& s, int& first, float om, float os, int ofirst) {
    if (om > m) {
        s = s * __builtin_amdgcn_exp2f((m - om) * c1) + os;
        m = om;
        first = ofirst;
    } else {
        s += om == -INFINITY ? os : os * __builtin_amdgcn_exp2f((om - m) * c1);
        if (om == m && ofirst < first) first = ofirst;
    }
}

// loss = sum / counted (NaN when no row counts or an input is bad), by one
// wave; parts are added in a fixed order
__device__ __forceinline__ void finish_loss(const double* part_loss, const int32_t* part_cnt,
                                            int64_t nparts, int lane, float* loss, int64_t* counts) {
    double L = 0.0;
    long long C = 0, V = 0, B = 0;
#pragma unroll 8
    for (int64_t k = lane; k < nparts; k += 64) {
        L += part_loss[k];
        C += part_cnt[3 * k];
        V += part_cnt[3 * k + 1];
        B |= part_cnt[3 * k + 2];
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        L += __shfl_xor(L, d, kWave);
        C += __shfl_xor(C, d, kWave);
        V += __shfl_xor(V, d, kWave);
        B |= __shfl_xor(B, d, kWave);
    }
    if (lane != 0) return;
    if (loss) loss[0] = (B || V == 0) ? __int_as_float(0x7fc00000) : (float)(L / (double)V);
    counts[0] = C;
    counts[1] = V;
    counts[2] = B;
}

// Joins the strips of R rows (512 / R at a time), then the rows' losses, and
// their mean and counts (loss_out and row_loss may be NULL).  R = 4 spreads
// few rows over more work-groups: 333 rows of 512 strips 15 -> 8 us.
template <int R>
__global__ __launch_bounds__(512) void head_join_kernel(Targets t, const float2* __restrict__ part, int64_t strips,
                                                        int32_t strip_classes, int64_t n, int64_t np,
                                                        float temperature, float c1, float* __restrict__ y,
                                                        float* __restrict__ prob,
                                                        const int32_t* __restrict__ flags, float* __restrict__ lse,
                                                        float* __restrict__ row_loss, double* part_loss,
                                                        int32_t* part_cnt, int32_t* done,
                                                        float* __restrict__ loss_out, int64_t* __restrict__ counts) {
    __shared__ float sm[8][R], ss[8][R];
    __shared__ int sa[8][R];
    constexpr int G = 64 / R;  // lanes of a wave that share a row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane % R, g = lane / R;
    const int64_t i = (int64_t)blockIdx.x * R + r;
    float m = -INFINITY, s = 0.f;
    int first = 0x7fffffff;  // the first strip with the maximum
    auto join_lanes = [&]() {
#pragma unroll
        for (int d = R; d < 64; d <<= 1) {
            const float om = __shfl_xor(m, d, kWave), os = __shfl_xor(s, d, kWave);
            const int of = __shfl_xor(first, d, kWave);
            // both sides join in the same order, so a row's lanes agree
            if (lane & d) {
                float m2 = om, s2 = os;
                int f2 = of;
                join(c1, m2, s2, f2, m, s, first);
                m = m2, s = s2, first = f2;
            } else {
                join(c1, m, s, first, om, os, of);
            }
        }
    };
    if (i < n) {
#pragma unroll 4
        for (int64_t k = wave * G + g; k < strips; k += 8 * G) {
            const float2 v = part[k * np + i];
            join(c1, m, s, first, v.x, v.y * past_rounding(v.x, c1), (int)k);
        }
    }
    join_lanes();
    if (g == 0) {
        sm[wave][r] = m;
        ss[wave][r] = s;
        sa[wave][r] = first;
    }
    __syncthreads();
    if (wave != 0) return;
    m = -INFINITY, s = 0.f, first = 0x7fffffff;
    for (int w = g; w < 8; w += G) join(c1, m, s, first, sm[w][r], ss[w][r], sa[w][r]);
    join_lanes();
    int st = 0;
    if (i < n) st = t.labels ? row_state<1>(t, i, 0) : flags[i];
    // the largest logit and the logarithm are not added before the target's
    // logit is taken off: a confident row's loss is far below its logits
    const float lns = log2f(s) * kLn2;
    float a = 0.f;
    if (!t.labels && st == 1) {
        // sum of q (ln q + (m - z) / T + ln s); an entry of probability zero
        // says nothing of its class (whose logit may be -inf)
        for (int k = g; k < t.k; k += G) {
            const float q = prob[i * t.k + k];
            if (!(q <= 0.f)) a += q * (logf(q) + ((m - y[i * t.k + k]) / temperature + lns));
        }
    }
#pragma unroll
    for (int d = R; d < 64; d <<= 1) a += __shfl_xor(a, d, kWave);
    double loss = 0.0;
    int hit = 0, valid = 0, bad = 0;
    if (g == 0 && i < n) {
        float v = 0.f;
        if (st == 1) {
            valid = 1;
            if (t.labels) {
                const float yl = y[i];
                v = m - yl + lns;
                hit = yl == m && !flags[i] && first == (int)(t.labels[i] / strip_classes);
            } else {
                v = a * temperature * temperature;
            }
            loss = (double)v;
        } else if (st == 2) {
            bad = 1;
            v = __int_as_float(0x7fc00000);
        }
        // see RowStats.  (A live row with a logit of +inf, or a largest one
        // whose m c1 is +inf, has nothing but NaN.)
        const float nan = __int_as_float(0x7fc00000);
        float l = INFINITY, f = s == s ? 0.f : s;
        if (st == 1) {
            l = fmaf(m, c1, log2f(s));
            f = l == -INFINITY ? (s > 0.f ? 1.f / s : nan) : __builtin_amdgcn_exp2f(-fmaf(m, c1, -l)) / s;
            if (l == INFINITY) l = nan;
        }
        lse[i] = l;
        (t.labels ? y : prob)[i * (t.labels ? 1 : t.k)] = f;
        if (row_loss) row_loss[i] = v;
    }
#pragma unroll
    for (int d = R / 2; d > 0; d >>= 1) {
        loss += __shfl_xor(loss, d, kWave);
        hit += __shfl_xor(hit, d, kWave);
        valid += __shfl_xor(valid, d, kWave);
        bad |= __shfl_xor(bad, d, kWave);
    }
    // the last work-group to arrive adds the parts, in their order
    int last = 0;
    if (lane == 0) {
        part_loss[blockIdx.x] = loss;
        part_cnt[3 * blockIdx.x] = hit;
        part_cnt[3 * blockIdx.x + 1] = valid;
        part_cnt[3 * blockIdx.x + 2] = bad;
    }
    if (!done) return;
    if (lane == 0) {
        __threadfence();
        last = atomicAdd(done, 1) == (int)gridDim.x - 1;
    }
    if (!__shfl(last, 0, kWave)) return;
    __threadfence();
    finish_loss(part_loss, part_cnt, gridDim.x, lane, loss_out, counts);
}

// owner[rows[i]] = i, where the rows are packed a block at a time
__global__ __launch_bounds__(256) void head_owner_kernel(const int64_t* __restrict__ rows, int64_t n,
                                                         int64_t hidden_rows, int32_t* owner) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i < n ? rows[i] : -1;
    if (row < 0 || row >= hidden_rows) return;
    __hip_atomic_store(owner + row, (int32_t)i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// d_hidden of a row that is listed more than once: each listing has a gradient
// of its own and one of them was kept.  All but one find another's number in
// owner and put NaN there, which is seen, and the one that was kept is not.
template <typename T>
__global__ __launch_bounds__(256) void head_repeated_kernel(const int64_t* __restrict__ rows, int64_t n,
                                                            int64_t hidden_rows, const int32_t* __restrict__ owner,
                                                            int64_t width, T* out, int64_t ldo) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i < n ? rows[i] : -1;
    if (row < 0 || row >= hidden_rows || owner[row] == (int32_t)i) return;
    for (int64_t d = 0; d < width; ++d) out[row * ldo + d] = from_float<T>(__int_as_float(0x7fc00000));
}

// finish_loss in a launch of its own (also of no rows at all)
__global__ __launch_bounds__(64) void head_finish_kernel(const double* part_loss, const int32_t* part_cnt,
                                                         int64_t nparts, float* __restrict__ loss,
                                                         int64_t* __restrict__ counts) {
    finish_loss(part_loss, part_cnt, nparts, threadIdx.x, loss, counts);
}

__global__ __launch_bounds__(256) void head_most_kernel(const float* __restrict__ dloss,
                                                        RowStats stats, int64_t n,
                                                        uint32_t* __restrict__ most) {
    // of non-negative floats the largest is the largest as an integer: the
    // order of the atomics does not matter.  Infinities and NaN are left out:
    // they are their rows' own shares, not a factor of every row
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    uint32_t m = i < n && stats.lse[i] != INFINITY ? __float_as_uint(fabsf(dloss[i])) : 0u;
    if (m >= 0x7f800000u) m = 0u;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t o = __shfl_xor(m, d, kWave);
        m = o > m ? o : m;
    }
    if ((threadIdx.x & 63) == 0 && m) atomicMax(most, m);
}

// 0 for a row that does not count, whatever dloss holds there: its G is zeros
// times this.  (Without a factor other than 0, infinity and NaN: 0 or NaN.)
__global__ __launch_bounds__(256) void head_row_scale_kernel(const float* __restrict__ dloss,
                                                             RowStats stats, int64_t n,
                                                             const uint32_t* __restrict__ most,
                                                             float* __restrict__ scale) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const float m = __uint_as_float(*most);
    scale[i] = stats.lse[i] == INFINITY ? 0.f : m > 0.f ? dloss[i] / m : dloss[i] * 0.f;
}

// G at a teacher's entries: the rounded p - q, q the entry's coefficient.
// (A label's place is known to the product's epilogue: one for a row.)
template <int DT, int PLANES>
__global__ __launch_bounds__(256) void head_subtract_kernel(Targets t, RowStats stats,
                                                            const float* __restrict__ y,
                                                            const float* __restrict__ coef,
                                                            const float* __restrict__ row_scale, float gscale,
                                                            float c1, int64_t n, int64_t v0, int64_t vc, uint16_t* G,
                                                            int64_t ldg, int64_t plane) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= n * t.k) return;
    const int64_t i = at / t.k;
    const int64_t v = teacher_at(t, i, (int)(at - i * t.k));
    if (v < v0 || v >= v0 + vc) return;
    const float q = coef[at];
    const float2 st = stats.of(i), b = base_of(st.x, c1);
    if (q < 0.f || st.x == INFINITY) return;
    const float s = row_scale ? row_scale[i] * gscale : gscale;
    uint16_t h[PLANES];
    planes_of<DT, PLANES>((exp2f(fmaf(y[at], b.x, -b.y)) * st.y - q) * s, h);
#pragma unroll
    for (int z = 0; z < PLANES; ++z) G[z * plane + i * ldg + (v - v0)] = h[z];
}

// The teacher's share of a part of the bias gradient (kBiasRows rows): the
// epilogue has summed p, this takes off q, unrounded both.  A work-group adds
// the part's entries in kBiasClasses of the classes in LDS, in whole units of
// 2^-40, so that the order does not matter (global atomics, of 200,000 rows of
// 5 entries in 47 classes, took 1.5 ms; this 12 us).
constexpr int kBiasClasses = 4096;
constexpr float kBiasUnit = 1099511627776.f;

__global__ __launch_bounds__(256) void head_bias_targets_kernel(Targets t, RowStats stats,
                                                                const float* __restrict__ coef,
                                                                const float* __restrict__ row_scale, float gscale,
                                                                int64_t n, int64_t v0, int64_t vc, int64_t vt,
                                                                float* __restrict__ part) {
    __shared__ unsigned long long sum[kBiasClasses];
    __shared__ int bad;
    const int64_t first = (int64_t)blockIdx.x * kBiasRows, c0 = (int64_t)blockIdx.y * kBiasClasses;
    const int classes = (int)(vc - c0 < kBiasClasses ? vc - c0 : kBiasClasses);
    const int rows = (int)(n - first < kBiasRows ? n - first : kBiasRows);  // none, of a padding part
    for (int c = threadIdx.x; c < classes; c += 256) sum[c] = 0;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    float* out = part + blockIdx.x * vt + c0;
    auto entries = [&](auto use) {
        for (int e = threadIdx.x; e < rows * t.k; e += 256) {
            const int64_t i = first + e / t.k, at = first * t.k + e;
            const int64_t c = teacher_at(t, i, e % t.k) - v0 - c0;
            if (c < 0 || c >= classes || coef[at] < 0.f || stats.lse[i] == INFINITY) continue;
            use((int)c, row_scale ? coef[at] * row_scale[i] : coef[at]);
        }
    };
    entries([&](int c, float q) {
        if (fabsf(q) < INFINITY) atomicAdd(sum + c, (unsigned long long)__float2ll_rn(q * kBiasUnit));
        else bad = 1;
    });
    __syncthreads();
    for (int c = threadIdx.x; c < classes; c += 256)
        if (sum[c]) out[c] -= gscale * (float)((double)(long long)sum[c] / (double)kBiasUnit);
    if (!bad) return;  // uniform
    __syncthreads();
    entries([&](int c, float q) {
        if (!(fabsf(q) < INFINITY)) out[c] = __int_as_float(0x7fc00000);
    });
}

// 16 waves share 64 columns.  sum: NULL, or [vc] of the blocks of rows before,
// in their order (first: none); only the last block writes the gradient.
template <typename T>
__global__ __launch_bounds__(1024) void head_bias_kernel(const float* __restrict__ part, int64_t nparts, int64_t vp,
                                                         int64_t vc, const float* __restrict__ alpha,
                                                         float* __restrict__ sum, int32_t first, int32_t last,
                                                         T* __restrict__ out) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (c < vc) {
#pragma unroll 4
        for (int64_t k = wave; k < nparts; k += 16) s += part[k * vp + c];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= vc) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][lane];
    if (!first) s += sum[c];
    if (last) out[c] = from_float<T>(s * *alpha);
    else sum[c] = s;
}

// Adds the splits' sums in order and applies alpha, 4 columns a lane: dW of a
// piece (rows in place), or dH (to the rows they belong to)
template <typename T>
__device__ __forceinline__ void sum_splits(const float* __restrict__ part, int64_t splits, int64_t stride,
                                           int64_t width, float a, bool keep, T* __restrict__ out) {
    for (int64_t d = threadIdx.x * 4; d < width; d += blockDim.x * 4) {
        float4_t s{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int64_t k = 0; k < splits; ++k) s += *reinterpret_cast<const float4_t*>(part + k * stride + d);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < width) out[d + e] = from_float<T>(keep ? s[e] * a : 0.f);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void head_weight_out_kernel(const float* __restrict__ part, int64_t splits,
                                                              int64_t vp, int64_t dp, int64_t width,
                                                              const float* __restrict__ alpha, T* __restrict__ out,
                                                              int64_t ldo) {
    const int64_t v = blockIdx.x;
    sum_splits(part + v * dp, splits, vp * dp, width, *alpha, true, out + v * ldo);
}

template <typename T>
__global__ __launch_bounds__(256) void head_hidden_out_kernel(const float* __restrict__ part, int64_t splits,
                                                              int64_t np, int64_t dp, int64_t width,
                                                              const int64_t* __restrict__ rows, int64_t hidden_rows,
                                                              RowStats stats,
                                                              const float* __restrict__ alpha, T* __restrict__ out,
                                                              int64_t ldo) {
    const int64_t i = blockIdx.x;
    const int64_t row = rows ? rows[i] : i;
    if (row < 0 || row >= hidden_rows) return;
    const bool keep = stats.lse[i] != INFINITY;  // a row that does not count gets zeros
    sum_splits(part + i * dp, splits, np * dp, width, *alpha, keep, out + row * ldo);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
int64_t ceil_div(int64_t x, int64_t a) { return (x + a - 1) / a; }

// work-groups of head_join_kernel up to which the last of them finishes the
// loss (each writes its L2's lines back for it: 1,024 of them take 29 us more
// against a launch of 5)
constexpr int64_t kJoinBlocks = 128;
// G of a piece: 16,384 rows x 100,003 classes at width 256 take 5.0 ms with
// 256 MiB, 4.70 with 512 and 4.54 with 1 GiB (fewer, fuller launches); at
// 8,192 x 131,072 x 4,096 it makes 1%.
constexpr int64_t kPieceBytes = (int64_t)1 << 30;
// Rows are taken in blocks where the scratch would otherwise grow with rows x
// classes: the strips' statistics of a forward block stay within kPartBytes
// (8 bytes a row and strip), and a backward block leaves G room for
// kLeastPiece classes a piece.  At most kBlockRows rows, so that no launch
// has 2^32 threads.
constexpr int64_t kPartBytes = (int64_t)512 << 20;
constexpr int64_t kLeastPiece = 4096;
constexpr int64_t kBlockRows = (int64_t)1 << 20;
constexpr int64_t kFewClasses = 1024;  // up to here G has a second plane
// Rows up to which head_few_kernel makes the logits.  Forward calls on 32,000 x
// 2,048, replayed in a graph, against the products (on packed W, where it has
// to be): f32 1 row 73 against 479 us, 64 rows 110 against 486, 128 (two
// readings of W) 227 against 486; 16-bit rows that are not 16-byte aligned 54
// against 117 at 1 row, 71 against 120 at 32; aligned ones, which need no
// packing, 33 against 50 at 1 row, 40 against 51 at 16.
constexpr int64_t kFewRows = 16, kFewPacked = 32, kFewF32 = 128;
constexpr int64_t kPackBytes = (int64_t)256 << 20;  // a packed piece of W

// A product's tile and the runs that its k is cut into: the least of
//   rounds of work-groups x (stages of a run + what a work-group costs besides)
// in stages of a 256-tile (1.6 us).  256-tiles run one to a CU, 128-tiles two,
// at 0.7 of their rate; a run's fp32 sums cost 16 stages to write and add up.
struct Plan {
    int tile;
    int64_t splits;
    double cost;
};

Plan plan(int64_t p, int64_t q, int64_t stages, int64_t most_splits, double besides) {
    Plan best{128, 1, 1e300};
    for (int tile = 256; tile >= 128; tile -= 128) {
        if (tile == 256 && (p <= 128 || q <= 128)) continue;  // padded to 128 only
        const int64_t tiles = ceil_div(p, tile) * ceil_div(q, tile);
        const int64_t slots = tile == 256 ? 256 : 512;
        const double step = tile == 256 ? 1.0 : 0.71, fixed = tile == 256 ? besides : 0.5 * besides;
        for (int64_t sp = 1; sp <= most_splits && (sp == 1 || tiles * sp <= 4 * slots); ++sp) {
            const double t = (double)ceil_div(tiles * sp, slots) *
                             ((double)ceil_div(stages, sp) * step + fixed + (sp > 1 ? 16 * step : 0));
            if (t < best.cost) best = Plan{tile, sp, t};
        }
    }
    return best;
}

// Sizes of a call, the same for the workspace query and the launch.
struct Shape {
    int64_t n, D, V;
    int64_t blocks, nb;  // blocks of rows, rows of a block
    int planes, gplanes;  // of the operands, of G
    bool split;       // f32 operands in three planes
    bool pack_w;      // W goes through a packed copy
    bool few;         // few rows: head_few_kernel makes the logits
    int64_t np, dp, vp;  // padded rows of a block, and width; classes of a piece
    int64_t ldg;         // pitch of G: rows start 256 bytes apart mod 4 KiB
    Plan logits, weight, hidden;
    int64_t strips, strip_classes;  // the forward's
};

bool weight_in_place(const grws_head* h) {
    return h->dtype != GRWS_F32 && h->ld_weight % 8 == 0 && h->width % 8 == 0 &&
           reinterpret_cast<uintptr_t>(h->weight) % 16 == 0;
}

// to whole 128-tiles, or 256-tiles where there is more than one of 128
int64_t pad(int64_t x) { return x <= 128 ? 128 : up(x, 256); }

Shape shape_of(const grws_head* h, bool backward) {
    Shape s{};
    s.n = h->n;
    s.D = h->width;
    s.V = h->classes;
    s.split = h->dtype == GRWS_F32;
    s.planes = s.split ? 3 : 1;
    s.gplanes = s.split ? 3 : s.V <= kFewClasses ? 2 : 1;
    s.pack_w = !weight_in_place(h);
    s.few = s.n <= (s.split ? kFewF32 : s.pack_w ? kFewPacked : kFewRows);
    s.dp = up(s.D, kK);
    s.vp = pad(s.V);
    int64_t rows = kBlockRows;
    auto limit = [&](int64_t bytes, int64_t row_bytes) {
        if (rows > bytes / row_bytes) rows = bytes / row_bytes;
    };
    limit(kPieceBytes, 2 * s.planes * s.dp);                                     // the packed rows
    if (backward) limit(kPieceBytes, 2 * s.gplanes * ((s.vp < kLeastPiece ? s.vp : kLeastPiece) + 128));
    else limit(kPartBytes, 8 * (s.vp / 64));
    limit((int64_t)1 << 31, 64 * ceil_div(h->k, 4) + 1);                         // threads of head_targets_kernel
    rows = rows < 256 ? 256 : rows / 256 * 256;
    s.blocks = ceil_div(s.n, rows);
    s.nb = s.blocks == 1 ? s.n : up(ceil_div(s.n, s.blocks), 256);
    s.blocks = ceil_div(s.n, s.nb);
    s.np = pad(s.nb);
    auto bound = [&](int64_t bytes, int64_t column_bytes) {
        int64_t most = bytes / column_bytes / 256 * 256;
        if (most < 256) most = 256;
        if (s.vp > most) s.vp = most;
    };
    if (backward) bound(kPieceBytes, 2 * s.gplanes * s.np);
    if (backward && s.blocks > 1) bound(kPieceBytes, 4 * s.dp);  // dW's sums over the blocks
    if (s.pack_w) bound(kPackBytes, 2 * s.planes * s.dp);
    bound((int64_t)1 << 29, 1);  // a launch's threads
    const int64_t seg = s.split ? 6 : 1, gseg = s.split ? 6 : s.gplanes;
    // the pieces: as few and as equal as the bound allows, or up to three
    // more where the tiles then fill the rounds better
    const int64_t fewest = ceil_div(s.V, s.vp), whole = s.vp;
    double least = 1e300;
    for (int64_t pieces = fewest; pieces < fewest + (fewest > 1 ? 4 : 1); ++pieces) {
        int64_t vp = fewest > 1 ? up(ceil_div(s.V, pieces), 256) : whole;
        if (vp > whole) vp = whole;
        const Plan l = plan(vp, s.np, seg * s.dp / kK, 1, 6);
        Plan w{}, d{};
        if (backward) {
            w = plan(s.D, vp, gseg * s.np / kK, ceil_div(s.np / kK, 4), 4);
            d = plan(s.dp, s.np, gseg * vp / kK, s.blocks > 1 ? 1 : ceil_div(vp / kK, 4), 4);
        }
        const double t = (double)ceil_div(s.V, vp) * (l.cost + w.cost + d.cost + 6);
        if (t < least) {
            least = t;
            s.vp = vp;
            s.logits = l;
            s.weight = w;
            s.hidden = d;
        }
    }
    if (backward && s.few && s.split) {
        // dH by head_few_dhidden_kernel: 2,048 waves, of at least 8 blocks of 16 classes
        int64_t sp = ceil_div(2048, s.dp / 64 * ceil_div(s.n, 64));
        const int64_t most = s.vp / 128;
        if (sp > most) sp = most;
        s.hidden.splits = sp < 2 ? 2 : sp;  // two at least: the runs are added up apart
    }
    s.strip_classes = s.few ? 32 : s.logits.tile / 2;
    s.strips = pad(s.V) / s.strip_classes;
    s.ldg = s.vp + 128;
    return s;
}

// Rows r0.. of a call (n of them) as a call of their own.
grws_head rows_of(const grws_head* h, int64_t r0, int64_t n) {
    grws_head b = *h;
    b.n = n;
    if (h->rows) {
        b.rows += r0;
    } else {
        b.hidden = static_cast<const char*>(h->hidden) + r0 * h->ld_hidden * dtype_size(h->dtype);
        b.hidden_rows -= r0;
    }
    if (h->k == 0) {
        b.labels += r0;
    } else {
        b.teacher_index = static_cast<const char*>(h->teacher_index) + r0 * h->k * (h->index_is_i64 ? 8 : 4);
        b.teacher_logits += r0 * h->k;
    }
    return b;
}

// The shape of a call's block of rows from r0 on.
Shape block_of(const Shape& s, int64_t r0) {
    Shape b = s;
    b.n = s.n - r0 < s.nb ? s.n - r0 : s.nb;
    if (s.blocks > 1) b.np = up(b.n, 256);
    return b;
}

int check_head(const grws_head* h) {
    GRWS_CHECK_ARG(h != nullptr, "head: null description");
    if (h->dtype != GRWS_F32 && h->dtype != GRWS_F16 && h->dtype != GRWS_BF16)
        return set_error(GRWS_E_DTYPE, "head: unsupported dtype %d", h->dtype);
    GRWS_CHECK_ARG(h->n >= 0 && h->n <= INT32_MAX && h->hidden_rows >= 0, "head: bad row count");
    GRWS_CHECK_ARG(h->width > 0 && h->width <= 65536, "head: width must be 1..65536");
    GRWS_CHECK_ARG(h->classes > 0 && h->classes <= INT32_MAX - 1024, "head: bad class count");
    GRWS_CHECK_ARG(h->ld_hidden >= h->width && h->ld_weight >= h->width && h->ld_hidden <= (1 << 21) &&
                       h->ld_weight <= (1 << 21),
                   "head: leading dimensions must be the width at least and 2^21 at most");
    GRWS_CHECK_ARG(h->k >= 0 && h->k <= 1024, "head: at most 1024 teacher entries a row");
    GRWS_CHECK_ARG(h->temperature > 0.f && h->temperature < INFINITY, "head: the temperature must be positive");
    if (h->n > 0) {
        GRWS_CHECK_ARG(h->hidden && h->weight, "head: null pointer");
        if (h->k == 0) {
            GRWS_CHECK_ARG(h->labels != nullptr, "head: null labels");
            GRWS_CHECK_ARG(h->temperature == 1.f, "head: labels take no temperature");
        } else {
            GRWS_CHECK_ARG(h->teacher_index && h->teacher_logits && !h->labels, "head: null teacher lists");
        }
    }
    return GRWS_OK;
}

Targets targets_of(const grws_head* h) {
    return Targets{h->labels, h->teacher_index, h->teacher_logits, h->rows, h->hidden_rows, h->classes,
                   h->k, h->index_is_i64};
}

struct FwdSpace {
    uint16_t *hp, *wp;
    float2* part;
    int32_t* flags;  // labels: StatsArgs::earlier; a teacher's lists: the rows' states
    double* pl;
    int32_t *pc, *done;
};

template <typename A>
void fwd_space(A& a, const Shape& s, FwdSpace* f) {
    auto take = [&](auto*& p, int64_t n) {
        using T = std::remove_reference_t<decltype(*p)>;
        if constexpr (std::is_same_v<A, Sizer>) a.template take<T>((size_t)n);
        else p = a.template take<T>((size_t)n);
    };
    if (!s.few) take(f->hp, s.planes * s.np * s.dp);
    if (s.pack_w && !s.few) take(f->wp, s.planes * s.vp * s.dp);
    take(f->part, s.strips * s.np);
    take(f->flags, s.nb);
    take(f->pl, s.n <= 8 ? 8 : ceil_div(s.n, 4));
    take(f->pc, s.n <= 8 ? 24 : 3 * ceil_div(s.n, 4));
    take(f->done, 1);
}

struct BwdSpace {
    uint16_t *hp, *wp, *G;
    float *dh, *dw, *bias, *bias_sum, *alpha, *scale;
    uint32_t* most;
    int32_t* owner;  // see head_repeated_kernel
};

template <typename A>
void bwd_space(A& a, const Shape& s, const grws_head* h, BwdSpace* f) {
    auto take = [&](auto*& p, int64_t n) {
        using T = std::remove_reference_t<decltype(*p)>;
        if constexpr (std::is_same_v<A, Sizer>) a.template take<T>((size_t)n);
        else p = a.template take<T>((size_t)n);
    };
    take(f->hp, s.planes * s.np * s.dp);
    if (s.pack_w && !(s.few && s.split)) take(f->wp, s.planes * s.vp * s.dp);
    take(f->G, s.gplanes * s.np * s.ldg);
    // several pieces: of all rows; several runs (of one block only): of each
    if (s.hidden.splits > 1 || s.vp < s.V) take(f->dh, s.hidden.splits * s.blocks * s.np * s.dp);
    if (s.weight.splits > 1 || s.blocks > 1) take(f->dw, s.weight.splits * s.vp * s.dp);
    take(f->bias, s.np / kBiasRows * s.vp);
    if (s.blocks > 1) take(f->bias_sum, s.vp);
    take(f->alpha, 1);
    take(f->scale, s.n);
    take(f->most, 1);
    if (h->rows) take(f->owner, h->hidden_rows);
}

// whether 8 elements of a row may be read as 16-byte vectors
bool rows_of_16(const void* p, int64_t ld, int32_t dtype) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % (dtype == GRWS_F32 ? 4 : 8) == 0;
}

int pack_hidden(const grws_head* h, const Shape& s, const Targets& t, uint16_t* hp, const Alpha& alpha,
                int32_t* done, int32_t* owner, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(s.np, 4));
    const int32_t vec = rows_of_16(h->hidden, h->ld_hidden, h->dtype);
    if (s.split)
        hipLaunchKernelGGL((head_pack_hidden_kernel<float, true>), grid, dim3(256), 0, stream, t,
                           static_cast<const float*>(h->hidden), h->ld_hidden, s.n, s.np, s.D, s.dp, vec, hp, alpha,
                           done, owner);
    else
        hipLaunchKernelGGL((head_pack_hidden_kernel<uint16_t, false>), grid, dim3(256), 0, stream, t,
                           static_cast<const uint16_t*>(h->hidden), h->ld_hidden, s.n, s.np, s.D, s.dp, vec, hp, alpha,
                           done, owner);
    GRWS_LAUNCH_CHECK();
    return GRWS_OK;
}

// The piece's rows of W as an operand, packed first where they have to be.
int weight_piece(const grws_head* h, const Shape& s, int64_t v0, int64_t vc, uint16_t* wp, bool strided, Opnd* o,
                 bool pack, hipStream_t stream) {
    if (!s.pack_w) {
        const char* p = static_cast<const char*>(h->weight) + v0 * h->ld_weight * 2;
        *o = strided ? Opnd{p, h->ld_weight * 2, 0, s.D, vc} : Opnd{p, h->ld_weight * 2, 0, vc, s.D};
        return GRWS_OK;
    }
    if (pack) {
        const dim3 grid((unsigned)ceil_div(vc, 4));
        const int32_t vec = rows_of_16(h->weight, h->ld_weight, h->dtype);
        if (s.split)
            hipLaunchKernelGGL((head_pack_weight_kernel<float, true>), grid, dim3(256), 0, stream,
                               static_cast<const float*>(h->weight) + v0 * h->ld_weight, h->ld_weight, vc, s.vp, s.D,
                               s.dp, vec, wp);
        else
            hipLaunchKernelGGL((head_pack_weight_kernel<uint16_t, false>), grid, dim3(256), 0, stream,
                               static_cast<const uint16_t*>(h->weight) + v0 * h->ld_weight, h->ld_weight, vc, s.vp,
                               s.D, s.dp, vec, wp);
        GRWS_LAUNCH_CHECK();
    }
    const char* p = reinterpret_cast<const char*>(wp);
    const int64_t plane = s.vp * s.dp * 2;
    *o = strided ? Opnd{p, s.dp * 2, plane, s.dp, vc} : Opnd{p, s.dp * 2, plane, vc, s.dp};
    return GRWS_OK;
}

Opnd hidden_operand(const Shape& s, const uint16_t* hp, bool strided) {
    const char* p = reinterpret_cast<const char*>(hp);
    const int64_t plane = s.np * s.dp * 2;
    return strided ? Opnd{p, s.dp * 2, plane, s.dp, s.np} : Opnd{p, s.dp * 2, plane, s.np, s.dp};
}

Gemm gemm_of(const Shape& s, const Plan& pl, const Opnd& P, const Opnd& Q, int64_t np, int64_t nq, int64_t k,
             int planes) {
    return Gemm{P, Q, planes == 3 ? 6 : planes, (int32_t)ceil_div(k, kK), (int32_t)ceil_div(np, pl.tile),
                (int32_t)ceil_div(nq, pl.tile), (int32_t)pl.splits};
}

template <typename T, int PLANES>
int launch_few(const grws_head* h, const FewArgs& a, hipStream_t stream) {
    const bool vec = rows_of_16(h->weight, h->ld_weight, h->dtype) && rows_of_16(h->hidden, h->ld_hidden, h->dtype);
    const dim3 grid((unsigned)ceil_div(a.vt, 128), (unsigned)ceil_div(a.n, 64));
#define GRWS_HEAD_FEW(NQ)                                                                                         \
    do {                                                                                                          \
        if (vec) hipLaunchKernelGGL((head_few_kernel<T, NQ, PLANES, true>), grid, dim3(256), 0, stream, a);        \
        else hipLaunchKernelGGL((head_few_kernel<T, NQ, PLANES, false>), grid, dim3(256), 0, stream, a);           \
    } while (0)
    if (a.n <= 16) GRWS_HEAD_FEW(1);
    else if (a.n <= 32) GRWS_HEAD_FEW(2);
    else GRWS_HEAD_FEW(4);
#undef GRWS_HEAD_FEW
    GRWS_LAUNCH_CHECK();
    return GRWS_OK;
}

// NAME<..., BP, BQ, WP, WQ> at a plan's tile
#define GRWS_HEAD_LAUNCH(PLAN, NAME, ARGS, ...)                                                                      \
    do {                                                                                                             \
        GRWS_CHECK_ARG((int64_t)ARGS.g.tp * ARGS.g.tq * 512 < (int64_t)1 << 32, "head: 2^32 threads or more");       \
        const dim3 grid_((unsigned)(ARGS.g.tp * ARGS.g.tq), (unsigned)ARGS.g.splits);                                \
        if (PLAN.tile == 256)                                                                                        \
            hipLaunchKernelGGL((NAME<__VA_ARGS__, 256, 256, 2, 4>), grid_, dim3(512), 0, stream, ARGS);              \
        else                                                                                                         \
            hipLaunchKernelGGL((NAME<__VA_ARGS__, 128, 128, 2, 2>), grid_, dim3(256), 0, stream, ARGS);              \
        GRWS_LAUNCH_CHECK();                                                                                         \
    } while (0)

// G of a piece of the classes and a block of the rows, and what the two
// products add of it to dW and dH.
int backward_block(const grws_head* h, const Shape& s, const BwdSpace& f, int64_t v0, int64_t vc, int64_t r0,
                   const RowStats& all_stats, const float* target_logit, const float* target_prob, bool per_row,
                   const Alpha& alpha, float c1, float gscale, void* d_hidden, int64_t ld_dh,
                   void* d_weight, int64_t ld_dw, void* d_bias, hipStream_t stream) {
    const Shape sb = block_of(s, r0);
    const grws_head hb = rows_of(h, r0, sb.n);
    const Targets t = targets_of(&hb);
    const size_t esz = dtype_size(h->dtype);
    const RowStats stats = all_stats.from(r0);
    const float* row_scale = per_row ? f.scale + r0 : nullptr;
    const bool first_rows = r0 == 0, last_rows = r0 + sb.n == s.n;
    const int64_t plane = sb.np * s.ldg;
    const int64_t vt = up(vc, s.few ? 128 : s.logits.tile);  // G's columns that are written
    if (s.blocks > 1) GRWS_TRY(pack_hidden(&hb, sb, t, f.hp, alpha, nullptr, nullptr, stream));
    Opnd W;
#define GRWS_HEAD_PLANES(X)                                  \
    do {                                                     \
        if (s.split) X(GRWS_BF16, 3);                        \
        else if (h->dtype == GRWS_F16 && s.gplanes == 1) X(GRWS_F16, 1); \
        else if (h->dtype == GRWS_F16) X(GRWS_F16, 2);       \
        else if (s.gplanes == 1) X(GRWS_BF16, 1);            \
        else X(GRWS_BF16, 2);                                \
    } while (0)
    if (s.few) {
        FewArgs a{};
        a.t = t;
        a.hidden = h->hidden, a.weight = h->weight, a.bias = h->bias;
        a.ldh = h->ld_hidden, a.ldw = h->ld_weight, a.n = s.n, a.np = s.np, a.width = s.D;
        a.v0 = v0, a.vend = v0 + vc, a.classes = s.V, a.c1 = c1;
        a.stats = stats, a.row_scale = row_scale, a.gscale = gscale, a.G = f.G, a.ldg = s.ldg, a.plane = plane;
        a.bias_part = d_bias ? f.bias : nullptr, a.vt = vt;
        if (s.split) GRWS_TRY((launch_few<float, 3>(h, a, stream)));
        else if (h->dtype == GRWS_F16 && s.gplanes == 1) GRWS_TRY((launch_few<_Float16, 1>(h, a, stream)));
        else if (h->dtype == GRWS_F16) GRWS_TRY((launch_few<_Float16, 2>(h, a, stream)));
        else if (s.gplanes == 1) GRWS_TRY((launch_few<__hip_bfloat16, 1>(h, a, stream)));
        else GRWS_TRY((launch_few<__hip_bfloat16, 2>(h, a, stream)));
    } else {
        GRWS_TRY(weight_piece(h, s, v0, vc, f.wp, false, &W, first_rows, stream));
        GradArgs a{gemm_of(s, s.logits, W, hidden_operand(sb, f.hp, false), vc, sb.np, s.dp, s.planes),
                   v0, s.V, sb.n, c1, h->bias,
                   h->dtype, stats, hb.labels, row_scale, gscale, f.G, s.ldg, plane,
                   d_bias ? f.bias : nullptr, vt};
#define GRWS_HEAD_GRAD(DT, PL) GRWS_HEAD_LAUNCH(s.logits, head_grad_kernel, a, DT, PL)
        GRWS_HEAD_PLANES(GRWS_HEAD_GRAD);
#undef GRWS_HEAD_GRAD
    }
    if (h->k > 0) {
        const dim3 grid((unsigned)ceil_div(sb.n * h->k, 256));
        const float *y = target_logit + r0 * h->k, *coef = target_prob + (s.n + r0) * h->k;
#define GRWS_HEAD_SUB(DT, PL)                                                                                      \
    hipLaunchKernelGGL((head_subtract_kernel<DT, PL>), grid, dim3(256), 0, stream, t, stats, y, coef, row_scale, gscale, \
                       c1, sb.n, v0, vc, f.G, s.ldg, plane)
        GRWS_HEAD_PLANES(GRWS_HEAD_SUB);
#undef GRWS_HEAD_SUB
        GRWS_LAUNCH_CHECK();
        if (d_bias) {
            const dim3 parts((unsigned)(sb.np / kBiasRows), (unsigned)ceil_div(vc, kBiasClasses));
            hipLaunchKernelGGL(head_bias_targets_kernel, parts, dim3(256), 0, stream, t, stats, coef, row_scale, gscale,
                               sb.n, v0, vc, vt, f.bias);
            GRWS_LAUNCH_CHECK();
        }
    }
    const char* gp = reinterpret_cast<const char*>(f.G);
    if (d_bias) {
        const int64_t nparts = sb.np / kBiasRows;
        const dim3 cg((unsigned)ceil_div(vc, 64));
        char* db = static_cast<char*>(d_bias) + v0 * esz;
#define GRWS_HEAD_BIAS(T)                                                                               \
    hipLaunchKernelGGL(head_bias_kernel<T>, cg, dim3(1024), 0, stream, f.bias, nparts, vt, vc, f.alpha, \
                       f.bias_sum, first_rows, last_rows, reinterpret_cast<T*>(db))
        if (h->dtype == GRWS_F32) GRWS_HEAD_BIAS(float);
        else if (h->dtype == GRWS_F16) GRWS_HEAD_BIAS(_Float16);
        else GRWS_HEAD_BIAS(__hip_bfloat16);
#undef GRWS_HEAD_BIAS
        GRWS_LAUNCH_CHECK();
    }
#undef GRWS_HEAD_PLANES
    if (d_weight) {
        char* out = static_cast<char*>(d_weight) + v0 * ld_dw * esz;
        const int32_t vec = reinterpret_cast<uintptr_t>(d_weight) % (4 * esz) == 0 && ld_dw % 4 == 0;
        const Opnd G{gp, s.ldg * 2, plane * 2, s.ldg, sb.np};
        WeightArgs w{gemm_of(s, s.weight, hidden_operand(sb, f.hp, true), G, s.D, vc, sb.np, s.gplanes),
                     f.alpha, out, ld_dw, vc, s.D, vec, s.weight.splits > 1 || s.blocks > 1 ? f.dw : nullptr,
                     s.vp, s.dp, first_rows};
        if (s.split) GRWS_HEAD_LAUNCH(s.weight, head_dweight_kernel, w, GRWS_BF16, GRWS_F32);
        else if (h->dtype == GRWS_F16) GRWS_HEAD_LAUNCH(s.weight, head_dweight_kernel, w, GRWS_F16, GRWS_F16);
        else GRWS_HEAD_LAUNCH(s.weight, head_dweight_kernel, w, GRWS_BF16, GRWS_BF16);
        if (w.part && last_rows) {  // before dH, whose operands would push the runs out of the L2
#define GRWS_HEAD_DW(T)                                                                                             \
    hipLaunchKernelGGL(head_weight_out_kernel<T>, dim3((unsigned)vc), dim3(256), 0, stream, f.dw, s.weight.splits,  \
                       s.vp, s.dp, s.D, f.alpha, reinterpret_cast<T*>(out), ld_dw)
            if (h->dtype == GRWS_F32) GRWS_HEAD_DW(float);
            else if (h->dtype == GRWS_F16) GRWS_HEAD_DW(_Float16);
            else GRWS_HEAD_DW(__hip_bfloat16);
#undef GRWS_HEAD_DW
            GRWS_LAUNCH_CHECK();
        }
    }
    if (d_hidden && s.few && s.split) {
        const FewHiddenArgs d{static_cast<const float*>(h->weight) + v0 * h->ld_weight, h->ld_weight, s.D, s.dp, s.n,
                              s.np, vc, f.G, s.ldg, plane, f.dh, (int32_t)s.hidden.splits, v0 == 0};
        const bool vec = rows_of_16(h->weight, h->ld_weight, h->dtype);
        const dim3 grid((unsigned)(s.dp / 64), (unsigned)ceil_div(s.hidden.splits, 4), (unsigned)ceil_div(s.n, 64));
#define GRWS_HEAD_FEW_DH(NQ)                                                                                     \
    do {                                                                                                         \
        if (vec) hipLaunchKernelGGL((head_few_dhidden_kernel<NQ, true>), grid, dim3(256), 0, stream, d);          \
        else hipLaunchKernelGGL((head_few_dhidden_kernel<NQ, false>), grid, dim3(256), 0, stream, d);             \
    } while (0)
        if (s.n <= 16) GRWS_HEAD_FEW_DH(1);
        else if (s.n <= 32) GRWS_HEAD_FEW_DH(2);
        else GRWS_HEAD_FEW_DH(4);
#undef GRWS_HEAD_FEW_DH
        GRWS_LAUNCH_CHECK();
    } else if (d_hidden) {
        GRWS_TRY(weight_piece(h, s, v0, vc, f.wp, true, &W, s.few, stream));
        const Opnd G{gp, s.ldg * 2, plane * 2, sb.np, vt};
        char* out = static_cast<char*>(d_hidden) + (h->rows ? 0 : r0 * ld_dh * esz);
        const int32_t vec = reinterpret_cast<uintptr_t>(out) % (4 * esz) == 0 && ld_dh % 4 == 0;
        HiddenArgs d{gemm_of(s, s.hidden, W, G, s.dp, sb.np, vc, s.gplanes), f.dh + (s.vp < s.V ? r0 * s.dp : 0),
                     sb.np, s.dp, v0 == 0, s.hidden.splits == 1 && v0 + vc == s.V, vec, f.alpha, out, ld_dh, sb.n, s.D,
                     hb.hidden_rows, hb.rows, stats};
        if (s.split) GRWS_HEAD_LAUNCH(s.hidden, head_dhidden_kernel, d, GRWS_BF16, GRWS_F32);
        else if (h->dtype == GRWS_F16) GRWS_HEAD_LAUNCH(s.hidden, head_dhidden_kernel, d, GRWS_F16, GRWS_F16);
        else GRWS_HEAD_LAUNCH(s.hidden, head_dhidden_kernel, d, GRWS_BF16, GRWS_BF16);
    }
    return GRWS_OK;
}

}  // namespace
}  // namespace grws

using namespace grws;

extern "C" size_t grws_head_fwd_workspace_bytes(const grws_head* h) {
    if (check_head(h) != GRWS_OK || h->n == 0) return 0;
    Sizer z;
    FwdSpace f{};
    fwd_space(z, shape_of(h, false), &f);
    return z.used;
}

extern "C" int grws_head_fwd(const grws_head* h, float* lse, float* target_logit, float* target_prob,
                             float* row_loss, float* loss, int64_t* counts, void* workspace, size_t workspace_bytes,
                             void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    GRWS_TRY(check_head(h));
    GRWS_CHECK_ARG(counts && (loss || row_loss || h->n == 0), "head: null output");
    if (h->n == 0) {
        hipLaunchKernelGGL(head_finish_kernel, dim3(1), dim3(64), 0, stream, nullptr, nullptr, (int64_t)0, loss,
                           counts);
        GRWS_LAUNCH_CHECK();
        return GRWS_OK;
    }
    GRWS_CHECK_ARG(lse && target_logit && (h->k == 0 || target_prob), "head: null output");
    const Shape s = shape_of(h, false);
    Carver cv(workspace, workspace_bytes);
    FwdSpace f{};
    fwd_space(cv, s, &f);
    if (!cv.ok) return set_error(GRWS_E_CAPACITY, "head: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    const float c1 = kLog2e / h->temperature;
    const int64_t join_rows = s.n <= 8 ? 1 : s.n <= 512 ? 4 : 16, joins = ceil_div(s.n, join_rows);
    const bool one = s.blocks == 1 && joins <= kJoinBlocks;
    for (int64_t r0 = 0; r0 < s.n; r0 += s.nb) {
        const Shape sb = block_of(s, r0);
        const grws_head hb = rows_of(h, r0, sb.n);
        const Targets t = targets_of(&hb);
        float* y = target_logit + r0 * (h->k > 0 ? h->k : 1);
        float* prob = h->k > 0 ? target_prob + r0 * h->k : nullptr;
        if (h->k > 0) {
            const dim3 grid((unsigned)ceil_div(sb.n * ((h->k + 3) / 4), 4));
            const int32_t vec = rows_of_16(h->hidden, h->ld_hidden, h->dtype) &&
                                rows_of_16(h->weight, h->ld_weight, h->dtype);
#define GRWS_HEAD_TARGETS(T)                                                                                        \
    hipLaunchKernelGGL(head_targets_kernel<T>, grid, dim3(256), 0, stream, t, static_cast<const T*>(hb.hidden),     \
                       h->ld_hidden, static_cast<const T*>(h->weight), h->ld_weight, static_cast<const T*>(h->bias), \
                       sb.n, s.D, vec, 1.f / h->temperature, prob, prob + s.n * h->k, y, f.flags)
            if (h->dtype == GRWS_F32) GRWS_HEAD_TARGETS(float);
            else if (h->dtype == GRWS_F16) GRWS_HEAD_TARGETS(_Float16);
            else GRWS_HEAD_TARGETS(__hip_bfloat16);
#undef GRWS_HEAD_TARGETS
            GRWS_LAUNCH_CHECK();
        }
        if (s.few) {
            FewArgs a{t, h->hidden, h->weight, h->bias, h->ld_hidden, h->ld_weight, s.n, s.np, s.D, 0, s.V, s.V, c1,
                      f.flags, f.part, y, f.flags, f.done};
            a.vt = pad(s.V);
            if (h->dtype == GRWS_F32) GRWS_TRY((launch_few<float, 0>(h, a, stream)));
            else if (h->dtype == GRWS_F16) GRWS_TRY((launch_few<_Float16, 0>(h, a, stream)));
            else GRWS_TRY((launch_few<__hip_bfloat16, 0>(h, a, stream)));
        } else {
            GRWS_TRY(pack_hidden(&hb, sb, t, f.hp, Alpha{}, f.done, nullptr, stream));
        }
        for (int64_t v0 = 0; v0 < s.V && !s.few; v0 += s.vp) {
            const int64_t vc = s.V - v0 < s.vp ? s.V - v0 : s.vp;
            Opnd W;
            // W in one piece stays packed for the blocks to come
            GRWS_TRY(weight_piece(h, s, v0, vc, f.wp, false, &W, r0 == 0 || s.vp < s.V, stream));
            StatsArgs a{gemm_of(s, s.logits, W, hidden_operand(sb, f.hp, false), vc, sb.np, s.dp, s.planes),
                        v0, s.V, sb.n, sb.np, c1,
                        h->bias, h->dtype, hb.labels, f.part, y, f.flags};
            if (h->dtype == GRWS_F16) GRWS_HEAD_LAUNCH(s.logits, head_stats_kernel, a, GRWS_F16);
            else GRWS_HEAD_LAUNCH(s.logits, head_stats_kernel, a, GRWS_BF16);
        }
        const int64_t at = r0 / join_rows;  // blocks are multiples of 256 rows
#define GRWS_HEAD_JOIN(R)                                                                                            \
    hipLaunchKernelGGL(head_join_kernel<R>, dim3((unsigned)ceil_div(sb.n, R)), dim3(512), 0, stream, t, f.part,      \
                       ceil_div(s.V, s.strip_classes), (int32_t)s.strip_classes, sb.n, sb.np, h->temperature, c1, y, \
                       prob, f.flags, lse + r0, row_loss ? row_loss + r0 : nullptr,                                 \
                       f.pl + at, f.pc + 3 * at, one ? f.done : nullptr, loss, counts)
        if (join_rows == 1) GRWS_HEAD_JOIN(1);
        else if (join_rows == 4) GRWS_HEAD_JOIN(4);
        else GRWS_HEAD_JOIN(16);
#undef GRWS_HEAD_JOIN
        GRWS_LAUNCH_CHECK();
    }
    if (!one) {
        hipLaunchKernelGGL(head_finish_kernel, dim3(1), dim3(64), 0, stream, f.pl, f.pc, joins, loss, counts);
        GRWS_LAUNCH_CHECK();
    }
    return GRWS_OK;
}

extern "C" int grws_head_plan(const grws_head* h, int32_t backward, int64_t* out) {
    clear_error();
    GRWS_TRY(check_head(h));
    GRWS_CHECK_ARG(out && h->n > 0, "head: nothing to plan");
    const Shape s = shape_of(h, backward != 0);
    const int64_t v[GRWS_HEAD_PLAN] = {s.blocks, s.nb, ceil_div(s.V, s.vp), s.vp, s.few, s.few ? 0 : s.logits.tile,
                                       s.weight.tile, s.weight.splits, s.hidden.tile, s.hidden.splits};
    for (int i = 0; i < GRWS_HEAD_PLAN; ++i) out[i] = v[i];
    return GRWS_OK;
}

extern "C" size_t grws_head_bwd_workspace_bytes(const grws_head* h) {
    if (check_head(h) != GRWS_OK || h->n == 0) return 0;
    Sizer z;
    BwdSpace f{};
    const Shape s = shape_of(h, true);
    bwd_space(z, s, h, &f);
    return z.used;
}

extern "C" int grws_head_bwd(const grws_head* h, const float* lse, const float* target_logit,
                             const float* target_prob, const int64_t* counts, const float* dloss, int32_t per_row,
                             void* d_hidden, int64_t ld_dh, void* d_weight, int64_t ld_dw, void* d_bias,
                             void* workspace, size_t workspace_bytes, void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    GRWS_TRY(check_head(h));
    GRWS_CHECK_ARG((!d_hidden || ld_dh >= h->width) && (!d_weight || ld_dw >= h->width),
                   "head: gradients' leading dimensions must be the width at least");
    if (h->n == 0) {
        const size_t e = dtype_size(h->dtype);
        if (d_weight)
            for (int64_t v = 0; v < (ld_dw == h->width ? 1 : h->classes); ++v)
                GRWS_TRY(fill_bytes_zero(static_cast<char*>(d_weight) + v * ld_dw * e,
                                         (ld_dw == h->width ? h->classes : 1) * h->width * e, stream));
        if (d_bias) GRWS_TRY(fill_bytes_zero(d_bias, h->classes * e, stream));
        return GRWS_OK;
    }
    GRWS_CHECK_ARG(lse && target_logit && counts && dloss && (h->k == 0 || target_prob), "head: null pointer");
    if (!d_hidden && !d_weight && !d_bias) return GRWS_OK;
    const Shape s = shape_of(h, true);
    Carver cv(workspace, workspace_bytes);
    BwdSpace f{};
    bwd_space(cv, s, h, &f);
    if (!cv.ok) return set_error(GRWS_E_CAPACITY, "head: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    const float c1 = kLog2e / h->temperature;
    const float gscale = h->dtype == GRWS_F16 ? 32768.f : 1.f;
    const RowStats stats = h->k > 0 ? RowStats{lse, target_prob, h->k} : RowStats{lse, target_logit, 1};
    if (per_row) {
        GRWS_TRY(fill_i32(reinterpret_cast<int32_t*>(f.most), 1, 0, stream));
        const dim3 grid((unsigned)ceil_div(s.n, 256));
        hipLaunchKernelGGL(head_most_kernel, grid, dim3(256), 0, stream, dloss, stats, s.n, f.most);
        GRWS_LAUNCH_CHECK();
        hipLaunchKernelGGL(head_row_scale_kernel, grid, dim3(256), 0, stream, dloss, stats, s.n, f.most, f.scale);
        GRWS_LAUNCH_CHECK();
    }
    const Alpha alpha{f.alpha, dloss, counts, per_row ? f.most : nullptr, h->temperature / gscale};
    int32_t* owner = d_hidden ? f.owner : nullptr;
    if (s.blocks == 1) {
        GRWS_TRY(pack_hidden(h, s, targets_of(h), f.hp, alpha, nullptr, owner, stream));
    } else if (owner) {
        hipLaunchKernelGGL(head_owner_kernel, dim3((unsigned)ceil_div(s.n, 256)), dim3(256), 0, stream, h->rows, s.n,
                           h->hidden_rows, owner);
        GRWS_LAUNCH_CHECK();
    }
    const size_t esz = dtype_size(h->dtype);
    // pieces of the classes, and of each the blocks of rows: W's piece is
    // packed once, dW's is complete after its blocks
    for (int64_t v0 = 0; v0 < s.V; v0 += s.vp) {
        const int64_t vc = s.V - v0 < s.vp ? s.V - v0 : s.vp;
        for (int64_t r0 = 0; r0 < s.n; r0 += s.nb)
            GRWS_TRY(backward_block(h, s, f, v0, vc, r0, stats, target_logit, target_prob, per_row, alpha, c1,
                                    gscale, d_hidden, ld_dh, d_weight, ld_dw, d_bias, stream));
    }
    if (d_hidden && s.hidden.splits > 1) {
#define GRWS_HEAD_DH(T)                                                                                              \
    hipLaunchKernelGGL(head_hidden_out_kernel<T>, dim3((unsigned)s.n), dim3(256), 0, stream, f.dh,               \
                       s.hidden.splits, s.np, s.dp, s.D, h->rows, h->hidden_rows, stats, f.alpha,                \
                       static_cast<T*>(d_hidden), ld_dh)
        if (h->dtype == GRWS_F32) GRWS_HEAD_DH(float);
        else if (h->dtype == GRWS_F16) GRWS_HEAD_DH(_Float16);
        else GRWS_HEAD_DH(__hip_bfloat16);
#undef GRWS_HEAD_DH
        GRWS_LAUNCH_CHECK();
    }
    if (owner) {
#define GRWS_HEAD_REPEATED(T)                                                                                        \
    hipLaunchKernelGGL(head_repeated_kernel<T>, dim3((unsigned)ceil_div(s.n, 256)), dim3(256), 0, stream, h->rows,   \
                       s.n, h->hidden_rows, owner, s.D, static_cast<T*>(d_hidden), ld_dh)
        if (h->dtype == GRWS_F32) GRWS_HEAD_REPEATED(float);
        else if (h->dtype == GRWS_F16) GRWS_HEAD_REPEATED(_Float16);
        else GRWS_HEAD_REPEATED(__hip_bfloat16);
#undef GRWS_HEAD_REPEATED
        GRWS_LAUNCH_CHECK();
    }
    return GRWS_OK;
}
