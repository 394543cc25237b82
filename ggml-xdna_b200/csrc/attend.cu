// Attention of new tokens over the paged cache (zest_kv_attend).
//
// The rows of one kv head are its new tokens' query heads, token by token:
// row r of a sequence is token r / G, head r % G of the group (G = heads /
// kv_heads). All of them read the same keys and values, so a tile of rows
// costs one read of the cache whatever G is.
//
// One pass over the keys with the running maximum m and sum l of a softmax in
// base 2 (the scale times log2 e folded into one multiply-add):
//   m' = max(m, s_j),  o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j,  l' alike.
//
// A long row of keys is cut into chunks that different blocks take. Few rows:
// the blocks of up to 8 chunks are a cluster and join their o, m and l through
// each other's shared memory. What more than one cluster, or (many rows) more
// than one block made of a row goes to the workspace, unnormalised, with its m
// and l, and kv_combine_kernel joins it in order.
#include "zest_kv.cuh"

#include <algorithm>
#include <cuda.h>
#include <cudaTypedefs.h>

namespace zest {

namespace {

constexpr uint64_t WAIT_LIMIT_NS = 1000000000ull;  // 1 s
constexpr int ROWS = 16;                           // query rows of a tile of the few-rows kernel
constexpr int KEYS = 64;                           // keys of a stage
constexpr float LOG2E = 1.44269504088896340736f;

struct attend_args {
    zest_kv_batch b;
    const uint16_t *q;
    int64_t ldq, pages;
    const uint16_t *v;  // this layer's values, for the rows that see a NaN or infinity others do not
    int64_t page_stride, token_stride, head_stride;
    int heads, group, d, page_size, causal;
    int64_t window;
    float scale_log2;
    uint16_t *out;
    int64_t ldo;
    float *y;
    int64_t ldy;
    uint16_t *a_next;
    int64_t lda;
    int64_t chunk;      // many rows: keys a block takes, a multiple of 128
    int splits;         // parts of a row that go to the workspace (1: none does, the result is whole)
    int join;           // few rows: blocks of a cluster, each with an equal part of the keys (then splits is 1)
    int by_rows;        // many rows: every head's last rows first, not one head's after another's
    int wide;           // few rows: a box has a head's columns whole
    float2 *ml;         // [splits][T * heads]: m and l (m NaN: a wait ran out and the part is none)
    float *part;        // [splits][T * heads][DP]: o
    unsigned *err;
};

// The keys that rows of tokens [t_lo, t_hi] see: any of them [lo, hi), all of them [clo, chi).
struct key_span {
    int lo, hi, clo, chi;
};

__device__ __forceinline__ int row_lo(const attend_args &A, const kv_seq &s, int t) {
    return A.causal && A.window ? (int) max((int64_t) 0, (int64_t) s.kv - s.n + t - A.window + 1) : 0;
}

__device__ __forceinline__ int row_hi(const attend_args &A, const kv_seq &s, int t) {
    return A.causal ? max(0, s.kv - s.n + t + 1) : s.kv;
}

__device__ __forceinline__ key_span span_of(const attend_args &A, const kv_seq &s, int t_lo, int t_hi) {
    return { row_lo(A, s, t_lo), row_hi(A, s, t_hi), row_lo(A, s, t_hi), row_hi(A, s, t_lo) };
}

// Eight results of one row: rounded to the cache's type, and as the next
// matmul's operand.
template <bool F16>
__device__ __forceinline__ uint4 round8(const float (&o)[8]) {
    return make_uint4(kv_bits2<F16>(o[0], o[1]), kv_bits2<F16>(o[2], o[3]), kv_bits2<F16>(o[4], o[5]),
                      kv_bits2<F16>(o[6], o[7]));
}

__device__ __forceinline__ uint4 pack8(const float (&o)[8]) {
    uint8_t enc[9];
    uint32_t bf[4];
    encode_block(o, enc, bf);
    return make_uint4(bf[0], bf[1], bf[2], bf[3]);
}

__device__ __forceinline__ void store8_f32(const attend_args &A, int64_t t, int head, int c, const float (&o)[8]) {
    float4 *y = reinterpret_cast<float4 *>(A.y + t * A.ldy + (int64_t) head * A.d + c);
    y[0] = make_float4(o[0], o[1], o[2], o[3]);
    y[1] = make_float4(o[4], o[5], o[6], o[7]);
}

// As asked for: in the cache's type, in f32, and as the next matmul's operand.
template <bool F16>
__device__ __forceinline__ void store8(const attend_args &A, int64_t t, int head, int c, const float (&o)[8]) {
    const int64_t col = (int64_t) head * A.d + c;
    if (A.out) *reinterpret_cast<uint4 *>(A.out + t * A.ldo + col) = round8<F16>(o);
    if (A.y) store8_f32(A, t, head, c, o);
    if (A.a_next) *reinterpret_cast<uint4 *>(A.a_next + t * A.lda + col) = pack8(o);
}

// A NaN or infinite value that some rows of a tile see and others do not is
// taken as zero in the tile's product (0 times it would reach every row) and
// added here to a row that sees keys [lo, hi), from those of them outside
// [clo, chi), which every row sees.
template <bool F16>
__device__ __forceinline__ void add_not_finite(const attend_args &A, int s, int kv_head, int c, int lo, int hi, int clo,
                                               int chi, float (&o)[8]) {
#pragma unroll 1
    for (int j = lo; j < hi; j++) {
        if (j >= clo && j < chi) {
            j = chi - 1;
            continue;
        }
        const int64_t page = A.b.table[s * A.b.table_stride + j / A.page_size];
        if (page < 0 || page >= A.pages) continue;
        const uint16_t *v =
            A.v + page * A.page_stride + j % A.page_size * A.token_stride + kv_head * A.head_stride + c;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float x = kv_value<F16>(v[i]);
            if (!(fabsf(x) <= 3.4028234e38f)) o[i] += x;
        }
    }
}

// --- m16n8k16 on a warp (few rows: the cache's bytes bound it, not the MMAs) ---

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                     "{%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                     "{%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// One lane arrives for a warp whose lanes have all come this far. They are
// together again behind it: warp-wide (.aligned) instructions want that, and a
// branch that one lane takes does not promise it by itself.
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    __syncwarp();
}

// 2^x by the hardware's approximation (relative error about 2^-22).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Both halves' exponents all ones, per half: NaN or infinite.
template <bool F16>
__device__ __forceinline__ bool bad_half(uint32_t h) {
    const uint32_t m = F16 ? 0x7c00u : 0x7f80u;
    return (h & m) == m;
}

// Whether one of eight halves is NaN or infinite: one more in an exponent of
// all ones carries into the sign's place.
template <bool F16>
__device__ __forceinline__ bool any_bad(const uint4 &w) {
    const uint32_t m = F16 ? 0x7c007c00u : 0x7f807f80u, one = F16 ? 0x04000400u : 0x00800080u;
    return (((w.x & m) + one) | ((w.y & m) + one) | ((w.z & m) + one) | ((w.w & m) + one)) & 0x80008000u;
}

// A stage's bytes, and as many stages as fill an SM with its 3, 2 or 1 blocks
// (by padded head size): 192 KB of keys and values in flight or in use.
template <int DP>
struct few_rows {
    static constexpr int HALF = KEYS * DP * 2;  // K or V of a stage
    static constexpr int STAGE = 2 * HALF;
    static constexpr int STAGES = DP == 64 ? 4 : 3;
    static constexpr int SMEM = 1024 + STAGES * STAGE;
};

constexpr int FEW_THREADS = 160;  // four warps of products, one that copies

// A block: up to 16 rows of one kv head of one sequence over one chunk of
// keys. Warp 4 brings 64 keys a stage by TMA in boxes of min(page, 64) keys
// (64-column blocks of 128-byte rows, swizzled; all of a head's blocks in one
// box where it is whole blocks: a box costs the TMA unit about 45 clocks
// besides 2 a row, and 32 sequences in pages of 16 took 142 us with a box a
// block); warps 0-3 take 16 keys of a stage each, with a running m, l and o of
// their own, joined at the end. Bound by HBM: 32 tokens over up to 8,192 keys
// (8 kv heads of 128, pages of 16) 119 us, 5.5 TB/s; one over 131,072 88 us, 6.0
// TB/s; over 1,000 by its latencies, 10.5 us.
template <int DP, bool F16>
__global__ void __launch_bounds__(FEW_THREADS) kv_attend_few_kernel(const __grid_constant__ CUtensorMap tk,
                                                                    const __grid_constant__ CUtensorMap tv,
                                                                    const __grid_constant__ attend_args A) {
    using C = few_rows<DP>;
    extern __shared__ uint8_t dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>(((uintptr_t) dyn + 1023) & ~(uintptr_t) 1023);
    __shared__ uint64_t full[C::STAGES], empty[C::STAGES];
    __shared__ int stop, not_finite;
    __shared__ float m_sh[4][ROWS], l_sh[4][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = blockIdx.z, split = blockIdx.x;  // the part of the keys (in a cluster, the block's rank)
    const int kv_head = blockIdx.y;

    const kv_seq s = kv_seq_of(A.b, A.page_size, seq);
    if (!s.ok) {
        if (threadIdx.x == 0) atomicOr(A.err, ZEST_ERR_BAD_SEQ);
        return;
    }
    const int rows = s.n * A.group;  // at most ROWS
    if (rows == 0) return;
    const key_span sp = span_of(A, s, 0, s.n - 1);
    // this block's keys: from the first of the span's 64-key block on, by chunks
    const int64_t first = (int64_t) sp.lo / KEYS * KEYS, blocks = (max((int64_t) sp.hi - first, (int64_t) 0) + KEYS - 1) / KEYS;
    const int64_t chunk = (blocks + gridDim.x - 1) / gridDim.x * KEYS;
    const int64_t from = min(first + blockIdx.x * chunk, (int64_t) sp.hi), to = min((int64_t) sp.hi, from + chunk);
    const int steps = to > from ? (int) ((to - from + KEYS - 1) / KEYS) : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 4);
        }
        stop = 0;
        not_finite = 0;
        fence_barrier_init();
    }
    __syncthreads();

    if (warp == 4) {
        // a lane brings one box: of K, then of V
        const int box = min(A.page_size, KEYS), boxes = KEYS / box, blocks = A.wide ? 1 : DP / 64;
        const int which = lane / boxes, kb = lane % boxes;
        const bool mine = which < 2 * blocks;
        const int col = which % blocks;
        const bool is_v = which >= blocks;
        const CUtensorMap *map = is_v ? &tv : &tk;
        const int at = (is_v ? C::HALF : 0) + kb * box * (DP * 2) + col * (box * 128);
        auto page_of = [&](int i) {
            const int64_t key = from + (int64_t) i * KEYS + kb * box;
            // a page that no row sees is outside the tensor: zeros (its entry may be none)
            if (!mine || i >= steps || key >= to || (key / A.page_size + 1) * A.page_size <= sp.lo) return (int) A.pages;
            const int p = A.b.table[seq * A.b.table_stride + key / A.page_size];
            if (p < 0 || p >= A.pages) {
                atomicOr(A.err, ZEST_ERR_BAD_PAGE);
                return (int) A.pages;
            }
            return p;
        };
        int page = page_of(0), i = 0;
        for (; i < steps; i++) {
            const int st = i % C::STAGES;
            const int next = page_of(i + 1);
            const bool ok = i < C::STAGES ||
                            mbar_wait_bounded(&empty[st], (i / C::STAGES - 1) & 1, (volatile int *) &stop, WAIT_LIMIT_NS);
            if (!__all_sync(0xffffffffu, ok)) {
                if (lane == 0) {
                    stop = 1;
                    atomicOr(A.err, ERR_TIMEOUT);
                }
                break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&full[st], C::STAGE);
            __syncwarp();
            if (mine) {
                const int token = (int) ((from + (int64_t) i * KEYS + kb * box) % A.page_size);
                uint8_t *dst = ring + st * C::STAGE + at;
                if (A.wide) tma_load_5d(dst, map, &full[st], 0, token, 0, kv_head, page);
                else tma_load_4d(dst, map, &full[st], col * 64, token, kv_head, page);
            }
            page = next;
        }
        // the last copies land before the block ends, whatever the others do
        for (int k = max(0, i - C::STAGES); k < i; k++)
            mbar_wait_bounded(&full[k % C::STAGES], (k / C::STAGES) & 1, nullptr, WAIT_LIMIT_NS);
        __syncwarp();
        __syncthreads();
        if (A.join > 1) {
            cluster_sync();
            cluster_sync();
        }
        return;
    }

    // this lane's two rows of the tile, and what they see
    const int g = lane >> 2, tq = lane & 3;
    int lo[2], hi[2];
    const uint16_t *qp[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int r = g + 8 * e;
        lo[e] = hi[e] = 0;
        qp[e] = nullptr;
        if (r < rows) {
            const int t = r / A.group;
            lo[e] = row_lo(A, s, t);
            hi[e] = row_hi(A, s, t);
            qp[e] = A.q + (s.q0 + (int64_t) t) * A.ldq + (int64_t) (kv_head * A.group + r % A.group) * A.d;
        }
    }
    uint32_t qf[DP / 16][4];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int c = ks * 16 + (e >> 1) * 8 + tq * 2;
            qf[ks][e] = qp[e & 1] && c < A.d ? *reinterpret_cast<const uint32_t *>(qp[e & 1] + c) : 0;
        }
    float o[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = { -INFINITY, -INFINITY }, l[2] = { 0.0f, 0.0f };
    bool bad = false, timeout = false;
    // where this lane's row of K's and of V's fragments lies in a stage, and how
    // far on the next column block is
    const int box = min(A.page_size, KEYS), block = box * 128;
    const int k_key = warp * 16 + (lane >> 4) * 8 + (lane & 7), v_key = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
    const int k_at = k_key / box * (box * DP * 2) + k_key % box * 128;
    const int v_at = C::HALF + v_key / box * (box * DP * 2) + v_key % box * 128;

    for (int i = 0; i < steps; i++) {
        const int st = i % C::STAGES;
        if (!mbar_wait_bounded(&full[st], (i / C::STAGES) & 1, (volatile int *) &stop, WAIT_LIMIT_NS)) {
            timeout = true;
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, timeout)) {
            if (lane == 0) {
                stop = 1;
                atomicOr(A.err, ERR_TIMEOUT);
            }
            timeout = true;
            break;
        }
        const uint32_t stage = smem_u32(ring + st * C::STAGE);
        const int k0 = warp * 16;  // this warp's keys of the stage
        const int64_t key0 = from + (int64_t) i * KEYS + k0;
        float sc[2][4] = {};
        {
            const int odd = (lane >> 3) & 1;
            const uint32_t row = stage + k_at;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ks++) {
                uint32_t b[4];
                const int unit = (ks * 2 + odd) & 7;
                ldmatrix_x4(b, row + (ks / 4) * block + ((unit ^ (lane & 7)) << 4));
                mma16816<F16>(sc[0], qf[ks], b[0], b[1]);
                mma16816<F16>(sc[1], qf[ks], b[2], b[3]);
            }
        }
        // does every row see every key of this warp's?
        // (rows past the last hold zero queries, and their results go nowhere)
        const bool masked = key0 < sp.clo || key0 + 16 > min((int64_t) sp.chi, to);
        if (masked) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t key = key0 + n * 8 + tq * 2 + (e & 1);
                    if (key < lo[e >> 1] || key >= hi[e >> 1] || key >= to) sc[n][e] = -INFINITY;
                }
            __syncwarp();
        }
        float f[2];
        bool moved = false;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float mx = fmaxf(fmaxf(sc[0][2 * e], sc[0][2 * e + 1]), fmaxf(sc[1][2 * e], sc[1][2 * e + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(m[e], mx * A.scale_log2);
            f[e] = mx == m[e] ? 1.0f : exp2_fast(m[e] - mx);  // m = -inf: 0
            moved |= mx != m[e];
            m[e] = mx;
        }
        uint32_t p[4];
        {
            float ps[2][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float base = m[e >> 1] == -INFINITY ? 0.0f : m[e >> 1];
#pragma unroll
                for (int n = 0; n < 2; n++) ps[n][e] = exp2_fast(__fmaf_rn(sc[n][e], A.scale_log2, -base));
            }
#pragma unroll
            for (int e = 0; e < 2; e++)
                l[e] = l[e] * f[e] + ((ps[0][2 * e] + ps[0][2 * e + 1]) + (ps[1][2 * e] + ps[1][2 * e + 1]));
            p[0] = kv_bits2<F16>(ps[0][0], ps[0][1]);
            p[1] = kv_bits2<F16>(ps[0][2], ps[0][3]);
            p[2] = kv_bits2<F16>(ps[1][0], ps[1][1]);
            p[3] = kv_bits2<F16>(ps[1][2], ps[1][3]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int j = 0; j < DP / 8; j++) {
                o[j][0] *= f[0];
                o[j][1] *= f[0];
                o[j][2] *= f[1];
                o[j][3] *= f[1];
            }
        }
        {
            const int right = lane >> 4;
            const uint32_t row = stage + v_at;
#pragma unroll
            for (int j = 0; j < DP / 8; j += 2) {
                uint32_t b[4];
                const int unit = (j + right) & 7;
                ldmatrix_x4_t(b, row + (j / 8) * block + ((unit ^ (lane & 7)) << 4));
                if (masked) {
                    // a key that not every row sees: its NaN and infinities apart (add_not_finite)
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int64_t k = key0 + (e & 1) * 8 + tq * 2 + h;
                            const uint32_t half = (b[e] >> (16 * h)) & 0xffffu;
                            if ((k < sp.clo || k >= sp.chi || k >= to) && bad_half<F16>(half)) {
                                b[e] &= h ? 0x0000ffffu : 0xffff0000u;
                                bad |= k < to;
                            }
                        }
                    __syncwarp();
                }
                mma16816<F16>(o[j], p, b[0], b[1]);
                mma16816<F16>(o[j + 1], p, b[2], b[3]);
            }
        }
        warp_arrive(&empty[st]);
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) not_finite = 1;
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    // every stage has been read: the ring holds the four warps' o now
    __syncthreads();
    constexpr int LD = DP + 4;
    float *os = reinterpret_cast<float *>(ring);
    static_assert(4 * ROWS * LD * 4 <= C::STAGES * C::STAGE, "the joined rows fit the ring");
#pragma unroll
    for (int j = 0; j < DP / 8; j++)
#pragma unroll
        for (int e = 0; e < 2; e++)
            *reinterpret_cast<float2 *>(os + (warp * ROWS + g + 8 * e) * LD + j * 8 + tq * 2) =
                make_float2(o[j][2 * e], o[j][2 * e + 1]);
    if (tq == 0)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            m_sh[warp][g + 8 * e] = m[e];
            l_sh[warp][g + 8 * e] = l[e];
        }
    __syncwarp();
    named_barrier(1, 128);
    const int row = threadIdx.x >> 3;
    float mx = -INFINITY, w[4], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) mx = fmaxf(mx, m_sh[k][row]);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        w[k] = m_sh[k][row] == -INFINITY ? 0.0f : exp2_fast(m_sh[k][row] - mx);
        sum += w[k] * l_sh[k][row];
    }
    const int t = row / A.group, head = kv_head * A.group + row % A.group;
    const int64_t tok = s.q0 + (int64_t) t, slot = split * (A.b.T * A.heads) + tok * A.heads + head;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const bool live = row < rows && !stop;  // a wait that ran out leaves the rows as they were
#pragma unroll
    for (int i = 0; i < DP / 64; i++) {
        const int c = (threadIdx.x & 7) * 8 + 64 * i;
        float x[8] = {};
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __fmaf_rn(os[(k * ROWS + row) * LD + c + e], w[k], x[e]);
        if (not_finite && live && c < A.d) {
            const int a = (int) max((int64_t) row_lo(A, s, t), from), z = (int) min((int64_t) row_hi(A, s, t), to);
            add_not_finite<F16>(A, seq, kv_head, c, a, z, sp.clo, max(sp.clo, sp.chi), x);
        }
        if (A.join > 1) {  // over the first warp's part, which this thread alone reads
            float4 *dst = reinterpret_cast<float4 *>(os + row * LD + c);
            dst[0] = make_float4(x[0], x[1], x[2], x[3]);
            dst[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else if (live && c < A.d) {
            if (A.splits > 1) {
                float4 *dst = reinterpret_cast<float4 *>(A.part + slot * DP + c);
                dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] *= inv;
                store8<F16>(A, tok, head, c, x);
            }
        }
    }
    if (A.join == 1) {
        if (row < rows && A.splits > 1 && (threadIdx.x & 7) == 0) A.ml[slot] = make_float2(stop ? NAN : mx, sum);
        return;
    }
    // the cluster's chunks joined in order, the rows' columns dealt to its blocks
    __shared__ float2 ml_sh[ROWS];
    if ((threadIdx.x & 7) == 0) ml_sh[row] = make_float2(stop ? NAN : mx, sum);
    __syncwarp();
    cluster_sync();
    for (int u = split * 128 + threadIdx.x; u < rows * (DP / 8); u += A.join * 128) {
        const int jr = u / (DP / 8), c = u % (DP / 8) * 8;
        if (c >= A.d) continue;
        float2 part[8];
        float top = -INFINITY, total = 0.0f, x[8] = {};
        bool whole = true;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < A.join) {
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                             : "=f"(part[k].x), "=f"(part[k].y)
                             : "r"(map_to_rank(&ml_sh[jr], k))
                             : "memory");
                whole = whole && part[k].x == part[k].x;
                top = fmaxf(top, part[k].x);
            }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < A.join) {
                const float f = part[k].x == -INFINITY ? 0.0f : exp2_fast(part[k].x - top);
                total += f * part[k].y;
                float4 a, b;
                const uint32_t src = map_to_rank(os + jr * LD + c, k);
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w)
                             : "r"(src)
                             : "memory");
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w)
                             : "r"(src + 16)
                             : "memory");
                const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = __fmaf_rn(v[e], f, x[e]);
            }
        const int64_t jtok = s.q0 + (int64_t) (jr / A.group);
        const int jhead = kv_head * A.group + jr % A.group;
        if (!whole) continue;
        const float scale = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= scale;
        store8<F16>(A, jtok, jhead, c, x);
    }
    __syncwarp();
    cluster_sync();  // nobody's shared memory goes while another reads it
}

// --- many rows: tcgen05 -------------------------------------------------------------

// Shapes by padded head size. A block's query tiles of 128 rows share each tile
// of keys and values, and one score buffer in TMEM in turn: it is free again as
// soon as a tile's rows are in registers, so the other tile's scores are made
// while these take their exponentials, and the tensor cores and the
// exponential units both work throughout. (A buffer of each tile's own, with P
// over it as the first form had it, holds the next scores back until P has
// been used: 229 us where this took 199 for 2,048 tokens over 8,192.)
// Measured: 2,048 tokens, 32 heads of 128 on 8, over 8,192 190 us (1,260
// TFLOP/s), over 32,768 900 us (1,190, at the power limit: 1.6 GHz); 24 heads of
// 256 on 4 over themselves 65-70 us; ragged prompts of up to 700 tokens, 32
// heads of 64: 61 us. A tile takes 2,600 clocks at 128 columns, where its MMAs
// take 2,048: the exponentials and their conversions (2,150 of two warps a
// scheduler) and a tile's first loads from TMEM bound it; a block pays 6 to 8 us
// besides for its set-up, its first tiles' way and its results.
template <int DP>
struct many_rows {
    static constexpr int NQ = DP == 256 ? 1 : 2;    // query tiles of a block
    static constexpr int BN = DP == 256 ? 64 : 128; // keys of a tile
    static constexpr int PART = 64;                 // keys whose weights are handed over at once
    static constexpr int PARTS = BN / PART;
    // One query tile leaves TMEM room for Q: its 64 KB of shared memory hold two
    // tiles more of keys and values, and the scores' MMAs, 64 keys wide, read half
    // as many bytes
    static constexpr bool Q_TMEM = NQ == 1;
    static constexpr int Q_BYTES = 128 * DP * 2;
    static constexpr int KV_BYTES = BN * DP * 2;
    static constexpr int KS = DP == 128 ? 3 : 4, VS = DP == 64 ? 4 : DP == 128 ? 2 : 3;  // tiles of K and of V in flight or in use
    static constexpr int SMEM = 1024 + (Q_TMEM ? 0 : NQ * Q_BYTES) + (KS + VS) * KV_BYTES;
    static_assert(!Q_TMEM || Q_BYTES == (VS - 1) * KV_BYTES, "Q comes in through V's slots but the first");
    static constexpr int SOFTMAX = NQ * 128;        // threads: one a row
    static constexpr int THREADS = SOFTMAX + 128;   // and a warp each for Q K^T, P V, K's copies and V's
    // Buffers of P: two where one query tile has the block to itself, since the
    // next scores' MMAs (1,000 clocks at 256 columns) go ahead of P's otherwise
    static constexpr int NP = NQ > 1 ? 1 : 2;
    // TMEM columns: O of each query tile, the scores, P of each query tile, Q
    static constexpr int O_COL = 0, S_COL = NQ * DP, P_COL = S_COL + BN, Q_COL = P_COL + NQ * NP * BN / 2, COLS = 512;
    static_assert(Q_COL + (Q_TMEM ? DP / 2 : 0) <= COLS, "TMEM holds O, S, P and Q");
    // a softmax warp looks at V(i) having seen the product of tile i - NP done
    static_assert(VS >= NP, "V(i - VS) has been used when a softmax warp waits for V(i)");
};

// A rise of the running maximum below this (in powers of two) leaves the
// weights relative to the old one: they stay within 2^8, and o is not touched.
constexpr float LAZY = 8.0f;

// Two f32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void unpack2(uint64_t p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A warp's wait: one look, and the rest, for at most WAIT_LIMIT_NS or until
// *gone, out of line. The same answer in every lane; a wait that runs out sets
// *gone and the error bit.
__device__ __forceinline__ bool wait_on(uint64_t *bar, uint32_t parity, volatile int *gone, unsigned *err) {
    const uint64_t t0 = global_ns();
    bool ok = false;
    for (uint32_t it = 1; !ok; it++) {
        ok = mbar_try_wait(bar, parity);
        if (!ok && (it & 63u) == 0 && (*gone || global_ns() - t0 > WAIT_LIMIT_NS)) break;
    }
    __syncwarp();
    if (__all_sync(0xffffffffu, ok)) return true;
    *gone = 1;
    atomicOr(err, ERR_TIMEOUT);
    return false;
}

__device__ __forceinline__ bool wait_soon(uint64_t *bar, uint32_t parity, volatile int *gone, unsigned *err) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_on(bar, parity, gone, err);
}

// 2^u and 2^w without the exponential unit: x = n + f, n the nearest integer
// (adding 1.5 * 2^23 leaves it in the low mantissa bits), 2^f by a polynomial
// of degree 4 on [-1/2, 1/2] whose relative error, fitted to be even
// (iteratively reweighted least squares), is 2^-18.5; n added to the exponent.
// Zero below 2^-126; u, w < 127 and not NaN.
__device__ __forceinline__ void exp2_poly(float &u, float &w) {
    const float R = 12582912.0f;  // 1.5 * 2^23
    const uint64_t x = pack2(fmaxf(u, -126.0f), fmaxf(w, -126.0f));
    const uint64_t t = add2(x, pack2(R, R)), n = add2(t, pack2(-R, -R));
    const uint64_t f = fma2(n, pack2(-1.0f, -1.0f), x);
    uint64_t p = pack2(9.5701022e-3f, 9.5701022e-3f);
    p = fma2(p, f, pack2(5.5917859e-2f, 5.5917859e-2f));
    p = fma2(p, f, pack2(2.4024744e-1f, 2.4024744e-1f));
    p = fma2(p, f, pack2(6.9312179e-1f, 6.9312179e-1f));
    p = fma2(p, f, pack2(9.9999928e-1f, 9.9999928e-1f));
    float tu, tw, pu, pw;
    unpack2(t, tu, tw);
    unpack2(p, pu, pw);
    u = u < -126.0f ? 0.0f : __uint_as_float(__float_as_uint(pu) + (__float_as_uint(tu) << 23));
    w = w < -126.0f ? 0.0f : __uint_as_float(__float_as_uint(pw) + (__float_as_uint(tw) << 23));
}

// The weights of 64 keys: x in as bits of scores, 2^(x scale + base) rounded to
// the cache's type into p, their f32 sums into s0 and s1. Rounded because the
// MMA takes both operands in 16 bits of one type: half a step of each weight,
// 1.4 times the distance from 64-bit arithmetic that one rounding of the result
// has (bf16 2.35e-3 against 1.66e-3); l sums the weights before that rounding,
// whose errors have no bias for it to share. One pair of eight by
// polynomial: the exponential unit (16 a clock and SM) is what the rows wait
// for. Clocks for 128 keys of a warp alone and of two warps a scheduler, with
// the maximum before: 1,676 and 2,334 with none, 1,536 and 2,146 with one of
// eight, 1,451 and 2,258 with one of four.
template <bool F16>
__device__ __forceinline__ void weights(const uint32_t *x, float scale, float base, uint32_t (&p)[32], uint64_t &s0,
                                        uint64_t &s1) {
    const uint64_t m = pack2(scale, scale), c = pack2(base, base);
#pragma unroll
    for (int e = 0; e < 32; e++) {
        float u, w;
        unpack2(fma2(pack2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), m, c), u, w);
        if (e % 8 == 7) {
            exp2_poly(u, w);
        } else {
            u = exp2_fast(u);
            w = exp2_fast(w);
        }
        if (e & 1) s1 = add2(s1, pack2(u, w));
        else s0 = add2(s0, pack2(u, w));
        p[e] = kv_bits2<F16>(u, w);
    }
}

// A block: NQ x 128 rows of one kv head of one sequence over one chunk of
// keys. S = Q K^T into TMEM; each softmax thread owns a row: it takes the
// row's scores from TMEM, keeps m and l, and leaves the weights P in TMEM, from
// where O += P V takes them as its A operand. O stays in TMEM
// and is touched by the threads only when a row's maximum rises by more than
// 2^8, and at the end.
template <int DP, bool F16>
__global__ void __launch_bounds__(many_rows<DP>::THREADS, 1)
    kv_attend_many_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                          const __grid_constant__ CUtensorMap tv, const __grid_constant__ attend_args A) {
    using C = many_rows<DP>;
    constexpr int NQ = C::NQ, NP = C::NP, BN = C::BN, KS = C::KS, VS = C::VS, PARTS = C::PARTS;
    extern __shared__ uint8_t dyn[];
    uint8_t *const tiles_sm = reinterpret_cast<uint8_t *>(((uintptr_t) dyn + 1023) & ~(uintptr_t) 1023);
    uint8_t *const k_sm = tiles_sm + (C::Q_TMEM ? 0 : NQ * C::Q_BYTES), *const v_sm = k_sm + KS * C::KV_BYTES;
    uint8_t *const q_sm = C::Q_TMEM ? v_sm + C::KV_BYTES : tiles_sm;
    // Every barrier's phases are waited for one after another by whoever waits
    // for it: a parity tells a phase from the one before it, not from the next.
    __shared__ uint64_t q_in, q_full, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[NQ], s_free, p_full[NQ][NP][PARTS],
        pv_done[NQ][NP], drained[2];
    __shared__ uint32_t tmem_sh;
    __shared__ int stop, not_finite;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the last rows see the most keys: first; and neighbours on the same keys
    const int units = A.heads / A.group * A.splits, tiles = gridDim.x / units, seq = blockIdx.y;
    const int unit = A.by_rows ? blockIdx.x % units : blockIdx.x / tiles;
    const int tile = tiles - 1 - (A.by_rows ? blockIdx.x / units : blockIdx.x % tiles);
    const int kv_head = unit / A.splits, split = unit % A.splits;

    const kv_seq s = kv_seq_of(A.b, A.page_size, seq);
    if (!s.ok) {
        if (threadIdx.x == 0) atomicOr(A.err, ZEST_ERR_BAD_SEQ);
        return;
    }
    const int per_tile = 128 / A.group;  // whole tokens of a query tile
    const int t0 = min((int64_t) tile * NQ * per_tile, (int64_t) s.n), t1 = min(t0 + NQ * per_tile, s.n);
    if (t0 >= t1) return;
    const int nq = NQ > 1 && t0 + per_tile < t1 ? 2 : 1;  // query tiles that have rows
    const key_span sp = span_of(A, s, t0, t1 - 1);
    const int from = (int) min((int64_t) sp.lo / KEYS * KEYS + split * A.chunk, (int64_t) sp.hi);
    const int to = (int) min((int64_t) sp.hi, from + A.chunk), n = max(0, (to - from + BN - 1) / BN);
    if (n == 0 && split > 0) return;

    constexpr int W_QK = C::SOFTMAX / 32, W_PV = W_QK + 1, W_COPY = W_QK + 2;
    if (threadIdx.x == 0) {
        mbar_init(&q_in, 1);
        mbar_init(&q_full, 4);
        for (int i = 0; i < KS; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VS; i++) {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < NQ; i++) {
            mbar_init(&s_full[i], 1);
            for (int b = 0; b < NP; b++) {
                for (int h = 0; h < PARTS; h++) mbar_init(&p_full[i][b][h], 4);
                mbar_init(&pv_done[i][b], 1);
            }
        }
        mbar_init(&s_free, 4);
        mbar_init(&drained[0], 1);
        mbar_init(&drained[1], 1);
        stop = 0;
        not_finite = 0;
        fence_barrier_init();
    }
    __syncwarp();
    if (warp == W_QK) {
        tmem_alloc(&tmem_sh, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;
    volatile int *const gone = &stop;
    // Q of 256 columns on its way to tensor memory: through shared memory, or (a
    // row cut into parts, where all blocks run at once) each row's thread reads
    // it. 2,048 tokens of 2,048, 24 heads: 64 us and 69; 128 tokens over 8,192, in
    // five parts: 60 us and 45, the tiles then taking 2,200 clocks for 1,240.
    const bool q_tma = !C::Q_TMEM || A.splits == 1;

    // A row of scores lives in registers: the softmax warps take the others'
    // share (384 threads of 168 at launch: 256 of 208 and 128 of 80 are no more).
    if (NQ > 1 && warp >= W_QK) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp >= W_COPY) {
        // Q and K by one warp, V by the other: a box of min(page, 64) keys by 64
        // columns a lane. Lanes issue their boxes one after another, about 100
        // clocks each, and a tile costs some 600 besides.
        const bool is_v = warp > W_COPY;
        const int box = min(A.page_size, KEYS), boxes = BN / box, kb = lane % boxes, col = lane / boxes * 64;
        const int shift = __ffs(A.page_size) - 1;  // a power of two
        const CUtensorMap *map = is_v ? &tv : &tk;
        uint8_t *const ring = is_v ? v_sm : k_sm;
        uint64_t *const full = is_v ? v_full : k_full, *const empty = is_v ? v_empty : k_empty;
        const int slots = is_v ? VS : KS;
        if (!is_v && q_tma && n > 0 && lane == 0) {
            mbar_arrive_expect_tx(&q_in, nq * (DP / 64) * per_tile * A.group * 128);
            for (int q = 0; q < nq; q++)
                for (int c = 0; c < DP / 64; c++)
                    tma_load_3d(q_sm + q * C::Q_BYTES + c * (128 * 128), &tq, &q_in, c * 64, kv_head * A.group,
                                s.q0 + t0 + q * per_tile);
        }
        __syncwarp();
        const bool has = col < DP;
        const int *const table = A.b.table + (int64_t) seq * A.b.table_stride;
        const int first_page = sp.lo >> shift;
        // this lane's box of tile i holds keys that a row sees (the entry of a page without may be none)
        auto seen = [&](int key) { return has && key < to && key >> shift >= first_page; };
        auto entry = [&](int i) {
            const int key = from + i * BN + kb * box;
            return seen(key) ? table[key >> shift] : -1;
        };
        int page = entry(0), i = 0, at = 0, phase = 1;  // phase: of the slot's last use
        for (; i < n; i++) {
            const int next = entry(i + 1);  // looked at a tile later
            if (i >= slots && !wait_soon(&empty[at], phase, gone, A.err)) break;
            if (C::Q_TMEM && q_tma && is_v && i == 1 && !wait_soon(&q_full, 0, gone, A.err)) break;  // Q has left the slots
            if (lane == 0) mbar_arrive_expect_tx(&full[at], C::KV_BYTES);
            __syncwarp();
            if (has) {
                const int key = from + i * BN + kb * box;
                if (page < 0 || page >= A.pages) {
                    if (seen(key)) atomicOr(A.err, ZEST_ERR_BAD_PAGE);
                    page = (int) A.pages;  // outside the tensor: zeros
                }
                tma_load_4d(ring + at * C::KV_BYTES + col / 64 * (BN * 128) + kb * box * 128, map, &full[at], col,
                            key & (A.page_size - 1), kv_head, page);
            }
            page = next;
            if (++at == slots) {
                at = 0;
                phase ^= 1;
            }
        }
        // the last copies land before the block ends, whatever the others do
        for (int k = max(0, i - slots); k < i; k++)
            mbar_wait_bounded(&full[k % slots], (k / slots) & 1, nullptr, WAIT_LIMIT_NS);
        if (!is_v && q_tma && n > 0) mbar_wait_bounded(&q_in, 0, nullptr, WAIT_LIMIT_NS);
    } else if (warp == W_QK || warp == W_PV) {
        // The scores' MMAs and the products' by a warp each: a wait or a commit
        // takes 100 to 250 clocks before the next MMA issues, and the tensor
        // cores, which hold but a few MMAs ahead, work for the other warp
        // meanwhile. The whole warp walks the loop, so that addresses and
        // descriptors are uniform (an MMA issues in a few clocks, not in 80);
        // one elected thread issues. A descriptor's address counts 16 bytes in
        // its low word, and no tile passes its 18 bits.
        constexpr uint32_t TYPE = F16 ? 0 : (1u << 7) | (1u << 10);
        auto wait = [&](uint64_t *bar, uint32_t phase) {
            const bool ok = wait_soon(bar, phase & 1, gone, A.err);
            tc_fence_after();
            return ok;
        };
        bool ok = true;
        if (warp == W_QK && n > 0) {
            constexpr uint32_t ID = (1u << 4) | TYPE | ((uint32_t) (BN >> 3) << 17) | (8u << 24);
            const uint64_t q_desc = sw128_desc(q_sm), k_desc = sw128_desc(k_sm);
            uint32_t used = 0;  // score tiles so far: the next waits until the last is in registers
            ok = wait(C::Q_TMEM ? &q_full : &q_in, 0);
            for (int i = 0; ok && i < n; i++) {
                const int at = i % KS;
                const uint64_t kt = k_desc + at * (C::KV_BYTES >> 4);
                if (!(ok = wait(&k_full[at], i / KS))) break;
                for (int q = 0; q < nq; q++) {
                    if (used > 0 && !(ok = wait(&s_free, used - 1))) break;
                    used++;
                    const uint64_t qt = q_desc + q * (C::Q_BYTES >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < DP / 16; ks++) {
                            const uint64_t kd = kt + ((ks / 4 * (BN * 128) + ks % 4 * 32) >> 4);
                            if (C::Q_TMEM) tc_mma_f16_ts(tmem + C::S_COL, tmem + C::Q_COL + ks * 8, kd, ID, ks > 0);
                            else tc_mma_bf16(tmem + C::S_COL, qt + ((ks / 4 * (128 * 128) + ks % 4 * 32) >> 4), kd, ID, ks > 0);
                        }
                        tc_commit(&s_full[q]);
                        if (q == nq - 1 && i + KS < n) tc_commit(&k_empty[at]);  // (else nobody waits for it)
                    }
                }
            }
        } else if (n > 0) {
            constexpr uint32_t ID = (1u << 4) | TYPE | (1u << 16) | ((uint32_t) (DP >> 3) << 17) | (8u << 24);
            const uint64_t v_desc = sw128_desc_mn(v_sm, BN * 128);
            for (int i = 0; ok && i < n; i++) {
                const int at = i % VS;
                const uint64_t vt = v_desc + at * (C::KV_BYTES >> 4);
                if (!(ok = wait(&v_full[at], i / VS))) break;
                for (int q = 0; ok && q < nq; q++) {
                    const uint32_t p_at = tmem + C::P_COL + (q * NP + i % NP) * (BN / 2);
#pragma unroll
                    for (int h = 0; h < PARTS; h++) {
                        if (!(ok = wait(&p_full[q][i % NP][h], i / NP))) break;
                        if (elect_one()) {
#pragma unroll
                            for (int ks = h * (C::PART / 16); ks < (h + 1) * (C::PART / 16); ks++)
                                tc_mma_f16_ts(tmem + C::O_COL + q * DP, p_at + ks * 8, vt + (ks * 16 * 128 >> 4), ID,
                                              i > 0 || ks > 0);
                            if (h == PARTS - 1) {
                                tc_commit(&pv_done[q][i % NP]);
                                if (q == nq - 1 && i + VS < n) tc_commit(&v_empty[at]);
                            }
                        }
                    }
                }
            }
        }
        if (!ok) {  // what was issued still ends before TMEM goes
            if (elect_one()) tc_commit(&drained[warp - W_QK]);
            mbar_wait_bounded(&drained[warp - W_QK], 0, nullptr, WAIT_LIMIT_NS);
        }
        __syncwarp();
    } else if (warp < W_QK) {
        if (NQ > 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int q = warp / 4, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t) (warp % 4 * 32) << 16;
        const uint32_t o_at = tmem + lanes + C::O_COL + q * DP;
        const int tq0 = t0 + q * per_tile, tq1 = min(tq0 + per_tile, t1);
        const int t = tq0 + row / A.group;
        const bool valid = row < per_tile * A.group && t < t1;
        const int lo = valid ? row_lo(A, s, t) : 0, hi = valid ? row_hi(A, s, t) : 0;
        // tiles [i0, i1) are seen whole by every row of the block
        const int i0 = max(0, sp.clo - from + BN - 1) / BN, i1 = max(0, min(sp.chi, to) - from) / BN;
        bool ok = q < nq;
        if (C::Q_TMEM && n > 0) {  // the row of Q, two values a column
            if (q_tma) ok = wait_soon(&q_in, 0, gone, A.err);
            if (ok) {
                const uint8_t *const staged = q_sm + row * 128;
                const uint16_t *const src =
                    A.q + (s.q0 + (int64_t) (valid ? t : 0)) * A.ldq + (kv_head * A.group + (valid ? row % A.group : 0)) * A.d;
                uint32_t x[DP / 64][32];  // all loads under way at once
#pragma unroll
                for (int c = 0; c < DP; c += 8) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (q_tma) w = *reinterpret_cast<const uint4 *>(staged + c / 64 * (128 * 128) + ((c / 8 ^ row) % 8 << 4));
                    else if (c < A.d) w = *reinterpret_cast<const uint4 *>(src + c);
                    uint32_t *const at = &x[c / 64][c % 64 / 2];
                    at[0] = w.x, at[1] = w.y, at[2] = w.z, at[3] = w.w;
                }
                __syncwarp();
#pragma unroll
                for (int c = 0; c < DP / 64; c++) tmem_st_32x32b_x32(tmem + lanes + C::Q_COL + c * 32, x[c]);
                tmem_st_wait();
                tc_fence_before();
                fence_proxy_async_shared();
                warp_arrive(&q_full);
            }
        }
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; ok && i < n; i++) {
            if (!(ok = wait_soon(&s_full[q], i & 1, gone, A.err))) break;
            tc_fence_after();
            uint32_t x[BN / 32][32];
#pragma unroll
            for (int c = 0; c < BN / 32; c++) tmem_ld_32x32b_x32(tmem + lanes + C::S_COL + c * 32, x[c]);
#pragma unroll
            for (int c = 0; c < BN / 32; c++) tmem_ld_wait(x[c]);
            tc_fence_before();
            warp_arrive(&s_free);
            // the last product of P's buffer is done: P may go
            if (i >= NP) {
                if (!(ok = wait_soon(&pv_done[q][i % NP], (i / NP - 1) & 1, gone, A.err))) break;
                tc_fence_after();
            }
            if (i < i0 || i >= i1) {
                const int key0 = from + i * BN, z = min(hi, to) - key0;
                if (A.window) {
                    const int a = lo - key0;
#pragma unroll
                    for (int c = 0; c < BN / 32; c++)
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (c * 32 + e < a) x[c][e] = 0xff800000u;
                }
#pragma unroll
                for (int c = 0; c < BN / 32; c++)
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (c * 32 + e >= z) x[c][e] = 0xff800000u;
                // keys that not every row of the block sees: their NaN and
                // infinities out of the tile of values (add_not_finite). The
                // first query tile's warps do it for both: its product goes
                // before the second's, so every row's waits on its own product
                // put the cleaned tile and the flag before what it reads
                if (q == 0) {
                    if (!(ok = wait_soon(&v_full[i % VS], (i / VS) & 1, gone, A.err))) break;
                    uint8_t *vt = v_sm + i % VS * C::KV_BYTES;
                    const int c0 = sp.clo - key0, c1 = min(sp.chi, to) - key0;
                    bool found = false;
#pragma unroll 4
                    for (int e = row; e < C::KV_BYTES / 16; e += 128) {
                        const int key = e / 8 % BN;
                        uint4 w = *reinterpret_cast<uint4 *>(vt + e * 16);
                        if ((key >= c0 && key < c1) || !any_bad<F16>(w)) continue;
                        uint32_t h[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if (bad_half<F16>(h[k])) h[k] &= 0xffff0000u;
                            if (bad_half<F16>(h[k] >> 16)) h[k] &= 0x0000ffffu;
                        }
                        *reinterpret_cast<uint4 *>(vt + e * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                        found |= key0 + key < to;
                    }
                    if (found) not_finite = 1;
                    fence_proxy_async_shared();
                }
                __syncwarp();
            }
            float top[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
            for (int c = 0; c < BN / 32; c++)
#pragma unroll
                for (int e = 0; e < 32; e += 8)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        top[k] = max3_nan(top[k], __uint_as_float(x[c][e + k]), __uint_as_float(x[c][e + 4 + k]));
            float mx = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]) * A.scale_log2;
            float base = m == -INFINITY ? 0.0f : -m;
            // or NaN; a row past the last holds what lay there and moves no other's
            const bool rose = valid && !(mx <= m + LAZY);
            if (__any_sync(0xffffffffu, rose)) {
                if (i > 0 && NP > 1) {  // and the last product into o
                    if (!(ok = wait_soon(&pv_done[q][(i - 1) % NP], ((i - 1) / NP) & 1, gone, A.err))) break;
                    tc_fence_after();
                }
                // a NaN or an infinite score: the row's weights are NaN, as the formula's
                const bool odd = !(mx < INFINITY);
                mx = odd ? m : fmaxf(m, mx);
                if (i > 0) {  // o relative to the new maxima
                    const float f = mx == m ? 1.0f : exp2_fast(m - mx);
#pragma unroll 1
                    for (int c = 0; c < DP / 32; c++) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_at + c * 32, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_32x32b_x32(o_at + c * 32, o);
                    }
                    l *= f;
                }
                m = mx;
                base = odd ? NAN : m == -INFINITY ? 0.0f : -m;
            }
            uint64_t s0 = 0, s1 = 0;
#pragma unroll
            for (int h = 0; h < PARTS; h++) {
                uint32_t p[32];
                weights<F16>(x[2 * h], A.scale_log2, base, p, s0, s1);
                tmem_st_32x32b_x32(tmem + lanes + C::P_COL + (q * NP + i % NP) * (BN / 2) + h * 32, p);
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(&p_full[q][i % NP][h]);
            }
            float sa, sb;
            unpack2(add2(s0, s1), sa, sb);
            l += sa + sb;
        }
        // the last product
        if (ok && n > 0) {
            ok = wait_soon(&pv_done[q][(n - 1) % NP], ((n - 1) / NP) & 1, gone, A.err);
            tc_fence_after();
        }
        const int head = kv_head * A.group + row % A.group;
        const int64_t tok = s.q0 + (int64_t) t;
        if (ok) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (not_finite) {
#pragma unroll 1
                for (int c = 0; c < DP; c += 8) {
                    float r[8];
                    __syncwarp();
                    tmem_ld_32x32b_x8(o_at + c, r);
                    if (valid && c < A.d)
                        add_not_finite<F16>(A, seq, kv_head, c, max(lo, from), min(hi, to), sp.clo, max(sp.clo, sp.chi), r);
                    __syncwarp();
                    tmem_st_32x32b_x8(o_at + c, r);
                }
            }
            // Rolled, since every block comes through here once and pays for
            // each line of code. 16-bit results go through shared memory (the
            // query tile's, whose scores are all made, or the tiles', all used), a
            // row of DP a thread, 16 bytes at unit ^ (row % 8), and out of it in
            // whole rows.
            uint8_t *const rows16 = q_sm + q * C::Q_BYTES + warp % 4 * 32 * (DP * 2);
            const bool whole = A.splits == 1;
            const int rows = min(32, (tq1 - tq0) * A.group - warp % 4 * 32);  // of this warp's that hold something
#pragma unroll 1
            for (int pass = 0; pass < (whole && A.a_next ? 2 : 1); pass++) {  // A.out and the rest; A.a_next
                __syncwarp();
#pragma unroll 1
                for (int c = 0; c < DP; c += 64) {
                    uint32_t o[2][32];
                    __syncwarp();  // rows that hold nothing skip the stores, not the loads
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (n > 0) tmem_ld_32x32b_x32(o_at + c + 32 * h, o[h]);
                        else
#pragma unroll
                            for (int e = 0; e < 32; e++) o[h][e] = 0;
                    if (n > 0) {
                        tmem_ld_wait(o[0]);
                        tmem_ld_wait(o[1]);
                    }
                    auto eights = [&](auto store) {  // of eight columns' values each
#pragma unroll
                        for (int e = 0; e < 64; e += 8) {
                            float r[8];
#pragma unroll
                            for (int k = 0; k < 8; k++) r[k] = __uint_as_float(o[e / 32][e % 32 + k]) * inv;
                            store(e, r);
                        }
                    };
                    uint8_t *const at = rows16 + lane * (DP * 2) + c * 2;
                    if (!whole) {
                        // unnormalised to the workspace, whose rows have room for DP
                        // values: 32 columns at a time, a line of a row by 8 lanes
                        // (128 tokens over 8,192, heads of 128: 36 us with a row a lane, 32 so)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                *reinterpret_cast<uint4 *>(rows16 + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                                    make_uint4(o[h][4 * e], o[h][4 * e + 1], o[h][4 * e + 2], o[h][4 * e + 3]);
                            __syncwarp();
                            const int r1 = warp % 4 * 32 + lane / 8, u = lane % 8;
                            int g = r1 % A.group;
                            float *dst = A.part + (split * (A.b.T * A.heads) + (s.q0 + (int64_t) (tq0 + r1 / A.group)) * A.heads +
                                                   kv_head * A.group + g) * DP + c + 32 * h + u * 4;
                            const int64_t wrap = (int64_t) (A.heads - A.group) * DP;
#pragma unroll
                            for (int r = lane / 8; r < 32; r += 4) {
                                if (r < rows)
                                    *reinterpret_cast<uint4 *>(dst) =
                                        *reinterpret_cast<const uint4 *>(rows16 + r * 128 + ((u ^ (r & 7)) << 4));
                                dst += 4 * DP;
                                for (g += 4; g >= A.group; g -= A.group) dst += wrap;
                            }
                        }
                    } else if (!valid) {
                    } else if (pass == 1) {
                        eights([&](int e, const float (&r)[8]) {
                            *reinterpret_cast<uint4 *>(at + ((e / 8 ^ (lane & 7)) << 4)) = pack8(r);
                        });
                    } else {
                        if (A.out)
                            eights([&](int e, const float (&r)[8]) {
                                *reinterpret_cast<uint4 *>(at + ((e / 8 ^ (lane & 7)) << 4)) = round8<F16>(r);
                            });
                        if (A.y)
                            eights([&](int e, const float (&r)[8]) {
                                if (c + e < A.d) store8_f32(A, tok, head, c + e, r);
                            });
                    }
                }
                uint16_t *const base = pass == 0 ? A.out : A.a_next;
                if (!whole || !base) continue;
                __syncwarp();
                const int64_t ld = pass == 0 ? A.ldo : A.lda;
                constexpr int UNITS = DP / 8, AT_ONCE = 32 / UNITS, N = 4;
                const int u = lane % UNITS;
                const int r1 = warp % 4 * 32 + lane / UNITS;  // this lane's first row of the tile
                int g = r1 % A.group;
                uint16_t *dst = base + (s.q0 + (int64_t) (tq0 + r1 / A.group)) * ld + (kv_head * A.group + g) * A.d + u * 8;
                const int64_t wrap = ld - (int64_t) A.group * A.d;  // from a token's last head to the next's first
                const bool has = u * 8 < A.d;
#pragma unroll 1
                for (int r0 = lane / UNITS; r0 < rows; r0 += N * AT_ONCE) {
                    uint4 v[N];
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        const int r = (r0 + k * AT_ONCE) & 31;
                        v[k] = *reinterpret_cast<const uint4 *>(rows16 + r * (DP * 2) + ((u ^ (r & 7)) << 4));
                    }
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        if (has && r0 + k * AT_ONCE < rows) *reinterpret_cast<uint4 *>(dst) = v[k];
                        dst += AT_ONCE * A.d;
                        for (g += AT_ONCE; g >= A.group; g -= A.group) dst += wrap;
                    }
                }
            }
        }
        if (A.splits > 1 && valid) A.ml[split * (A.b.T * A.heads) + tok * A.heads + head] = make_float2(ok ? m : NAN, l);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_QK) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// The parts of each row joined in order, eight columns a thread. Few rows: the
// block's groups of threads take every GROUPS-th part of one row and meet in
// shared memory, so that 37 parts cost five loads one after another. A row one
// of whose parts is none (m is NaN, which no maximum is) stays as it was.
template <int DP, bool F16, bool FEW>
__global__ void __launch_bounds__(128) kv_combine_kernel(const __grid_constant__ attend_args A, int tile_rows) {
    constexpr int PER_ROW = DP / 8, GROUPS = 128 / PER_ROW;
    const int seq = blockIdx.z, kv_head = blockIdx.y, group = threadIdx.x / PER_ROW;
    const kv_seq s = kv_seq_of(A.b, A.page_size, seq);
    if (!s.ok) return;
    const int64_t rows = (int64_t) s.n * A.group;
    const int64_t r = FEW ? blockIdx.x : (int64_t) blockIdx.x * GROUPS + group;
    const int c = threadIdx.x % PER_ROW * 8;
    if (FEW ? r >= rows : r >= rows || c >= A.d) return;
    int n = A.splits;
    if (!FEW) {  // the chunks of the row's tile, counted as its blocks counted them
        const int64_t r0 = r / tile_rows * tile_rows;
        const key_span sp = span_of(A, s, (int) (r0 / A.group), (int) ((min(r0 + tile_rows, rows) - 1) / A.group));
        const int64_t span = sp.hi - (int64_t) sp.lo / KEYS * KEYS;
        n = span > 0 ? (int) ((span + A.chunk - 1) / A.chunk) : 1;
    }
    const int t = (int) (r / A.group), head = kv_head * A.group + (int) (r % A.group);
    const int64_t tok = s.q0 + (int64_t) t, stride = A.b.T * A.heads, slot = tok * A.heads + head;
    float mx = -INFINITY, sum = 0.0f, x[8] = {};
    const int first = FEW ? group : 0, step = FEW ? GROUPS : 1;
    bool whole = true;
    for (int i = first; i < n; i += step) {
        const float m = A.ml[i * stride + slot].x;
        whole = whole && m == m;
        mx = fmaxf(mx, m);
    }
#pragma unroll 4
    for (int i = first; i < n; i += step) {
        const float2 ml = A.ml[i * stride + slot];
        const float w = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - mx);
        const float4 *p = reinterpret_cast<const float4 *>(A.part + (i * stride + slot) * DP + c);
        const float4 a = p[0], b = p[1];
        sum += w * ml.y;
        const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __fmaf_rn(v[e], w, x[e]);
    }
    if (FEW) {
        __shared__ float sh[GROUPS][DP + 4];
        __shared__ float2 ml_sh[GROUPS];
        if (c == 0) ml_sh[group] = make_float2(whole ? mx : NAN, sum);
#pragma unroll
        for (int e = 0; e < 8; e++) sh[group][c + e] = x[e];
        __syncthreads();
        if (group > 0 || c >= A.d) return;
        float top = -INFINITY;
        whole = true;
        for (int g = 0; g < GROUPS; g++) {
            whole = whole && ml_sh[g].x == ml_sh[g].x;
            top = fmaxf(top, ml_sh[g].x);
        }
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.0f;
        for (int g = 0; g < GROUPS; g++) {
            const float w = ml_sh[g].x == -INFINITY ? 0.0f : exp2_fast(ml_sh[g].x - top);
            sum += w * ml_sh[g].y;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __fmaf_rn(sh[g][c + e], w, x[e]);
        }
    }
    if (!whole) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= inv;
    store8<F16>(A, tok, head, c, x);
}

// --- host ------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p) : nullptr;
    }();
    return fn;
}

// One layer's pool as (value, token of a page, kv head, page), in boxes of 64
// values by min(page, 64) tokens; wide: as (value of a block of 64, token,
// block, kv head, page), in boxes of whole heads (whole blocks of 64 only: a
// partial one would reach into the next head). Columns past d and pages past
// the pool read zeros.
bool pool_tmap(CUtensorMap *m, const zest_kv_cache *kv, const void *base, bool wide) {
    auto fn = encode_fn();
    if (!fn) return false;
    // a dimension of one entry is never stepped over: any valid stride does
    const int64_t hs = kv->kv_heads > 1 ? kv->head_stride : 8 * 32, ps = kv->pages > 1 ? kv->page_stride : 8 * 32;
    const cuuint64_t tokens = (cuuint64_t) kv->page_size, heads = (cuuint64_t) kv->kv_heads, pages = (cuuint64_t) kv->pages;
    const cuuint32_t box_keys = (cuuint32_t) std::min(kv->page_size, KEYS), blocks = (cuuint32_t) kv->d / 64;
    cuuint64_t dims[5] = { (cuuint64_t) kv->d, tokens, heads, pages, 1 };
    cuuint64_t strides[4] = { (cuuint64_t) kv->token_stride * 2, (cuuint64_t) hs * 2, (cuuint64_t) ps * 2, 16 };
    cuuint32_t box[5] = { 64, box_keys, 1, 1, 1 };
    if (wide) {
        const cuuint64_t wide_dims[5] = { 64, tokens, blocks, heads, pages };
        const cuuint64_t wide_strides[4] = { (cuuint64_t) kv->token_stride * 2, 128, (cuuint64_t) hs * 2,
                                             (cuuint64_t) ps * 2 };
        std::copy(wide_dims, wide_dims + 5, dims);
        std::copy(wide_strides, wide_strides + 4, strides);
        box[2] = blocks;
    }
    cuuint32_t estr[5] = { 1, 1, 1, 1, 1 };
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, wide ? 5 : 4, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The batch with bounds no looser than its arrays allow: they shape the launch.
zest_kv_batch tightened(const zest_kv_cache *kv, const zest_kv_batch *b) {
    zest_kv_batch t = *b;
    t.max_q = std::min(t.max_q, t.T);
    t.max_kv = std::min(t.max_kv, t.table_stride * kv->page_size);
    return t;
}

// How a call runs: its row tiles, and the chunks its keys are cut into.
struct attend_plan {
    int dp, tile_rows, splits, join;
    bool many, wide, by_rows;
    int64_t row_tiles, chunk, ws_ml, ws_part;
};

// Up to 16 rows of a kv head go to the few-rows kernel: the cache's bytes
// bound it, and its smaller blocks keep more of them in flight. More rows go
// to the tensor-core tiles.
// The keys are cut so that the blocks fill the GPU once; where sequences may
// differ in length, up to four times for balance, in chunks of 1,024 keys or
// more (32 tokens over up to 8,192: 132 us filling it twice, 119 four times, 128
// eight times). Never below 128 keys a block (512 for many rows). Up to 8 blocks
// that have an SM each join as one cluster, without a second launch; more go
// through the workspace (as clusters of 4 the 32 tokens took 128 us, and one
// token over 131,072 keys 127 for 91: clusters wait for a GPC's SMs together).
// Many rows: where rows differ much in the keys they see, the blocks with the
// most run first, of all heads, so that the last to start are short (2,048
// tokens of 2,048: 72 us one head after another, 58 so; over 8,192: 199 and
// 190). With long keys all blocks are alike, and neighbours on one head's keys
// find them in L2 (over 32,768: 910 and 928; heads of 256 over 8,192: 290 and 307).
attend_plan plan_attend(const zest_kv_cache *kv, const zest_kv_batch *b, const zest_kv_attn *at) {
    attend_plan p;
    p.dp = kv->d <= 64 ? 64 : kv->d <= 128 ? 128 : 256;
    const int64_t group = at->heads / kv->kv_heads;
    p.many = b->max_q * group > ROWS;
    p.wide = !p.many && kv->d % 64 == 0 && kv->d == p.dp;
    p.tile_rows = p.many ? (int) ((p.dp == 256 ? 1 : 2) * (128 / group) * group) : ROWS;
    p.row_tiles = std::max<int64_t>(1, up(b->max_q * group, p.tile_rows));
    const int64_t units = std::max<int64_t>(1, b->n_seqs * (int64_t) kv->kv_heads * p.row_tiles);
    const int64_t per_sm = p.many ? 1 : p.dp == 64 ? 3 : p.dp == 128 ? 2 : 1;
    int64_t span = b->max_kv;
    if (at->causal && at->window)  // which may start inside a block of keys
        span = std::min(span, std::min(at->window, span) + std::min<int64_t>(b->max_q, p.tile_rows) + KEYS - 1);
    p.by_rows = p.dp < 256 && span < 8 * b->max_q;
    const int64_t once = std::max<int64_t>(1, 148 * per_sm / units), least = p.many ? 512 : 128;
    int64_t splits = once;
    if (b->n_seqs > 1) splits = std::max(once, std::min(148 * per_sm * 4 / units, up(span, 1024)));
    splits = std::max<int64_t>(1, std::min(splits, up(span, least)));
    p.chunk = 0;
    p.join = 1;
    if (p.many) {
        p.chunk = std::max<int64_t>(1, up(up(span, splits), 2 * KEYS)) * 2 * KEYS;
        splits = std::max<int64_t>(1, up(span, p.chunk));
    } else if (splits <= 8 && splits * units <= 148) {
        p.join = (int) splits;
        splits = 1;
    }
    p.splits = (int) splits;
    p.ws_ml = p.ws_part = 0;
    if (p.splits > 1) {
        p.ws_ml = up((int64_t) p.splits * b->T * at->heads * 8, 256) * 256;
        p.ws_part = (int64_t) p.splits * b->T * at->heads * p.dp * 4;
    }
    return p;
}

const char *attend_fault(const zest_kv_cache *kv, const zest_kv_batch *b, const zest_kv_attn *at) {
    if (!at) return "nothing to attend with";
    if (at->heads < 1 || at->heads % kv->kv_heads || at->heads / kv->kv_heads > 128)
        return "heads are a multiple of the kv heads, at most 128 times";
    if (!(at->scale > 0.0f) || std::isinf(at->scale * LOG2E)) return "scale is not positive and finite";
    if (at->window < 0 || (at->window > 0 && !at->causal)) return "a window is positive and causal";
    const attend_plan p = plan_attend(kv, b, at);
    if (p.row_tiles * kv->kv_heads * p.splits > 0x7fffffff || b->max_q * (at->heads / kv->kv_heads) > 0x7fffffff)
        return "too many rows, or too many heads for the keys";
    return nullptr;
}

// A step's queries as (value, head, token), in boxes of 64 values of a group
// of heads and as many whole tokens as 128 rows hold.
bool query_tmap(CUtensorMap *m, const attend_args &a) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = { (cuuint64_t) a.d, (cuuint64_t) a.heads, (cuuint64_t) a.b.T };
    cuuint64_t strides[2] = { (cuuint64_t) a.d * 2, (cuuint64_t) a.ldq * 2 };
    cuuint32_t box[3] = { 64, (cuuint32_t) a.group, (cuuint32_t) (128 / a.group) };
    cuuint32_t estr[3] = { 1, 1, 1 };
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<uint16_t *>(a.q), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A kernel's dynamic shared memory allowed, on each device before its first launch there.
template <typename K>
bool allow_smem(K kernel, int bytes, uint64_t &ready) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (dev < 64 && (__atomic_load_n(&ready, __ATOMIC_RELAXED) >> dev & 1)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    if (dev < 64) __atomic_fetch_or(&ready, 1ull << dev, __ATOMIC_RELAXED);
    return true;
}

template <int DP, bool F16>
int launch_attend(const zest_kv_cache *kv, const CUtensorMap &tk, const CUtensorMap &tv, const attend_args &a,
                  const attend_plan &p, cudaStream_t st) {
    const char *call = "zest_kv_attend";
    static uint64_t few_ready = 0, many_ready = 0;
    if (p.many) {
        using C = many_rows<DP>;
        CUtensorMap tq;
        if (!query_tmap(&tq, a)) return kv_refuse(call, "the queries' strides make no tensor map");
        if (!allow_smem(kv_attend_many_kernel<DP, F16>, C::SMEM, many_ready)) return check_launch(call);
        const dim3 grid((unsigned) (p.row_tiles * kv->kv_heads * p.splits), a.b.n_seqs);
        kv_attend_many_kernel<DP, F16><<<grid, C::THREADS, C::SMEM, st>>>(tq, tk, tv, a);
    } else {
        using C = few_rows<DP>;
        if (!allow_smem(kv_attend_few_kernel<DP, F16>, C::SMEM, few_ready)) return check_launch(call);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.splits * p.join, kv->kv_heads, a.b.n_seqs);
        cfg.blockDim = dim3(FEW_THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = st;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = p.join;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, kv_attend_few_kernel<DP, F16>, tk, tv, a);
    }
    if (check_launch(call)) return -1;
    const int64_t rows = a.b.max_q * a.group;
    if (p.splits == 1 || rows == 0) return 0;  // (of no rows, the kernel above has looked for sequences that have some)
    if (p.many)
        kv_combine_kernel<DP, F16, false><<<dim3((unsigned) up(rows, 128 / (DP / 8)), kv->kv_heads, a.b.n_seqs), 128, 0, st>>>(
            a, p.tile_rows);
    else
        kv_combine_kernel<DP, F16, true><<<dim3((unsigned) rows, kv->kv_heads, a.b.n_seqs), 128, 0, st>>>(a, p.tile_rows);
    return check_launch(call);
}

}  // namespace

}  // namespace zest

using namespace zest;

extern "C" {

int64_t zest_kv_attend_workspace(const zest_kv_cache *kv, const zest_kv_batch *batch, const zest_kv_attn *at) {
    const char *call = "zest_kv_attend_workspace";
    if (const char *why = kv_cache_fault(kv, 0)) return kv_refuse(call, why);
    if (const char *why = kv_batch_fault(batch)) return kv_refuse(call, why);
    const zest_kv_batch b = tightened(kv, batch);
    if (const char *why = attend_fault(kv, &b, at)) return kv_refuse(call, why);
    const attend_plan p = plan_attend(kv, &b, at);
    return p.ws_ml + p.ws_part;
}

int zest_kv_attend(const zest_kv_cache *kv, int64_t layer, const zest_kv_batch *batch, const zest_kv_attn *at,
                   void *workspace, size_t workspace_bytes, unsigned *err, void *stream) {
    const char *call = "zest_kv_attend";
    if (const char *why = kv_cache_fault(kv, layer)) return kv_refuse(call, why);
    if (const char *why = kv_batch_fault(batch)) return kv_refuse(call, why);
    const zest_kv_batch b = tightened(kv, batch);
    if (const char *why = attend_fault(kv, &b, at)) return kv_refuse(call, why);
    if (!err) return kv_refuse(call, "no device error word");
    if (b.T == 0 || b.n_seqs == 0) return 0;  // nothing to read or write: whatever the pointers
    const int64_t wide = (int64_t) at->heads * kv->d;
    auto rows = [&](const void *p, int64_t ld, int64_t unit) { return ld >= wide && ld % unit == 0 && !((uintptr_t) p & 15); };
    if (!at->q || !rows(at->q, at->ldq, 8)) return kv_refuse(call, "q rows cover the heads and are 16-byte aligned");
    if (!at->out && !at->y && !at->a_next) return kv_refuse(call, "no output");
    if ((at->out && !rows(at->out, at->ldo, 8)) || (at->y && !rows(at->y, at->ldy, 4)) ||
        (at->a_next && !rows(at->a_next, at->lda, 8)))
        return kv_refuse(call, "output rows cover the heads and are 16-byte aligned");
    const attend_plan p = plan_attend(kv, &b, at);
    const int64_t need = p.ws_ml + p.ws_part;
    if (need > 0 && (!workspace || ((uintptr_t) workspace & 15) || (int64_t) workspace_bytes < need))
        return kv_refuse(call, "the workspace is smaller than zest_kv_attend_workspace says, or not 16-byte aligned");
    const int64_t off = kv->layers > 1 ? layer * kv->layer_stride : 0;
    CUtensorMap tk, tv;
    if (!pool_tmap(&tk, kv, (const uint16_t *) kv->k + off, p.wide) ||
        !pool_tmap(&tv, kv, (const uint16_t *) kv->v + off, p.wide))
        return kv_refuse(call, "the pools' strides make no tensor map");
    attend_args a;
    a.b = b;
    a.q = (const uint16_t *) at->q;
    a.ldq = at->ldq;
    a.pages = kv->pages;
    a.v = (const uint16_t *) kv->v + off;
    a.page_stride = kv->pages > 1 ? kv->page_stride : 0;
    a.token_stride = kv->token_stride;
    a.head_stride = kv->kv_heads > 1 ? kv->head_stride : 0;
    a.heads = at->heads;
    a.group = at->heads / kv->kv_heads;
    a.d = kv->d;
    a.page_size = kv->page_size;
    a.causal = at->causal != 0;
    a.window = std::min(at->window, int64_t(1) << 32);  // wider than any sequence is as wide as it gets
    a.scale_log2 = at->scale * LOG2E;
    a.out = (uint16_t *) at->out;
    a.ldo = at->ldo;
    a.y = at->y;
    a.ldy = at->ldy;
    a.a_next = at->a_next;
    a.lda = at->lda;
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.join = p.join;
    a.wide = p.wide;
    a.by_rows = p.by_rows;
    a.ml = (float2 *) workspace;
    a.part = (float *) ((uint8_t *) workspace + p.ws_ml);
    a.err = err;
    cudaStream_t st = (cudaStream_t) stream;
    const bool f16 = kv->type == ZEST_TYPE_F16;
    switch (p.dp) {
        case 64: return f16 ? launch_attend<64, true>(kv, tk, tv, a, p, st) : launch_attend<64, false>(kv, tk, tv, a, p, st);
        case 128: return f16 ? launch_attend<128, true>(kv, tk, tv, a, p, st) : launch_attend<128, false>(kv, tk, tv, a, p, st);
        default: return f16 ? launch_attend<256, true>(kv, tk, tv, a, p, st) : launch_attend<256, false>(kv, tk, tv, a, p, st);
    }
}

}  // extern "C"
