// The paged key/value cache's own operations: a step's keys and values
// written to their pages (zest_kv_append), and the bookkeeping between steps
// (zest_kv_grow, _fork, _free, _compact), all on the device: a serving loop
// needs no copy of the tables on the host.
#include "zest_kv.cuh"

#include <algorithm>
#include <cstdio>

namespace zest {

int kv_refuse(const char *call, const char *why) {
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", call, why);
    return set_error(msg);
}

namespace {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

constexpr int AP_WARPS = 8;

// The sequence that row t may belong to: the last whose first row is t or
// before it, by a search that 32 lanes make together (each step cuts the
// range by 32), its bounds loaded with the last step. index -1: none.
struct found_seq {
    int index;
    kv_seq s;
};

__device__ __forceinline__ found_seq kv_find_seq(const zest_kv_batch &b, int page_size, int t, int lane) {
    int lo = 0, hi = b.n_seqs;
    while (true) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        int a = 0, e = 0, kv = 0;
        if (at < hi) {
            a = b.q_start[at];
            if (step == 1) {
                e = b.q_start[at + 1];
                kv = b.kv_len[at];
            }
        }
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && a <= t);
        if (!m) return { -1, {} };  // only ever in the first step: later ranges start at a sequence that holds
        const int k = 31 - __clz(m);
        lo += k * step;
        hi = min(hi, lo + step);
        if (step == 1) {
            a = __shfl_sync(0xffffffffu, a, k);
            e = __shfl_sync(0xffffffffu, e, k);
            kv = __shfl_sync(0xffffffffu, kv, k);
            return { lo, kv_seq_from(b, page_size, a, e, kv) };
        }
    }
}

struct append_args {
    zest_kv_batch b;
    zest_kv_new in;
    uint16_t *k, *v;  // this layer
    int64_t page_stride, token_stride, head_stride, pages;
    int page_size, page_shift, kv_heads, d, q_heads;
    float inv_d;
    unsigned *err;
};

// Head rows of a token that a warp has in flight.
template <int NC>
constexpr int AP_ROWS = NC == 1 ? 6 : 3;

// What a token's heads share of the rotation: out = x * co + partner * si for
// this lane's values (si negative for the first of a pair), and where a quad's
// partners lie.
template <int NC>
struct turn_of {
    float co[NC][4], si[NC][4];
};

// One head row of d values, 4 a lane and 128 columns (NC = 1: d <= 128), after
// its norm (w: this lane's weights) and rotation, rounded and stored. The
// partners of a NeoX pair (n_dims / 2 apart) come back from shared memory.
// Sums and rotations in f32 with explicitly rounded products; the scale is
// 1 / sqrt to 2 units in the last place (rsqrtf): far below the one rounding
// to 16 bits.
template <int NC, bool F16>
__device__ __forceinline__ void append_row(float (&v)[NC][4], const append_args &A, const float (&w)[NC][4],
                                           const turn_of<NC> &f, float4 *buf, uint16_t *dst, bool turn) {
    const int lane = threadIdx.x & 31, d = A.d;
    const bool neox = A.in.mode == ZEST_ROPE_NEOX;
    const int n_dims = A.in.rope ? A.in.n_dims : 0, half = n_dims / 2;
    if (turn && A.in.eps >= 0.0f) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) ss = __fmaf_rn(v[c][e], v[c][e], ss);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float sc = rsqrtf(__fmaf_rn(ss, A.inv_d, A.in.eps));
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[c][e] = __fmul_rn(__fmul_rn(v[c][e], sc), w[c][e]);
    }
    if (turn && n_dims) {
        if (neox) {
            __syncwarp();
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (4 * lane + 128 * c < d) buf[lane + 32 * c] = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
            __syncwarp();
        }
        const float *row = reinterpret_cast<const float *>(buf);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int j0 = 4 * lane + 128 * c;
            if (j0 >= n_dims) continue;
            float x[4];
            if (!neox) {
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = v[c][e ^ 1];
            } else if (half % 4 == 0) {  // four values on one side of the middle, their partners side by side too
                const float4 q = buf[(j0 < half ? j0 + half : j0 - half) / 4];
                x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = j0 + e;
                    x[e] = j < n_dims ? row[j < half ? j + half : j - half] : 0.0f;
                }
            }
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = __fadd_rn(__fmul_rn(v[c][e], f.co[c][e]), __fmul_rn(x[e], f.si[c][e]));
            v[c][0] = o[0];
            v[c][1] = o[1];
            if (j0 + 2 < n_dims) {  // n_dims may end in the middle of a quad
                v[c][2] = o[2];
                v[c][3] = o[3];
            }
        }
    }
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int j = 4 * lane + 128 * c;
        if (j < d)
            *reinterpret_cast<uint2 *>(dst + j) =
                make_uint2(kv_bits2<F16>(v[c][0], v[c][1]), kv_bits2<F16>(v[c][2], v[c][3]));
    }
}

// A block's share of a token's head rows (q, k, v), up to AP_ROWS a warp, all
// loaded before anything is known of the token's sequence: the search for it
// and the page's number are two loads, one after the other, that the rows'
// loads run beside. 2,048 tokens of 32 + 8 + 8 heads of 128 take 27.5 us, 2.8
// TB/s: two thirds of the issue slots are taken, by the norm's sums over lanes
// and the rotation's exchange (24.6 us without the norm), and four blocks' 32
// warps an SM are what the rows in registers leave room for: at 64 registers a
// thread, 40 bytes of which spill (27.0 us; three blocks of 80 registers, which
// spill none, 28.8). 32 tokens: 3.9 us, those loads' latency.
template <int NC, bool F16>
__global__ void __launch_bounds__(AP_WARPS * 32, NC == 1 ? 4 : 2) kv_append_kernel(const __grid_constant__ append_args A) {
    constexpr int N = AP_ROWS<NC>;
    __shared__ float4 buf[AP_WARPS][NC * 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = A.d;
    const int q_rows = A.q_heads, k_rows = q_rows + A.kv_heads, rows = k_rows + A.kv_heads;
    const int step = gridDim.y * AP_WARPS;
    const bool neox = A.in.mode == ZEST_ROPE_NEOX;
    const int n_dims = A.in.rope ? A.in.n_dims : 0, half = n_dims / 2;
    for (int64_t t = blockIdx.x; t < A.b.T; t += gridDim.x) {
        const float *qx = A.in.q + t * A.in.ldq, *kx = A.in.k + t * A.in.ldk, *vx = A.in.v + t * A.in.ldv;
        for (int r0 = blockIdx.y * AP_WARPS + warp; r0 < rows; r0 += N * step) {
            float v[N][NC][4];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int r = r0 + k * step;
                const float *x = r < q_rows ? qx + r * d : r < k_rows ? kx + (r - q_rows) * d : vx + (r - k_rows) * d;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int j = 4 * lane + 128 * c;
                    const float4 f =
                        r < rows && j < d ? *reinterpret_cast<const float4 *>(x + j) : make_float4(0, 0, 0, 0);
                    v[k][c][0] = f.x, v[k][c][1] = f.y, v[k][c][2] = f.z, v[k][c][3] = f.w;
                }
            }
            turn_of<NC> turn = {};
            float w[2][NC][4];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int j0 = 4 * lane + 128 * c;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = j0 + e, p = neox ? (j < half ? j : j - half) : j >> 1;
                    if (j < n_dims) {
                        const float2 f = *reinterpret_cast<const float2 *>(A.in.rope + t * n_dims + 2 * p);
                        turn.co[c][e] = f.x;
                        turn.si[c][e] = (neox ? j < half : (j & 1) == 0) ? -f.y : f.y;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float *src = h ? A.in.k_norm : A.in.q_norm;
                    const float4 f = src && j0 < d ? *reinterpret_cast<const float4 *>(src + j0) : make_float4(1, 1, 1, 1);
                    w[h][c][0] = f.x, w[h][c][1] = f.y, w[h][c][2] = f.z, w[h][c][3] = f.w;
                }
            }
            const found_seq at_seq = kv_find_seq(A.b, A.page_size, (int) t, lane);
            const kv_seq &sq = at_seq.s;
            if (at_seq.index < 0) break;
            if (!sq.ok) {
                if (lane == 0) atomicOr(A.err, ZEST_ERR_BAD_SEQ);
                break;
            }
            const int i = (int) (t - sq.q0), pos = sq.kv - sq.n + i;
            if (i >= sq.n) break;  // behind the last sequence
            int64_t at = -1;       // the token's place in the pools, in values
            if (pos < 0) {
                if (lane == 0) atomicOr(A.err, ZEST_ERR_BAD_SEQ);
            } else {
                const int64_t page = A.b.table[at_seq.index * A.b.table_stride + (pos >> A.page_shift)];
                if (page < 0 || page >= A.pages) {
                    if (lane == 0) atomicOr(A.err, ZEST_ERR_BAD_PAGE);
                } else {
                    at = page * A.page_stride + (pos & (A.page_size - 1)) * A.token_stride;
                }
            }
            uint16_t *qo = reinterpret_cast<uint16_t *>(A.in.q_out) + t * A.in.ldqo;
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int r = r0 + k * step;
                if (r >= rows || (r >= q_rows && at < 0)) continue;
                if (r < q_rows) append_row<NC, F16>(v[k], A, w[0], turn, buf[warp], qo + r * d, true);
                else
                    append_row<NC, F16>(v[k], A, w[1], turn, buf[warp],
                                        r < k_rows ? A.k + at + (r - q_rows) * A.head_stride
                                                   : A.v + at + (r - k_rows) * A.head_stride,
                                        r < k_rows);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------

// The tables' part of each page operation is one block's work: ranks of free
// and live pages by block scans over refs, 16 pages a thread and step, so a
// pool of 16,384 pages is one step. Bound by latency, not bytes: one dependent
// load after another, so loads that do not depend go out together.
constexpr int PG_THREADS = 1024, PG_PER = 16, PG_STEP = PG_THREADS * PG_PER;

struct pages_shared {
    int warp[32];
    int total;
    int bad;
    int off[ZEST_KV_MAX_SEQS + 1];   // before each sequence: pages taken by the earlier ones
    int held[ZEST_KV_MAX_SEQS];      // its pages before the call (grow); its fresh page (fork)
    int who[ZEST_KV_MAX_SEQS];
};

// This thread's exclusive prefix over the block of v; total: all of it.
__device__ __forceinline__ int block_scan(int v, pages_shared &sh, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sh.warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = sh.warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sh.warp[lane] = w;
    }
    __syncthreads();
    const int before = x - v + (warp ? sh.warp[warp - 1] : 0);
    total = sh.warp[31];
    __syncthreads();
    return before;
}

// The free (or, live = true, held) pages in [from, pages) in rising order:
// f(rank, page) for each with rank < limit. Every thread calls it; returns how
// many there are up to the step where the limit was passed.
template <typename F>
__device__ __forceinline__ int64_t each_page(const int32_t *refs, int64_t from, int64_t pages, bool live,
                                             int64_t limit, pages_shared &sh, F f) {
    const bool vec = ((uintptr_t) refs & 15) == 0;
    int64_t seen = 0;
    for (int64_t base = from & ~(int64_t) 3; base < pages && seen < limit; base += PG_STEP) {
        const int64_t p0 = base + (int64_t) threadIdx.x * PG_PER;
        int4 r[PG_PER / 4];
#pragma unroll
        for (int i = 0; i < PG_PER / 4; i++) {
            const int64_t p = p0 + 4 * i;
            if (vec && p + 4 <= pages) r[i] = *reinterpret_cast<const int4 *>(refs + p);
            else
                r[i] = make_int4(p < pages ? refs[p] : 0, p + 1 < pages ? refs[p + 1] : 0,
                                 p + 2 < pages ? refs[p + 2] : 0, p + 3 < pages ? refs[p + 3] : 0);
        }
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < PG_PER / 4; i++)
            bits |= ((r[i].x != 0) | (r[i].y != 0) << 1 | (r[i].z != 0) << 2 | (r[i].w != 0) << 3) << (4 * i);
        if (!live) bits = ~bits;
        // only pages of [from, pages)
        const int64_t n = min(max(pages - p0, (int64_t) 0), (int64_t) PG_PER), skip = max(from - p0, (int64_t) 0);
        bits &= (1u << n) - 1u;
        bits = skip < PG_PER ? bits & ~((1u << skip) - 1u) : 0u;
        int total;
        int64_t rank = seen + block_scan(__popc(bits), sh, total);
        while (bits && rank < limit) {
            f(rank++, p0 + __ffs(bits) - 1);
            bits &= bits - 1;
        }
        seen += total;
    }
    return seen;
}

struct pages_args {
    zest_kv_tables in, out;
    int64_t pages;
    int page_size, n;
    const int32_t *a, *b;  // seq and add; src and dst
    int32_t *ws;           // moves: count, then (from, to) pairs; compact: [1 + 2 * pages] then the map
    unsigned *err;
};

// n values copied by one block, four 16-byte loads a thread in flight.
__device__ __forceinline__ void copy_values(int32_t *dst, const int32_t *src, int64_t n) {
    if (dst == src) return;
    int64_t done = 0;
    if ((((uintptr_t) dst | (uintptr_t) src) & 15) == 0) {
        const int64_t n4 = n / 4;
        for (int64_t base = threadIdx.x; base < n4; base += 4 * PG_THREADS) {
            int4 x[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (base + i * PG_THREADS < n4) x[i] = reinterpret_cast<const int4 *>(src)[base + i * PG_THREADS];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (base + i * PG_THREADS < n4) reinterpret_cast<int4 *>(dst)[base + i * PG_THREADS] = x[i];
        }
        done = 4 * n4;
    }
    for (int64_t i = done + threadIdx.x; i < n; i += PG_THREADS) dst[i] = src[i];
}

// out := in, by one block (in and out may be the same).
__device__ __forceinline__ void copy_tables(const pages_args &A) {
    copy_values(A.out.refs, A.in.refs, A.pages);
    copy_values(A.out.table, A.in.table, A.in.seqs * A.in.table_stride);
    copy_values(A.out.len, A.in.len, A.in.seqs);
}

// The same by many blocks, ahead of the operation's own, for tables that one
// block would take longer over than a launch costs (above 64 Ki entries).
__global__ void __launch_bounds__(256) kv_copy_tables_kernel(const __grid_constant__ pages_args A) {
    const int64_t at = blockIdx.x * (int64_t) blockDim.x + threadIdx.x, step = (int64_t) gridDim.x * blockDim.x;
    if (A.in.refs != A.out.refs)
        for (int64_t i = at; i < A.pages; i += step) A.out.refs[i] = A.in.refs[i];
    if (A.in.table != A.out.table)
        for (int64_t i = at; i < A.in.seqs * A.in.table_stride; i += step) A.out.table[i] = A.in.table[i];
    if (A.in.len != A.out.len)
        for (int64_t i = at; i < A.in.seqs; i += step) A.out.len[i] = A.in.len[i];
}

// out := in, and the sequences named into sh.who; sh.bad gets bits where one
// is out of range or, with `once`, appears twice. Ends with the block in step
// and the copies visible to it.
__device__ __forceinline__ void begin(const pages_args &A, const int32_t *who, bool once, pages_shared &sh) {
    const int i = threadIdx.x, mine = i < A.n ? who[i] : 0;
    if (i == 0) sh.bad = 0;
    if (i < A.n) sh.who[i] = mine;
    copy_tables(A);
    __syncthreads();
    bool bad = i < A.n && (mine < 0 || mine >= A.in.seqs);
    if (once)  // every pair, dealt over the block
        for (int e = i; e < A.n * A.n; e += PG_THREADS) {
            const int a = e / A.n, b = e % A.n;
            bad |= a < b && sh.who[a] == sh.who[b];
        }
    if (bad) atomicOr(&sh.bad, (int) ZEST_ERR_BAD_SEQ);
}

// The bits found so far; true: stop, out stays what copy_tables made it.
__device__ __forceinline__ bool give_up(const pages_args &A, pages_shared &sh) {
    __syncthreads();
    const int bad = sh.bad;
    __syncthreads();
    if (bad && threadIdx.x == 0) {
        atomicOr(A.err, (unsigned) bad);
        if (A.ws) A.ws[0] = 0;
    }
    return bad != 0;
}

__global__ void __launch_bounds__(PG_THREADS) kv_grow_kernel(const __grid_constant__ pages_args A) {
    __shared__ pages_shared sh;
    begin(A, A.a, true, sh);
    if (give_up(A, sh)) return;
    int need = 0, now = 0;
    const int i = threadIdx.x;
    if (i < A.n) {
        const int64_t len = A.out.len[sh.who[i]], add = A.b[i], ps = A.page_size;
        const int64_t held = (len + ps - 1) / ps, want = (len + add + ps - 1) / ps;
        if (len < 0 || add < 0 || len + add > 0x7fffffff || want > A.in.table_stride)
            atomicOr(&sh.bad, (int) ZEST_ERR_BAD_SEQ);
        else {
            need = (int) (want - held);
            now = (int) (len + add);
            sh.held[i] = (int) held;
        }
    }
    if (give_up(A, sh)) return;
    // a thousand sequences of at most 2^31 tokens: the sum of needs may pass 32 bits, so it is bounded first
    int total;
    const int before = block_scan(min(need, (1 << 20)), sh, total);
    const bool huge = __syncthreads_or(need > (1 << 20));
    if (i < A.n) sh.off[i] = before;
    if (threadIdx.x == 0) sh.off[A.n] = total;
    __syncthreads();
    const int64_t there = each_page(A.out.refs, 0, A.pages, false, total, sh, [](int64_t, int64_t) {});
    if (threadIdx.x == 0 && (huge || there < total)) atomicOr(&sh.bad, (int) ZEST_ERR_NO_PAGES);
    if (give_up(A, sh)) return;
    each_page(A.out.refs, 0, A.pages, false, total, sh, [&](int64_t rank, int64_t page) {
        int lo = 0, hi = A.n;  // the sequence with off[lo] <= rank < off[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (sh.off[mid] <= rank) lo = mid;
            else hi = mid;
        }
        A.out.table[sh.who[lo] * A.out.table_stride + sh.held[lo] + rank - sh.off[lo]] = (int32_t) page;
        A.out.refs[page] = 1;
    });
    if (i < A.n) A.out.len[sh.who[i]] = now;
}

__global__ void __launch_bounds__(PG_THREADS) kv_free_kernel(const __grid_constant__ pages_args A) {
    __shared__ pages_shared sh;
    begin(A, A.a, false, sh);
    if (give_up(A, sh)) return;
    const int64_t w = A.out.table_stride, n = A.n * w;
    for (int64_t e = threadIdx.x; e < n; e += blockDim.x) {
        // taken out by exchange: of a sequence named twice, one finds the page
        const int page = atomicExch(&A.out.table[sh.who[e / w] * w + e % w], -1);
        if (page < 0) continue;
        if (page >= A.pages || atomicSub(&A.out.refs[page], 1) <= 0) {
            if (page < A.pages) atomicAdd(&A.out.refs[page], 1);
            atomicOr(A.err, ZEST_ERR_BAD_PAGE);
        }
    }
    for (int i = threadIdx.x; i < A.n; i += blockDim.x) A.out.len[sh.who[i]] = 0;
}

__global__ void __launch_bounds__(PG_THREADS) kv_fork_kernel(const __grid_constant__ pages_args A) {
    __shared__ pages_shared sh;
    begin(A, A.b, true, sh);  // dst, left in sh.who
    __syncthreads();
    const int i = threadIdx.x, ps = A.page_size;
    int len = 0, src = 0, part = 0;
    if (i < A.n && !sh.bad) {
        src = A.a[i];
        const bool in_range = src >= 0 && src < A.in.seqs;
        len = in_range ? A.out.len[src] : 0;
        if (!in_range || len < 0 || (len + (int64_t) ps - 1) / ps > A.in.table_stride || A.out.len[sh.who[i]] != 0) {
            atomicOr(&sh.bad, (int) ZEST_ERR_BAD_SEQ);
            len = 0;
        }
        part = len % ps != 0;
    }
    if (give_up(A, sh)) return;
    int total;
    const int before = block_scan(part, sh, total);
    if (i < A.n) sh.off[i] = before;
    if (threadIdx.x == 0) sh.off[A.n] = total;
    __syncthreads();
    // every page that will be shared or copied has to be one; a warp a pair
    const int64_t w = A.out.table_stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int k = warp; k < A.n; k += PG_THREADS / 32) {
        const int64_t from = A.a[k], pages = (A.out.len[from] + (int64_t) ps - 1) / ps;
        for (int64_t j = lane; j < pages; j += 32) {
            const int page = A.out.table[from * w + j];
            if (page < 0 || page >= A.pages) atomicOr(&sh.bad, (int) ZEST_ERR_BAD_PAGE);
        }
    }
    const int64_t there = each_page(A.out.refs, 0, A.pages, false, total, sh, [](int64_t, int64_t) {});
    if (threadIdx.x == 0 && there < total) atomicOr(&sh.bad, (int) ZEST_ERR_NO_PAGES);
    if (give_up(A, sh)) return;
    // the rank-th free page goes to the rank-th pair with a part page: by rank, then by pair
    each_page(A.out.refs, 0, A.pages, false, total, sh, [&](int64_t rank, int64_t page) {
        sh.held[rank] = (int) page;
    });
    __syncthreads();
    if (i < A.n && part) {
        const int fresh = sh.held[sh.off[i]];
        A.ws[1 + 2 * sh.off[i]] = A.out.table[src * w + len / ps];
        A.ws[2 + 2 * sh.off[i]] = fresh;
        A.out.refs[fresh] = 1;
    }
    if (threadIdx.x == 0) A.ws[0] = total;
    __syncthreads();
    for (int k = warp; k < A.n; k += PG_THREADS / 32) {
        const int64_t from = A.a[k], to = sh.who[k], l = A.out.len[from], whole = l / ps;
        if (from == to) continue;  // an empty sequence copied onto itself
        for (int64_t j = lane; j < w; j += 32) {
            int page = -1;
            if (j < whole) {
                page = A.out.table[from * w + j];
                atomicAdd(&A.out.refs[page], 1);
            } else if (j == whole && l % ps) {
                page = sh.held[sh.off[k]];
            }
            A.out.table[to * w + j] = page;
        }
    }
    __syncthreads();
    if (i < A.n) A.out.len[sh.who[i]] = len;
}

// Whether one of the table's entries that thread `at` of `step` looks at is no
// page of the pool (an entry below zero holds none).
__device__ __forceinline__ bool no_page(const pages_args &A, int64_t at, int64_t step) {
    const int64_t n = A.in.seqs * A.in.table_stride, n4 = ((uintptr_t) A.in.table & 15) ? 0 : n / 4;
    bool bad = false;
#pragma unroll 4
    for (int64_t i = at; i < n4; i += step) {
        const int4 p = reinterpret_cast<const int4 *>(A.in.table)[i];
        bad |= max(max(p.x, p.y), max(p.z, p.w)) >= A.pages;
    }
    for (int64_t i = 4 * n4 + at; i < n; i += step) bad |= A.in.table[i] >= A.pages;
    return bad;
}

// Tables that one block would take longer over than a launch costs are looked
// over by many, ahead of the plan: what they find in ws[0], cleared before.
constexpr int64_t CHECKED_APART = 1 << 16;

__global__ void __launch_bounds__(256) kv_check_table_kernel(const __grid_constant__ pages_args A) {
    if (no_page(A, blockIdx.x * (int64_t) blockDim.x + threadIdx.x, (int64_t) gridDim.x * blockDim.x)) A.ws[0] = 1;
}

// ws: count of moves, (from, to) pairs, and behind 1 + 2 * pages the new
// number of each page. The table is rewritten by the copying kernel, whose
// many blocks suit its size. An entry that is no page: nothing moves, and every
// page keeps its number.
__global__ void __launch_bounds__(PG_THREADS) kv_compact_kernel(const __grid_constant__ pages_args A) {
    __shared__ pages_shared sh;
    const bool apart = A.in.seqs * A.in.table_stride > CHECKED_APART;
    const bool bad = apart ? A.ws[0] != 0 : no_page(A, threadIdx.x, PG_THREADS);
    copy_values(A.out.refs, A.in.refs, A.pages);
    copy_values(A.out.len, A.in.len, A.in.seqs);
    int32_t *map = A.ws + 1 + 2 * A.pages;
    const int64_t all = A.pages;
    for (int64_t i = threadIdx.x; i < all; i += blockDim.x) map[i] = (int32_t) i;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) {
            atomicOr(A.err, ZEST_ERR_BAD_PAGE);
            A.ws[0] = 0;
        }
        return;
    }
    const int64_t live = each_page(A.out.refs, 0, all, true, all, sh, [](int64_t, int64_t) {});
    const int64_t holes = each_page(A.out.refs, 0, live, false, all, sh, [&](int64_t rank, int64_t page) {
        A.ws[2 + 2 * rank] = (int32_t) page;
    });
    __syncthreads();
    each_page(A.out.refs, live, all, true, all, sh, [&](int64_t rank, int64_t page) {
        const int to = A.ws[2 + 2 * rank], count = A.out.refs[page];
        A.ws[1 + 2 * rank] = (int32_t) page;
        map[page] = to;
        A.out.refs[to] = count;
        A.out.refs[page] = 0;
    });
    if (threadIdx.x == 0) A.ws[0] = (int32_t) holes;
}

struct move_args {
    const int32_t *ws;
    uint16_t *pool[2];
    int64_t layers, layer_stride, page_stride, token_stride, head_stride, pages;
    int page_size, kv_heads, d;
    int flat;                     // a page's values lie in one run
    int64_t pieces;               // of a page
    const int32_t *table_in;      // compact: its entries renumbered by the map (null: none)
    int32_t *table_out;
    int64_t entries;
};

constexpr int MV_THREADS = 256, MV_PIECE = MV_THREADS * 4;  // 16-byte vectors: 16 KB

// Each move's page in each layer, K and V, in pieces of 16 KB: four 16-byte
// loads a thread in flight before the first store. Reads and writes each
// byte once; no page is both read and written. Bound by HBM: 360 MB
// of 512 pages in 12 layers read and written in 137 us with the plan, 5.2 TB/s.
__global__ void __launch_bounds__(MV_THREADS) kv_move_kernel(const __grid_constant__ move_args A) {
    const int64_t moves = A.ws[0], units = moves * A.layers * 2 * A.pieces;
    const int64_t vecs = (int64_t) A.page_size * A.kv_heads * (A.d / 8);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t piece = u % A.pieces, q = u / A.pieces, kv = q & 1, r = q >> 1;
        const int64_t layer = r % A.layers, m = r / A.layers;
        uint16_t *pool = A.pool[kv] + layer * A.layer_stride;
        const uint16_t *src = pool + A.ws[1 + 2 * m] * A.page_stride;
        uint16_t *dst = pool + A.ws[2 + 2 * m] * A.page_stride;
        uint4 x[4];
        int64_t at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t v = piece * MV_PIECE + i * MV_THREADS + threadIdx.x;
            at[i] = -1;
            if (v < vecs) {
                if (A.flat) {
                    at[i] = v * 8;
                } else {
                    const int dv = A.d / 8, c = (int) (v % dv), h = (int) (v / dv % A.kv_heads);
                    at[i] = v / dv / A.kv_heads * A.token_stride + h * A.head_stride + c * 8;
                }
                x[i] = *reinterpret_cast<const uint4 *>(src + at[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (at[i] >= 0) *reinterpret_cast<uint4 *>(dst + at[i]) = x[i];
    }
    if (A.table_in) {
        const int32_t *map = A.ws + 1 + 2 * A.pages;
        for (int64_t e = blockIdx.x * (int64_t) MV_THREADS + threadIdx.x; e < A.entries;
             e += (int64_t) gridDim.x * MV_THREADS) {
            const int p = A.table_in[e];
            A.table_out[e] = p >= 0 && p < A.pages ? map[p] : p;
        }
    }
}

int launch_moves(const zest_kv_cache *kv, const int32_t *ws, int64_t most, const int32_t *table_in,
                 int32_t *table_out, int64_t entries, cudaStream_t st, const char *what) {
    move_args m;
    m.ws = ws;
    m.pool[0] = (uint16_t *) kv->k;
    m.pool[1] = (uint16_t *) kv->v;
    m.layers = kv->layers;
    m.layer_stride = kv->layers > 1 ? kv->layer_stride : 0;
    m.page_stride = kv->pages > 1 ? kv->page_stride : 0;
    m.token_stride = kv->token_stride;
    m.head_stride = kv->kv_heads > 1 ? kv->head_stride : 0;
    m.pages = kv->pages;
    m.page_size = kv->page_size;
    m.kv_heads = kv->kv_heads;
    m.d = kv->d;
    const int64_t d = kv->d, ps = kv->page_size, kh = kv->kv_heads;
    m.flat = (kv->token_stride == kh * d && (kh == 1 || kv->head_stride == d)) ||
             (kv->token_stride == d && (kh == 1 || kv->head_stride == ps * d));
    m.pieces = (ps * kh * (d / 8) + MV_PIECE - 1) / MV_PIECE;
    m.table_in = table_in;
    m.table_out = table_out;
    m.entries = entries;
    const int64_t units = std::max<int64_t>(most * m.layers * 2 * m.pieces, (entries + MV_THREADS - 1) / MV_THREADS);
    kv_move_kernel<<<(int) std::min<int64_t>(std::max<int64_t>(units, 1), 148 * 8), MV_THREADS, 0, st>>>(m);
    return check_launch(what);
}

const char *tables_fault(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out) {
    if (const char *why = kv_cache_fault(kv, 0)) return why;
    if (!in || !out || !in->refs || !in->table || !in->len || !out->refs || !out->table || !out->len)
        return "no tables";
    if (in->seqs < 1 || in->seqs > 0x7fffffff || in->table_stride < 1 || in->table_stride > 0x7fffffff)
        return "no sequences, or no room for pages";
    if (out->seqs != in->seqs || out->table_stride != in->table_stride) return "in and out differ in size";
    return nullptr;
}

// The checks that the operations on n named sequences share.
const char *named_fault(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, int n,
                        const int32_t *a, const int32_t *b, const unsigned *err) {
    if (const char *why = tables_fault(kv, in, out)) return why;
    if (n < 0 || n > ZEST_KV_MAX_SEQS) return "0 to 1024 sequences a call";
    if (n > 0 && (!a || !b)) return "no sequence numbers";
    if (!err) return "no device error word";
    return nullptr;
}

pages_args args_of(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, int n,
                   const int32_t *a, const int32_t *b, void *ws, unsigned *err) {
    return { *in, *out, kv->pages, kv->page_size, n, a, b, (int32_t *) ws, err };
}

// Large tables copied by many blocks first; the operation then works in place.
int copy_first(pages_args &a, cudaStream_t st, const char *call) {
    const int64_t n = a.in.seqs * (a.in.table_stride + 1) + a.pages;
    if (n <= (1 << 16) || (a.in.refs == a.out.refs && a.in.table == a.out.table && a.in.len == a.out.len)) return 0;
    kv_copy_tables_kernel<<<(int) std::min<int64_t>((n + 1023) / 1024, 148 * 8), 256, 0, st>>>(a);
    a.in = a.out;
    return check_launch(call);
}

}  // namespace

}  // namespace zest

using namespace zest;

extern "C" {

int zest_kv_append(const zest_kv_cache *kv, int64_t layer, const zest_kv_batch *batch, const zest_kv_new *in,
                   unsigned *err, void *stream) {
    const char *call = "zest_kv_append";
    if (const char *why = kv_cache_fault(kv, layer)) return kv_refuse(call, why);
    if (const char *why = kv_batch_fault(batch)) return kv_refuse(call, why);
    if (!in || !err) return kv_refuse(call, "no new rows, or no device error word");
    const int64_t d = kv->d, wide = kv->kv_heads * d;
    auto good = [](const float *p, int64_t ld, int64_t n) { return p && ld >= n && ld % 4 == 0 && !((uintptr_t) p & 15); };
    if (batch->T > 0 && (!good(in->k, in->ldk, wide) || !good(in->v, in->ldv, wide)))
        return kv_refuse(call, "k and v rows cover the heads and are 16-byte aligned");
    if (in->q) {
        if (in->heads < 1 || in->heads > 65535 || !good(in->q, in->ldq, in->heads * d) || !in->q_out ||
            ((uintptr_t) in->q_out & 15) || in->ldqo < in->heads * d || in->ldqo % 8)
            return kv_refuse(call, "q rows cover the heads, and q and q_out are 16-byte aligned");
    }
    if (in->eps != in->eps || std::isinf(in->eps)) return kv_refuse(call, "eps is not a number");
    if (((uintptr_t) in->q_norm & 15) || ((uintptr_t) in->k_norm & 15))
        return kv_refuse(call, "norm weights are not 16-byte aligned");
    if (in->rope) {
        if (in->mode != ZEST_ROPE_NORMAL && in->mode != ZEST_ROPE_NEOX) return kv_refuse(call, "unsupported rope mode");
        if (in->n_dims <= 0 || in->n_dims % 2 || in->n_dims > d) return kv_refuse(call, "n_dims even and within d");
        if ((uintptr_t) in->rope & 7) return kv_refuse(call, "the rope table is not 8-byte aligned");
    }
    if (batch->T == 0 || batch->n_seqs == 0) return 0;
    append_args a;
    a.b = *batch;
    a.in = *in;
    const int64_t at = kv->layers > 1 ? layer * kv->layer_stride : 0;
    a.k = (uint16_t *) kv->k + at;
    a.v = (uint16_t *) kv->v + at;
    a.page_stride = kv->pages > 1 ? kv->page_stride : 0;
    a.token_stride = kv->token_stride;
    a.head_stride = kv->kv_heads > 1 ? kv->head_stride : 0;
    a.pages = kv->pages;
    a.page_size = kv->page_size;
    a.kv_heads = kv->kv_heads;
    a.d = kv->d;
    a.inv_d = 1.0f / (float) kv->d;
    a.page_shift = 4;
    while (1 << a.page_shift < kv->page_size) a.page_shift++;
    a.q_heads = in->q ? in->heads : 0;
    a.err = err;
    // a token's heads over as many blocks as give a warp AP_ROWS of them; few
    // tokens: over more, down to one row a warp
    const int rows = a.q_heads + 2 * a.kv_heads, most = (rows + AP_WARPS - 1) / AP_WARPS;
    const int each = AP_WARPS * (d <= 128 ? AP_ROWS<1> : AP_ROWS<2>), least = (rows + each - 1) / each;
    const int gx = (int) std::min<int64_t>(batch->T, 1 << 20);
    const dim3 grid(gx, (int) std::min<int64_t>(most, std::max<int64_t>(least, 148 * 8 / gx)));
    cudaStream_t st = (cudaStream_t) stream;
    const bool f16 = kv->type == ZEST_TYPE_F16;
    if (d <= 128 && f16) kv_append_kernel<1, true><<<grid, AP_WARPS * 32, 0, st>>>(a);
    else if (d <= 128) kv_append_kernel<1, false><<<grid, AP_WARPS * 32, 0, st>>>(a);
    else if (f16) kv_append_kernel<2, true><<<grid, AP_WARPS * 32, 0, st>>>(a);
    else kv_append_kernel<2, false><<<grid, AP_WARPS * 32, 0, st>>>(a);
    return check_launch(call);
}

int64_t zest_kv_pages_workspace(const zest_kv_cache *kv) {
    if (const char *why = kv_cache_fault(kv, 0)) return kv_refuse("zest_kv_pages_workspace", why);
    // fork: at most a move a pair; compact: at most half the pages move, and the map
    return 4 * (std::max<int64_t>(1 + 3 * kv->pages, 1 + 2 * ZEST_KV_MAX_SEQS) + 3);
}

int zest_kv_grow(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, int n,
                 const int32_t *seq, const int32_t *add, unsigned *err, void *stream) {
    if (const char *why = named_fault(kv, in, out, n, seq, add, err)) return kv_refuse("zest_kv_grow", why);
    pages_args a = args_of(kv, in, out, n, seq, add, nullptr, err);
    if (copy_first(a, (cudaStream_t) stream, "zest_kv_grow")) return -1;
    kv_grow_kernel<<<1, PG_THREADS, 0, (cudaStream_t) stream>>>(a);
    return check_launch("zest_kv_grow");
}

int zest_kv_free(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, int n,
                 const int32_t *seq, unsigned *err, void *stream) {
    if (const char *why = named_fault(kv, in, out, n, seq, seq, err)) return kv_refuse("zest_kv_free", why);
    pages_args a = args_of(kv, in, out, n, seq, seq, nullptr, err);
    if (copy_first(a, (cudaStream_t) stream, "zest_kv_free")) return -1;
    kv_free_kernel<<<1, PG_THREADS, 0, (cudaStream_t) stream>>>(a);
    return check_launch("zest_kv_free");
}

int zest_kv_fork(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, int n,
                 const int32_t *src, const int32_t *dst, void *workspace, unsigned *err, void *stream) {
    if (const char *why = named_fault(kv, in, out, n, src, dst, err)) return kv_refuse("zest_kv_fork", why);
    if (!workspace || ((uintptr_t) workspace & 15)) return kv_refuse("zest_kv_fork", "no 16-byte aligned workspace");
    pages_args a = args_of(kv, in, out, n, src, dst, workspace, err);
    if (copy_first(a, (cudaStream_t) stream, "zest_kv_fork")) return -1;
    kv_fork_kernel<<<1, PG_THREADS, 0, (cudaStream_t) stream>>>(a);
    if (check_launch("zest_kv_fork")) return -1;
    if (n == 0) return 0;
    return launch_moves(kv, (const int32_t *) workspace, n, nullptr, nullptr, 0, (cudaStream_t) stream, "zest_kv_fork");
}

int zest_kv_compact(const zest_kv_cache *kv, const zest_kv_tables *in, const zest_kv_tables *out, void *workspace,
                    unsigned *err, void *stream) {
    if (const char *why = tables_fault(kv, in, out)) return kv_refuse("zest_kv_compact", why);
    if (!err) return kv_refuse("zest_kv_compact", "no device error word");
    if (!workspace || ((uintptr_t) workspace & 15)) return kv_refuse("zest_kv_compact", "no 16-byte aligned workspace");
    const pages_args a = args_of(kv, in, out, 0, nullptr, nullptr, workspace, err);
    const int64_t entries = in->seqs * in->table_stride;
    cudaStream_t st = (cudaStream_t) stream;
    if (entries > CHECKED_APART) {
        cudaMemsetAsync(workspace, 0, 4, st);
        kv_check_table_kernel<<<(int) std::min<int64_t>((entries / 4 + 255) / 256, 148 * 8), 256, 0, st>>>(a);
        if (check_launch("zest_kv_compact")) return -1;
    }
    kv_compact_kernel<<<1, PG_THREADS, 0, st>>>(a);
    if (check_launch("zest_kv_compact")) return -1;
    return launch_moves(kv, (const int32_t *) workspace, kv->pages / 2, in->table, out->table, entries, st,
                        "zest_kv_compact");
}

}  // extern "C"
