// Attention of a tree (or chain) of drafted tokens over a paged cache.
//
// For token i of a sequence and query head h of kv head g:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(q.k_j - m),  m = max_j q.k_j
// over the positions j that token i sees: every position before ctx_len, and
// of the T drafted ones behind it those that its mask row names.  A row that
// sees nothing gives 0.
//
// The T * rep query rows of a kv head share its K/V rows, so they are the rows
// of one matrix product, and each K/V row is read once for all of them.  Three
// kernels share the work, all with the online softmax (running maximum, sum and
// output per row): attention_tree_rows.cu for up to 32 rows and
// attention_tree_tc.cu for more, over bf16 and int8 caches, and the one below
// for f32 caches.  Where (sequence, kv head, row tile) are too few for the SMs
// the context is split too, and tree_join_kernel joins the splits in split order,
// so results do not depend on the schedule.
//
// The products run on the tensor cores and keep f32's accuracy by splitting
// the f32 operand into a sum of terms of the other's type:
//   bf16 cache: q and p as three bf16 terms (2^-26), two for p when q and out
//     are bf16 (2^-18, against the output's 2^-9);
//   int8 cache: codes are exact in f16; q (over a power of two of its row's
//     magnitude) and p * v_scale (over a power of two of its row's) as two
//     f16 terms (2^-22); k_scale multiplies the scores;
//   f32 cache: both operands as two tf32 terms (2^-22).
// A bf16 q is one term as it is (in f16 elements below 2^-14 of the row's
// largest lose what is below 2^-25 of it).
//
// The kernel below: a CTA takes up to 16 * WR rows and a run of 32-position tiles,
// keeps S and the sums of P.V in registers; WR of its four warps divide the rows,
// the 4/WR others the positions of a tile, joined at the end.  The order of
// head_dim in the products is free as long as both operands use the same, so a
// lane takes 8 consecutive elements of a K row (one shared-memory load) as its B
// fragments, and 4 consecutive elements of each of its V rows as the B fragments
// of 4 column tiles.  Row pitches are chosen so that these loads are free of bank
// conflicts.  Splitting K and V into terms and three products per element, not
// memory, bound it: 8 sequences x 4 rows at 2000 positions, 32 kv heads of 128, take
// 208 us (2.6 TB/s).
#include "attention_tree.cuh"

#include <cuda_fp16.h>

#include <algorithm>

#include "attention_tree_dev.cuh"
#include "tcgen05.cuh"

namespace sb {

namespace {

constexpr int TA_THREADS = 128;

constexpr int TA_TILE = 32, TA_STAGES = 2;

template <int HD>
constexpr int ta_pitch() {
    return HD == 128 ? 528 : 272;  // of a row, bytes
}
template <int HD>
constexpr size_t ta_ring_bytes() {
    // the join: O, m and l of every row of every position group
    return std::max((size_t)TA_STAGES * TA_TILE * 2 * ta_pitch<HD>(), (size_t)64 * (HD + 2) * 4);
}
template <int HD, bool BF16, int WR>
constexpr size_t ta_smem_bytes() {
    return ta_ring_bytes<HD>() + (size_t)(BF16 ? 1 : 2) * (HD / 8) * 32 * 16 * WR;
}

// QT: terms of q (a bf16 element is one tf32 term); p, K and V are two.
template <int HD, bool BF16, int WR>
__global__ void __launch_bounds__(TA_THREADS) tree_attn_kernel(const TreeAttnArgs a) {
    constexpr int QT = BF16 ? 1 : 2, PT = 2, P = ta_pitch<HD>();
    constexpr int TILE = TA_TILE, STAGES = TA_STAGES, WP = 4 / WR, PW = TILE / WP;  // positions a warp takes of a tile
    constexpr int NT = PW / 8;                                                      // its column tiles of S
    constexpr int KS = HD / 8;
    constexpr int ROWS = 16 * WR;
    constexpr int CPR = HD / 4;  // 16-byte chunks of a K or V row
    constexpr int STAGE = TILE * 2 * P;
    constexpr int NO = HD / 8;  // column tiles of O

    extern __shared__ __align__(16) uint8_t sm[];
    uint4 *qf = reinterpret_cast<uint4 *>(sm + ta_ring_bytes<HD>());  // [WR][QT][KS][32] A fragments of q
    __shared__ __align__(8) unsigned long long bars[STAGES];
    pdl_launch_dependents();  // the join's blocks wait for this kernel's end

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gid = lane >> 2, c4 = lane & 3;
    const int wr = warp % WR, wp = warp / WR;
    const int nkv = a.c.pg.n_kv;
    const int split = blockIdx.x % a.n_splits, rt = blockIdx.x / a.n_splits;
    const int g = blockIdx.y, b = blockIdx.z;
    const int total_rows = a.T * a.rep;
    const int row0 = rt * ROWS;

    const int cap = a.c.pg.max_pages * a.c.pg.page_size;
    const int ctx = min(max(a.ctx_len[b], 0), cap);
    const int n_new = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
    const int n_vis = min(n_new, cap - ctx);  // tokens behind the table have no rows to be seen
    // the last token of this CTA's rows; under the j <= i rule nothing behind it is read
    const int last_i = min((min(row0 + ROWS, total_rows) - 1) / a.rep, n_new - 1);
    const int len = (int)min((long long)cap, (long long)ctx + (a.mask ? n_new : last_i + 1));
    const int ntiles = (len + TILE - 1) / TILE;
    const int per = (ntiles + a.n_splits - 1) / a.n_splits;
    const int t0 = min(split * per, ntiles), t1 = min(t0 + per, ntiles);

    // threads 0-31 copy a tile's K rows, 32-63 its V rows (bulk copies), each with the cache row found a tile ahead
    if (tid == 0) {
#pragma unroll
        for (int k = 0; k < STAGES; k++) mbar_init(smem_u32(&bars[k]), 2 * TILE);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    auto row_of = [&](int t) {
        const int p = t * TILE + (tid & (TILE - 1));
        return tid < 2 * TILE && p < len ? kv_row(a.c.pg, b, g, p) : -1ll;
    };
    auto issue = [&](int t, long long row) {
        if (tid >= 2 * TILE) return;
        float *dst = reinterpret_cast<float *>(sm + (size_t)(t % STAGES) * STAGE + tid * P);
        const uint32_t bar = smem_u32(&bars[t % STAGES]);
        if (row >= 0) {
            mbar_expect_tx(bar, HD * 4);
            tma_load_1d(smem_u32(dst), static_cast<const float *>(tid < TILE ? a.c.k : a.c.v) + (size_t)row * HD, HD * 4, bar);
        } else {  // rows behind the end (or on no page) read as zeros
#pragma unroll 4
            for (int i = 0; i < HD; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            fence_proxy_async_smem();  // a later copy may take the place
            mbar_arrive(bar);
        }
    };
    if (t0 < t1) issue(t0, row_of(t0));
    long long ahead = row_of(t0 + 1);

    // ---- q fragments
    const int ra = row0 + wr * 16 + gid, rb = ra + 8;
    auto qrow = [&](int r, int d) -> float {  // element d of q row r
        if (r >= total_rows) return 0.0f;
        const int t = r / a.rep, h = r - t * a.rep;
        const size_t o = (size_t)((size_t)b * a.T + t) * a.ldq + (size_t)(g * a.rep + h) * HD + d;
        return BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[o]) : static_cast<const float *>(a.q)[o];
    };
    if (wp == 0) {
        for (int ch = 0; ch < HD / 32; ch++) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int d = ch * 32 + c4 * 8 + 2 * s;
                float v[4] = {qrow(ra, d), qrow(rb, d), qrow(ra, d + 1), qrow(rb, d + 1)};
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) u[k] = tf32_rna(v[k]), v[k] = __fsub_rn(v[k], __uint_as_float(u[k]));
                    qf[((wr * QT + t) * KS + ch * 4 + s) * 32 + lane] = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        }
    }

    const int ia = ra < total_rows && ra / a.rep < n_new ? ra / a.rep : -1;
    const int ib = rb < total_rows && rb / a.rep < n_new ? rb / a.rep : -1;
    float o[NO][4];
#pragma unroll
    for (int n = 0; n < NO; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[n][e] = 0.0f;
    float ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;  // l: this lane's share of the sum

    bool ok = true;  // a wait that gives up (2 s) ends this thread's later ones
    for (int t = t0; t < t1; t++) {
        if (ok) ok = mbar_wait_long(smem_u32(&bars[t % STAGES]), ((t - t0) / STAGES) & 1);
        __syncthreads();
        if (t + 1 < t1) issue(t + 1, ahead);
        ahead = row_of(t + 2);

        const uint8_t *kt = sm + (size_t)(t % STAGES) * STAGE + wp * PW * P;
        const uint8_t *vt = sm + (size_t)(t % STAGES) * STAGE + TILE * P + wp * PW * P;

        // ---- S = q K^T
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = 0.0f;
#pragma unroll
        for (int ch = 0; ch < HD / 32; ch++) {
            uint32_t kh[NT][8], kl[NT][8];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float4 *p = reinterpret_cast<const float4 *>(kt + (n * 8 + gid) * P + (ch * 32 + c4 * 8) * 4);
                const float4 x = p[0], y = p[1];
                const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    kh[n][e] = tf32_rna(v[e]);
                    kl[n][e] = tf32_rna(__fsub_rn(v[e], __uint_as_float(kh[n][e])));
                }
            }
#pragma unroll
            for (int st = 0; st < 4; st++) {
#pragma unroll
                for (int q = 0; q < QT; q++) {
                    const uint4 f = qf[((wr * QT + q) * KS + ch * 4 + st) * 32 + lane];
                    const uint32_t af[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma_tf32(s[n], af, kh[n][2 * st], kh[n][2 * st + 1]);
                        if (q == 0) mma_tf32(s[n], af, kl[n][2 * st], kl[n][2 * st + 1]);
                    }
                }
            }
        }

        // ---- scores in powers of two; what a row does not see is -inf
        const long long base = (long long)t * TILE;
        const bool tail = base + TILE > ctx;
        unsigned long long va = ~0ull, vb = ~0ull;
        if (tail) {
            va = visible_bits(a, b, ia, ctx, n_vis, base) >> (wp * PW);
            vb = visible_bits(a, b, ib, ctx, n_vis, base) >> (wp * PW);
        }
        float na = ma, nb = mb;
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] *= LOG2E;
            if (tail) {
                const int bit = n * 8 + 2 * c4;
                if (!((va >> bit) & 1)) s[n][0] = -INFINITY;
                if (!((va >> (bit + 1)) & 1)) s[n][1] = -INFINITY;
                if (!((vb >> bit) & 1)) s[n][2] = -INFINITY;
                if (!((vb >> (bit + 1)) & 1)) s[n][3] = -INFINITY;
            }
            na = fmaxf(na, fmaxf(s[n][0], s[n][1]));
            nb = fmaxf(nb, fmaxf(s[n][2], s[n][3]));
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, d));
            nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, d));
        }
        float alpha_a = ma == -INFINITY ? 0.0f : ex2(ma - na), alpha_b = mb == -INFINITY ? 0.0f : ex2(mb - nb);
        ma = na, mb = nb;
        const float za = na == -INFINITY ? 0.0f : na, zb = nb == -INFINITY ? 0.0f : nb;
        la *= alpha_a, lb *= alpha_b;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            s[n][0] = ex2(s[n][0] - za), s[n][1] = ex2(s[n][1] - za);
            s[n][2] = ex2(s[n][2] - zb), s[n][3] = ex2(s[n][3] - zb);
            la += s[n][0] + s[n][1];
            lb += s[n][2] + s[n][3];
        }
        // ---- a non-finite V element of a drafted row must not reach rows that do not see it (0 * inf): when a
        // tail tile holds any, their products go row by row under the mask and zeros take their place below
        if (tail) {
            bool bad = false;
            uint8_t *tile_v = sm + (size_t)(t % STAGES) * STAGE + TILE * P;
            for (int i = tid; i < TILE * CPR; i += TA_THREADS) {
                const uint4 w = *reinterpret_cast<const uint4 *>(tile_v + (i / CPR) * P + (i % CPR) * 16);
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) bad |= (x[e] & 0x7f800000u) == 0x7f800000u;
            }
            if (__syncthreads_or(bad)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        for (int k = 0; k < 4; k++) {
                            const int pos = n * 8 + 2 * k + e;
                            const float pa = __shfl_sync(0xffffffffu, s[n][e], gid * 4 + k);
                            const float pb = __shfl_sync(0xffffffffu, s[n][2 + e], gid * 4 + k);
                            const bool sa = (va >> pos) & 1, sb = (vb >> pos) & 1;
#pragma unroll
                            for (int m = 0; m < NO; m++)
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    const int d = (m >> 2) * 32 + c4 * 8 + h * 4 + (m & 3);
                                    const float x = *reinterpret_cast<const float *>(vt + pos * P + d * 4);
                                    if (isfinite(x)) continue;
                                    // (their row's rescaling below leaves an infinity or a NaN as it is)
                                    if (sa) o[m][h] = fmaf(pa, x, o[m][h]), alpha_a = alpha_a > 0.0f ? alpha_a : 1.0f;
                                    if (sb) o[m][2 + h] = fmaf(pb, x, o[m][2 + h]), alpha_b = alpha_b > 0.0f ? alpha_b : 1.0f;
                                }
                        }
                __syncthreads();
                for (int i = tid; i < TILE * HD; i += TA_THREADS) {
                    float *p = reinterpret_cast<float *>(tile_v + (i / HD) * P) + i % HD;
                    if (!isfinite(*p)) *p = 0.0f;
                }
                fence_proxy_async_smem();
                __syncthreads();
            }
        }

        // ---- O = O * alpha + P V.  The tile's products start from zero and join O in an f32 FMA: the tensor cores
        // truncate as they accumulate, which over a long context would add up (1e-5 at 4096 positions).
        uint32_t af[NT][PT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float v[4] = {s[n][0], s[n][2], s[n][1], s[n][3]};
#pragma unroll
            for (int q = 0; q < PT; q++)
#pragma unroll
                for (int k = 0; k < 4; k++) af[n][q][k] = tf32_rna(v[k]), v[k] = __fsub_rn(v[k], __uint_as_float(af[n][q][k]));
        }
#pragma unroll
        for (int m = 0; m < HD / 32; m++) {
            float d[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) d[j][e] = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float4 x = *reinterpret_cast<const float4 *>(vt + (n * 8 + 2 * c4) * P + (m * 32 + gid * 4) * 4);
                const float4 y = *reinterpret_cast<const float4 *>(vt + (n * 8 + 2 * c4 + 1) * P + (m * 32 + gid * 4) * 4);
                const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t b0 = tf32_rna(xs[j]), b1 = tf32_rna(ys[j]);
#pragma unroll
                    for (int q = 0; q < PT; q++) mma_tf32(d[j], af[n][q], b0, b1);
                    mma_tf32(d[j], af[n][0], tf32_rna(__fsub_rn(xs[j], __uint_as_float(b0))),
                             tf32_rna(__fsub_rn(ys[j], __uint_as_float(b1))));
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float(&x)[4] = o[m * 4 + j];
                x[0] = fmaf(x[0], alpha_a, d[j][0]), x[1] = fmaf(x[1], alpha_a, d[j][1]);
                x[2] = fmaf(x[2], alpha_b, d[j][2]), x[3] = fmaf(x[3], alpha_b, d[j][3]);
            }
        }
    }
    if (!ok) wait_failed(a.errors, WAIT_TREE_F32);
    __syncthreads();

    // ---- whole sums of l; O in units of exp(-m)
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) la += __shfl_xor_sync(0xffffffffu, la, d), lb += __shfl_xor_sync(0xffffffffu, lb, d);
    // ---- the position groups of a row, joined in order; then the splits
    float *red = reinterpret_cast<float *>(sm);                 // [WP][ROWS][HD]
    float *rm = red + 64 * HD, *rl = rm + 64;                   // [WP][ROWS] each
    {
        const int r = wp * ROWS + wr * 16 + gid;
        if (c4 == 0) rm[r] = ma, rl[r] = la, rm[r + 8] = mb, rl[r + 8] = lb;
        // column tiles 4m .. 4m+3 are dims m*32 + c4*8 .. +7 (halves j and 4+j)
#pragma unroll
        for (int m = 0; m < HD / 32; m++) {
            float4 *pa = reinterpret_cast<float4 *>(red + (size_t)r * HD + m * 32 + c4 * 8);
            float4 *pb = reinterpret_cast<float4 *>(red + (size_t)(r + 8) * HD + m * 32 + c4 * 8);
            pa[0] = make_float4(o[4 * m][0], o[4 * m + 1][0], o[4 * m + 2][0], o[4 * m + 3][0]);
            pa[1] = make_float4(o[4 * m][1], o[4 * m + 1][1], o[4 * m + 2][1], o[4 * m + 3][1]);
            pb[0] = make_float4(o[4 * m][2], o[4 * m + 1][2], o[4 * m + 2][2], o[4 * m + 3][2]);
            pb[1] = make_float4(o[4 * m][3], o[4 * m + 1][3], o[4 * m + 2][3], o[4 * m + 3][3]);
        }
    }
    __syncthreads();

    const size_t tile = ((size_t)b * nkv + g) * (gridDim.x / a.n_splits) + rt;
    tree_finish<HD, BF16, WP, ROWS, TA_THREADS>(a, red, rm, rl, min(ROWS, total_rows - row0), row0, b, g, n_new, split, tile);
}

template <int HD, bool BF16, int WR>
int ta_inst(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    auto kern = tree_attn_kernel<HD, BF16, WR>;
    static int limit[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!limit[dev & 63]) SB_TRY(allow_max_dynamic_smem(kern, &limit[dev & 63]));
    constexpr size_t smem = ta_smem_bytes<HD, BF16, WR>();
    SB_CHECK(smem <= (size_t)limit[dev & 63], SB_ERR_SHAPE, "tree attention: needs %zu B shared memory (limit %d)", smem,
             limit[dev & 63]);
    SB_CUDA_TRY(launch(kern, dim3(p.row_tiles * a.n_splits, a.c.pg.n_kv, a.B), dim3(TA_THREADS), smem, st, false, a));
    return SB_OK;
}
template <int HD, bool BF16>
int ta_rows(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    return p.rows == 16   ? ta_inst<HD, BF16, 1>(a, p, st)
           : p.rows == 32 ? ta_inst<HD, BF16, 2>(a, p, st)
                          : ta_inst<HD, BF16, 4>(a, p, st);
}
template <int HD>
int ta_hd(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    return a.bf16 ? ta_rows<HD, true>(a, p, st) : ta_rows<HD, false>(a, p, st);
}

// The join of the splits, in order; a thread has four elements of a row.  A
// kernel of its own, over all SMs: the last CTA of a tile to arrive took 60 us for
// 32 rows x 64 splits of 8 kv heads, this takes 3.  Its blocks are in place when
// the attention kernel ends.
constexpr int TJ_THREADS = 128, TJ_BATCH = 8;  // splits whose loads are in flight together
template <int HD, bool BF16>
__global__ void __launch_bounds__(TJ_THREADS) tree_join_kernel(const __grid_constant__ TreeAttnArgs a, int rows, int row_tiles, int chunks) {
    const int tile = blockIdx.x / chunks;
    const int r = (blockIdx.x - tile * chunks) * (TJ_THREADS / (HD / 4)) + threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4) * 4;
    const int bg = tile / row_tiles, row = (tile - bg * row_tiles) * rows + r;
    const int b = bg / a.c.pg.n_kv, g = bg - b * a.c.pg.n_kv;
    if (r >= rows || row >= a.T * a.rep) return;
    pdl_wait();
    const int n_new = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
    const size_t first = (size_t)tile * a.n_splits * rows + r;
    float M = -INFINITY, L = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < a.n_splits; s0 += TJ_BATCH) {
        float2 ml[TJ_BATCH];
        float4 y[TJ_BATCH];
#pragma unroll
        for (int i = 0; i < TJ_BATCH; i++) {
            const size_t at = first + (size_t)min(s0 + i, a.n_splits - 1) * rows;  // past the last: that one again, not used
            ml[i] = __ldcg(a.ml + at);
            y[i] = __ldcg(reinterpret_cast<const float4 *>(a.part + at * HD + d));
        }
#pragma unroll
        for (int i = 0; i < TJ_BATCH; i++) {
            if (s0 + i >= a.n_splits || (ml[i].x == -INFINITY && ml[i].y == 0.0f)) continue;
            const float n = fmaxf(M, ml[i].x);
            const float f = ex2(ml[i].x - n), k = M == -INFINITY ? 0.0f : ex2(M - n);
            M = n;
            L = fmaf(ml[i].y, f, L * k);
            x.x = fmaf(y[i].x, f, x.x * k), x.y = fmaf(y[i].y, f, x.y * k), x.z = fmaf(y[i].z, f, x.z * k), x.w = fmaf(y[i].w, f, x.w * k);
        }
    }
    tree_store4<HD, BF16>(a, b, g, row, d, x, L, n_new);
}
template <int HD>
int tj_hd(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    const int chunks = ceil_div(std::min(p.rows, a.T * a.rep), TJ_THREADS / (HD / 4));
    const dim3 grid((unsigned)((size_t)a.B * a.c.pg.n_kv * p.row_tiles * chunks));
    SB_CUDA_TRY(launch(a.bf16 ? tree_join_kernel<HD, true> : tree_join_kernel<HD, false>, grid, dim3(TJ_THREADS), 0, st, true, a,
                       p.rows, p.row_tiles, chunks));
    return SB_OK;
}

}  // namespace

TreeAttnPlan tree_attn_plan(const TreeAttnArgs &a, int max_len) {
    if (tree_attn_rows_wanted(a)) return tree_attn_rows_plan(a, max_len);
    if (tree_attn_tc_wanted(a)) return tree_attn_tc_plan(a, max_len);
    TreeAttnPlan p;
    const int rows = a.T * a.rep;
    p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    p.row_tiles = ceil_div(rows, p.rows);
    const long long base = (long long)a.B * a.c.pg.n_kv * p.row_tiles;
    p.n_splits = tree_splits(base, ceil_div(std::max(max_len, 1), TA_TILE), p.rows == 64 ? 1 : 2);
    return p;
}

int tree_tensor_maps(TreeAttnArgs &a, int max_rows) {
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    a.box_rows = 0;
    if (a.c.pg.page_size % 8 != 0) return SB_OK;
    static EncodeFn encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        SB_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        SB_CHECK(fn && q == cudaDriverEntryPointSuccess, SB_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    int rows = 8;
    while (rows < max_rows && a.c.pg.page_size % (2 * rows) == 0) rows *= 2;
    const bool i8 = a.c.dtype == SB_KV_I8;
    const int esz = i8 ? 1 : 2, inner = std::min(a.c.hd * esz, 128);
    const cuuint64_t dims[2] = {(cuuint64_t)a.c.hd, (cuuint64_t)a.c.pg.n_pages * a.c.pg.n_kv * a.c.pg.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)a.c.hd * esz};
    const cuuint32_t box[2] = {(cuuint32_t)(inner / esz), (cuuint32_t)rows}, estr[2] = {1, 1};
    for (int i = 0; i < 2; i++) {
        const CUresult r = encode(i ? &a.tmv : &a.tmk, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                  i ? a.c.v : a.c.k, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        SB_CHECK(r == CUDA_SUCCESS, SB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    }
    a.box_rows = rows;
    return SB_OK;
}

// Splits of the context for `base` CTAs and `tiles` steps of it: those that
// let the busiest SM finish first, counting for a split what it costs to start
// and join (about a tile and a half).
int tree_splits(long long base, int tiles, int resident) {
    const int sms = device_props().sm_count * resident;
    int best = 1;
    double cost = 1e30;
    for (int s = 1; s <= 64 && s <= tiles; s++) {
        const double per = ceil_div(tiles, s) + (s > 1 ? 2.5 : 1.0);
        const double c = (double)((base * s + sms - 1) / sms) * per;
        if (c < cost * 0.999) cost = c, best = s;
    }
    return best;
}

int tree_attn_launch(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    if (tree_attn_rows_wanted(a)) SB_TRY(tree_attn_rows_launch(a, st));
    else if (tree_attn_tc_wanted(a)) SB_TRY(tree_attn_tc_launch(a, p, st));
    else SB_TRY(a.c.hd == 128 ? ta_hd<128>(a, p, st) : ta_hd<64>(a, p, st));
    if (p.n_splits == 1) return SB_OK;
    return a.c.hd == 128 ? tj_hd<128>(a, p, st) : tj_hd<64>(a, p, st);
}

}  // namespace sb
