// Tree attention for few query rows per kv head (T * rep <= 32) over a bf16 or
// int8 cache: the ordinary decode step and small trees.  What it computes, and
// the terms that keep f32's accuracy, are described in attention_tree.cu.
//
// With few rows the time goes to reading the cache (two bytes or one per K and V
// element) and to the work per cached element, so the products are turned round:
// S^T = K q^T and O^T = V^T p^T have positions and dims as the 16-row side of
// mma.m16n8k16 and the query rows as its 8-column side, and nothing is padded
// beyond 8 rows.  Each cached element is turned into its operand once, for all
// rows.
//
// Warps work alone: a warp streams tiles of PW positions through its own ring
// (boxes of the tensor copy engine and an mbarrier per stage; single 16-byte
// copies where pages are not a multiple of 8 positions), keeps q's fragments, S, the sums and O in
// registers, and takes every fourth or sixth tile of its CTA's share of the
// context.  A row's reference maximum serves until a score exceeds it by 2^8 (a
// vote, no reduction), so the steady state has no shuffles; probabilities up to
// 2^8 still fit the f16 terms, which are scaled to at most 2^15.  Warps and then
// splits are joined in order.
//
// Tiles lie as the boxes leave them, 16-byte chunks of 128-byte rows XOR-ed with
// the row's lowest three bits.  Both fragment loads are free of bank conflicts
// all the same: the order of the positions within a tile and that of the output's
// dims over the lanes are free, and are taken such that the rows and chunks of a
// load's phase differ where they have to (tr_position, tr_chunk).  (Rows of 64
// bytes, int8 of head_dim 64, keep two-way conflicts.)
//
// Bound by latency: a warp's products, softmax and products follow one another, and
// an SM has room for 8 to 12 warps.  Its issue slots are 47 % busy (int8, 8 rows:
// about 1000 instructions per 32 positions, half of which turn codes into f16
// operands) and 22 % (bf16, 32 rows, 255 registers a thread).  32 sequences x 1 token
// at 2048 positions, 8 kv heads of 4 query heads, int8: 37 us (3.8 TB/s; 44 us with
// four warps per CTA and 16-byte copies).  26 tokens at 1100, 32 kv heads, bf16: 24 us.
//
// Up to 32 rows, beyond which it would read the cache twice.  With 32 rows this
// kernel and the 128-row one take, in us, f32 q, for 8 sequences at 2000: 32 kv heads,
// int8 95 and 131, bf16 118 and 143; 8 kv heads, int8 35 and 37, bf16 42 and 48.  For
// one sequence at 2000 the other is ahead: 32 kv heads, int8 26 and 24, bf16 29 and 26;
// 8 kv heads, int8 19 and 16, bf16 21 and 18 (bf16 q: 25 and 20, 19 and 16).  With 8
// rows this one is ahead throughout: 32 kv heads at 2000, one sequence, 14 and 23.
#include "attention_tree.cuh"

#include <cuda_fp16.h>

#include <algorithm>

#include "attention_tree_dev.cuh"
#include "tcgen05.cuh"

namespace sb {

namespace {

// Two CTAs per SM in any case: of 6 warps where a warp's registers allow it
// (one group of 8 rows), else of 4.
constexpr int tr_warps(int nr) { return nr == 1 ? 6 : 4; }

template <int HD, int DT>
struct TrCache {
    static constexpr int ESZ = DT == SB_KV_I8 ? 1 : 2;
    static constexpr int RB = HD * ESZ;                   // bytes of a row
    static constexpr int CPR = RB / 16;                   // 16-byte chunks of a row
    static constexpr int PW = DT == SB_KV_I8 ? 32 : 16;   // positions of a warp's tile
    static constexpr int STAGES = 2;
    static constexpr int TILE = PW * RB;
    static constexpr int STAGE = 2 * TILE;                // scales lie behind all stages
    static constexpr int SCALES = DT == SB_KV_I8 ? 2 * PW * 4 : 0;
};

// byte offset of chunk `col` of row `row` of a tile of PW rows
template <int RB, int PW>
__device__ __forceinline__ int tr_at(int row, int col) {
    if (RB == 64) return row * 64 + ((col ^ ((row >> 1) & 3)) << 4);
    return (RB == 256 ? (col >> 3) * PW * 128 : 0) + row * 128 + (((col & 7) ^ (row & 7)) << 4);
}
// position (of eight) that is row `i` of a fragment, and the other way round
template <int RB>
__device__ __forceinline__ int tr_position(int i) {
    return RB == 64 ? i : ((i & 1) << 2) | (i >> 1);
}
template <int RB>
__device__ __forceinline__ int tr_index(int p) {
    return RB == 64 ? p : ((p & 3) << 1) | (p >> 2);
}
// 16-byte chunk of V's row and first dim of the eight dims that lane group gid has of the md-th 64 dims
template <int HD, int DT>
__device__ __forceinline__ int tr_chunk(int md, int gid) {
    if (DT != SB_KV_I8) return md * 8 + (gid & 1) * 4 + (gid >> 1);
    return HD == 64 ? gid >> 1 : ((gid >> 1) & 1) * 4 + (gid >> 2) + md * 2;
}
template <int HD, int DT>
__device__ __forceinline__ int tr_dim(int md, int gid) {
    return DT == SB_KV_I8 ? tr_chunk<HD, DT>(md, gid) * 16 + (gid & 1) * 8 : tr_chunk<HD, DT>(md, gid) * 8;
}

template <int DT>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (DT == SB_KV_I8) mma_f16(d, a, b0, b1);
    else mma_bf16(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

constexpr size_t tr_join_bytes(int hd, int nr) { return (size_t)tr_warps(nr) * nr * 8 * (hd + 2) * 4; }
template <int HD, int DT, int NR>
constexpr size_t tr_ring_bytes() {
    return std::max((size_t)tr_warps(NR) * TrCache<HD, DT>::STAGES * (TrCache<HD, DT>::STAGE + TrCache<HD, DT>::SCALES), tr_join_bytes(HD, NR));
}
// q's fragments lie in shared memory where they would not leave enough registers
constexpr bool tr_q_shared(int nr, int qt) { return nr * qt > 3; }

template <int HD, int DT, bool BF16, int NR>
__global__ void __launch_bounds__(tr_warps(NR) * 32, 2) tree_attn_rows_kernel(const __grid_constant__ TreeAttnArgs a) {
    using C = TrCache<HD, DT>;
    constexpr int TR_WARPS = tr_warps(NR), TR_THREADS = TR_WARPS * 32;
    constexpr int QT = BF16 ? 1 : DT == SB_KV_BF16 ? 3 : 2;
    constexpr int PT = DT == SB_KV_BF16 && !BF16 ? 3 : 2;
    constexpr int PW = C::PW, MT = PW / 16, KS = HD / 16, RB = C::RB, ROWS = NR * 8;
    constexpr bool QS = tr_q_shared(NR, QT);

    extern __shared__ __align__(1024) uint8_t sm_raw[];
    uint8_t *sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) unsigned long long bars[TR_WARPS][C::STAGES];
    uint2 *qsm = reinterpret_cast<uint2 *>(sm + tr_ring_bytes<HD, DT, NR>());  // QS: [KS][NR][QT][32]
    float *fs = reinterpret_cast<float *>(qsm + KS * NR * QT * 32);             // QS: fr of all rows

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gid = lane >> 2, c4 = lane & 3;
    const int nkv = a.c.pg.n_kv;
    const int split = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
    const int total_rows = a.T * a.rep;
    pdl_launch_dependents();  // the join's blocks wait for this kernel's end

    // ---- q: rows nr*8 + gid, the dims of this lane, as they come; with QS a warp has one nr
    constexpr int NQ = QS ? 1 : NR, QW = BF16 ? HD / 8 : HD / 4;
    static_assert(!QS || NR <= TR_WARPS, "a warp per eight rows");
    uint32_t raw[NQ][QW];
#pragma unroll
    for (int k = 0; k < NQ; k++) {
        const int row = (QS ? warp : k) * 8 + gid, r = row < total_rows ? row : 0;  // rows past the last: zeroed below
        const int t = r / a.rep, h = r - t * a.rep;
        const size_t o = (size_t)((size_t)b * a.T + t) * a.ldq + (size_t)(g * a.rep + h) * HD;
        constexpr int RUN = DT == SB_KV_I8 ? 16 : 8;  // consecutive dims of a lane
        constexpr int E = BF16 ? 8 : 4;               // elements of a 16-byte load
#pragma unroll
        for (int j = 0; j < HD / (4 * RUN); j++)
#pragma unroll
            for (int e = 0; e < RUN; e += E) {
                const size_t d = o + j * 4 * RUN + c4 * RUN + e;
                const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.q) + d * (BF16 ? 2 : 4));
                const int at = (j * RUN + e) * 4 / E;
                raw[k][at] = v.x, raw[k][at + 1] = v.y, raw[k][at + 2] = v.z, raw[k][at + 3] = v.w;
            }
    }

    const int cap = a.c.pg.max_pages * a.c.pg.page_size;
    const int ctx = min(max(a.ctx_len[b], 0), cap);
    auto tokens = [&]() { return a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T; };  // (read where it is needed: a register less)
    const int len = ctx + min(tokens(), cap - ctx);
    const int ntiles = (len + PW - 1) / PW;
    const int per = (ntiles + a.n_splits - 1) / a.n_splits;
    const int t0 = min(split * per, ntiles) + warp, t1 = min(min(split * per, ntiles) + per, ntiles);

    uint8_t *ring = sm + (size_t)warp * C::STAGES * C::STAGE;
    float *scales = reinterpret_cast<float *>(sm + (size_t)TR_WARPS * C::STAGES * C::STAGE + (size_t)warp * C::STAGES * C::SCALES);
    const uint32_t bar = smem_u32(bars[warp]);
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < C::STAGES; s++) mbar_init(bar + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const int br = a.box_rows, bs = br ? __ffs(br) - 1 : 0;  // a power of two
    // the cache row of position `lane` of tile t, or with boxes that of its lane-th box; read a tile ahead
    auto row_of = [&](int t) {
        const int p = t * PW + (br ? lane * br : lane);
        return lane < PW && p < len ? kv_row(a.c.pg, b, g, p) : -1ll;
    };
    // What lies behind the sequence's end is not copied: nobody sees it.  Rows on no page read as zeros.
    auto issue = [&](int t, int st, long long row) {
        uint8_t *ks = ring + st * C::STAGE, *vs = ks + C::TILE;
        const int p0 = t * PW, cnt = min(PW, len - p0);
        if (br) {
            const int boxes = (cnt + br - 1) / br;
            const unsigned good = __ballot_sync(0xffffffffu, row >= 0) & ((1u << boxes) - 1);
            if (good != (1u << boxes) - 1) {
                for (int i = 0; i < boxes; i++)
                    if (!((good >> i) & 1))
                        for (int e = lane; e < br * C::CPR; e += 32) {
                            const int at = tr_at<RB, PW>(i * br + e / C::CPR, e % C::CPR);
                            *reinterpret_cast<uint4 *>(ks + at) = make_uint4(0, 0, 0, 0);
                            *reinterpret_cast<uint4 *>(vs + at) = make_uint4(0, 0, 0, 0);
                        }
                fence_proxy_async_smem();  // a later box may take the place
                __syncwarp();
            }
            if (lane == 0) mbar_expect_tx(bar + 8 * st, __popc(good) * br * 2 * RB);
            __syncwarp();
            if ((good >> lane) & 1) {
#pragma unroll
                for (int h = 0; h < (RB == 256 ? 2 : 1); h++) {
                    const int at = h * PW * 128 + lane * br * (RB == 64 ? 64 : 128);
                    tma_box(smem_u32(ks + at), &a.tmk, h * 64, (int)row, bar + 8 * st);
                    tma_box(smem_u32(vs + at), &a.tmv, h * 64, (int)row, bar + 8 * st);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < PW * C::CPR / 32; i++) {
                const int ch = i * 32 + lane, r = ch / C::CPR, col = ch % C::CPR;
                const long long x = __shfl_sync(0xffffffffu, row, r);
                const size_t off = x < 0 ? 0 : (size_t)x * RB + col * 16;
                const int n = x < 0 ? 0 : 16;
                cp_async16_fill(smem_u32(ks + tr_at<RB, PW>(r, col)), static_cast<const char *>(a.c.k) + off, n);
                cp_async16_fill(smem_u32(vs + tr_at<RB, PW>(r, col)), static_cast<const char *>(a.c.v) + off, n);
            }
        }
        if (DT == SB_KV_I8) {
            const long long first = __shfl_sync(0xffffffffu, row, lane >> bs);
            const long long x = first < 0 || lane >= cnt ? -1 : first + (lane & ((1 << bs) - 1));
            const size_t off = x < 0 ? 0 : (size_t)x;
            const int n = x < 0 ? 0 : 4;
            cp_async4_fill(smem_u32(scales + st * 2 * PW + lane), a.c.ks + off, n);
            cp_async4_fill(smem_u32(scales + st * 2 * PW + PW + lane), a.c.vs + off, n);
        }
    };
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; s++) {
        if (t0 + s * TR_WARPS < t1) issue(t0 + s * TR_WARPS, s, row_of(t0 + s * TR_WARPS));
        cp_commit();
    }
    long long ahead = row_of(t0 + (C::STAGES - 1) * TR_WARPS);

    // fragments b0, b1 of every k step (k step s of a K chunk: dims first + 4s + {0,1} and + {2,3} of the lane's run)
    uint2 qf[QS ? 1 : KS * NR * QT];
    float fr[NR][2];  // scores of rows 2*c4 and 2*c4+1 in powers of two
    if (!QS || warp < NR) {
#pragma unroll
        for (int k = 0; k < NQ; k++) {
            const int nr = QS ? warp : k;
            const bool in = nr * 8 + gid < total_rows;
            float x[HD / 4];
#pragma unroll
            for (int e = 0; e < HD / 4; e++) {
                const uint32_t w = raw[k][BF16 ? e / 2 : e];
                x[e] = !in ? 0.0f : __uint_as_float(!BF16 ? w : e & 1 ? w & 0xffff0000u : w << 16);
            }
            float scale = 1.0f, f = LOG2E;
            if (DT == SB_KV_I8) row_exponent(x, scale, f);
            if (QS) {
                if (c4 == 0) fs[nr * 8 + gid] = f;
            } else {  // rows 2*c4 and 2*c4+1 are those of the lanes with that gid
                fr[k][0] = __shfl_sync(0xffffffffu, f, 8 * c4), fr[k][1] = __shfl_sync(0xffffffffu, f, 8 * c4 + 4);
            }
#pragma unroll
            for (int s = 0; s < KS; s++) {
                uint32_t u[QT], w[QT];
                if (DT == SB_KV_I8) {
                    split_f16x2<QT>(x[4 * s] * scale, x[4 * s + 1] * scale, u);
                    split_f16x2<QT>(x[4 * s + 2] * scale, x[4 * s + 3] * scale, w);
                } else {
                    split_bf16x2<QT>(x[4 * s], x[4 * s + 1], u);
                    split_bf16x2<QT>(x[4 * s + 2], x[4 * s + 3], w);
                }
#pragma unroll
                for (int q = 0; q < QT; q++) {
                    if (QS) qsm[((s * NR + nr) * QT + q) * 32 + lane] = make_uint2(u[q], w[q]);
                    else qf[QS ? 0 : (s * NR + k) * QT + q] = make_uint2(u[q], w[q]);
                }
            }
        }
    }
    if (QS) {
        __syncthreads();
#pragma unroll
        for (int nr = 0; nr < NR; nr++) fr[nr][0] = fs[nr * 8 + 2 * c4], fr[nr][1] = fs[nr * 8 + 2 * c4 + 1];
    }

    float o[HD / 16][NR][4];
    float m[NR][2], l[NR][2], wlim[NR][2], kw[NR][2];
#pragma unroll
    for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int nr = 0; nr < NR; nr++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][nr][e] = 0.0f;
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
        for (int e = 0; e < 2; e++) m[nr][e] = -INFINITY, l[nr][e] = 0.0f, wlim[nr][e] = 0.0f, kw[nr][e] = 0.0f;

    int st = 0;
    uint32_t phase = 0;
    bool ok = true;  // a wait that gives up (2 s) ends the later ones of its warp
    for (int t = t0; t < t1; t += TR_WARPS) {
        cp_wait<C::STAGES - 2>();
        if (br && ok) ok = __all_sync(0xffffffffu, mbar_wait_long(bar + 8 * st, phase));
        __syncwarp();
        {
            const int nt = t + (C::STAGES - 1) * TR_WARPS, ns = st == 0 ? C::STAGES - 1 : st - 1;
            if (nt < t1) issue(nt, ns, ahead);
            cp_commit();
            ahead = row_of(nt + TR_WARPS);
        }
        const uint8_t *kt = ring + st * C::STAGE;
        uint8_t *vt = ring + st * C::STAGE + C::TILE;
        const float *sck = scales + st * 2 * PW, *scv = sck + PW;
        st = st + 1 == C::STAGES ? 0 : st + 1;
        if (st == 0) phase ^= 1;

        // ---- S^T = K q^T: s[mt][nr][e]: position mt*16 + pg + 8*(e>>1), row nr*8 + 2*c4 + (e&1)
        const int pg = tr_position<RB>(gid);
        float s[MT][NR][4];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[mt][nr][e] = 0.0f;
            const int ra = mt * 16 + pg;
            constexpr int GS = DT == SB_KV_I8 ? 4 : 2;  // k steps of a 16-byte chunk
#pragma unroll
            for (int j = 0; j < KS / GS; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(kt + tr_at<RB, PW>(ra, 4 * j + c4));
                const uint4 y = *reinterpret_cast<const uint4 *>(kt + tr_at<RB, PW>(ra + 8, 4 * j + c4));
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < GS; i++) {
                    uint32_t af[4];
                    if (DT == SB_KV_I8) {
                        const uint32_t u = xw[i] ^ 0x80808080u, v = yw[i] ^ 0x80808080u;
                        af[0] = code2_f16(u, 0x4140), af[2] = code2_f16(u, 0x4342);
                        af[1] = code2_f16(v, 0x4140), af[3] = code2_f16(v, 0x4342);
                    } else {
                        af[0] = xw[2 * i], af[2] = xw[2 * i + 1], af[1] = yw[2 * i], af[3] = yw[2 * i + 1];
                    }
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int q = 0; q < QT; q++) {
                            const int at = ((j * GS + i) * NR + nr) * QT + q;
                            const uint2 f = QS ? qsm[at * 32 + lane] : qf[QS ? 0 : at];
                            mma16<DT>(s[mt][nr], af, f.x, f.y);
                        }
                }
            }
        }

        // ---- scores in powers of two; what a row does not see is -inf
        const int base = t * PW;
        const bool tail = base + PW > ctx;
        bool up = false;
        float sk[MT][2], sv[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                sk[mt][h] = DT == SB_KV_I8 ? sck[mt * 16 + h * 8 + pg] : 1.0f;
                sv[mt][h] = DT == SB_KV_I8 ? scv[mt * 16 + h * 8 + pg] : 1.0f;
            }
        unsigned seen[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; nr++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                seen[nr][e] = ~0u;
                if (tail) {
                    const int r = nr * 8 + 2 * c4 + e;
                    const int i = r < total_rows && r / a.rep < tokens() ? r / a.rep : -1;
                    seen[nr][e] = (unsigned)visible_bits(a, b, i, ctx, len - ctx, base);
                }
            }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float &x = s[mt][nr][e];
                    x *= DT == SB_KV_I8 ? fr[nr][e & 1] * sk[mt][e >> 1] : LOG2E;
                    if (tail && !((seen[nr][e & 1] >> (mt * 16 + (e >> 1) * 8 + pg)) & 1)) x = -INFINITY;
                    up |= x > m[nr][e & 1] + 8.0f;
                }
        float alpha[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) alpha[nr][0] = alpha[nr][1] = 1.0f;
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = m[nr][e];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) x = fmaxf(x, fmaxf(s[mt][nr][e], s[mt][nr][2 + e]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    // a row whose own scores are in range keeps its reference, whatever the warp's other rows see
                    if (x > m[nr][e] + 8.0f) {
                        const float down = m[nr][e] - x;  // -inf at first
                        alpha[nr][e] = ex2(down);
                        l[nr][e] *= alpha[nr][e];
                        m[nr][e] = x;
                        if (DT == SB_KV_I8 && wlim[nr][e] > 0.0f) {
                            // the weights so far have shrunk, and the largest of them (kw below) with them: kw rises as far
                            // (clamped as below), so that a large v_scale which has lost its weight takes no bits from others
                            const int ex = (int)(__float_as_uint(wlim[nr][e]) >> 23) - 8;
                            const int lower = min((int)fminf(-down, 256.0f), max(ex - 16, 0));
                            wlim[nr][e] = __uint_as_float((uint32_t)(ex - lower + 8) << 23);
                            kw[nr][e] = __uint_as_float((uint32_t)(254 - (ex - lower) + 7) << 23);
                            alpha[nr][e] = ex2(down + (float)lower);
                        }
                    }
                }
        }
        bool over = false;
#pragma unroll
        for (int nr = 0; nr < NR; nr++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float z = m[nr][e] == -INFINITY ? 0.0f : m[nr][e];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float &x = s[mt][nr][2 * h + e];
                        x = ex2(x - z);
                        l[nr][e] += x;
                        if (DT == SB_KV_I8) {
                            // a row that does not see a position takes nothing from its scale either
                            x = !tail || ((seen[nr][e] >> (mt * 16 + h * 8 + pg)) & 1) ? x * sv[mt][h] : 0.0f;
                            over |= fabsf(x) > wlim[nr][e];
                        }
                    }
            }
        if (DT == SB_KV_I8) {
            // p * v_scale times a power of two kw: at most 2^15, at least 2^7 for the largest when kw was chosen
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nr = 0; nr < NR; nr++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = 0.0f;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) x = fmaxf(x, fmaxf(fabsf(s[mt][nr][e]), fabsf(s[mt][nr][2 + e])));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        if (x > wlim[nr][e]) {
                            const int ex = min(max((int)(__float_as_uint(x) >> 23), 16), 240);  // biased exponent
                            const float k = __uint_as_float((uint32_t)(254 - ex + 7) << 23);
                            alpha[nr][e] *= kw[nr][e] > 0.0f ? k / kw[nr][e] : 0.0f;
                            kw[nr][e] = k;
                            wlim[nr][e] = __uint_as_float((uint32_t)(ex + 8) << 23);
                        }
                    }
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nr = 0; nr < NR; nr++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[mt][nr][e] *= kw[nr][e & 1];
        }

        // ---- a non-finite V element of a drafted row must not reach rows that do not see it (0 * inf): when a tail
        // tile holds any, their products go one by one under the mask and zeros take their place below
        if (DT != SB_KV_I8 && tail) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < PW * C::CPR / 32; i++) {
                const uint4 w = *reinterpret_cast<const uint4 *>(vt + (i * 32 + lane) * 16);
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) bad |= (x[e] & 0x7f800000u) == 0x7f800000u || (x[e] & 0x7f80u) == 0x7f80u;
            }
            if (__any_sync(0xffffffffu, bad)) {
                for (int pos = 0; pos < PW; pos++) {
                    const int src = tr_index<RB>(pos & 7) * 4 + c4;
                    float p[NR][2];
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            p[nr][e] = 0.0f;
#pragma unroll
                            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    const float y = __shfl_sync(0xffffffffu, s[mt][nr][2 * h + e], src);
                                    if (pos >> 3 == mt * 2 + h) p[nr][e] = y;
                                }
                        }
#pragma unroll
                    for (int i = 0; i < HD / 16; i++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int d = tr_dim<HD, DT>(i >> 2, gid) + 2 * (i & 3) + h;
                            const float x = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(vt + tr_at<RB, PW>(pos, d >> 3) + (d & 7) * 2));
                            if (isfinite(x)) continue;
#pragma unroll
                            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                                for (int e = 0; e < 2; e++)
                                    if ((seen[nr][e] >> pos) & 1) {
                                        o[i][nr][2 * h + e] = fmaf(p[nr][e], x, o[i][nr][2 * h + e]);
                                        alpha[nr][e] = alpha[nr][e] > 0.0f ? alpha[nr][e] : 1.0f;
                                    }
                        }
                }
                __syncwarp();
                for (int i = lane; i < PW * HD; i += 32) {
                    uint16_t *p = reinterpret_cast<uint16_t *>(vt) + i;
                    if ((*p & 0x7f80) == 0x7f80) *p = 0;
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
        }

        // ---- O^T = O^T * alpha + V^T p^T; the tile's products start from zero (the tensor cores truncate as they
        // accumulate, which over a long context would add up)
        uint2 pf[MT][NR][PT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nr = 0; nr < NR; nr++) {
                uint32_t u[PT], w[PT];
                if (DT == SB_KV_I8) split_f16x2<PT>(s[mt][nr][0], s[mt][nr][1], u), split_f16x2<PT>(s[mt][nr][2], s[mt][nr][3], w);
                else split_bf16x2<PT>(s[mt][nr][0], s[mt][nr][1], u), split_bf16x2<PT>(s[mt][nr][2], s[mt][nr][3], w);
#pragma unroll
                for (int q = 0; q < PT; q++) pf[mt][nr][q] = make_uint2(transpose8x8(u[q]), transpose8x8(w[q]));
            }
#pragma unroll
        for (int md = 0; md < HD / 64; md++) {
            uint32_t av[MT][4][4];  // [k step][16-dim tile][fragment]: tile i: dims tr_dim(md, gid) + 2i, + 2i+1
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const int r = mt * 16;  // k index 2*c4 (+1, +8, +9) is this position:
                const int ra = r + tr_position<RB>(2 * c4), rb = r + tr_position<RB>(2 * c4 + 1), ch = tr_chunk<HD, DT>(md, gid);
                if (DT == SB_KV_I8) {
                    const int hi = (gid & 1) * 8;
                    uint2 w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        w[k] = *reinterpret_cast<const uint2 *>(vt + tr_at<RB, PW>((k & 1 ? rb : ra) + (k >> 1) * 8, ch) + hi);
                        w[k].x ^= 0x80808080u, w[k].y ^= 0x80808080u;
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t w0 = h ? w[0].y : w[0].x, w1 = h ? w[1].y : w[1].x, w2 = h ? w[2].y : w[2].x, w3 = h ? w[3].y : w[3].x;
                        const uint32_t x01 = __byte_perm(w0, w1, 0x5140), x23 = __byte_perm(w0, w1, 0x7362);
                        const uint32_t y01 = __byte_perm(w2, w3, 0x5140), y23 = __byte_perm(w2, w3, 0x7362);
                        av[mt][2 * h][0] = code2_f16(x01, 0x4140), av[mt][2 * h][1] = code2_f16(x01, 0x4342);
                        av[mt][2 * h + 1][0] = code2_f16(x23, 0x4140), av[mt][2 * h + 1][1] = code2_f16(x23, 0x4342);
                        av[mt][2 * h][2] = code2_f16(y01, 0x4140), av[mt][2 * h][3] = code2_f16(y01, 0x4342);
                        av[mt][2 * h + 1][2] = code2_f16(y23, 0x4140), av[mt][2 * h + 1][3] = code2_f16(y23, 0x4342);
                    }
                } else {
                    uint4 w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        w[k] = *reinterpret_cast<const uint4 *>(vt + tr_at<RB, PW>((k & 1 ? rb : ra) + (k >> 1) * 8, ch));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t w0 = (&w[0].x)[i], w1 = (&w[1].x)[i], w2 = (&w[2].x)[i], w3 = (&w[3].x)[i];
                        av[mt][i][0] = __byte_perm(w0, w1, 0x5410), av[mt][i][1] = __byte_perm(w0, w1, 0x7632);
                        av[mt][i][2] = __byte_perm(w2, w3, 0x5410), av[mt][i][3] = __byte_perm(w2, w3, 0x7632);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int q = 0; q < PT; q++) mma16<DT>(d, av[mt][i], pf[mt][nr][q].x, pf[mt][nr][q].y);
                    float(&x)[4] = o[md * 4 + i][nr];
                    x[0] = fmaf(x[0], alpha[nr][0], d[0]), x[1] = fmaf(x[1], alpha[nr][1], d[1]);
                    x[2] = fmaf(x[2], alpha[nr][0], d[2]), x[3] = fmaf(x[3], alpha[nr][1], d[3]);
                }
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    if (!ok && lane == 0) wait_failed(a.errors, WAIT_TREE_ROWS);
    __syncthreads();

    // ---- O in units of exp(-m), whole sums; the warps' shares, then the splits, joined in order
    float *red = reinterpret_cast<float *>(sm);  // [warps][ROWS][HD]
    float *rm = red + TR_WARPS * ROWS * HD, *rl = rm + TR_WARPS * ROWS;
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float x = l[nr][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            const int r = warp * ROWS + nr * 8 + 2 * c4 + e;
            if (gid == 0) rm[r] = m[nr][e], rl[r] = x;
            const float k = DT == SB_KV_I8 ? (kw[nr][e] > 0.0f ? 1.0f / kw[nr][e] : 0.0f) : 1.0f;
#pragma unroll
            for (int i = 0; i < HD / 16; i++)
                *reinterpret_cast<float2 *>(red + (size_t)r * HD + tr_dim<HD, DT>(i >> 2, gid) + 2 * (i & 3)) =
                    make_float2(o[i][nr][e] * k, o[i][nr][2 + e] * k);
        }
    __syncthreads();
    const size_t tile = (size_t)b * nkv + g;
    tree_finish<HD, BF16, TR_WARPS, ROWS, TR_THREADS>(a, red, rm, rl, min(ROWS, total_rows), 0, b, g, tokens(), split, tile);
}

template <int HD, int DT, bool BF16, int NR>
int tr_inst(const TreeAttnArgs &a, cudaStream_t st) {
    constexpr int QT = BF16 ? 1 : DT == SB_KV_BF16 ? 3 : 2;
    auto kern = tree_attn_rows_kernel<HD, DT, BF16, NR>;
    static int limit[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!limit[dev & 63]) SB_TRY(allow_max_dynamic_smem(kern, &limit[dev & 63]));
    constexpr size_t smem = 1024 + tr_ring_bytes<HD, DT, NR>() + (tr_q_shared(NR, QT) ? (size_t)(HD / 16) * NR * QT * 256 + NR * 32 : 0);
    SB_CHECK(smem <= (size_t)limit[dev & 63], SB_ERR_SHAPE, "tree attention: needs %zu B shared memory (limit %d)", smem,
             limit[dev & 63]);
    SB_CUDA_TRY(launch(kern, dim3(a.n_splits, a.c.pg.n_kv, a.B), dim3(tr_warps(NR) * 32), smem, st, false, a));
    return SB_OK;
}
template <int HD, int DT, bool BF16>
int tr_rows(const TreeAttnArgs &a, cudaStream_t st) {
    const int rows = a.T * a.rep;
    return rows <= 8 ? tr_inst<HD, DT, BF16, 1>(a, st) : rows <= 16 ? tr_inst<HD, DT, BF16, 2>(a, st) : tr_inst<HD, DT, BF16, 4>(a, st);
}
template <int HD>
int tr_dt(const TreeAttnArgs &a, cudaStream_t st) {
    if (a.c.dtype == SB_KV_I8) return a.bf16 ? tr_rows<HD, SB_KV_I8, true>(a, st) : tr_rows<HD, SB_KV_I8, false>(a, st);
    return a.bf16 ? tr_rows<HD, SB_KV_BF16, true>(a, st) : tr_rows<HD, SB_KV_BF16, false>(a, st);
}

}  // namespace

bool tree_attn_rows_wanted(const TreeAttnArgs &a) { return a.c.dtype != SB_KV_F32 && a.T * a.rep <= 32; }

TreeAttnPlan tree_attn_rows_plan(const TreeAttnArgs &a, int max_len) {
    TreeAttnPlan p;
    const int rows = a.T * a.rep;
    p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    const int pw = a.c.dtype == SB_KV_I8 ? 32 : 16;
    const long long base = (long long)a.B * a.c.pg.n_kv;
    p.n_splits = tree_splits(base, ceil_div(std::max(max_len, 1), pw * tr_warps(p.rows / 8)), 2);
    return p;
}

int tree_attn_rows_launch(const TreeAttnArgs &in, cudaStream_t st) {
    TreeAttnArgs a = in;
    SB_TRY(tree_tensor_maps(a, a.c.dtype == SB_KV_I8 ? 32 : 16));
    return a.c.hd == 128 ? tr_dt<128>(a, st) : tr_dt<64>(a, st);
}

}  // namespace sb
