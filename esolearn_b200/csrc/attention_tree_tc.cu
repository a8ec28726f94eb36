// Tree attention for many query rows per kv head (T * rep > 32: large trees,
// prompts behind a cached prefix) over a bf16 or int8 cache, on the tcgen05
// tensor cores.  What it computes is described in attention_tree.cu.
//
// A CTA takes 128 query rows of one kv head and a run of 128-position tiles.
// Per tile S = q K^T and O = p V are two 128 x 128 products whose operands are
// sums of 16-bit terms, accumulated in TMEM:
//   int8 cache: the codes as exact f16; q (over a power of two of its row's
//     magnitude) as two f16 terms (one when q is bf16); k_scale multiplies the
//     scores; p * v_scale, over a power of two of the largest that the row sees,
//     as two f16 terms;
//   bf16 cache: K and V as they are, q and p as three bf16 terms (one and two
//     when q is bf16).
// Each tile's O starts from zero and is added to the row's sums in registers in
// f32: the tensor cores truncate as they accumulate.
//
// Roles (16 warps, one CTA per SM; registers are moved to where they are needed):
//   warps 0-7: softmax.  Thread = (row, half of the tile's columns).  Reads its
//     64 scores from TMEM, agrees with the thread of the other half on the row's
//     reference maximum (a whole power of two, which serves until a score exceeds
//     it by 2^8), and writes p's terms over the scores as the A operand of the
//     second product.
//   warps 8-11: sums.  Thread = row; adds each tile's O to the row's sums.  int8:
//     also turn V's codes into f16.
//   warps 12-14: loaders.  int8: bulk copies of K's codes, turned into f16, and
//     the scales; bf16: TMA boxes (pages of a multiple of eight positions).
//   warp 15: one thread issues the products: q K^T of tile t before p V of tile
//     t-1, so the first runs under the softmax of t-1.
// TMEM: three score tiles (p over them) and O; two where p has three terms (bf16
// cache, f32 q); two, q and O where shared memory has no room for q (int8 cache,
// f32 q, head_dim 128).
//
// Shared-memory operands use the 128-byte swizzle: rows of 64 16-bit elements
// (128 bytes, of 128 rows; head_dim 128 is two such blocks), piece c of row r
// at c ^ (r % 8).  That is K-major for q and K (along hd) and MN-major for V
// (along positions), so all rows are copied as they come, whole 128-byte lines
// at a time: a copy that scatters a line over several (the unswizzled core
// matrices) took 39 clocks per warp instruction.
//
// A tile's products take 1536 clocks (bf16 cache, bf16 q) or 2048 (int8, f32 q: its
// 10,600 warp instructions also take 2700 issue slots per scheduler), yet it takes
// 4000 and 5000: the chain scores - softmax - p V - sums of a tile, of which too
// little runs under the next one's, and the shared schedulers bound it (tensor cores
// 45 % and 31 % busy, issue slots 43 % and 45 %).  Looking pages and scales up a tile
// further ahead cost 10 %: more instructions.  512 tokens behind 8192, 8 kv heads of
// 4, bf16: 136 to 144 us (490 TFLOP/s, each product counted once), with f32 q 201 to
// 221; 32 tokens x 8 sequences up to 4096, 8 kv heads of 8, int8, f32 q: 113 to 125 us
// (290 TFLOP/s).
#include "attention_tree.cuh"

#include <algorithm>
#include <type_traits>

#include "attention_tree_dev.cuh"
#include "clock_pace.cuh"
#include "tcgen05.cuh"

namespace sb {

namespace {

constexpr int TT_THREADS = 512, TT_ROWS = 128, TT_TILE = 128;
constexpr int TT_SOFTMAX_WARPS = 8, TT_LOADERS = 3, TT_LOAD0 = 12, TT_MMA = 15;
// Registers of a thread, 128 at launch: 2 * softmax + sums + (loaders and products) = 4 * 128.  What they save is
// spills, and which role gains from more differs: 512 tokens behind 8192, bf16 cache and q, take 140 to 150 us with 144,
// 152 and 72 and 139 with 152, 152 and 56, which leaves a bf16 cache with f32 q as it is (214 both); 256 rows x 8
// sequences at 2000, 8 kv heads, int8, take 68.7 us with 144, 152 and 72 and 68.1 with 144, 160 and 64.
constexpr int tt_regs_softmax(int dt, bool bf16) { return dt != SB_KV_I8 && bf16 ? 152 : 144; }
constexpr int tt_regs_sums(int dt) { return dt == SB_KV_I8 ? 160 : 152; }
constexpr int tt_regs_rest(int dt, bool bf16) { return 4 * 128 - 2 * tt_regs_softmax(dt, bf16) - tt_regs_sums(dt); }
constexpr int TT_GROUPS = (16 + TT_LOADERS - 1) / TT_LOADERS;  // groups of eight positions of a tile that a loader has
constexpr int TT_SCALES = 4;  // tiles whose scales are kept
// p * v_scale * 2^kw, the weights' f16 terms, is below 2^TT_KW when kw is chosen and at most 2^TT_KW_MAX while it serves.
constexpr float TT_KW = 7.0f, TT_KW_MAX = 14.0f;

template <int HD, int DT, bool BF16>
struct TtShape {
    // terms of q and of p: f32's accuracy with an f32 q (bf16 terms hold 8 bits each, f16 terms 11); where q and the output
    // are bf16, p's two bf16 terms leave 2^-18, well below the output's rounding
    static constexpr int QT = BF16 ? 1 : DT == SB_KV_BF16 ? 3 : 2;
    static constexpr int PT = DT == SB_KV_BF16 && !BF16 ? 3 : 2;
    // q in TMEM where shared memory has no room for it; TMEM then has room for two score tiles instead of three, as it has where p has three terms
    static constexpr bool QTMEM = DT == SB_KV_I8 && !BF16 && HD == 128;
    static constexpr int NSB = QTMEM || PT == 3 ? 2 : 3;
    static constexpr int T_S = PT * 64;             // TMEM columns of a score tile, 128, and of p's terms, which take its place
    static constexpr int NS = 2;                    // stages of K and of V
    static constexpr int T_Q = 256, T_O = 384;      // TMEM columns; scores from 0
    static constexpr int MAT = 128 * HD * 2;        // bytes of a 128-row 16-bit tile
    static constexpr int STAGE = 2 * MAT;           // V then K
    static constexpr int Q_OFF = NS * STAGE;
    // int8: codes as they come: two runs (tiles) for every loader's groups of K, one for every sums warp's of V
    static constexpr int RAWK = TT_GROUPS * 8 * HD, RAWV = 4 * 8 * HD;
    static constexpr int RAW_OFF = Q_OFF + (QTMEM ? 0 : QT * MAT);
    static constexpr int SC_OFF = RAW_OFF + (DT == SB_KV_I8 ? TT_LOADERS * 2 * RAWK + 4 * RAWV : 0);  // int8: [TT_SCALES][k scale, v scale, log2 v scale][128]
    static constexpr int SC_BYTES = DT == SB_KV_I8 ? TT_SCALES * 3 * 128 * 4 : 0;
    static constexpr int EX_OFF = SC_OFF + SC_BYTES;  // [2][2][128]: row maxima of the halves; int8: of log2(p * v_scale) too
    static constexpr int AL_OFF = EX_OFF + 2 * 2 * 128 * (DT == SB_KV_I8 ? 8 : 4);  // [4][128] bytes: log2 of the sums' rescaling
    static constexpr int BAR_OFF = AL_OFF + 4 * 128;
    static constexpr int BYTES = BAR_OFF + 448;
    static constexpr int JOIN = 128 * (HD + 2) * 4;  // the row sums at the end, over the stages and q
    static_assert(NSB * T_S <= (QTMEM ? T_Q : T_O), "TMEM columns");
    static_assert(JOIN <= SC_OFF, "the row sums must fit the tiles");
    static_assert(RAWK % 128 == 0 && RAWV % 128 == 0, "bulk copies");
};

// Shared-memory descriptor of a 128-byte-swizzled operand: groups of eight rows
// 1024 bytes apart (SBO), 64-element blocks `lbo` bytes apart (MN-major only).
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t lbo) {
    return umma_sdesc(addr, lbo, 1024) | ((uint64_t)2 << 61);
}
// Byte offset of 16-byte piece c (of 8 elements) of row r of a [128][hd] tile.
__device__ __forceinline__ int sw128(int r, int c) { return (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

// Instruction descriptor of kind::f16: f32 accumulator, A and B of the same
// 16-bit type, M = 128, N = n; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t idesc_f16(int n, bool bf16, bool b_mn) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]),
          "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]),
          "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&r)[16]) { tmem_ld16(taddr, reinterpret_cast<uint32_t *>(&r[0])); }
// wait for this thread's tcgen05.ld; no use of the registers may move before it
template <int N>
__device__ __forceinline__ void tmem_ld_done(float (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+f"(r[i]));
}
// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// (x, y) as TERMS pairs of 16-bit terms
template <int DT, int TERMS>
__device__ __forceinline__ void split2(uint64_t v, uint32_t (&o)[TERMS]) {
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        const float2 x = unpack2(v);
        float2 h;
        if (DT == SB_KV_I8) {
            const __half2 p = __floats2half2_rn(x.x, x.y);
            o[t] = *reinterpret_cast<const uint32_t *>(&p);
            h = __half22float2(p);
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x.x, x.y);
            o[t] = *reinterpret_cast<const uint32_t *>(&p);
            h = make_float2(__uint_as_float(o[t] << 16), __uint_as_float(o[t] & 0xffff0000u));
        }
        if (t + 1 < TERMS) v = fma2(pack2(h.x, h.y), pack2(-1.0f, -1.0f), v);
    }
}
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

template <int HD, int DT, bool BF16>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_attn_tc_kernel(const __grid_constant__ TreeAttnArgs a) {
    using C = TtShape<HD, DT, BF16>;
    constexpr int QT = C::QT, MAT = C::MAT, NS = C::NS;
    extern __shared__ __align__(1024) uint8_t sm[];
    // (no static shared memory: the tiles start on a 1024-byte boundary and nearly fill the SM)
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(sm + C::BAR_OFF + 208);
    pdl_launch_dependents();  // the join's blocks wait for this kernel's end
    int *s_bad = reinterpret_cast<int *>(sm + C::BAR_OFF + 216);  // [2] bf16: a tail tile's V holds non-finite elements
    static_assert(C::NS == 2 && TT_LOADERS == 3 && TT_SCALES * 8 + 136 <= 208, "barriers and small words");

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nkv = a.c.pg.n_kv;
    const int split = blockIdx.x % a.n_splits, rt = blockIdx.x / a.n_splits;
    const int g = blockIdx.y, b = blockIdx.z;
    const int total_rows = a.T * a.rep, row0 = rt * TT_ROWS;

    const uint32_t base = smem_u32(sm);
    const uint32_t bars = base + C::BAR_OFF;
    const uint32_t s_full = bars, p_full = bars + 24, pv_done = bars + 48;  // [3]: of tile t at t % NSB
    const uint32_t k_full = bars + 72, v_full = bars + 88;  // [2]: at t % NS
    const uint32_t sc_full = bars + 136;  // [TT_SCALES]
    const uint32_t q_full = bars + 336;
    // [2]: V of tail tile t has landed, at t % NS.  One barrier for both stages would not do: a loader may lag a whole tile
    // behind the one that issues the copies, whose next phase would then hide the one that it waits for.
    const uint32_t tail_full = bars + 104;
    const uint32_t raw_k = bars + 352, raw_v = bars + 400;  // [TT_LOADERS][2], [4]
    if (tid == 0) {
        for (int i = 0; i < 3; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, TT_SOFTMAX_WARPS + 4);  // p of the tile is there, O of the tile before added
            mbar_init(pv_done + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, TT_LOADERS);
            mbar_init(v_full + 8 * i, DT == SB_KV_I8 ? 4 : TT_LOADERS);
            s_bad[i] = 0;
        }
        for (int i = 0; i < TT_SCALES; i++) mbar_init(sc_full + 8 * i, TT_LOADERS);
        mbar_init(q_full, TT_SOFTMAX_WARPS);
        for (int i = 0; i < 2; i++) mbar_init(tail_full + 8 * i, 1);
        for (int i = 0; i < 2 * TT_LOADERS; i++) mbar_init(raw_k + 8 * i, 1);
        for (int i = 0; i < 4; i++) mbar_init(raw_v + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TT_MMA) tmem_alloc(&s_tmem, 512);

    const int cap = a.c.pg.max_pages * a.c.pg.page_size;
    const int ctx = min(max(a.ctx_len[b], 0), cap);
    const int n_new = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
    const int n_vis = min(n_new, cap - ctx);  // tokens behind the table have no rows to be seen
    // the last token of these rows; under the j <= i rule nothing behind it is read
    const int last_i = min((min(row0 + TT_ROWS, total_rows) - 1) / a.rep, n_new - 1);
    const int len = (int)min((long long)cap, (long long)ctx + (a.mask ? n_new : last_i + 1));
    const int ntiles = (len + TT_TILE - 1) / TT_TILE;
    const int per = (ntiles + a.n_splits - 1) / a.n_splits;
    const int t0 = min(split * per, ntiles), nt = min(per, ntiles - t0);

    // ---- loaders: a warp has groups of eight positions of a tile (int8 scales and bf16 rows: lw, lw+3, ..; int8 codes: six
    // on end); the lanes of an instruction cover
    // whole rows
    constexpr int CPR = HD * (DT == SB_KV_I8 ? 1 : 2) / 16;  // 16-byte pieces of a cached row
    constexpr int LPI = 32 / CPR;                            // rows of an instruction
    constexpr int NI = 8 / LPI;                              // instructions of a group
    static_assert(TT_GROUPS <= 8, "a lane looks two rows up");
    const int lw = warp - TT_LOAD0, piece = lane % CPR, sub = lane / CPR;
    // this lane's look-up of a tile: position lane%8 of groups lane/8 and lane/8 + 4
    auto look_up = [&](int t) {
        int r[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int grp = lw + (h * 4 + (lane >> 3)) * TT_LOADERS, p = (t0 + t) * TT_TILE + grp * 8 + (lane & 7);
            r[h] = grp < 16 && t < nt && p < len ? (int)kv_row(a.c.pg, b, g, p) : -1;
        }
        return make_int2(r[0], r[1]);
    };
    // int8, bulk copies of n groups from `first` on of a tile to `dst`: as few as the pages allow where they hold a
    // multiple of eight positions (a warp's copies are issued one after the other, 200 clocks each), else row by row
    auto copy_codes = [&](const void *cache, int t, int first, int n, uint32_t dst, uint32_t bar) {
        const char *src = static_cast<const char *>(cache);
        if (a.c.pg.page_size % 8 == 0) {
            const int grp = first + lane, p = (t0 + t) * TT_TILE + grp * 8;
            const int row = lane < n && grp < 16 && p < len ? (int)kv_row(a.c.pg, b, g, p) : -1;
            const int before = __shfl_up_sync(0xffffffffu, row, 1);
            const bool lead = row >= 0 && (lane == 0 || before < 0 || row != before + 8);  // a run of groups begins here
            const unsigned who = __ballot_sync(0xffffffffu, row >= 0), leads = __ballot_sync(0xffffffffu, lead);
            if (lane == 0) mbar_expect_tx(bar, __popc(who) * 8 * HD);
            __syncwarp();
            if (lead) {  // (n < 32: a lane behind the run always ends it)
                const int groups = __ffs((leads | ~who) >> (lane + 1));
                tma_load_1d(dst + lane * 8 * HD, src + (size_t)row * HD, groups * 8 * HD, bar);
            }
        } else {
            int r[2], cnt = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int i = h * 4 + (lane >> 3), grp = first + i, p = (t0 + t) * TT_TILE + grp * 8 + (lane & 7);
                r[h] = i < n && grp < 16 && p < len ? (int)kv_row(a.c.pg, b, g, p) : -1;
                cnt += __popc(__ballot_sync(0xffffffffu, r[h] >= 0));
            }
            if (lane == 0) mbar_expect_tx(bar, cnt * HD);
            __syncwarp();
            if (r[0] >= 0) tma_load_1d(dst + lane * HD, src + (size_t)r[0] * HD, HD, bar);
            if (r[1] >= 0) tma_load_1d(dst + (32 + lane) * HD, src + (size_t)r[1] * HD, HD, bar);
        }
    };
    // and their conversion.  Eight lanes take two rows: of 128-byte rows the even one's first and the odd one's last 64
    // bytes, then the other halves, so that loads and both stores always hit eight different bank groups.
    auto put_codes = [&](const uint8_t *src, uint8_t *dst, int grp) {
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int odd = (lane >> 2) & 1, rr = (lane >> 3) * 2 + odd;
            const int pc = (lane & 3) + (NI == 2 ? ((odd ^ j) << 2) : 0);
            uint4 w = *reinterpret_cast<const uint4 *>(src + rr * HD + pc * 16);
            w.x ^= 0x80808080u, w.y ^= 0x80808080u, w.z ^= 0x80808080u, w.w ^= 0x80808080u;
            uint8_t *at = dst + (pc >> 2) * 16384 + (grp * 8 + rr) * 128;
            *reinterpret_cast<uint4 *>(at + ((((2 * pc) & 7) ^ rr) << 4)) =
                make_uint4(code2_f16(w.x, 0x4140), code2_f16(w.x, 0x4342), code2_f16(w.y, 0x4140), code2_f16(w.y, 0x4342));
            *reinterpret_cast<uint4 *>(at + ((((2 * pc + 1) & 7) ^ rr) << 4)) =
                make_uint4(code2_f16(w.z, 0x4140), code2_f16(w.z, 0x4342), code2_f16(w.w, 0x4140), code2_f16(w.w, 0x4342));
        }
    };
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // ---- q's terms to TMEM or shared memory
    const int quad = warp & 3, half = warp >> 2;  // (half: softmax warps)
    const int rl = quad * 32 + lane, row = row0 + rl;
    const bool in = row < total_rows;
    const int token = in ? row / a.rep : 0;
    const int iv = in && token < n_new ? token : -1;
    float f = LOG2E;
    float *ex = reinterpret_cast<float *>(sm + C::EX_OFF), *exw = ex + 512;
    signed char *al = reinterpret_cast<signed char *>(sm + C::AL_OFF);
    if (warp < TT_SOFTMAX_WARPS) {
        const size_t at = (size_t)((size_t)b * a.T + token) * a.ldq + (size_t)(g * a.rep + (in ? row - token * a.rep : 0)) * HD + half * (HD / 2);
        auto load8 = [&](int d, float (&x)[8]) {
            if (!in) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = 0.0f;
            } else if (BF16) {
                const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.q) + at + d);
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) x[2 * e] = __uint_as_float(u[e] << 16), x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
            } else {
                const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at + d);
                const float4 w = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at + d + 4);
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            }
        };
        float scale = 1.0f;
        if (DT == SB_KV_I8) {
            float m = 0.0f;
            for (int d = 0; d < HD / 2; d += 8) {
                float x[8];
                load8(d, x);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = fabsf(x[e]);
                    if (y < INFINITY) m = fmaxf(m, y);
                }
            }
            ex[half * 128 + rl] = m;
            pair_sync(1 + quad);
            m = fmaxf(m, ex[(half ^ 1) * 128 + rl]);
            pair_sync(1 + quad);
            const int e = min(max((int)(__float_as_uint(m) >> 23), 2), 252);
            scale = __uint_as_float((uint32_t)(254 - e) << 23);
            f = LOG2E * __uint_as_float((uint32_t)e << 23);
        }
        for (int d = 0; d < HD / 2; d += 16) {
            uint32_t u[QT][8];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float x[8];
                load8(d + 8 * e, x);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t w[QT];
                    if (DT == SB_KV_I8) split_f16x2<QT>(x[2 * i] * scale, x[2 * i + 1] * scale, w);
                    else split_bf16x2<QT>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
                    for (int q = 0; q < QT; q++) u[q][4 * e + i] = w[q];
                }
            }
            const int dim = half * (HD / 2) + d;
#pragma unroll
            for (int q = 0; q < QT; q++) {
                if (C::QTMEM) {
                    tmem_st8(tmem + ((uint32_t)(quad * 32) << 16) + C::T_Q + q * (HD / 2) + dim / 2, u[q]);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        *reinterpret_cast<uint4 *>(sm + C::Q_OFF + q * MAT + sw128(rl, dim / 8 + e)) =
                            make_uint4(u[q][4 * e], u[q][4 * e + 1], u[q][4 * e + 2], u[q][4 * e + 3]);
                }
            }
        }
        if (C::QTMEM) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
    }

    float m = -INFINITY, l = 0.0f, kw = 0.0f;  // softmax: weights are 2^(score - m + kw), m and kw whole
    // A wait that gives up (2 s) ends all later ones of its warp; the warps still go through their loops, so that no
    // barrier between warps is left waiting.
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_long(bar, parity));
    };
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    float *red = reinterpret_cast<float *>(sm), *rm = red + 128 * HD, *rs = rm + 128;

    if (warp < TT_SOFTMAX_WARPS) {
        // =================================================== softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(tt_regs_softmax(DT, BF16)));
        for (int t = 0; t < nt; t++) {
            const int buf = t & 1;
            const int sb = t % C::NSB;
            const uint32_t S = tmem + lanes + sb * C::T_S;
            const int pos0 = (t0 + t) * TT_TILE + half * 64;
            const bool tail = pos0 + 64 > ctx;
            unsigned long long vis = ~0ull;
            if (tail) vis = visible_bits(a, b, iv, ctx, n_vis, pos0);
            if (DT == SB_KV_I8) wait(sc_full + 8 * (t % TT_SCALES), (t / TT_SCALES) & 1);
            wait(s_full + 8 * sb, (t / C::NSB) & 1);
            tc_fence_after();
            uint64_t s[32];  // pairs of scores
            {
                float x[2][32];
                tmem_ld32(S + half * 64, x[0]);
                tmem_ld32(S + half * 64 + 32, x[1]);
                tmem_ld_done(x[0]);
                tmem_ld_done(x[1]);
#pragma unroll
                for (int j = 0; j < 32; j++) s[j] = pack2(x[j >> 4][(j & 15) * 2], x[j >> 4][(j & 15) * 2 + 1]);
            }
            const float *sc = reinterpret_cast<const float *>(sm + C::SC_OFF) + (t % TT_SCALES) * 384 + half * 64;
            if (DT == SB_KV_I8) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const ulonglong2 k4 = *reinterpret_cast<const ulonglong2 *>(sc + 2 * j);
                    s[j] = mul2(s[j], k4.x), s[j + 1] = mul2(s[j + 1], k4.y);
                }
            }
            if (tail) {
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    float2 x = unpack2(s[j]);
                    if (!((vis >> (2 * j)) & 1)) x.x = -INFINITY;
                    if (!((vis >> (2 * j + 1)) & 1)) x.y = -INFINITY;
                    s[j] = pack2(x.x, x.y);
                }
            }
            const uint64_t f2 = pack2(f, f);
            float top;
            {
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const float2 x = unpack2(s[j]);
                    m4[j & 3] = max3(m4[j & 3], x.x, x.y);
                }
                top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            }
            // int8: the largest log2(2^score |v_scale|) of what the row sees in this tile, to within one
            float wtop = -INFINITY;
            if (DT == SB_KV_I8) {
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const ulonglong2 v4 = *reinterpret_cast<const ulonglong2 *>(sc + 256 + 2 * j);
                    const float2 x = unpack2(fma2(s[j], f2, v4.x)), y = unpack2(fma2(s[j + 1], f2, v4.y));
                    m4[j & 2] = max3(m4[j & 2], x.x, x.y), m4[(j & 2) + 1] = max3(m4[(j & 2) + 1], y.x, y.y);
                }
                wtop = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            }
            // the row's other half; behind this barrier both have their scores in registers
            ex[(buf * 2 + half) * 128 + rl] = top;
            if (DT == SB_KV_I8) exw[(buf * 2 + half) * 128 + rl] = wtop;
            pair_sync(1 + quad);
            top = fmaxf(top, ex[(buf * 2 + (half ^ 1)) * 128 + rl]) * f;
            if (DT == SB_KV_I8) wtop = fmaxf(wtop, exw[(buf * 2 + (half ^ 1)) * 128 + rl]);
            const float m_old = m;
            const float kw_old = kw;
            if (top > m + 8.0f) m = ceilf(top);
            if (DT == SB_KV_I8 && m > -INFINITY) {
                // kw keeps p * v_scale * 2^kw in f16's range, by what the row sees and what weight it gives it: a large
                // scale of little weight costs the others nothing.  It rises with m, by which older weights have shrunk, and
                // is chosen anew where this tile's weights would leave the range.  (Rows that see nothing here: wtop -inf.)
                const float e = ceilf(wtop - m);
                if (m_old > -INFINITY) kw += m - m_old;
                if (m_old == -INFINITY || kw + e > TT_KW_MAX) kw = TT_KW - e;
                kw = fminf(fmaxf(kw, -100.0f), 96.0f);
            }
            // (2^-127 and less is as good as nothing; ex2 gives 0)
            const float la = m_old == -INFINITY ? -127.0f : fmaxf((m_old - m) + (kw - kw_old), -127.0f);
            const float alpha = la > -127.0f ? ex2(la) : 0.0f;
            if (half == 0) al[(t & 3) * 128 + rl] = (signed char)la;
            const float off = m == -INFINITY ? 0.0f : kw - m;
            const uint64_t off2 = pack2(off, off);
            uint64_t l2 = pack2(0.0f, 0.0f);
            auto weights = [&](auto masked) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t term[C::PT][8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float2 x = unpack2(fma2(s[c * 8 + j], f2, off2));
                        uint64_t p = pack2(ex2(x.x), ex2(x.y));
                        l2 = add2(l2, p);
                        if (DT == SB_KV_I8) {
                            p = mul2(p, *reinterpret_cast<const uint64_t *>(sc + 128 + c * 16 + 2 * j));
                            if (masked.value) {  // a row that does not see a position takes nothing from its scale either
                                float2 w = unpack2(p);
                                if (!((vis >> (c * 16 + 2 * j)) & 1)) w.x = 0.0f;
                                if (!((vis >> (c * 16 + 2 * j + 1)) & 1)) w.y = 0.0f;
                                p = pack2(w.x, w.y);
                            }
                        }
                        uint32_t u[C::PT];
                        split2<DT>(p, u);
#pragma unroll
                        for (int q = 0; q < C::PT; q++) term[q][j] = u[q];
                    }
#pragma unroll
                    for (int q = 0; q < C::PT; q++) tmem_st8(S + q * 64 + half * 32 + c * 8, term[q]);
                }
            };
            if (DT == SB_KV_I8 && tail) weights(std::true_type{});
            else weights(std::false_type{});
            {
                const float2 x = unpack2(l2);
                l = fmaf(l, alpha, x.x + x.y);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * sb);
        }
    } else if (warp < TT_LOAD0) {
        // =================================================== sums
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(tt_regs_sums(DT)));
        float o[HD];
#pragma unroll
        for (int i = 0; i < HD; i++) o[i] = 0.0f;
        if (lane == 0) mbar_arrive(p_full);
        // int8: these warps also turn V's codes (four groups each) into f16, two tiles ahead of the sums
        uint8_t *raw = sm + C::RAW_OFF + TT_LOADERS * 2 * C::RAWK + quad * C::RAWV;
        int vcopied = 0, vgot = 0;
        auto put_v = [&](int t) {  // V of tile t, and the copies for t + 1
            wait(raw_v + 8 * quad, t & 1);
            if (ok) vgot = t + 1;
#pragma unroll 1
            for (int i = 0; i < 4; i++) put_codes(raw + i * 8 * HD, sm + (t % NS) * C::STAGE, quad * 4 + i);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(v_full + 8 * (t % NS));
            if (ok && t + 1 < nt) copy_codes(a.c.v, t + 1, quad * 4, 4, smem_u32(raw), raw_v + 8 * quad), vcopied++;
        };
        if (DT == SB_KV_I8 && nt > 0) {
            copy_codes(a.c.v, 0, quad * 4, 4, smem_u32(raw), raw_v + 8 * quad), vcopied++;
            put_v(0);
            if (nt > 1) put_v(1);
        }
        for (int t = 0; t < nt; t++) {
            const int buf = t & 1;
            wait(pv_done + 8 * (t % C::NSB), (t / C::NSB) & 1);
            tc_fence_after();
            const int la = al[(t & 3) * 128 + rl];
            const float alpha = la > -127 ? ex2((float)la) : 0.0f;
#pragma unroll
            for (int c = 0; c < HD; c += 16) {
                float d[16];
                tmem_ld16f(tmem + lanes + C::T_O + c, d);
                tmem_ld_done(d);
#pragma unroll
                for (int i = 0; i < 16; i++) o[c + i] = fmaf(o[c + i], alpha, d[i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * ((t + 1) % C::NSB));
            if (DT == SB_KV_I8 && t + 2 < nt) put_v(t + 2);
            if (DT == SB_KV_BF16 && *reinterpret_cast<volatile int *>(&s_bad[buf])) {
                // the tile's non-finite V elements (zeros in the product) reach the rows that see them
                const int p0 = (t0 + t) * TT_TILE;
                for (int h = 0; h < 2; h++) {
                    const unsigned long long vis = visible_bits(a, b, iv, ctx, n_vis, p0 + h * 64);
                    for (int j = 0; j < 64; j++) {
                        const int p = p0 + h * 64 + j;
                        if (p >= len || !((vis >> j) & 1)) continue;
                        const long long r = kv_row(a.c.pg, b, g, p);
                        if (r < 0) continue;
                        const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(a.c.v) + (size_t)r * HD;
#pragma unroll
                        for (int i = 0; i < HD; i++) {
                            const float x = __bfloat162float(src[i]);
                            if (!isfinite(x)) o[i] += x;
                        }
                    }
                }
            }
        }
        if (vgot < vcopied) mbar_wait_long(raw_v + 8 * quad, vgot & 1);  // a copy in flight must not outlive the CTA
        // (every product has been done, so the tiles' memory is free)
#pragma unroll
        for (int i = 0; i < HD; i += 4) *reinterpret_cast<float4 *>(red + (size_t)rl * HD + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    } else if (warp < TT_LOAD0 + TT_LOADERS) {
        // =================================================== loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(tt_regs_rest(DT, BF16)));
        // K of tile t goes where K of t-NS was, once q K^T of t-NS is done; V where V of t-NS was, once p V of t-NS is.
        if (DT == SB_KV_I8) {
            // codes of K, two tiles ahead, and the scales
            uint8_t *raw = sm + C::RAW_OFF + lw * 2 * C::RAWK;
            const uint32_t bar = raw_k + 16 * lw;
            int issued = 0, got = 0;
            auto copy = [&](int t) {
                copy_codes(a.c.k, t, lw * TT_GROUPS, TT_GROUPS, smem_u32(raw + (t & 1) * C::RAWK), bar + 8 * (t & 1));
                issued++;
            };
            if (nt > 0) copy(0);
            if (nt > 1) copy(1);
            int2 r1 = look_up(0), r2;  // rows of tile t+1; scales of tile t (0 where there is no row)
            float2 sk, sv;
            auto fetch_scales = [&](int2 r) {
                sk = make_float2(a.c.ks[max(r.x, 0)], a.c.ks[max(r.y, 0)]);
                sv = make_float2(a.c.vs[max(r.x, 0)], a.c.vs[max(r.y, 0)]);
                if (r.x < 0) sk.x = sv.x = 0.0f;
                if (r.y < 0) sk.y = sv.y = 0.0f;
            };
            fetch_scales(r1);
            r1 = look_up(1);
            for (int t = 0; t < nt; t++) {
                const int stage = t % NS, slot = t % TT_SCALES;
                if (t >= NS) wait(s_full + 8 * ((t - NS) % C::NSB), ((t - NS) / C::NSB) & 1);
                // (the scales in this slot, of tile t-4, have been read: p V of t-4, which waits for all of its weights, was
                // issued before q K^T of t-2)
                float *sc = reinterpret_cast<float *>(sm + C::SC_OFF) + slot * 384 + (lane & 7);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int grp = lw + (h * 4 + (lane >> 3)) * TT_LOADERS;
                    const float k1 = h ? sk.y : sk.x, v1 = h ? sv.y : sv.x;
                    const int e = (int)(__float_as_uint(v1) << 1 >> 24);  // |v1| < 2^(e - 126); what is not finite reaches its output anyhow
                    if (grp < 16) sc[grp * 8] = k1, sc[128 + grp * 8] = v1, sc[256 + grp * 8] = e == 255 ? -150.0f : (float)(e - 126);
                }
                fetch_scales(r1);
                r2 = look_up(t + 2);
                wait(bar + 8 * (t & 1), (t >> 1) & 1);
                if (ok) got = t + 1;
#pragma unroll
                for (int i = 0; i < TT_GROUPS; i++)
                    if (lw * TT_GROUPS + i < 16)
                        put_codes(raw + (t & 1) * C::RAWK + i * 8 * HD, sm + stage * C::STAGE + MAT, lw * TT_GROUPS + i);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(k_full + 8 * stage), mbar_arrive(sc_full + 8 * slot);
                if (ok && t + 2 < nt) copy(t + 2);
                r1 = r2;
            }
            if (!ok) {  // copies in flight must not outlive the CTA
                for (int i = got; i < issued; i++) mbar_wait_long(bar + 8 * (i & 1), (i >> 1) & 1);
            }
        } else {
            // step 2t: K of tile t, step 2t+1: V of tile t: TMA boxes, or rows copied one by one (pages of no multiple of
            // eight positions), which arrive under the next two steps.  V of a tile with drafted rows is looked at.
            constexpr int LAG = 2;
            const int box = a.box_rows;
            int2 rows = make_int2(-1, -1);
            unsigned hand = 0;  // steps whose arrival follows their copies, newest in bit 0
            unsigned tail_phase = 0;  // of tail_full, a bit per stage
            // row of this lane's box of a tile, looked up a tile ahead
            const int part = lane / (HD / 64), blk = lane % (HD / 64);
            auto box_row = [&](int t) {
                const int p = (t0 + t) * TT_TILE + part * box;
                const long long r = part * box < TT_TILE && t < nt && p < len ? kv_row(a.c.pg, b, g, p) : -1;
                return r < 0 ? a.c.pg.n_pages * a.c.pg.n_kv * a.c.pg.page_size : (int)r;
            };
            int y = box > 0 && lw == 0 ? box_row(0) : 0, y_next = 0;
            for (int n = 0; n < 2 * nt + LAG; n++) {
                const int t = n >> 1, stage = t % NS;
                const bool isv = n & 1;
                const uint32_t full = (isv ? v_full : k_full) + 8 * stage;
                hand <<= 1;
                bool tail = false;
                if (n < 2 * nt) {
                    if (t >= NS) wait((isv ? pv_done : s_full) + 8 * ((t - NS) % C::NSB), ((t - NS) / C::NSB) & 1);
                    uint8_t *dst = sm + stage * C::STAGE + (isv ? 0 : MAT);
                    tail = isv && (t0 + t + 1) * TT_TILE > ctx;
                    if (ok && box > 0) {
                        if (lw == 0) {
                            if (!isv) y_next = box_row(t + 1);
                            const uint32_t bar = tail ? tail_full + 8 * stage : full;
                            if (lane == 0) mbar_expect_tx(bar, MAT);
                            __syncwarp();
                            if (part * box < TT_TILE) tma_box(smem_u32(dst) + blk * 16384 + part * box * 128, isv ? &a.tmv : &a.tmk, blk * 64, y, bar);
                            if (isv) y = y_next;
                        } else if (!tail && lane == 0) {
                            mbar_arrive(full);
                        }
                    } else if (ok) {
                        hand |= tail ? 0 : 1;
                        if (!isv) rows = look_up(t);
#pragma unroll
                        for (int i = 0; i < TT_GROUPS; i++) {
                            const int grp = lw + i * TT_LOADERS;
#pragma unroll
                            for (int j = 0; j < NI; j++) {
                                const int row = __shfl_sync(0xffffffffu, i < 4 ? rows.x : rows.y, (i & 3) * 8 + j * LPI + sub);
                                if (grp >= 16) continue;
                                const char *src = static_cast<const char *>(isv ? a.c.v : a.c.k) + (row < 0 ? 0 : ((size_t)row * CPR + piece) * 16);
                                // rows behind the end (or on no page) are zeros
                                cp_async16_fill(smem_u32(dst) + sw128(grp * 8 + j * LPI + sub, piece), src, row < 0 ? 0 : 16);
                            }
                        }
                    }
                    cp_commit();
                    if (ok && tail) {
                        // A non-finite V element of a drafted row must not reach rows that do not see it (0 * inf): it is a
                        // zero in the product, and the sums add it where it is seen.
                        if (box > 0) wait(tail_full + 8 * stage, (tail_phase >> stage) & 1);
                        else cp_wait<0>();
                        __syncwarp();
                        tail_phase ^= 1u << stage;
                        bool bad = false;
#pragma unroll 4
                        for (int i = 0; i < TT_GROUPS * NI; i++) {
                            const int grp = lw + (i / NI) * TT_LOADERS;
                            if (grp >= 16) break;
                            uint4 *at = reinterpret_cast<uint4 *>(dst + sw128(grp * 8 + (i % NI) * LPI + sub, piece));
                            const uint4 w = *at;
                            uint32_t x[4] = {w.x, w.y, w.z, w.w};
                            bool here = false;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u, here = true;
                                if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0xffffu, here = true;
                            }
                            if (here) *at = make_uint4(x[0], x[1], x[2], x[3]), bad = true;
                        }
                        if (bad) s_bad[t & 1] = 1;  // stays set: a later tile of its parity only looks in vain
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0 && ok) mbar_arrive(full);
                    }
                } else {
                    cp_commit();
                }
                if (n >= LAG && ((hand >> LAG) & 1)) {
                    cp_wait<LAG>();
                    fence_proxy_async_smem();
                    __syncwarp();
                    const int m = n - LAG;
                    if (lane == 0) mbar_arrive((m & 1 ? v_full : k_full) + 8 * ((m >> 1) % NS));
                }
            }
            cp_wait<0>();
        }
    } else {
        // =================================================== products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(tt_regs_rest(DT, BF16)));
        if (lane == 0) {
        ok = mbar_wait_long(q_full, 0);
        const uint32_t id_s = idesc_f16(TT_TILE, DT == SB_KV_BF16, false), id_o = idesc_f16(HD, DT == SB_KV_BF16, true);
        // Products are issued no faster than they run (64 clocks; 32 for head_dim 64's second one): a product that waits
        // for the tensor cores holds up the barrier polls of the softmax warps beside this one (2000 clocks a tile).
        // The wait, of at most 62 * 21 clocks, is bounded twice: by the clock, whose differences are taken modulo its 2^32,
        // and by the number of readings.
        auto clock32 = []() {
            uint32_t c;
            asm volatile("mov.u32 %0, %%clock;" : "=r"(c)::"memory");
            return c;
        };
        uint32_t pace_from = 0;
        auto pace = [&](int n) {
            if ((n & 3) == 3)
                for (int i = 0; i < 1024 && !clocks_passed(pace_from, clock32(), 62 * (n - 2)); i++) {
                }
        };
        for (int t = 0; t <= nt && ok; t++) {
            if (t < nt) {
                const int buf = t % C::NSB, stage = t % NS;
                ok = mbar_wait_long(k_full + 8 * stage, (t / NS) & 1);
                // the scores' columns are free once p V of tile t-NSB has read its terms from them
                if (ok && t >= C::NSB) ok = mbar_wait_long(pv_done + 8 * buf, (t / C::NSB - 1) & 1);
                if (!ok) break;
                tc_fence_after();
                pace_from = clock32();
                const uint64_t kd = sw128_desc(base + stage * C::STAGE + MAT, 16);
#pragma unroll
                for (int q = QT - 1; q >= 0; q--) {  // small terms first: less is cut off
                    const uint64_t qd = sw128_desc(base + C::Q_OFF + q * MAT, 16);
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const int at = (k >> 2) * (16384 >> 4) + (k & 3) * 2;  // 64 elements a block, 32 bytes a step
                        if (C::QTMEM) umma_ts(tmem + buf * C::T_S, tmem + C::T_Q + q * (HD / 2) + k * 8, kd + at, id_s, q != QT - 1 || k > 0);
                        else umma_ss(tmem + buf * C::T_S, qd + at, kd + at, id_s, q != QT - 1 || k > 0);
                        pace((QT - 1 - q) * (HD / 16) + k);
                    }
                }
                umma_commit(s_full + 8 * buf);
            }
            if (t > 0) {
                const int buf = (t - 1) % C::NSB, stage = (t - 1) % NS;
                ok = mbar_wait_long(v_full + 8 * stage, ((t - 1) / NS) & 1) && mbar_wait_long(p_full + 8 * buf, ((t - 1) / C::NSB) & 1);
                if (!ok) break;
                tc_fence_after();
                pace_from = clock32();
                const uint64_t vd = sw128_desc(base + stage * C::STAGE, 16384);
#pragma unroll
                for (int q = C::PT - 1; q >= 0; q--)
#pragma unroll
                    for (int k = 0; k < TT_TILE / 16; k++) {
                        umma_ts(tmem + C::T_O, tmem + buf * C::T_S + q * 64 + k * 8, vd + k * (2048 >> 4), id_o, q != C::PT - 1 || k > 0);
                        pace((C::PT - 1 - q) * (TT_TILE / 16) + k);
                    }
                umma_commit(pv_done + 8 * buf);
            }
        }
        if (ok && nt > 0) ok = mbar_wait_long(pv_done + 8 * ((nt - 1) % C::NSB), ((nt - 1) / C::NSB) & 1);
        }
    }
    if (!ok) wait_failed(a.errors, WAIT_TREE_TC);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == TT_MMA) tmem_dealloc(tmem, 512);

    // ---- the output or the splits' join
    if (warp < TT_SOFTMAX_WARPS) ex[half * 128 + rl] = l;
    __syncthreads();
    if (warp < 4) rm[rl] = m == -INFINITY ? m : m - kw, rs[rl] = ex[rl] + ex[128 + rl];
    __syncthreads();
    const size_t tile = ((size_t)b * nkv + g) * (gridDim.x / a.n_splits) + rt;
    tree_finish<HD, BF16, 1, TT_ROWS, TT_THREADS>(a, red, rm, rs, min(TT_ROWS, total_rows - row0), row0, b, g, n_new, split, tile);
}

template <int HD, int DT, bool BF16>
int tt_inst(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    auto kern = tree_attn_tc_kernel<HD, DT, BF16>;
    static int limit[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!limit[dev & 63]) SB_TRY(allow_max_dynamic_smem(kern, &limit[dev & 63]));
    // one CTA per SM: all of TMEM belongs to it
    constexpr int smem = std::max(TtShape<HD, DT, BF16>::BYTES, 118 * 1024);
    SB_CHECK(smem <= limit[dev & 63], SB_ERR_SHAPE, "tree attention: needs %d B shared memory (limit %d)", smem, limit[dev & 63]);
    SB_CUDA_TRY(launch(kern, dim3(p.row_tiles * a.n_splits, a.c.pg.n_kv, a.B), dim3(TT_THREADS), smem, st, false, a));
    return SB_OK;
}
template <int HD>
int tt_dt(const TreeAttnArgs &a, const TreeAttnPlan &p, cudaStream_t st) {
    if (a.c.dtype == SB_KV_I8) return a.bf16 ? tt_inst<HD, SB_KV_I8, true>(a, p, st) : tt_inst<HD, SB_KV_I8, false>(a, p, st);
    return a.bf16 ? tt_inst<HD, SB_KV_BF16, true>(a, p, st) : tt_inst<HD, SB_KV_BF16, false>(a, p, st);
}

}  // namespace

bool tree_attn_tc_wanted(const TreeAttnArgs &a) { return a.c.dtype != SB_KV_F32 && a.T * a.rep > 32; }

TreeAttnPlan tree_attn_tc_plan(const TreeAttnArgs &a, int max_len) {
    TreeAttnPlan p;
    p.rows = TT_ROWS;
    p.row_tiles = ceil_div(a.T * a.rep, TT_ROWS);
    const long long base = (long long)a.B * a.c.pg.n_kv * p.row_tiles;
    p.n_splits = tree_splits(base, ceil_div(std::max(max_len, 1), TT_TILE));
    return p;
}

int tree_attn_tc_launch(const TreeAttnArgs &args, const TreeAttnPlan &p, cudaStream_t st) {
    TreeAttnArgs a = args;
    if (a.c.dtype == SB_KV_BF16) SB_TRY(tree_tensor_maps(a, TT_TILE));
    return a.c.hd == 128 ? tt_dt<128>(a, p, st) : tt_dt<64>(a, p, st);
}

}  // namespace sb
