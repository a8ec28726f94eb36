// Writing, moving and reading rows of a paged K/V cache (kv_cache.cuh).
//
// Quantised rows follow quantize_symmetric's rule (quantize.rs:16-32) row by row, in
// f32 without contraction, but for their scale: scale = max|x| * (1 / 127), code =
// x * (1 / scale) rounded half away from zero and held to [-127, 127].
// quantize_symmetric divides by 127; the product is what tensor programs make of a
// division by a constant, so that rows agree with theirs bit for bit, and lies
// within one unit in the last place of the quotient.
#include "kv_cache.cuh"

#include <algorithm>

namespace sb {

namespace {

// 16 bytes of values: 4 f32 or 8 bf16
template <bool BF16>
struct Io;
template <>
struct Io<false> {
    using T = float;
    static constexpr int E = 4;
    __device__ static void open(uint4 u, float (&x)[4]) {
        x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
    }
    __device__ static void store(float *p, const float (&x)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(lo)) |
           ((uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi)) << 16);
}
template <>
struct Io<true> {
    using T = __nv_bfloat16;
    static constexpr int E = 8;
    __device__ static void open(uint4 u, float (&x)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    __device__ static void store(T *p, const float (&x)[8]) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(bf16x2(x[0], x[1]), bf16x2(x[2], x[3]), bf16x2(x[4], x[5]), bf16x2(x[6], x[7]));
    }
};

// round half away from zero, NaN -> 0, held to [-127, 127]
__device__ __forceinline__ int quant_code(float x, float inv) {
    const float r = roundf(__fmul_rn(x, inv));
    return isnan(r) ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

constexpr int APPEND_THREADS = 256;

// A lane holds 16 bytes of a head's row, a group of lanes the whole row; a group
// takes HEADS heads of a (b, t) row (q heads first, then k, then v), so that
// their loads are in flight together and the row's cos and sin are read once.
// Bound by memory, with 62 % of the issue slots taken: 4096 rows of 64 + 2 * 8
// heads of 128, f32 to int8, 310 MB in 62 us (5.0 TB/s); to bf16 54 us (5.9 TB/s),
// to f32 55 us (6.1 TB/s).  Rows looped over with the next one's loads ahead took
// 78 us to int8, eight heads a group 90.
template <int HD, bool BF16>
struct Append {
    static constexpr int E = Io<BF16>::E;
    static constexpr int LPH = HD / E;               // lanes per head
    static constexpr int G = APPEND_THREADS / LPH;   // groups
    static constexpr int HEADS = 4;                  // per group
};

template <int HD, bool BF16, int DT>
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(const KvAppendArgs a) {
    using T = typename Io<BF16>::T;
    using P = Append<HD, BF16>;
    constexpr int E = P::E, LPH = P::LPH, G = P::G, HEADS = P::HEADS;
    const int lane = threadIdx.x % LPH, grp = threadIdx.x / LPH;
    const int row = blockIdx.x;
    const int b = row / a.T, t = row - b * a.T;
    const int nkv = a.c.pg.n_kv, nh = a.n_heads;
    const int heads = nh + 2 * nkv;
    const int h0 = blockIdx.y * G * HEADS + grp;

    pdl_wait();
    pdl_launch_dependents();
    const int ctx = a.ctx_len[b];
    const int nn = a.n_new ? a.n_new[b] : a.T;
    const int dep = a.depth ? a.depth[(size_t)b * a.depth_ld + t] : t;
    const T *q = static_cast<const T *>(a.q) + (size_t)row * a.ldq + lane * E;
    const T *k = static_cast<const T *>(a.k) + (size_t)row * a.ldk + lane * E;
    const T *v = static_cast<const T *>(a.v) + (size_t)row * a.ldv + lane * E;
    uint4 raw[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const int h = min(h0 + i * G, heads - 1);  // past the last head: that head again, not used
        const int g = h < nh ? h : h < nh + nkv ? h - nh : h - nh - nkv;
        raw[i] = *reinterpret_cast<const uint4 *>((h < nh ? q : h < nh + nkv ? k : v) + g * HD);
    }
    const bool live = ctx >= 0 && t < nn;
    float cs[E / 2], sn[E / 2];
    bool turned = live;
    if (a.cos) {
        const long long p = (long long)ctx + dep;
        turned = live && p >= 0 && p < a.rope_len;
        const size_t o = turned ? (size_t)p * (HD / 2) + lane * (E / 2) : 0;
        if constexpr (E == 8) {
            const float4 c4 = *reinterpret_cast<const float4 *>(a.cos + o), s4 = *reinterpret_cast<const float4 *>(a.sin + o);
            cs[0] = c4.x, cs[1] = c4.y, cs[2] = c4.z, cs[3] = c4.w;
            sn[0] = s4.x, sn[1] = s4.y, sn[2] = s4.z, sn[3] = s4.w;
        } else {
            const float2 c2 = *reinterpret_cast<const float2 *>(a.cos + o), s2 = *reinterpret_cast<const float2 *>(a.sin + o);
            cs[0] = c2.x, cs[1] = c2.y, sn[0] = s2.x, sn[1] = s2.y;
        }
    }
    const long long at = kv_row(a.c.pg, b, 0, (long long)ctx + t);
    const long long r0 = turned ? at : -1;
    T *qo = static_cast<T *>(a.q_out) + (size_t)row * nh * HD + lane * E;
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const int h = h0 + i * G;
        if (h - grp >= heads) break;  // the same for the whole block
        float x[E];
        Io<BF16>::open(raw[i], x);
        if (h < nh + nkv && a.cos) {
#pragma unroll
            for (int j = 0; j < E / 2; j++) {
                const float x0 = x[2 * j], x1 = x[2 * j + 1];
                x[2 * j] = __fsub_rn(__fmul_rn(x0, cs[j]), __fmul_rn(x1, sn[j]));
                x[2 * j + 1] = __fadd_rn(__fmul_rn(x0, sn[j]), __fmul_rn(x1, cs[j]));
            }
        }
        if (h < nh) {
#pragma unroll
            for (int j = 0; j < E; j++) x[j] = r0 >= 0 ? __fmul_rn(x[j], a.q_scale) : 0.0f;
            Io<BF16>::store(qo + h * HD, x);
        }
        // the other heads' rows of a warp go on together: a row's maximum is taken over its lanes
        const bool put = h >= nh && h < heads && r0 >= 0;
        if (!__any_sync(0xffffffffu, put)) continue;
        const bool isk = h < nh + nkv;
        const size_t r = put ? (size_t)r0 + (size_t)((isk ? h : h - nkv) - nh) * a.c.pg.page_size : 0;
        void *dst = isk ? a.c.k : a.c.v;
        if (DT == SB_KV_I8) {
            float m = fabsf(x[0]);
#pragma unroll
            for (int j = 1; j < E; j++) m = fmaxf(m, fabsf(x[j]));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = __fmul_rn(m, 1.0f / 127.0f), inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
            uint32_t w[E / 4];
#pragma unroll
            for (int j = 0; j < E / 4; j++) w[j] = 0;
#pragma unroll
            for (int j = 0; j < E; j++) w[j >> 2] |= (uint32_t)(quant_code(x[j], inv) & 0xff) << (8 * (j & 3));
            if (!put) continue;
            int8_t *d = static_cast<int8_t *>(dst) + r * HD + lane * E;
            if constexpr (E == 8) *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t *>(d) = w[0];
            if (lane == 0) (isk ? a.c.ks : a.c.vs)[r] = s;
        } else if (put && DT == SB_KV_F32) {
            float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(dst) + r * HD + lane * E);
#pragma unroll
            for (int j = 0; j < E / 4; j++) d[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        } else if (put) {
            uint2 *d = reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(dst) + r * HD + lane * E);
#pragma unroll
            for (int j = 0; j < E / 4; j++) d[j] = make_uint2(bf16x2(x[4 * j], x[4 * j + 1]), bf16x2(x[4 * j + 2], x[4 * j + 3]));
        }
    }
}

// Each thread owns one 16-byte column (or one scale) of the rows and moves it
// for the whole path: rows are read eight at a time before any of them is
// written.  The path ascends and path[i] >= i, so no row is written before the
// batch that reads it.  Bound by latency (path, page table, row, one after the
// other), so all loads of a batch are issued together: a row that does not move
// is read and not written (32 sequences of 8 kv heads: about 4 us).
__global__ void kv_commit_kernel(const KvCacheArgs c, const int *ctx_len, const int *path, int path_ld,
                                 const int *n_accept, int row16) {
    const int b = blockIdx.y;
    const int per_head = 2 * row16 + (c.dtype == SB_KV_I8 ? 2 : 0);  // k columns, v columns, scales
    const int e = blockIdx.x * blockDim.x + threadIdx.x;
    const int g = e / per_head, col = e - g * per_head;
    if (g >= c.pg.n_kv) return;
    pdl_wait();
    pdl_launch_dependents();
    const int ctx = ctx_len[b], n = min(n_accept[b], path_ld);
    const int *pb = path + (size_t)b * path_ld;
    const bool scale = col >= 2 * row16;
    char *base = static_cast<char *>(col < row16 ? c.k : c.v);
    const int cc = col < row16 ? col : col - row16;
    float *sbase = col == 2 * row16 ? c.ks : c.vs;
    for (int i0 = 0; i0 < (ctx < 0 ? 0 : n); i0 += 8) {
        uint4 v[8];
        int p[8];
        long long from[8], to[8];
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = pb[min(i0 + j, path_ld - 1)];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            from[j] = kv_row(c.pg, b, g, (long long)ctx + p[j]);
            to[j] = kv_row(c.pg, b, g, (long long)ctx + i0 + j);
            if (i0 + j >= n || p[j] < 0 || p[j] == i0 + j || from[j] < 0) to[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const size_t f = from[j] < 0 ? 0 : (size_t)from[j];
            if (scale)
                v[j].x = __float_as_uint(sbase[f]);
            else
                v[j] = *reinterpret_cast<const uint4 *>(base + (f * row16 + cc) * 16);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (to[j] < 0) continue;
            if (scale)
                sbase[to[j]] = __uint_as_float(v[j].x);
            else
                *reinterpret_cast<uint4 *>(base + ((size_t)to[j] * row16 + cc) * 16) = v[j];
        }
    }
}

// HD/4 lanes per cached row, four elements a lane, so that f32 rows leave in
// whole 16-byte lanes.  A block takes READ_UNROLL times as many (position, head)
// rows as it has lane groups, in the order in which they are written: its writes
// are one contiguous run, and all its reads are in flight together: bound by
// memory, 8 x 8192 positions of 8 heads of 128 from int8 to f32 in 110 us (6.1 TB/s).
constexpr int READ_THREADS = 256, READ_UNROLL = 4;

template <int DT>
__device__ __forceinline__ float4 read4(const void *base, size_t at) {
    if (DT == SB_KV_F32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
    if (DT == SB_KV_BF16) {
        const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(base) + at);
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    }
    const char4 c = *reinterpret_cast<const char4 *>(static_cast<const int8_t *>(base) + at);
    return make_float4((float)c.x, (float)c.y, (float)c.z, (float)c.w);
}
__device__ __forceinline__ float4 scaled(float4 x, float s, bool in) {
    return in ? make_float4(x.x * s, x.y * s, x.z * s, x.w * s) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}

template <int HD, int DT, bool BF16>
__global__ void __launch_bounds__(READ_THREADS) kv_read_kernel(const KvCacheArgs c, const int *start, int n, void *k_out,
                                                               void *v_out) {
    constexpr int LPR = HD / 4;
    constexpr int RPB = READ_THREADS / LPR;
    const int b = blockIdx.y, lane = threadIdx.x % LPR;
    const int nkv = c.pg.n_kv;
    const long long first = (long long)blockIdx.x * (RPB * READ_UNROLL), all = (long long)n * nkv;
    const int p0 = (int)(first / nkv), g0 = (int)(first - (long long)p0 * nkv);
    pdl_wait();
    pdl_launch_dependents();
    const int s0 = start ? start[b] : 0;
    long long r[READ_UNROLL];
    float4 k[READ_UNROLL], v[READ_UNROLL];
    float ks[READ_UNROLL], vs[READ_UNROLL];
#pragma unroll
    for (int i = 0; i < READ_UNROLL; i++) {
        const int e = g0 + threadIdx.x / LPR + i * RPB, dp = e / nkv;
        r[i] = kv_row(c.pg, b, e - dp * nkv, (long long)s0 + p0 + dp);
    }
#pragma unroll
    for (int i = 0; i < READ_UNROLL; i++) {
        const size_t f = r[i] < 0 ? 0 : (size_t)r[i];  // a position outside reads row 0 and leaves zeros
        k[i] = read4<DT>(c.k, f * HD + lane * 4);
        v[i] = read4<DT>(c.v, f * HD + lane * 4);
        ks[i] = DT == SB_KV_I8 ? c.ks[f] : 1.0f;
        vs[i] = DT == SB_KV_I8 ? c.vs[f] : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < READ_UNROLL; i++) {
        const long long at = first + threadIdx.x / LPR + i * RPB;
        if (at >= all) continue;
        const size_t o = ((size_t)b * all + at) * HD + lane * 4;
        const float4 kx = scaled(k[i], ks[i], r[i] >= 0), vx = scaled(v[i], vs[i], r[i] >= 0);
        if (BF16) {
            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(k_out) + o) = make_uint2(bf16x2(kx.x, kx.y), bf16x2(kx.z, kx.w));
            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(v_out) + o) = make_uint2(bf16x2(vx.x, vx.y), bf16x2(vx.z, vx.w));
        } else {
            *reinterpret_cast<float4 *>(static_cast<float *>(k_out) + o) = kx;
            *reinterpret_cast<float4 *>(static_cast<float *>(v_out) + o) = vx;
        }
    }
}

template <int HD, bool BF16>
int append_io(const KvAppendArgs &a, cudaStream_t st) {
    using P = Append<HD, BF16>;
    const dim3 grid((unsigned)(a.B * a.T), (unsigned)ceil_div(a.n_heads + 2 * a.c.pg.n_kv, P::G * P::HEADS));
    auto kern = a.c.dtype == SB_KV_I8    ? kv_append_kernel<HD, BF16, SB_KV_I8>
                : a.c.dtype == SB_KV_F32 ? kv_append_kernel<HD, BF16, SB_KV_F32>
                                         : kv_append_kernel<HD, BF16, SB_KV_BF16>;
    SB_CUDA_TRY(launch(kern, grid, dim3(APPEND_THREADS), 0, st, true, a));
    return SB_OK;
}
template <int HD>
int append_hd(const KvAppendArgs &a, cudaStream_t st) {
    return a.bf16 ? append_io<HD, true>(a, st) : append_io<HD, false>(a, st);
}

template <int HD, int DT>
int read_dt(const KvCacheArgs &c, int B, const int *start, int n, int out_bf16, void *k_out, void *v_out, cudaStream_t st) {
    constexpr int rows = READ_THREADS / (HD / 4) * READ_UNROLL;
    const long long blocks = ((long long)n * c.pg.n_kv + rows - 1) / rows;
    SB_CHECK(blocks <= 0x7fffffffll, SB_ERR_SHAPE, "sb_kv_read: n %d", n);
    const dim3 grid((unsigned)blocks, (unsigned)B);
    if (out_bf16)
        SB_CUDA_TRY(launch(kv_read_kernel<HD, DT, true>, grid, dim3(READ_THREADS), 0, st, true, c, start, n, k_out, v_out));
    else
        SB_CUDA_TRY(launch(kv_read_kernel<HD, DT, false>, grid, dim3(READ_THREADS), 0, st, true, c, start, n, k_out, v_out));
    return SB_OK;
}

template <int HD>
int read_hd(const KvCacheArgs &c, int B, const int *start, int n, int out_bf16, void *k_out, void *v_out, cudaStream_t st) {
    if (c.dtype == SB_KV_I8) return read_dt<HD, SB_KV_I8>(c, B, start, n, out_bf16, k_out, v_out, st);
    if (c.dtype == SB_KV_F32) return read_dt<HD, SB_KV_F32>(c, B, start, n, out_bf16, k_out, v_out, st);
    return read_dt<HD, SB_KV_BF16>(c, B, start, n, out_bf16, k_out, v_out, st);
}

}  // namespace

int kv_append_launch(const KvAppendArgs &a, cudaStream_t st) {
    return a.c.hd == 128 ? append_hd<128>(a, st) : append_hd<64>(a, st);
}

int kv_commit_launch(const KvCacheArgs &c, int B, const int *ctx_len, const int *path, int path_ld,
                     const int *n_accept, cudaStream_t st) {
    const int esz = c.dtype == SB_KV_F32 ? 4 : c.dtype == SB_KV_BF16 ? 2 : 1;
    const int row16 = c.hd * esz / 16;
    const int cols = c.pg.n_kv * (2 * row16 + (c.dtype == SB_KV_I8 ? 2 : 0));
    SB_CUDA_TRY(launch(kv_commit_kernel, dim3(ceil_div(cols, 64), B), dim3(64), 0, st, true, c, ctx_len, path, path_ld,
                       n_accept, row16));
    return SB_OK;
}

int kv_read_launch(const KvCacheArgs &c, int B, const int *start, int n, int out_bf16, void *k_out, void *v_out,
                   cudaStream_t st) {
    return c.hd == 128 ? read_hd<128>(c, B, start, n, out_bf16, k_out, v_out, st)
                       : read_hd<64>(c, B, start, n, out_bf16, k_out, v_out, st);
}

}  // namespace sb
