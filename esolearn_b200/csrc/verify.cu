// Verification of drafted tokens (speculative sampling), one cluster of CTAs
// per sequence.
//
// Node 0 is the sequence's last token; node i > 0 is a drafted token under
// node parents[i] < i.  The walk starts at node 0.  At a node with target
// probabilities p = softmax(logits[node] / T) its children are tried in order;
// w = p, W = 1 at first.
//   with the draft's probabilities q = draft[node] (the children were drawn from
//   it independently): child x is accepted when u W q(x) < w(x); otherwise
//   w <- max(w - W q, 0), W <- sum w.  With a the sum of the W so far, w is
//   max(p - a q, 0): one pass over the row per rejection, no stored w;
//   without (the children are given tokens): accepted when u W < w(x);
//   otherwise W <- W - w(x), w(x) <- 0: no pass at all.
// An accepted child is the next node.  Where no child is accepted the next
// token is the y with the largest w(y) / noise(y), lowest index first; for
// noise ~ Exp(1) that draws y from w / W.  If nothing is left of w, from p.
// T < 1e-8 is greedy: the child that is the row's argmax (ties -> last index,
// generate.rs:167-173) is accepted, and the argmax is the next token.
//
// The rows of nodes that the walk does not reach are not waited for.  A row is
// split over the CTAs of its cluster and copied once into their shared memory
// (bulk copies where rows are 16-byte aligned), from which all passes over it
// read.  Maxima, sums and candidates are exchanged through distributed shared
// memory and joined in a fixed order, so that every CTA takes the same decisions
// from the same bits.  A step is bound by latency (copy, block and cluster
// reduction): where there is room the first child's row is on its way while its
// parent's step runs, and the noise is fetched into L2 from the start.
//
// With few rows altogether (verify_all_rows below) the maxima and sums of every
// node's row are taken first, by a kernel over all SMs, and the walk then needs
// a row only where it ends, once and straight from memory: it reads more than the
// walk would and is still faster, since its steps no longer wait for one another's
// rows.
#include "verify.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "pipeline.cuh"

namespace sb {

namespace {

namespace cg = cooperative_groups;

constexpr int VT = 512;
constexpr int MAX_ROW = 184 * 1024;  // bytes of shared memory for rows
constexpr int MAX_CS = 16;

struct Best {
    float v;
    int i;
};
// larger value first; of equal ones the lower index (last = false) or the higher
__device__ __forceinline__ Best better(Best a, Best b, bool last) {
    if (b.i < 0) return a;
    if (a.i < 0 || b.v > a.v || (b.v == a.v && (last ? b.i > a.i : b.i < a.i))) return b;
    return a;
}

struct Shared {
    float2 stat[2][MAX_CS];  // one slot per rank, two rounds in turn
    Best best[2][MAX_CS];
    float2 wstat[VT / 32];
    Best wbest[VT / 32];
    int first[VERIFY_MAX_NODES];  // first child and next sibling (N: none)
    int next[VERIFY_MAX_NODES];
    int parents[VERIFY_MAX_NODES];
    int tokens[VERIFY_MAX_NODES];
    float u[VERIFY_MAX_NODES];
    float lx[VERIFY_MAX_NODES];  // logits[node][token of child i]
    float qx[VERIFY_MAX_NODES];
    int rejected[VERIFY_MAX_NODES];
    float2 pm[VERIFY_MAX_NODES];  // PRE: (max, sum) of every node's row
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Exponents are (x - max) c everywhere, in sums, joins and probabilities: x c - max c in one FMA would round max c, by
// more than one at low temperatures, and scale the sum against the probabilities.
// (max, sum of 2^((x - max) c)) of two parts
__device__ __forceinline__ float2 join_stat(float2 a, float2 b, float c) {
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, 0.0f);
    return make_float2(m, a.y * (a.x == -INFINITY ? 0.0f : ex2((a.x - m) * c)) + b.y * (b.x == -INFINITY ? 0.0f : ex2((b.x - m) * c)));
}
__device__ __forceinline__ void prefetch_l2(const float *p, int bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// (max, sum of 2^((x - max) c)) of up to 8192 columns of a row: part[row][chunk].
constexpr int ST = 256, SE = 32;
template <bool VEC>
__global__ void __launch_bounds__(ST) verify_stats_kernel(const float *logits, long long ld, int V, int chunks, float c, float2 *part) {
    __shared__ float2 sh[ST / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / chunks;
    const int v0 = (blockIdx.x - r * chunks) * ST * SE, len = min(ST * SE, V - v0);
    const float *row = logits + (size_t)r * ld + v0;
    float x[SE];
#pragma unroll
    for (int k = 0; k < SE; k += 4) {
        const int v = VEC ? (k * ST + tid * 4) : 0;
        if (VEC && v + 4 <= len) {
            const float4 y = __ldg(reinterpret_cast<const float4 *>(row + v));
            x[k] = y.x, x[k + 1] = y.y, x[k + 2] = y.z, x[k + 3] = y.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int w = VEC ? v + e : (k + e) * ST + tid;
                x[k + e] = w < len ? __ldg(row + w) : -INFINITY;
            }
        }
    }
    pdl_launch_dependents();
    float2 st = make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int k = 0; k < SE; k++) st.x = fmaxf(st.x, x[k]);
    if (st.x > -INFINITY) {
#pragma unroll
        for (int k = 0; k < SE; k++) st.y += ex2((x[k] - st.x) * c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) st = join_stat(st, make_float2(__shfl_xor_sync(0xffffffffu, st.x, o), __shfl_xor_sync(0xffffffffu, st.y, o)), c);
    if (lane == 0) sh[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = lane < ST / 32 ? sh[lane] : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int o = ST / 64; o > 0; o >>= 1) st = join_stat(st, make_float2(__shfl_xor_sync(0xffffffffu, st.x, o), __shfl_xor_sync(0xffffffffu, st.y, o)), c);
        if (lane == 0) part[blockIdx.x] = st;
    }
}

// VEC: rows, and the noise and the draft's rows, are 16-byte aligned.
// `two`: shared memory holds two rows' columns.  PRE: every row's maximum and sum
// come as `chunks` parts from verify_stats_kernel.
template <bool VEC, bool PRE>
__global__ void __launch_bounds__(VT, 1) verify_kernel(const VerifyArgs a, int two, const float2 *part, int chunks) {
    extern __shared__ __align__(16) float sm_rows[];
    __shared__ Shared s;
    __shared__ __align__(8) unsigned long long bars[2];
    cg::cluster_group cl = cg::this_cluster();
    const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / cs;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = ((a.V + cs - 1) / cs + 3) & ~3;
    const int w0 = min(rank * per, a.V), len = min(w0 + per, a.V) - w0;  // this CTA's columns
    const int len4 = (len + 3) & ~3;
    const bool greedy = a.temperature < 1e-8f;
    const float c = greedy ? 1.0f : 1.4426950408889634f / a.temperature;
    const float *noise = a.noise ? a.noise + (size_t)b * a.ld_noise + w0 : nullptr;
    const float *rows = a.logits + (size_t)b * a.N * a.ld + w0;

    // columns behind the end are -inf (the last copy of a row takes whole 16 bytes; what is left of it is set below)
    const int bulk = VEC ? len & ~3 : 0;
    if (tid == 0) {
        mbar_init(smem_u32(&bars[0]), 1);
        mbar_init(smem_u32(&bars[1]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // A CTA's shared memory may be written by another only once it has started: all arrive here and wait, with the first
    // row's copy and the tree's tables between, before the first exchange.
    if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    unsigned phase[2] = {0, 0};
    // starts the copy of a node's row (its 16-byte part) into buffer `buf`; thread 0
    auto start = [&](int n, int buf) {
        if (bulk > 0 && tid == 0) {
            const uint32_t bar = smem_u32(&bars[buf]);
            mbar_expect_tx(bar, bulk * 4);
            tma_load_1d(smem_u32(sm_rows + buf * per), rows + (size_t)n * a.ld, bulk * 4, bar);
        }
    };
    // the rest of the row by plain copies; then the whole row is there
    auto finish = [&](int n, int buf) {
        float *dst = sm_rows + buf * per;
        const float *src = rows + (size_t)n * a.ld;
        for (int v = bulk + tid; v < len4; v += VT) dst[v] = v < len ? src[v] : -INFINITY;
        if (bulk > 0) {
            if (!mbar_wait(smem_u32(&bars[buf]), phase[buf])) wait_failed(a.errors, WAIT_VERIFY);
            phase[buf] ^= 1;
        }
        __syncthreads();
    };
    if (!PRE) start(0, 0);
    for (int i = tid; i < a.N; i += VT) {
        s.parents[i] = i == 0 ? -1 : a.parents[(size_t)b * a.parents_ld + i];
        s.tokens[i] = a.tokens[(size_t)b * a.N + i];
        s.u[i] = greedy ? 0.0f : a.u[(size_t)b * a.N + i];
        s.first[i] = a.N;
    }
    if (VEC && tid == 32 && !greedy && bulk > 0) prefetch_l2(noise, bulk * 4);
    __syncthreads();
    for (int i = tid; i < a.N; i += VT) {
        const int p = s.parents[i];
        int n = a.N;
        if (p >= 0 && p < i) {
            atomicMin(&s.first[p], i);
            n = i + 1;
            while (n < a.N && s.parents[n] != p) n++;
        }
        s.next[i] = n;
        if (PRE && p >= 0 && p < i) {
            const int t = s.tokens[i];
            const bool in = t >= 0 && t < a.V;
            s.lx[i] = in ? (rows - w0)[(size_t)p * a.ld + t] : -INFINITY;
            if (a.draft) s.qx[i] = in ? a.draft[((size_t)b * a.N + p) * a.ld_draft + t] : 0.0f;
        }
    }
    if (PRE) {
        pdl_wait();
        for (int i = warp; i < a.N; i += VT / 32) {
            float2 st = make_float2(-INFINITY, 0.0f);
            for (int k = lane; k < chunks; k += 32) st = join_stat(st, __ldcg(part + ((size_t)b * a.N + i) * chunks + k), c);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) st = join_stat(st, make_float2(__shfl_xor_sync(0xffffffffu, st.x, o), __shfl_xor_sync(0xffffffffu, st.y, o)), c);
            if (lane == 0) s.pm[i] = st;
        }
    }
    __syncthreads();
    if (cs > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

    auto cluster_sync = [&]() {
        if (cs > 1) cl.sync();
        else __syncthreads();
    };
    int round = 0;
    // joins over the block, then over the cluster; every thread gets the result
    auto all_stat = [&](float2 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = join_stat(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)), c);
        if (lane == 0) s.wstat[warp] = v;
        __syncthreads();
        if (warp == 0) {
            v = lane < VT / 32 ? s.wstat[lane] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v = join_stat(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)), c);
            if (lane < cs) *cl.map_shared_rank(&s.stat[round & 1][rank], lane) = v;
        }
        cluster_sync();
        v = (lane & 15) < cs ? s.stat[round & 1][lane & 15] : make_float2(-INFINITY, 0.0f);
        for (int o = cs / 2; o > 0; o >>= 1) v = join_stat(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)), c);
        v.x = __shfl_sync(0xffffffffu, v.x, 0), v.y = __shfl_sync(0xffffffffu, v.y, 0);
        round++;
        return v;
    };
    auto all_sum = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) s.wstat[warp].x = v;
        __syncthreads();
        if (warp == 0) {
            v = lane < VT / 32 ? s.wstat[lane].x : 0.0f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane < cs) cl.map_shared_rank(&s.stat[round & 1][rank], lane)->x = v;
        }
        cluster_sync();
        v = (lane & 15) < cs ? s.stat[round & 1][lane & 15].x : 0.0f;
        for (int o = cs / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        v = __shfl_sync(0xffffffffu, v, 0);
        round++;
        return v;
    };
    auto all_best = [&](Best v, bool last) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(0xffffffffu, v.v, o), __shfl_xor_sync(0xffffffffu, v.i, o)}, last);
        if (lane == 0) s.wbest[warp] = v;
        __syncthreads();
        if (warp == 0) {
            v = lane < VT / 32 ? s.wbest[lane] : Best{-INFINITY, -1};
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(0xffffffffu, v.v, o), __shfl_xor_sync(0xffffffffu, v.i, o)}, last);
            if (lane < cs) *cl.map_shared_rank(&s.best[round & 1][rank], lane) = v;
        }
        cluster_sync();
        v = (lane & 15) < cs ? s.best[round & 1][lane & 15] : Best{-INFINITY, -1};
        for (int o = cs / 2; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(0xffffffffu, v.v, o), __shfl_xor_sync(0xffffffffu, v.i, o)}, last);
        v.v = __shfl_sync(0xffffffffu, v.v, 0), v.i = __shfl_sync(0xffffffffu, v.i, 0);
        round++;
        return v;
    };
    // four values of a global row of this CTA's columns; `whole`: all of them are there (a load without a condition,
    // so that those of several steps are in flight together), else `fill` behind the end
    auto four = [&](const float *row, int v, float fill, auto whole) {
        if constexpr (whole.value) {
            if (VEC) return __ldg(reinterpret_cast<const float4 *>(row + v));
            return make_float4(__ldg(row + v), __ldg(row + v + 1), __ldg(row + v + 2), __ldg(row + v + 3));
        } else {
            float4 y = make_float4(fill, fill, fill, fill);
            if (v < len) y.x = row[v];
            if (v + 1 < len) y.y = row[v + 1];
            if (v + 2 < len) y.z = row[v + 2];
            return y;
        }
    };
    // f(column, four elements, whole) over this thread's columns of `node`'s row: from buffer `buf`, or, with PRE, from memory
    auto over_row = [&](int node, int buf, auto f) {
        const float4 *x = reinterpret_cast<const float4 *>(sm_rows + buf * per);
        const float *g = rows + (size_t)node * a.ld;
        const int end = len & ~3;
        int v = tid * 4;
#pragma unroll 4
        for (; v < end; v += VT * 4) f(v, PRE ? four(g, v, 0.0f, std::true_type{}) : x[v >> 2], std::true_type{});
        if (v < len4) f(v, PRE ? four(g, v, -INFINITY, std::false_type{}) : x[v >> 2], std::false_type{});
    };

    int node = 0, count = 1, buf = 0;
    bool ahead = false;  // the other buffer's copy (of the first child's row) has not been waited for
    if (rank == 0 && tid == 0) a.path[(size_t)b * a.N] = 0;
    for (;;) {
        const float *row = rows - w0 + (size_t)node * a.ld;
        const float *drow = a.draft ? a.draft + ((size_t)b * a.N + node) * a.ld_draft : nullptr;
        const int child = s.first[node];
        if (!PRE && two && child < a.N) start(child, buf ^ 1), ahead = true;
        for (int i = tid; i < (PRE ? 0 : a.N); i += VT) {
            if (i == 0 || s.parents[i] != node) continue;
            const int t = s.tokens[i];
            const bool in = t >= 0 && t < a.V;
            s.lx[i] = in ? row[t] : -INFINITY;
            if (drow) s.qx[i] = in ? drow[t] : 0.0f;
        }
        if (!PRE) finish(node, buf);
        int go = -1, nrej = 0;
        Best pick = {-INFINITY, -1};
        if (greedy) {
            over_row(node, buf, [&](int v, float4 x, auto whole) {
                const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; e++)  // columns ascend: the last of equal ones stays
                    if ((whole.value || v + e < len) && y[e] >= pick.v) pick = Best{y[e], w0 + v + e};
            });
            pick = all_best(pick, true);
            for (int i = child; i < a.N && go < 0; i = s.next[i])
                if (s.tokens[i] == pick.i) go = i;
        } else {
            float2 st = make_float2(-INFINITY, 0.0f);
            if (PRE) st = s.pm[node];
            if (!PRE) over_row(node, buf, [&](int, float4 x, auto) { st.x = fmaxf(st.x, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w))); });
            if (!PRE && st.x > -INFINITY) {
                over_row(node, buf, [&](int, float4 x, auto) {
                    st.y += (ex2((x.x - st.x) * c) + ex2((x.y - st.x) * c)) + (ex2((x.z - st.x) * c) + ex2((x.w - st.x) * c));
                });
            }
            if (!PRE) st = all_stat(st);
            const float m = st.x, inv = st.y > 0.0f ? 1.0f / st.y : 0.0f;
            auto prob = [&](float y) { return y > -INFINITY ? ex2((y - m) * c) * inv : 0.0f; };
            float sum_a = 0.0f, left = 1.0f;
            for (int i = child; i < a.N; i = s.next[i]) {
                float w = prob(s.lx[i]);
                if (drow) {
                    w = fmaxf(w - sum_a * s.qx[i], 0.0f);
                    if (s.u[i] * left * s.qx[i] < w) {
                        go = i;
                        break;
                    }
                    sum_a += left;
                    nrej++;
                    if (s.next[i] < a.N) {  // another child follows: it needs what is left
                        float t = 0.0f;
                        over_row(node, buf, [&](int v, float4 x, auto whole) {
                            const float4 q = four(drow + w0, v, 0.0f, whole);
                            t += (fmaxf(prob(x.x) - sum_a * q.x, 0.0f) + fmaxf(prob(x.y) - sum_a * q.y, 0.0f)) +
                                 (fmaxf(prob(x.z) - sum_a * q.z, 0.0f) + fmaxf(prob(x.w) - sum_a * q.w, 0.0f));
                        });
                        left = all_sum(t);
                    }
                } else {
                    for (int k = 0; k < nrej; k++)
                        if (s.rejected[k] == s.tokens[i]) w = 0.0f;
                    if (s.u[i] * left < w) {
                        go = i;
                        break;
                    }
                    left -= w;
                    __syncthreads();  // all have read the list
                    if (tid == 0) s.rejected[nrej] = s.tokens[i];
                    __syncthreads();
                    nrej++;
                }
            }
            if (go < 0) {
                for (int pass = 0; pass < 2; pass++) {
                    pick = Best{-INFINITY, -1};
                    auto race = [&](int v, const float(&y)[4], float4 e4, auto whole) {
                        const float n[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {  // columns ascend: the first of equal ones stays
                            const float t = y[e] > 0.0f ? __fdividef(y[e], n[e]) : 0.0f;
                            if ((whole.value || v + e < len) && t > pick.v) pick = Best{t, w0 + v + e};
                        }
                    };
                    if (pass == 0 && drow) {
                        over_row(node, buf, [&](int v, float4 x, auto whole) {
                            const float4 e4 = four(noise, v, 0.0f, whole), q = four(drow + w0, v, 0.0f, whole);
                            race(v, {prob(x.x) - sum_a * q.x, prob(x.y) - sum_a * q.y, prob(x.z) - sum_a * q.z, prob(x.w) - sum_a * q.w}, e4, whole);
                        });
                    } else {
                        const int gone = pass == 0 ? nrej : 0;
                        over_row(node, buf, [&](int v, float4 x, auto whole) {
                            const float4 e4 = four(noise, v, 0.0f, whole);
                            float y[4] = {prob(x.x), prob(x.y), prob(x.z), prob(x.w)};
                            for (int r = 0; r < gone; r++) {
                                const int k = s.rejected[r] - w0 - v;
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (k == e) y[e] = 0.0f;
                            }
                            race(v, y, e4, whole);
                        });
                    }
                    pick = all_best(pick, false);
                    if (pick.v > 0.0f) break;  // the same in every CTA
                }
            }
        }
        __syncthreads();  // the row, lx, qx and the list are free again
        if (ahead && (go < 0 || go != child)) {
            // a row that was not needed after all: its copy has to land before its buffer or the CTA goes
            if (bulk > 0 && !mbar_wait(smem_u32(&bars[buf ^ 1]), phase[buf ^ 1])) wait_failed(a.errors, WAIT_VERIFY);
            phase[buf ^ 1] ^= 1;
        }
        if (go < 0) {
            if (rank == 0) {
                if (tid == 0) {
                    a.n_accept[b] = count;
                    a.next[b] = max(pick.i, 0);
                }
                for (int i = count + tid; i < a.N; i += VT) a.path[(size_t)b * a.N + i] = -1;
            }
            break;
        }
        if (ahead && go == child) buf ^= 1;
        else if (!PRE) start(go, buf);
        ahead = false;
        node = go;
        if (rank == 0 && tid == 0) a.path[(size_t)b * a.N + count] = node;
        count++;
    }
    cluster_sync();  // no CTA leaves while another may still write to its shared memory
}

}  // namespace

// Rows of all nodes first: where reading them all takes less than the walk's
// steps, of about 4 us each (all rows of 1e8 bytes take 30 us).  With the draft's
// probabilities walks are long, since its tokens are mostly accepted.  Walk against
// all rows first, in us, V 128256 where not said:
//   chains with probabilities: 1 x 6 nodes, V 32000: 21.5, 10.0; 16 x 6, V 32000:
//     25.6, 12.1; 8 x 9 (3.7e7 bytes): 45, 21.5;
//   given tokens: 1 x 2, V 32000: 10.8, 9.8; 8 x 2: 14.2, 13.0; 32 x 2 (3.3e7 bytes):
//     23.4, 23.2; 4 x 26 (5.3e7): 22.5, 25.5; 32 x 6 (9.9e7): 28.9, 38.0;
//     32 x 26 (4.3e8): 34.7, 85;
//   a single node: 10.4, 9.9; 8 of them 10.6, 11.2.
bool verify_all_rows(const VerifyArgs &a) {
    return a.temperature >= 1e-8f && a.N > 1 && (double)a.B * a.N * a.V * 4 < (a.draft ? 1.0e8 : 4.0e7);
}
int verify_chunks(const VerifyArgs &a) { return ceil_div(a.V, ST * SE); }

int verify_launch(const VerifyArgs &a, float2 *part, cudaStream_t st) {
    const bool greedy = a.temperature < 1e-8f;
    auto aligned = [](const float *p, long long ld) { return ld % 4 == 0 && ((uintptr_t)p & 15) == 0; };
    const bool vec = aligned(a.logits, a.ld) && (greedy || (aligned(a.noise, a.ld_noise) && (!a.draft || aligned(a.draft, a.ld_draft))));
    const bool pre = part != nullptr;
    auto kern = pre ? (vec ? verify_kernel<true, true> : verify_kernel<false, true>) : (vec ? verify_kernel<true, false> : verify_kernel<false, false>);
    static bool ready[64][4] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    bool &done = ready[dev & 63][vec + 2 * pre];
    if (!done) {
        SB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        SB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_ROW));
        done = true;
    }
    if (pre) {
        const float c = 1.4426950408889634f / a.temperature;
        const dim3 grid((unsigned)(verify_chunks(a) * a.B * a.N));
        SB_CUDA_TRY(launch(vec ? verify_stats_kernel<true> : verify_stats_kernel<false>, grid, dim3(ST), 0, st, false, a.logits, a.ld, a.V,
                           verify_chunks(a), c, part));
    }
    // CTAs per sequence: as many as the SMs hold at once while each has 4096 columns, and at least what a row needs.
    // Clusters of 16 find room in few places: 8 chains of 8, V 128256, took 38.5 us with 16 and 29 with 8.
    int cs = 1;
    while (cs < 8 && a.B * cs * 2 <= device_props().sm_count && a.V >= 4096 * cs * 2) cs *= 2;
    while (!pre && cs < MAX_CS && (long long)(a.V / cs + 4) * 4 > MAX_ROW) cs *= 2;
    const long long per = ((a.V + cs - 1) / cs + 3) & ~3;
    SB_CHECK(pre || per * 4 <= MAX_ROW, SB_ERR_SHAPE, "verify: V %d", a.V);
    // the first child's row ahead: where both rows fit and the other CTAs of an SM are not in its way
    const int two = !pre && per * 8 <= MAX_ROW && (a.B * cs <= device_props().sm_count || per * 16 <= MAX_ROW);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.B * cs));
    cfg.blockDim = dim3(VT);
    cfg.dynamicSmemBytes = pre ? 0 : (size_t)per * 4 * (two ? 2 : 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pre ? 2 : 1;
    SB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, two, const_cast<const float2 *>(part), verify_chunks(a)));
    return SB_OK;
}

}  // namespace sb
