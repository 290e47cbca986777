// key_blocks.hip — which blocks of keys a query block's attention reads: per block a bound of every key in it,
// per query block an upper bound of the logits it can reach in each block, and the blocks of the largest.
//
// A block's keys lie, dim by dim, between lo and hi, so q . k <= sum_d max(q_d hi_d, q_d lo_d) for each of them.
// With q split by sign that sum is one product, [max(q, 0) | min(q, 0)] . [hi | lo] over 2 D values. Both sides
// are quantized like every other row here (amax / 127 per row, ties to even), so the product is exact
// in int32 whatever its order, and the two multiplications by the scales are the only roundings: the score and
// the selection are one well-defined answer, ties going to the lowest block.
//   score(query block, n) = max over its rows r (tokens x heads of the kv head) of (dot(r, n) * qs_r), times ks_n
// in f32 (rounded twice; the scale of the block is positive, so it may come after the maximum).
#include <math.h>

#include "attn_keys.h"

namespace e2mi {

struct BoundsArgs {
    const uint16_t *k;
    int64_t ldk;
    int Mk;
    const int32_t *k_start, *k_len;
    int max_k, KV, NB;
    int8_t *bounds;  // [B][NB][KV][2 D]: hi, lo
    float *scale;    // [B][NB][KV]
};

template <class T>
__device__ inline float value_of(uint16_t bits) { return (float)__builtin_bit_cast(T, bits); }

// One workgroup a block and kv head: its 64 keys' rows read once in 16-byte chunks (HBM-bound), the extremes
// joined through LDS.
template <class T, int D>
__global__ __launch_bounds__(256) void k_block_bounds(BoundsArgs a) {
    constexpr int CH = D / 8, RG = 256 / CH;  // chunks of a row, rows read at once
    __shared__ float s_hi[RG][D], s_lo[RG][D];
    __shared__ float s_amax[4];
    const int tid = threadIdx.x, n = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    int ks, nk;
    if (!key_range(a.k_start, a.k_len, b, a.max_k, a.Mk, ks, nk) || n * kKeyBlock >= nk) return;
    const int keys = min(kKeyBlock, nk - n * kKeyBlock);
    const int ch = tid % CH, rg = tid / CH;
    const uint16_t *kp = a.k + ((int64_t)ks + n * kKeyBlock) * a.ldk + (int64_t)kvh * D + ch * 8;
    float hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; e++) hi[e] = -INFINITY, lo[e] = INFINITY;
#pragma unroll
    for (int r = 0; r < kKeyBlock; r += RG) {
        if (r + rg < keys) {
            const uint4 x = *(const uint4 *)(kp + (int64_t)(r + rg) * a.ldk);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float f = value_of<T>((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
                hi[e] = fmaxf(hi[e], f);
                lo[e] = fminf(lo[e], f);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) s_hi[rg][ch * 8 + e] = hi[e], s_lo[rg][ch * 8 + e] = lo[e];
    __syncthreads();
    constexpr int PER = D > 256 ? 2 : 1;
    float h[PER], l[PER], am = 0.f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        h[i] = -INFINITY, l[i] = INFINITY;
        const int d = tid + 256 * i;
        if (d < D) {
#pragma unroll
            for (int r = 0; r < RG; r++) h[i] = fmaxf(h[i], s_hi[r][d]), l[i] = fminf(l[i], s_lo[r][d]);
            am = fmaxf(am, fmaxf(fabsf(h[i]), fabsf(l[i])));
        }
    }
    am = group_max<64>(am);
    if ((tid & 63) == 0) s_amax[tid >> 6] = am;
    __syncthreads();
    const QScale q = qscale(fmaxf(fmaxf(s_amax[0], s_amax[1]), fmaxf(s_amax[2], s_amax[3])));
    const int64_t slot = ((int64_t)b * a.NB + n) * a.KV + kvh;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int d = tid + 256 * i;
        if (d < D) {
            a.bounds[slot * 2 * D + d] = (int8_t)qbyte(h[i], q.inv);
            a.bounds[slot * 2 * D + D + d] = (int8_t)qbyte(l[i], q.inv);
        }
    }
    if (tid == 0) a.scale[slot] = q.sc;
}

struct SelectArgs {
    const uint16_t *q;
    int64_t ldq;
    int Mq;
    const int8_t *bounds;
    const float *kscale;
    const int32_t *q_start, *q_len, *k_len;
    int max_q, max_k, KV, G, NB, NQ, q_block, n_sel, n_first, n_local, causal;
    int group;   // rows set aside for a query block in a tile of 32: 4, 8, 16 or 32
    float *scores;  // [B][NQ][KV][NB]
    int32_t *sel;   // [B][NQ][KV][n_sel]
};

// Scores: a workgroup takes 32 / group query blocks (of up to 32 rows each; a query block of more rows takes
// all 32, tile after tile) against its share of the blocks, a wave 32 blocks at a time.
template <class T, int D>
__global__ __launch_bounds__(256) void k_block_scores(SelectArgs a) {
    constexpr int K2 = 2 * D, PITCH = K2 + 16;
    __shared__ __align__(16) int8_t s_q[32 * PITCH];
    __shared__ float s_sc[32];
    __shared__ int s_last[32];  // last key a row sees (-1: none)
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, half = lane >> 5;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int per = 32 / a.group;
    const int shares = (a.NB + 127) / 128;
    const int share = (int)(blockIdx.x % (unsigned)shares), qb0 = (int)(blockIdx.x / (unsigned)shares) * per;
    int qs, nq;
    if (!row_range(a.q_start, a.q_len, b, a.max_q, a.Mq, qs, nq)) return;
    if ((int64_t)qb0 * a.q_block >= nq) return;
    const int nk = max(0, min(a.k_len[b], a.max_k));
    const int n0 = share * 128 + w * 32;  // this wave's blocks
    const int n = n0 + (lane & 31);
    const int R = a.q_block * a.G;  // rows of a query block
    float best[8];
#pragma unroll
    for (int i = 0; i < 8; i++) best[i] = -INFINITY;
    v4i bf[K2 / 32];
    const bool some = n0 * kKeyBlock < nk;
    if (some) {
        const int64_t slot = ((int64_t)b * a.NB + min(n, (nk - 1) / kKeyBlock)) * a.KV + kvh;
#pragma unroll
        for (int s = 0; s < K2 / 32; s++) bf[s] = *(const v4i *)(a.bounds + slot * K2 + 32 * s + 16 * half);
    }
    for (int r0 = 0; r0 < (a.group == 32 ? R : 1); r0 += 32) {
        if (r0) __syncthreads();
        // quantize this tile's rows, a wave 8 of them
        for (int i = w; i < 32; i += 4) {
            const int blk = qb0 + i / a.group, in = r0 + i % a.group;
            const int64_t tok = (int64_t)blk * a.q_block + in / a.G;
            const bool row = in < R && tok < nq;
            float x[D / 64];
            float am = 0.f;
            const uint16_t *qp = a.q + (qs + (row ? tok : 0)) * a.ldq + (int64_t)(kvh * a.G + in % a.G) * D;
#pragma unroll
            for (int e = 0; e < D / 64; e++) {
                x[e] = row ? value_of<T>(qp[lane + 64 * e]) : 0.f;
                am = fmaxf(am, fabsf(x[e]));
            }
            const QScale q = qscale(group_max<64>(am));
#pragma unroll
            for (int e = 0; e < D / 64; e++) {
                const int v = qbyte(x[e], q.inv);
                s_q[i * PITCH + lane + 64 * e] = (int8_t)(v > 0 ? v : 0);
                s_q[i * PITCH + D + lane + 64 * e] = (int8_t)(v < 0 ? v : 0);
            }
            if (lane == 0) {
                s_sc[i] = q.sc;
                s_last[i] = !row ? -1 : a.causal ? (int)tok + nk - nq : nk - 1;
            }
        }
        __syncthreads();
        if (!some) continue;
        v16i acc = {};
#pragma unroll
        for (int s = 0; s < K2 / 32; s++)
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const v4i *)(s_q + (lane & 31) * PITCH + 32 * s + 16 * half), bf[s], acc, 0, 0, 0);
        // lane: block n; register r: row 8 (r / 4) + 4 half + r % 4; best[] holds runs of 4 rows
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = 8 * (r >> 2) + 4 * half + (r & 3);
            const float v = n * kKeyBlock <= s_last[row] ? __fmul_rn((float)acc[r], s_sc[row]) : -INFINITY;
            best[r >> 2] = fmaxf(best[r >> 2], v);
        }
    }
    if (!some) return;
    // runs of 4 rows: register i of half h is rows 8 i + 4 h .. + 3
    float other[4];
#pragma unroll
    for (int i = 0; i < 4; i++) other[i] = xor_lane<32>(best[i]);
    const float ks = n * kKeyBlock < nk ? a.kscale[((int64_t)b * a.NB + n) * a.KV + kvh] : 0.f;
    auto put = [&](int blk, float v) {
        if (n * kKeyBlock < nk && (int64_t)(qb0 + blk) * a.q_block < nq)
            a.scores[(((int64_t)b * a.NQ + qb0 + blk) * a.KV + kvh) * a.NB + n] = __fmul_rn(v, ks);
    };
    if (a.group == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) put(2 * i + half, best[i]);
        return;
    }
    if (half) return;
    float run[4];
#pragma unroll
    for (int i = 0; i < 4; i++) run[i] = fmaxf(best[i], other[i]);  // rows 8 i .. 8 i + 7
    if (a.group == 8) {
#pragma unroll
        for (int i = 0; i < 4; i++) put(i, run[i]);
    } else if (a.group == 16) {
        put(0, fmaxf(run[0], run[1]));
        put(1, fmaxf(run[2], run[3]));
    } else {
        put(0, fmaxf(fmaxf(run[0], run[1]), fmaxf(run[2], run[3])));
    }
}

// An order-preserving unsigned key of a score; NaN (an infinite bound times 0) comes last of those that may be taken.
__device__ inline uint32_t order_key(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    if (v != v) return 1;
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return k < 1 ? 1 : k > 0xfffffffeu ? 0xfffffffeu : k;
}

// The n_sel largest: the n_sel-th largest key by bisection of its 32 bits (counts by ballots over keys held in
// registers), then everything above it and the first of its equals, in block order. W waves a list, RPL keys
// a lane: key 64 (w RPL + j) + lane is register j of wave w.
template <int W, int RPL>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void k_block_top(SelectArgs a, int64_t lists) {
    constexpr int WG = W > 4 ? W : 4;  // waves a workgroup
    __shared__ int s_n[W > 1 ? 2 : 1][W];
    const int lane = threadIdx.x & 63, w = W > 1 ? threadIdx.x >> 6 : 0;
    const int64_t id = (int64_t)blockIdx.x * (WG / W) + (W > 1 ? 0 : threadIdx.x >> 6);
    if (id >= lists) return;
    const int qb = (int)(id / a.KV % a.NQ), b = (int)(id / a.KV / a.NQ);
    int32_t *out = a.sel + id * a.n_sel;
    int qs, nq;
    const bool has = row_range(a.q_start, a.q_len, b, a.max_q, a.Mq, qs, nq) && (int64_t)qb * a.q_block < nq;
    const int nk = max(0, min(a.k_len[b], a.max_k));
    const int t0 = qb * a.q_block, t1 = min(t0 + a.q_block, nq) - 1;
    const int far = !has ? -1 : a.causal ? min(t1 + nk - nq, nk - 1) : nk - 1;  // last key any row sees
    const int p0 = t0 + nk - nq, p1 = t1 + nk - nq;  // where the block's queries stand among the keys
    // local blocks: floor division, p may be negative where a sequence has fewer keys than queries
    const int l0 = (p0 >> 6) - (a.n_local - 1), l1 = (p1 >> 6) + (a.causal ? 0 : a.n_local - 1);
    const float *sc = a.scores + id * a.NB;
    uint32_t key[RPL];
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        const int n = 64 * (w * RPL + j) + lane;
        key[j] = 0;
        if (n < a.NB && (int64_t)n * kKeyBlock <= far)
            key[j] = n < a.n_first || (a.n_local > 0 && n >= l0 && n <= l1) ? 0xffffffffu : order_key(sc[n]);
    }
    int flip = 0;
    auto total = [&](int mine, int &before) {  // over the list's waves
        before = 0;
        if constexpr (W == 1) {
            return mine;
        } else {
            if (lane == 0) s_n[flip][w] = mine;
            __syncthreads();
            int all = 0;
            for (int i = 0; i < W; i++) {
                const int v = s_n[flip][i];
                before += i < w ? v : 0;
                all += v;
            }
            flip ^= 1;
            return all;
        }
    };
    auto count = [&](uint32_t from) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < RPL; j++) c += __popcll(__ballot(key[j] >= from));
        return c;
    };
    int before;
    uint32_t cut = 1;
    int above = 0;  // keys > cut that are taken; equals fill the rest
    if (total(count(1), before) > a.n_sel) {
        cut = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = cut | (1u << bit);
            if (total(count(c), before) >= a.n_sel) cut = c;
        }
        above = cut == 0xffffffffu ? 0 : total(count(cut + 1), before);
    } else {
        above = total(count(2), before);
    }
    const int room = a.n_sel - above;  // of the keys equal to cut
    // places: equals before this wave, taken before this wave
    int equal = 0, over = 0;
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        equal += __popcll(__ballot(key[j] == cut));
        over += __popcll(__ballot(key[j] > cut));
    }
    int eq_before, over_before;
    total(equal, eq_before);
    const int n_over = total(over, over_before);
    (void)n_over;
    int eq = eq_before, at = over_before + min(eq_before, room);
    const uint64_t low = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        const uint64_t me = __ballot(key[j] == cut);
        const bool take = key[j] > cut || (key[j] == cut && eq + __popcll(me & low) < room);
        const uint64_t mt = __ballot(take);
        if (take) out[at + __popcll(mt & low)] = 64 * (w * RPL + j) + lane;
        eq += __popcll(me);
        at += __popcll(mt);
    }
    // the rest of the list; the last wave's `at` is the number taken
    if (w == W - 1)
        for (int i = at + lane; i < a.n_sel; i += 64) out[i] = -1;
}

template <class T, int D>
static int launch_bounds_of(hipStream_t st, const BoundsArgs &a, int B) {
    hipLaunchKernelGGL((k_block_bounds<T, D>), dim3(a.NB, a.KV, B), dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "block bounds launch");
}
template <class T, int D>
static int launch_scores(hipStream_t st, const SelectArgs &a, int B) {
    const int64_t tiles = ((int64_t)a.NQ * a.group + 31) / 32, grid = tiles * ((a.NB + 127) / 128);
    if (grid > 0x7fffffff) {
        set_error("block_select: too many rows for a launch");
        return -1;
    }
    hipLaunchKernelGGL((k_block_scores<T, D>), dim3((unsigned)grid, a.KV, B), dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "block scores launch");
}

#define E2MI_BY_TYPE(call, dtype, D, ...)                                                             \
    ((dtype) == E2MI_F16 ? ((D) == 64 ? call<_Float16, 64>(__VA_ARGS__) : (D) == 128 ? call<_Float16, 128>(__VA_ARGS__) \
                            : (D) == 256 ? call<_Float16, 256>(__VA_ARGS__) : call<_Float16, 512>(__VA_ARGS__))          \
                         : ((D) == 64 ? call<__bf16, 64>(__VA_ARGS__) : (D) == 128 ? call<__bf16, 128>(__VA_ARGS__)     \
                            : (D) == 256 ? call<__bf16, 256>(__VA_ARGS__) : call<__bf16, 512>(__VA_ARGS__)))

static bool head_fits(int dtype, int D) {
    return (dtype == E2MI_F16 || dtype == E2MI_BF16) && (D == 64 || D == 128 || D == 256 || D == 512);
}
constexpr int kMaxBlocks = 32768;  // blocks of a sequence that a selection ranks (2^21 keys)

}  // namespace e2mi

using namespace e2mi;

extern "C" int e2mi_block_bounds(e2mi_stream stream, int dtype, const uint16_t *k, int64_t ldk, int Mk, const int32_t *k_start,
                                 const int32_t *k_len, int B, int max_k, int KV, int D, int8_t *bounds, float *scale) {
    if (!head_fits(dtype, D) || Mk < 0 || B < 0 || B > 65535 || max_k < 0 || max_k > 0x7fffff00 || KV <= 0 || KV > 65535) {
        set_error("block_bounds: needs f16 or bf16 rows, head_dim 64, 128, 256 or 512 and B, KV <= 65535 (type %d B=%d Mk=%d max_k=%d "
                  "KV=%d D=%d)", dtype, B, Mk, max_k, KV, D);
        return -1;
    }
    if (!k || !aligned16(k) || ldk < (int64_t)KV * D || ldk % 8 || ldk > (1LL << 28) || !k_start || !k_len || !bounds ||
        !aligned16(bounds) || !scale) {
        set_error("block_bounds: needs row ranges, 16-byte aligned k rows (pitch >= KV * D in multiples of 8) and bounds, and scales");
        return -1;
    }
    if (!Mk || !B || !max_k) return 0;
    const BoundsArgs a = {k, ldk, Mk, k_start, k_len, max_k, KV, (max_k + kKeyBlock - 1) / kKeyBlock, bounds, scale};
    return E2MI_BY_TYPE(launch_bounds_of, dtype, D, (hipStream_t)stream, a, B);
}

extern "C" size_t e2mi_block_select_workspace_bytes(int B, int max_q, int max_k, int KV, int q_block) {
    if (B <= 0 || max_q <= 0 || max_k <= 0 || KV <= 0 || q_block <= 0) return 0;
    return (size_t)B * (((size_t)max_q + q_block - 1) / q_block) * KV * (((size_t)max_k + kKeyBlock - 1) / kKeyBlock) * 4;
}

extern "C" int e2mi_block_select(e2mi_stream stream, int dtype, const uint16_t *q, int64_t ldq, int Mq, const int8_t *bounds,
                                 const float *scale, const int32_t *q_start, const int32_t *q_len, const int32_t *k_len, int B,
                                 int max_q, int max_k, int H, int KV, int D, int q_block, int n_sel, int n_first, int n_local,
                                 int causal, int32_t *sel, void *workspace, size_t workspace_bytes) {
    if (!head_fits(dtype, D) || Mq < 0 || B < 0 || B > 65535 || max_q < 0 || max_k < 0 || max_k > kMaxBlocks * kKeyBlock || H <= 0 ||
        KV <= 0 || KV > 65535 || H % KV || H > 65535 || q_block <= 0 || q_block > 1024 || n_sel <= 0 || n_sel > kMaxSelect ||
        (int64_t)max_q * (H / KV) > 0x7fffff00 || (int64_t)Mq * (H / KV) > 0x7fffff00) {
        set_error("block_select: needs f16 or bf16 rows, head_dim 64, 128, 256 or 512, H %% KV == 0, max_k <= %d, 1 <= q_block <= 1024, 1 <= "
                  "n_sel <= %d (type %d B=%d Mq=%d max_q=%d max_k=%d H=%d KV=%d D=%d q_block=%d n_sel=%d)", kMaxBlocks * kKeyBlock,
                  kMaxSelect, dtype, B, Mq, max_q, max_k, H, KV, D, q_block, n_sel);
        return -1;
    }
    // blocks that a query block's own places touch at most, with the neighbours on each side asked for
    const int64_t local = n_local > 0 ? (q_block - 1 + kKeyBlock - 1) / kKeyBlock + 1 + (int64_t)(n_local - 1) * (causal ? 1 : 2) : 0;
    if (n_first < 0 || n_local < 0 || (int64_t)n_first + local > n_sel) {
        set_error("block_select: n_first + the local blocks (%lld) must fit in n_sel (n_first=%d n_local=%d n_sel=%d)", (long long)local,
                  n_first, n_local, n_sel);
        return -1;
    }
    if (!q || !aligned16(q) || ldq < (int64_t)H * D || ldq % 8 || ldq > (1LL << 28) || !q_start || !q_len || !k_len || !sel ||
        (max_k && (!bounds || !scale || !aligned16(bounds)))) {
        set_error("block_select: needs row ranges, 16-byte aligned q rows (pitch >= H * D in multiples of 8), bounds, scales and sel");
        return -1;
    }
    const size_t need = e2mi_block_select_workspace_bytes(B, max_q, max_k, KV, q_block);
    if (need && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < need)) {
        set_error("block_select: needs a workspace of %zu bytes (%zu given)", need, workspace_bytes);
        return -1;
    }
    if (!B || !max_q) return 0;
    const int G = H / KV, R = q_block * G;
    SelectArgs a = {};
    a.q = q, a.ldq = ldq, a.Mq = Mq, a.bounds = bounds, a.kscale = scale, a.q_start = q_start, a.q_len = q_len, a.k_len = k_len;
    a.max_q = max_q, a.max_k = max_k, a.KV = KV, a.G = G, a.NB = (max_k + kKeyBlock - 1) / kKeyBlock;
    a.NQ = (max_q + q_block - 1) / q_block, a.q_block = q_block, a.n_sel = n_sel, a.n_first = n_first, a.n_local = n_local;
    a.causal = causal != 0, a.scores = (float *)workspace, a.sel = sel;
    a.group = R <= 4 ? 4 : R <= 8 ? 8 : R <= 16 ? 16 : 32;
    const hipStream_t st = (hipStream_t)stream;
    if (a.NB && Mq && E2MI_BY_TYPE(launch_scores, dtype, D, st, a, B)) return -1;
    const int64_t lists = (int64_t)B * a.NQ * KV;
    if (lists > 0x7fffffff) {
        set_error("block_select: too many lists for a launch");
        return -1;
    }
    const unsigned n = (unsigned)lists;
    if (a.NB <= 512) hipLaunchKernelGGL((k_block_top<1, 8>), dim3((n + 3) / 4), dim3(256), 0, st, a, lists);
    else if (a.NB <= 2048) hipLaunchKernelGGL((k_block_top<1, 32>), dim3((n + 3) / 4), dim3(256), 0, st, a, lists);
    else if (a.NB <= 8192) hipLaunchKernelGGL((k_block_top<4, 32>), dim3(n), dim3(256), 0, st, a, lists);
    else hipLaunchKernelGGL((k_block_top<16, 32>), dim3(n), dim3(1024), 0, st, a, lists);
    return check_hip(hipGetLastError(), "block selection launch");
}
