// attn_keys.hip — attention of packed sequences over a prefix that all of them share, and over blocks of 64
// keys that a list selects for each block of queries (16-bit rows, V transposed, GQA, optionally causal).
//
// A row here is one token of one head. The G = H / KV heads of a kv head read the same keys, so a token's G
// rows lie side by side in a tile: single tokens of grouped heads fill it G times as far, and K and V are
// read once for all of them. Row r of a sequence is token r / G, head kvh * G + r % G.
//
// One pass with the running maximum m and sum l of a softmax (base 2, logits times scale * log2 e):
//   t = c2 q.k,  m' = max(m, t),  o = 2^(m - m') o + sum 2^(t - m') v,  l = 2^(m - m') l + sum 2^(t - m')
// in f32, the probabilities rounded to the rows' type for the second product (half a step of each, with
// random signs: as far off as the output's own rounding). Keys may be shared out: each share leaves (o, m, l),
// and k_keys_merge joins them in the order of the shares, so results do not depend on timing.
//
// S^T = K Q^T by 32x32x16 MFMA with the 32 keys in an order (bits 2 and 3 of the index exchanged) that leaves
// in a lane's registers 8 j .. 8 j + 7 the consecutive keys 16 j + 8 half + 0 .. 7 of one row, which is the
// operand order of O^T += V^T P^T: probabilities go from registers to the next product, V^T is read in
// 16-byte chunks of 8 keys.
#include <math.h>

#include "attn_keys.h"

namespace e2mi {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <class T>
struct Half8;
template <>
struct Half8<_Float16> {
    typedef h8 type;
    static __device__ inline f16v mma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Half8<__bf16> {
    typedef b8 type;
    static __device__ inline f16v mma(b8 a, b8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

enum { kOwnRows = 0, kAllRows = 1, kSelected = 2 };  // whose rows against which keys (k_keys_few)

// One tile of the running softmax: 16 logits of one row per lane (its partner lane ^ 32 holds the other 16).
// The running maximum moves only when a tile exceeds it by more than kTau, so p <= 2^kTau and most tiles need
// no rescale of o: the same softmax, divided by the same sum at the end. Returns the rescale.
constexpr float kTau = 8.f;
template <class T>
__device__ __forceinline__ float softmax_step(const float (&s)[16], float c, float &mrun, float &lrun,
                                              typename Half8<T>::type (&pb)[2]) {
    float mloc = s[0];
#pragma unroll
    for (int r = 1; r < 16; r++) mloc = fmaxf(mloc, s[r]);
    mloc = fmaxf(mloc, xor_lane<32>(mloc));
    const float mc = mloc * c;
    float alpha = 1.f;
    if (mc > mrun + kTau) {
        alpha = __builtin_amdgcn_exp2f(mrun - mc);
        mrun = mc;
    }
    const float ms = mrun == -INFINITY ? 0.f : mrun;  // no key yet: every p is 0
    float psum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -ms));
        psum += p;
        pb[r >> 3][r & 7] = (T)p;
    }
    lrun = lrun * alpha + psum;
    return alpha;
}

// 8 consecutive values at any 2-byte address (V^T's pitch may be odd): one 16-byte load, unaligned
template <class T>
__device__ inline typename Half8<T>::type load8(const uint16_t *p) {
    struct __attribute__((packed, aligned(2))) Any {
        typename Half8<T>::type v;
    };
    return ((const Any *)p)->v;
}

__device__ inline int swap23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// Writes a row's context (a lane holds dims 32 t + 8 g + 4 half + 0..3 of its row, o already divided by the
// sum): 16-bit rows, and per 128 dims the quantized pair of the O projection.
template <class T, int D>
__device__ __forceinline__ void write_row(const KeysArgs &a, const f16v (&o)[D / 32], int64_t m, int h, int half) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    if (a.ctx) {
        T *y = (T *)a.ctx + m * a.ldc + (int64_t)h * D + 4 * half;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4 v = {(T)o[t][4 * g], (T)o[t][4 * g + 1], (T)o[t][4 * g + 2], (T)o[t][4 * g + 3]};
                *(v4 *)(y + 32 * t + 8 * g) = v;
            }
    }
    if constexpr (D % 128 == 0) {
        if (a.cq) {
            const int64_t row = m * a.H + h;
#pragma unroll
            for (int blk = 0; blk < D / 128; blk++) {
                float am = 0.f;
#pragma unroll
                for (int t = 4 * blk; t < 4 * blk + 4; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++) am = fmaxf(am, fabsf(o[t][r]));
                am = fmaxf(am, xor_lane<32>(am));
                const QScale qs = qscale(am);
#pragma unroll
                for (int t = 4 * blk; t < 4 * blk + 4; t++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *(uint32_t *)(a.cq + row * D + 32 * t + 8 * g + 4 * half) =
                            pack4_magic(o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3], qs.inv);
                if (half == 0) a.cs[row * (D / 128) + blk] = qs.sc;
            }
        }
    }
}

// The blocks of a selection list that hold keys this tile may see, compacted in list order into LDS; returns
// their number (every thread of the workgroup). blocks: those below it may be read.
__device__ inline int read_list(const int32_t *sel, int n_sel, int blocks, int *list, int *count) {
    if (threadIdx.x < 64) {
        int n = 0;
        for (int i = 0; i < n_sel; i += 64) {
            const int e = i + (int)threadIdx.x < n_sel ? sel[i + threadIdx.x] : -1;
            const bool keep = e >= 0 && e < blocks;
            const uint64_t mask = __ballot(keep);
            if (keep) list[n + __popcll(mask & ((1ull << threadIdx.x) - 1))] = e;
            n += __popcll(mask);
        }
        if (threadIdx.x == 0) *count = n;
    }
    __syncthreads();
    return *count;
}

// 32 rows a workgroup; its four waves take every fourth key tile of 32 and are joined through LDS. Fragments
// go from global memory to registers: a tile's K and V^T are read by one wave only, so LDS would hold them for
// nobody else, and the reads in flight are bounded by registers, not by LDS.
template <class T, int D, int MODE>
__global__ __launch_bounds__(256, D == 512 ? 1 : 2) void k_keys_few(KeysArgs a) {
    typedef typename Half8<T>::type V8;
    constexpr int NQ = D / 16, NO = D / 32;
    extern __shared__ __align__(16) float few_smem[];  // two waves' o (join); the list (kSelected)
    __shared__ float s_m[4][32], s_l[4][32];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, half = lane >> 5;
    const int kvh = blockIdx.y, b = blockIdx.z, G = a.G;
    const int part = (int)(blockIdx.x % (unsigned)a.parts), tile = (int)(blockIdx.x / (unsigned)a.parts);

    int qs = 0, nq = a.Mq, ks = 0, nk = 0;
    if constexpr (MODE != kAllRows) {
        if (!row_range(a.q_start, a.q_len, b, a.max_q, a.Mq, qs, nq)) return;
        if (a.own.rows) key_range(a.k_start, a.k_len, b, a.max_k, a.own.rows, ks, nk);
    }
    // this tile's rows
    int tok0 = 0, ntok = nq, r0 = tile * 32;
    if constexpr (MODE == kSelected) {
        const int per = (a.q_block * G + 31) / 32;
        tok0 = tile / per * a.q_block;
        ntok = min(a.q_block, nq - tok0);
        r0 = tile % per * 32;
    }
    const int rows = ntok * G;
    if (r0 >= rows) return;
    const int r = r0 + (lane & 31), rc = min(r, rows - 1);
    const int tok = tok0 + rc / G, h = kvh * G + rc % G;
    const int64_t m = (int64_t)qs + tok;
    const int back = nk - nq;  // token i stands at own key i + back
    const int last = a.causal ? tok + back : nk - 1;
    const int far = a.causal ? min(nk, tok0 + (min(r0 + 31, rows - 1)) / G + back + 1) : nk;  // own keys any row here sees

    // its key tiles
    int n_pre = 0, n_own = 0;
    int *list = (int *)few_smem;
    if constexpr (MODE == kSelected) {
        const int32_t *sel = a.sel + (((int64_t)b * a.NQ + tok0 / a.q_block) * a.KV + kvh) * a.n_sel;
        n_own = 2 * read_list(sel, a.n_sel, far > 0 ? (far + kKeyBlock - 1) / kKeyBlock : 0, list, &s_count);
    } else {
        n_pre = (a.pre.rows + 31) / 32;
        if (MODE == kOwnRows && far > 0) n_own = (far + 31) / 32;
    }
    const int n = n_pre + n_own;
    const int t0 = (int)((int64_t)n * part / a.parts), t1 = (int)((int64_t)n * (part + 1) / a.parts);

    V8 qf[NQ];
    {
        const uint16_t *qp = a.q + m * a.ldq + (int64_t)h * D + 8 * half;
#pragma unroll
        for (int s = 0; s < NQ; s++) qf[s] = *(const V8 *)(qp + 16 * s);
    }
    f16v o[NO];
#pragma unroll
    for (int t = 0; t < NO; t++) o[t] = (f16v){};
    float mrun = -INFINITY, lrun = 0.f;

    for (int t = t0 + w; t < t1; t += 4) {
        const bool pre = t < n_pre;
        const KeySet &src = pre ? a.pre : a.own;
        int key0;
        if constexpr (MODE == kSelected) key0 = list[t >> 1] * kKeyBlock + (t & 1) * 32;
        else key0 = (pre ? t : t - n_pre) * 32;
        const int lim = pre ? src.rows : nk;  // keys of this range
        if (MODE == kSelected && key0 >= lim) continue;
        const int64_t base = pre ? 0 : ks;
        const uint16_t *kp = src.k + (base + min(key0 + swap23(lane & 31), lim - 1)) * src.ldk + (int64_t)kvh * D + 8 * half;
        f16v st = (f16v){};
#pragma unroll
        for (int s = 0; s < NQ; s++) st = Half8<T>::mma(*(const V8 *)(kp + 16 * s), qf[s], st);
        float tv[16];
#pragma unroll
        for (int i = 0; i < 16; i++) tv[i] = st[i];
        const bool short_tile = key0 + 32 > lim;
        if (short_tile || (!pre && a.causal)) {
            const int top = pre ? lim - 1 : min(last, lim - 1);
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (key0 + 16 * (i >> 3) + 8 * half + (i & 7) > top) tv[i] = -INFINITY;
        }
        V8 pb[2];
        const float alpha = softmax_step<T>(tv, a.c2, mrun, lrun, pb);
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < NO; i++) o[i] *= alpha;
        }
        const uint16_t *vp = src.vt + ((int64_t)kvh * D + (lane & 31)) * src.ldv + base + key0 + 8 * half;
        if (!short_tile) {
#pragma unroll
            for (int i = 0; i < 2 * NO; i++)
                o[i >> 1] = Half8<T>::mma(load8<T>(vp + (int64_t)(i >> 1) * 32 * src.ldv + 16 * (i & 1)), pb[i & 1], o[i >> 1]);
        } else {
            // values past the range are not read (they may lie past the tensor) and count as 0: a zero
            // probability times an infinity would be a NaN
            const int left = lim - key0 - 8 * half;
            for (int i = 0; i < 2 * NO; i++) {
                const int have = left - 16 * (i & 1);
                const uint16_t *x = vp + (int64_t)(i >> 1) * 32 * src.ldv + 16 * (i & 1);
                V8 vf = {};
                if (have >= 8) {
                    vf = load8<T>(x);
                } else {
#pragma unroll
                    for (int e = 0; e < 7; e++)
                        if (e < have) vf[e] = __builtin_bit_cast(T, x[e]);
                }
#pragma unroll
                for (int u = 0; u < NO; u++)
                    if (u == i >> 1) o[u] = Half8<T>::mma(vf, pb[i & 1], o[u]);
            }
        }
    }

    // join the four waves: a common maximum, then two by two through LDS
    float lsum = lrun + xor_lane<32>(lrun);
    if (half == 0) s_m[w][lane] = mrun, s_l[w][lane] = lsum;
    __syncthreads();  // the list is no longer read
    const int c = lane & 31;
    const float mall = fmaxf(fmaxf(s_m[0][c], s_m[1][c]), fmaxf(s_m[2][c], s_m[3][c]));
    auto share = [&](float mp) { return mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - mall); };
    lsum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) lsum += s_l[i][c] * share(s_m[i][c]);
    const float mine = share(mrun);
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] *= mine;
    constexpr int kWave = NO * 16 * 64;  // floats of one wave's o
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (w >= step && w < 2 * step) {
            float *buf = few_smem + (w - step) * kWave + lane;
#pragma unroll
            for (int i = 0; i < NO * 16; i++) buf[i * 64] = o[i >> 4][i & 15];
        }
        __syncthreads();
        if (w < step) {
            const float *buf = few_smem + w * kWave + lane;
#pragma unroll
            for (int i = 0; i < NO * 16; i++) o[i >> 4][i & 15] += buf[i * 64];
        }
        if (step > 1) __syncthreads();
    }
    if (w || r >= rows) return;
    if (a.part_o) {
        const int64_t row = ((int64_t)(a.part0 + part) * a.Mq + m) * a.H + h;
        // no key: nothing but the maximum says so; a NaN sum (NaN rows) takes the whole row with it
        if (half == 0) *(float2 *)(a.part_ml + row * 2) = make_float2(lsum == lsum ? mall : INFINITY, lsum);
        if (lsum == 0.f) return;
        float *y = a.part_o + row * D + 4 * half;
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *(float4 *)(y + 32 * i + 8 * g) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        return;
    }
    const float inv = lsum == 0.f ? 0.f : __fdiv_rn(1.f, lsum);
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] *= inv;
    write_row<T, D>(a, o, m, h, half);
}

// Joins the shares of a row: a wave a row, lane p holding share p's maximum and sum, then D / 64 dims a lane.
template <class T, int D>
__global__ __launch_bounds__(256) void k_keys_merge(KeysArgs a) {
    constexpr int VW = D / 64;
    typedef float vf __attribute__((ext_vector_type(VW)));
    typedef T vt __attribute__((ext_vector_type(VW)));
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, b = blockIdx.z;
    int qs, nq;
    if (!row_range(a.q_start, a.q_len, b, a.max_q, a.Mq, qs, nq)) return;
    const int64_t i = (int64_t)blockIdx.x * 4 + w;
    if (i >= (int64_t)nq * a.H) return;
    const int64_t row = (int64_t)qs * a.H + i, pitch = (int64_t)a.Mq * a.H;
    float mp = -INFINITY, lp = 0.f;
    if (lane < a.all_parts) {
        const float2 ml = *(const float2 *)(a.part_ml + (lane * pitch + row) * 2);
        mp = ml.x, lp = ml.y;
    }
    const float mall = group_max<64>(mp);
    const float wp = mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - mall);
    const float sum = group_sum<64>(wp * lp);
    vf o = {};
    for (int p = 0; p < a.all_parts; p++) {
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wp), p));
        if (__builtin_bit_cast(int, f) == 0) continue;  // a share without keys left no o
        const vf v = *(const vf *)(a.part_o + (p * pitch + row) * D + lane * VW);
        o += v * f;
    }
    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
    o *= inv;
    const int64_t m = qs + i / a.H, h = i % a.H;
    if (a.ctx) {
        vt y;
#pragma unroll
        for (int e = 0; e < VW; e++) y[e] = (T)o[e];
        *(vt *)((T *)a.ctx + m * a.ldc + h * D + lane * VW) = y;
    }
    if constexpr (D % 128 == 0) {
        if (a.cq) {
            constexpr int LB = 128 / VW;  // lanes of a 128-dim block
            float am = 0.f;
#pragma unroll
            for (int e = 0; e < VW; e++) am = fmaxf(am, fabsf(o[e]));
            am = group_max<LB>(am);
            const QScale q = qscale(am);
            typedef int8_t vq __attribute__((ext_vector_type(VW)));
            vq y;
#pragma unroll
            for (int e = 0; e < VW; e++) y[e] = (int8_t)qbits(o[e], q.inv);
            *(vq *)(a.cq + row * D + lane * VW) = y;
            if (lane % LB == 0) a.cs[row * (D / 128) + lane / LB] = q.sc;
        }
    }
}

// ---- host: plan, checks, launches

struct KeysPlan {
    bool apart = false;           // the prefix by rows of all sequences, their own keys by sequence
    int pre_parts = 0, parts = 1;  // shares of the prefix (apart) and of the other launch
    int all() const { return pre_parts + parts; }
    bool merged() const { return all() > 1; }
};

// Shares for a launch of `groups` workgroups whose longest walk is `tiles` key tiles of 32: enough to give every
// CU two workgroups, at least 8 tiles (two a wave) each.
static int key_shares(int64_t groups, int64_t tiles, int most) {
    const int64_t want = (2L * num_cus() + groups - 1) / groups;
    int64_t n = want < tiles / 8 ? want : tiles / 8;
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

static KeysPlan plan_prefix(int Mq, int P, int B, int max_q, int max_k, int H, int KV) {
    KeysPlan p;
    const int G = H / KV;
    const int64_t own_tiles = ((int64_t)max_k + 31) / 32, pre_tiles = ((int64_t)P + 31) / 32;
    const int64_t seq_groups = (((int64_t)max_q * G + 31) / 32) * KV * B;
    // sequences of less than a tile share the prefix's tiles
    p.apart = B > 1 && P > 0 && (int64_t)max_q * G < 32;
    if (p.apart) {
        p.pre_parts = key_shares(((int64_t)Mq * G + 31) / 32 * KV, pre_tiles, kMaxKeyParts / 2);
        p.parts = key_shares(seq_groups, own_tiles, kMaxKeyParts / 2);
    } else {
        p.parts = key_shares(seq_groups, own_tiles + pre_tiles, kMaxKeyParts);
    }
    return p;
}

static KeysPlan plan_blocks(int B, int max_q, int H, int KV, int q_block, int n_sel) {
    KeysPlan p;
    const int G = H / KV;
    const int64_t groups = (((int64_t)q_block * G + 31) / 32) * (((int64_t)max_q + q_block - 1) / q_block) * KV * B;
    p.parts = key_shares(groups, 2 * (int64_t)n_sel, kMaxKeyParts);
    return p;
}

static size_t part_bytes(const KeysPlan &p, int Mq, int H, int D) {
    return p.merged() ? (size_t)p.all() * Mq * H * (D + 2) * 4 : 0;
}

template <class T, int D, int MODE>
static int launch_few(hipStream_t st, const KeysArgs &a, int64_t tiles, int B) {
    constexpr size_t lds = (size_t)D * 128 * 2 > kMaxSelect * 4 ? (size_t)D * 128 * 2 : kMaxSelect * 4;
    if (tiles * a.parts > 0x7fffffff) {
        set_error("attention over keys: too many rows for a launch");
        return -1;
    }
    if (lds > 65536 && check_hip(hipFuncSetAttribute((const void *)k_keys_few<T, D, MODE>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "lds attribute"))
        return -1;
    hipLaunchKernelGGL((k_keys_few<T, D, MODE>), dim3((unsigned)(tiles * a.parts), a.KV, B), dim3(256), lds, st, a);
    return check_hip(hipGetLastError(), "attention launch");
}

template <class T, int D>
static int run_keys(hipStream_t st, KeysArgs a, const KeysPlan &p, void *workspace) {
    const int G = a.G;
    if (p.merged()) {
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + (size_t)p.all() * a.Mq * a.H * D;
    }
    a.all_parts = p.all();
    if (a.sel) {
        a.parts = p.parts;
        const int64_t tiles = ((int64_t)a.q_block * G + 31) / 32 * a.NQ;
        if (launch_few<T, D, kSelected>(st, a, tiles, a.B)) return -1;
    } else {
        if (p.apart) {
            a.parts = p.pre_parts;
            if (launch_few<T, D, kAllRows>(st, a, ((int64_t)a.Mq * G + 31) / 32, 1)) return -1;
            a.part0 = p.pre_parts;
            a.pre = {};
        }
        a.parts = p.parts;
        if (launch_few<T, D, kOwnRows>(st, a, ((int64_t)a.max_q * G + 31) / 32, a.B)) return -1;
    }
    if (!p.merged()) return 0;
    hipLaunchKernelGGL((k_keys_merge<T, D>), dim3((unsigned)(((int64_t)a.max_q * a.H + 3) / 4), 1, a.B), dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "attention merge launch");
}

static int run_keys(hipStream_t st, int dtype, int D, const KeysArgs &a, const KeysPlan &p, void *workspace) {
#define E2MI_KEYS(DIM)                                                         \
    case DIM:                                                                  \
        return dtype == E2MI_F16 ? run_keys<_Float16, DIM>(st, a, p, workspace) \
                                 : run_keys<__bf16, DIM>(st, a, p, workspace)
    switch (D) {
        E2MI_KEYS(64);
        E2MI_KEYS(128);
        E2MI_KEYS(256);
        default:
            return dtype == E2MI_F16 ? run_keys<_Float16, 512>(st, a, p, workspace) : run_keys<__bf16, 512>(st, a, p, workspace);
    }
#undef E2MI_KEYS
}

// sizes that the plans and the kernels' index arithmetic take
static bool sizes_fit(int Mq, int B, int max_q, int max_k, int H, int KV, int D) {
    return (D == 64 || D == 128 || D == 256 || D == 512) && Mq >= 0 && B >= 0 && B <= 65535 && max_q >= 0 && max_k >= 0 &&
           H > 0 && KV > 0 && KV <= 65535 && H % KV == 0 && H <= 65535 && (int64_t)Mq * (H / KV) < 0x7fffff00 &&
           (int64_t)max_q * (H / KV) < 0x7fffff00 && max_k < 0x7fffff00;
}

static int check_keys(const char *who, const char *what, const KeySet &s, int KV, int D) {
    if (s.rows < 0 || (s.rows && (!s.k || !s.vt || !aligned16(s.k) || (uintptr_t)s.vt % 2 || s.ldk < (int64_t)KV * D ||
                                  s.ldk % 8 || s.ldv < s.rows || s.ldk > (1LL << 28) || s.ldv > (1LL << 31)))) {
        set_error("%s: %s need 16-byte aligned k rows of a pitch >= KV * D in multiples of 8 and transposed v of a pitch >= "
                  "rows (rows=%d ldk=%lld ldv=%lld)", who, what, s.rows, (long long)s.ldk, (long long)s.ldv);
        return -1;
    }
    return 0;
}

static int check_call(const char *who, int dtype, const KeysArgs &a, int D, float scale) {
    if (dtype != E2MI_F16 && dtype != E2MI_BF16) {
        set_error("%s: needs f16 or bf16 rows (type %d)", who, dtype);
        return -1;
    }
    if (!sizes_fit(a.Mq, a.B, a.max_q, a.max_k, a.H, a.KV, D) || !(scale > 0.f) || !(scale < INFINITY)) {
        set_error("%s: needs head_dim 64, 128, 256 or 512, H %% KV == 0, B <= 65535 and a finite scale > 0 (B=%d Mq=%d max_q=%d "
                  "max_k=%d H=%d KV=%d D=%d scale=%g)", who, a.B, a.Mq, a.max_q, a.max_k, a.H, a.KV, D, (double)scale);
        return -1;
    }
    const int64_t w = (int64_t)a.H * D;
    if (!a.q || !aligned16(a.q) || a.ldq < w || a.ldq % 8 || a.ldq > (1LL << 28) || !a.q_start || !a.q_len || !a.k_start || !a.k_len) {
        set_error("%s: needs row ranges and 16-byte aligned q rows of a pitch >= H * D in multiples of 8", who);
        return -1;
    }
    if ((!a.ctx && !a.cq) || (a.cq != nullptr) != (a.cs != nullptr) || (a.cq && D % 128) || ((uintptr_t)a.cq & 7) ||
        (a.ctx && (!aligned16(a.ctx) || a.ldc < w || a.ldc % 8 || a.ldc > (1LL << 28)))) {
        set_error("%s: needs ctx (16-byte aligned, pitch >= H * D in multiples of 8) or ctx_q with ctx_s (8-byte aligned, head_dim a "
                  "multiple of 128)", who);
        return -1;
    }
    return check_keys(who, "keys", a.own, a.KV, D);
}

static int check_workspace(const char *who, size_t need, const void *ws, size_t have) {
    if (need && (!ws || !aligned16(ws) || have < need)) {
        set_error("%s: needs a 16-byte aligned workspace of %zu bytes (%zu given)", who, need, have);
        return -1;
    }
    return 0;
}

}  // namespace e2mi

using namespace e2mi;

extern "C" size_t e2mi_attention_prefix_workspace_bytes(int Mq, int P, int B, int max_q, int max_k, int H, int KV, int D) {
    if (!sizes_fit(Mq, B, max_q, max_k, H, KV, D) || P < 0 || !Mq || !B || !max_q) return 0;
    return part_bytes(plan_prefix(Mq, P, B, max_q, max_k, H, KV), Mq, H, D);
}

extern "C" int e2mi_attention_prefix(e2mi_stream stream, int dtype, const uint16_t *q, int64_t ldq, int Mq, const uint16_t *k,
                                     int64_t ldk, const uint16_t *vt, int64_t ldv, int Mk, const uint16_t *pk, int64_t ldpk,
                                     const uint16_t *pvt, int64_t ldpv, int P, const int32_t *q_start, const int32_t *q_len,
                                     const int32_t *k_start, const int32_t *k_len, int B, int max_q, int max_k, int H, int KV,
                                     int D, float scale, int causal, uint16_t *ctx, int64_t ldc, int8_t *ctx_q, float *ctx_s,
                                     void *workspace, size_t workspace_bytes) {
    KeysArgs a = {};
    a.q = q, a.ldq = ldq, a.Mq = Mq;
    a.own = {k, vt, ldk, ldv, Mk};
    a.pre = {pk, pvt, ldpk, ldpv, P};
    a.q_start = q_start, a.q_len = q_len, a.k_start = k_start, a.k_len = k_len;
    a.B = B, a.max_q = max_q, a.max_k = max_k, a.H = H, a.KV = KV;
    a.G = KV > 0 ? H / KV : 0;
    a.c2 = scale * 1.44269504088896341f, a.causal = causal != 0;
    a.ctx = ctx, a.ldc = ldc, a.cq = ctx_q, a.cs = ctx_s;
    if (check_call("attention_prefix", dtype, a, D, scale)) return -1;
    if (check_keys("attention_prefix", "prefix keys", a.pre, KV, D)) return -1;
    if (!Mq || !B || !max_q) return 0;
    const KeysPlan p = plan_prefix(Mq, P, B, max_q, max_k, H, KV);
    if (check_workspace("attention_prefix", part_bytes(p, Mq, H, D), workspace, workspace_bytes)) return -1;
    return run_keys((hipStream_t)stream, dtype, D, a, p, workspace);
}

extern "C" size_t e2mi_attention_blocks_workspace_bytes(int Mq, int B, int max_q, int H, int KV, int D, int q_block, int n_sel) {
    if (!sizes_fit(Mq, B, max_q, 0, H, KV, D) || q_block <= 0 || n_sel <= 0 || n_sel > kMaxSelect || !Mq || !B || !max_q) return 0;
    return part_bytes(plan_blocks(B, max_q, H, KV, q_block, n_sel), Mq, H, D);
}

extern "C" int e2mi_attention_blocks(e2mi_stream stream, int dtype, const uint16_t *q, int64_t ldq, int Mq, const uint16_t *k,
                                     int64_t ldk, const uint16_t *vt, int64_t ldv, int Mk, const int32_t *q_start,
                                     const int32_t *q_len, const int32_t *k_start, const int32_t *k_len, int B, int max_q,
                                     int max_k, int H, int KV, int D, int q_block, const int32_t *sel, int n_sel, float scale,
                                     int causal, uint16_t *ctx, int64_t ldc, int8_t *ctx_q, float *ctx_s, void *workspace,
                                     size_t workspace_bytes) {
    KeysArgs a = {};
    a.q = q, a.ldq = ldq, a.Mq = Mq;
    a.own = {k, vt, ldk, ldv, Mk};
    a.q_start = q_start, a.q_len = q_len, a.k_start = k_start, a.k_len = k_len;
    a.B = B, a.max_q = max_q, a.max_k = max_k, a.H = H, a.KV = KV;
    a.G = KV > 0 ? H / KV : 0;
    a.c2 = scale * 1.44269504088896341f, a.causal = causal != 0;
    a.ctx = ctx, a.ldc = ldc, a.cq = ctx_q, a.cs = ctx_s;
    a.sel = sel, a.q_block = q_block, a.n_sel = n_sel;
    if (check_call("attention_blocks", dtype, a, D, scale)) return -1;
    if (!sel || q_block <= 0 || q_block > 1024 || n_sel <= 0 || n_sel > kMaxSelect) {
        set_error("attention_blocks: needs lists of 1 to %d blocks for 1 to 1024 tokens (q_block=%d n_sel=%d)", kMaxSelect, q_block, n_sel);
        return -1;
    }
    if (!Mq || !B || !max_q) return 0;
    a.NQ = (max_q + q_block - 1) / q_block;
    const KeysPlan p = plan_blocks(B, max_q, H, KV, q_block, n_sel);
    if (check_workspace("attention_blocks", part_bytes(p, Mq, H, D), workspace, workspace_bytes)) return -1;
    return run_keys((hipStream_t)stream, dtype, D, a, p, workspace);
}
