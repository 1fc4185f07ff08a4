// ops_fattn_wide.hip — FLASH_ATTN_EXT whose keys are wider than its values: latent attention.
//
//   absorbed   K rows of 576 (the latent vector and the rotated channels), V = 512 of the same row's
//              channels, one (or a few) KV heads shared by all query heads; cache f16, q8_0 or q4_0
//   expanded   K rows of 192, V rows of 128, f16, a KV head a query head (or a group)
//
//   s_j = scale q.k_j [softcap tanh(s / softcap)] + slope mask_j,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),
//   sinks join the denominator once; a row whose mask leaves nothing gives 0.
//
// Precision: the result is f32 and callers ask for GGML_PREC_F32, so nothing is rounded to 11 bits on
// the way: q (scaled by a power of two into f16's range) and the softmax weights enter the f16 matrix
// units as two terms, high + low, each product twice: 22 bits, for a weight down to 2^-10 of the row's largest, below
// that 2^-32 of the largest; K and V are exact in f16, quantised
// ones as their integers: a block's step is applied in f32 to the products of K, and to the weights of V
// as their terms are formed. The rate that bounds the large cases is therefore half the f16 rate.
//
// All kernels: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_16x16x32_f16, so a lane holds scores and
// outputs of one query row (lane & 15): softmax state and rescaling are lane-local, and P^T goes from
// the score registers straight into the second product (its k index runs over the keys the lane has;
// V's rows follow by transposing LDS reads). Query rows of one KV head are flattened token-major, so a
// workgroup's rows are any mix of heads and tokens. Its waves share tiles of 32 keys in LDS, a ring
// filled by LDS-DMA ahead of use. With few rows the tiles are dealt out over `nsplit` workgroups
// (split, split + nsplit, ...: a padded tail of masked tiles is shared evenly) and joined by a second
// launch. Tiles that the mask hides from every row of the workgroup are never loaded.
#include "backend.h"
#include "quants.cuh"

#include <algorithm>
#include <type_traits>

namespace mx {

typedef _Float16 wh8 __attribute__((ext_vector_type(8)));
typedef _Float16 wh4 __attribute__((ext_vector_type(4)));
typedef _Float16 wh2 __attribute__((ext_vector_type(2)));
typedef float wf4 __attribute__((ext_vector_type(4)));
typedef uint16_t wu4 __attribute__((ext_vector_type(4)));
typedef __fp16 w16x4 __attribute__((vector_size(8)));
typedef __attribute__((address_space(3))) w16x4 * lds_w4;
typedef __attribute__((address_space(3))) void * lds_dma;

constexpr int FW_KT = 32;                    // keys of a tile
constexpr int FW_PIECE = FW_KT * 128;        // 64 channels of a tile in LDS, f16
constexpr int FW_TB = 32;                    // tokens of one entry of the mask's tile map
constexpr int FW_MAX_SPLIT = 256;
constexpr int FW_TILE = 0x3FFFFFFF;          // a listed tile's number; bit 30: the mask or the row's end cuts it
constexpr float FW_L2E = 1.4426950408889634f;   // scores, masks and sinks are taken to base 2 where they come in
enum { FW_LIVE = 1, FW_MIXED = 2 };          // tile map bits: some key is visible; some mask value is not 0

struct FwArgs {
    const char * q; size_t q1, q2, q3;       // f32 [DK, n_q, H, S]
    const char * k; size_t k1, k2, k3;
    const char * v; size_t v1, v2, v3;
    const char * mask; size_t m1, m2, m3; int mne2, mne3;   // f16 or null
    const float * sinks;
    char * dst; size_t d1, d2, d3;           // f32 [DV, H, n_q, S]
    float * opart, * mpart, * lpart;         // [nsplit][S * n_q * H][DV | 1 | 1]
    const uint8_t * map; int n_tb;           // [mne3][n_tb][n_tiles] tile map, or null
    int n_q, n_kv, H, G, Hkv, S, nsplit, n_tiles, vpiece;   // vpiece: 64s of channels of a K row before V
    float scale, softcap, max_bias, m0, m1f;   // to base 2: softcap, or scale where there is none
    uint32_t n_head_log2;
};

__device__ __forceinline__ uint4 ldu16(const char * p) { uint4 v; __builtin_memcpy(&v, p, 16); return v; }

// two values to f16, to nearest: what many small weights leave out then has either sign (cut off, 4096 weights of 2^-17 of
// the largest take 2e-5 from the result, 32768 of 2^-20 1e-4)
__device__ __forceinline__ wh2 fw_near(float x0, float x1) {
    typedef float wf2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector((wf2{x0, x1}), wh2);
}
// hi + lo = x to 22 bits, or to 2^-25 where x is below 2^-3 (f16's smallest step is 2^-24): the high term truncated, the
// remainder (exact in f32) rounded
__device__ __forceinline__ void split2(float x0, float x1, int j, wh8 & hi, wh8 & lo) {
    const wh2 h = __builtin_bit_cast(wh2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    const wh2 l = fw_near(x0 - (float) h[0], x1 - (float) h[1]);
    hi[j] = h[0]; hi[j + 1] = h[1];
    lo[j] = l[0]; lo[j + 1] = l[1];
}
// the same of the products x0 d0, x1 d1, h being x0 and x1 to f16: the high terms multiplied there, the remainder of the whole product
__device__ __forceinline__ void split2p(float x0, float x1, wh2 h, wh2 d, int j, wh8 & hi, wh8 & lo) {
    h *= d;
    const wh2 l = fw_near(__builtin_fmaf(x0, (float) d[0], -(float) h[0]), __builtin_fmaf(x1, (float) d[1], -(float) h[1]));
    hi[j] = h[0]; hi[j + 1] = h[1];
    lo[j] = l[0]; lo[j + 1] = l[1];
}
__device__ __forceinline__ void split8(const float (&x)[8], wh8 & hi, wh8 & lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) split2(x[j], x[j + 1], j, hi, lo);
}

// A tile in LDS: pieces of 64 channels, each [32 rows][128 B], so that an LDS-DMA instruction of a wave (64 x 16 B,
// consecutive in LDS) is eight rows of one piece. The eight 16-byte chunks of a row are XORed with swz(row): two
// rows cover the 64 banks, so the 16 rows a b128 read takes at one chunk, eight of each parity, get eight places each,
// and the transposing reads (eight rows x two neighbouring chunks at a time) four pairs for four rows of a parity
__device__ __forceinline__ int fw_swz(int row) { return (row & 6) | ((row >> 3) & 1); }

__device__ __forceinline__ wh4 lds_tr4(const char * a) {
    return __builtin_bit_cast(wh4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_w4) a));
}

// LDS-DMA of 16 bytes a lane, from base + off (a lane's) + soff to LDS `to` + 16 lane. The buffer form: the compiler
// counts it with the vector loads alone; behind the global form, which it takes for a flat access, every wait for an
// LDS read becomes a wait for all of them
struct FwSrc { __amdgpu_buffer_rsrc_t r; };
__device__ __forceinline__ FwSrc fw_src(const char * base) { return FwSrc{__builtin_amdgcn_make_buffer_rsrc((void *) base, 0, -1, 0x00027000)}; }
__device__ __forceinline__ void fw_dma(const FwSrc & s, int off, int soff, char * to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(s.r, (lds_dma) to, 16, off, soff, 0, 0);
}

template <int N> __device__ __forceinline__ void fw_vmcnt() {   // at most N vector memory operations outstanding
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Workgroup barrier behind this wave's LDS accesses, with LDS-DMA still on its way (__syncthreads waits for that too)
__device__ __forceinline__ void fw_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// over the four lanes of a row (lane ^ 16, ^ 32, ^ 48), in registers: the swaps exchange rows of 16 (halves of 32) of
// two copies, so their maximum (sum) is the pair's
template <bool SUM> __device__ __forceinline__ float fw_row4(float x) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = SUM ? __uint_as_float(a.x) + __uint_as_float(a.y) : fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return SUM ? __uint_as_float(a.x) + __uint_as_float(a.y) : fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
}

__device__ __forceinline__ uint32_t fw_row4_max(uint32_t x) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    u2 a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a.x, a.y);
    a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(a.x, a.y);
}

// element i of a cache row, for the plain loop below
template <int KV> __device__ __forceinline__ float fw_get(const char * row, int i) {
    if constexpr (KV == GGML_TYPE_F16) return h2f(*(const uint16_t *) (row + 2 * (size_t) i));
    else return dequant_one<KV>(row + (size_t) (i >> 5) * qsize_of<KV>(), i & 31);
}

// the factor of the mask
__device__ __forceinline__ float fw_slope(const FwArgs & p, uint32_t h) {
    return p.max_bias > 0.0f ? FW_L2E * (h < p.n_head_log2 ? powf(p.m0, h + 1) : powf(p.m1f, 2 * (h - p.n_head_log2) + 1)) : FW_L2E;
}

// What a workgroup works on: rows [r0, r0 + ROWS) of KV head hk of sequence seq, row r being token r / G
// and head hk G + r % G; tiles split, split + nsplit, ...
struct FwJob {
    int hk, seq, r0, nrow, split, nl;        // nl: tiles of the split
    const char * kb;
    __device__ __forceinline__ int tile(const FwArgs & p, int i) const { return split + min(i, nl - 1) * p.nsplit; }   // the split's i-th (its last)
    __device__ __forceinline__ int head(const FwArgs & p, int r) const { return hk * p.G + r % p.G; }
    __device__ __forceinline__ const char * mask_row(const FwArgs & p, int tok, int h) const {
        return p.mask + (size_t) tok * p.m1 + (size_t) (h % p.mne2) * p.m2 + (size_t) (seq % p.mne3) * p.m3;
    }
};

// (KV head, sequence) units: with a multiple of eight the workgroups of one unit stay on one XCD and
// share its L2; the last rows (most keys, under a causal mask) go first. FOLD, two workgroups a CU: those
// that take the second places of an XCD's 32 CUs run the other way, so that the last rows share a CU with
// the first ones
template <int ROWS, bool FOLD> __device__ __forceinline__ FwJob fw_job(const FwArgs & p) {
    FwJob j;
    j.nrow = p.n_q * p.G;
    const int nrb = (j.nrow + ROWS - 1) / ROWS, units = p.Hkv * p.S;
    int unit, rb;
    if (units % 8 == 0) { unit = blockIdx.x % 8 + 8 * (blockIdx.x / 8 / nrb); rb = blockIdx.x / 8 % nrb; }
    else { unit = blockIdx.x / nrb; rb = blockIdx.x % nrb; }
    if (!FOLD || units % 8 != 0 || gridDim.x > 512 || !(unit / 8 * nrb / 32 & 1)) rb = nrb - 1 - rb;
    j.hk = unit % p.Hkv;
    j.seq = unit / p.Hkv;
    j.r0 = rb * ROWS;
    j.split = blockIdx.y;
    j.nl = (p.n_tiles - j.split + p.nsplit - 1) / p.nsplit;
    j.kb = p.k + (size_t) j.hk * p.k2 + (size_t) j.seq * p.k3;
    return j;
}

// The split's tiles that some row of the workgroup looks at, in order, 64 at a time: lane l judges tile
// w0 + l from the map or, when the tokens are few, from their mask rows (every wave for itself)
struct FwTiles {
    uint64_t live, mixed;
    int w0;
    template <int ROWS> __device__ __forceinline__ void window(const FwArgs & p, const FwJob & j) {
        const int lane = threadIdx.x & 63, l = w0 + lane, tile = j.split + l * p.nsplit;
        uint32_t f = 0;
        if (l < j.nl) {
            const int t_lo = j.r0 / p.G, t_hi = (min(j.r0 + ROWS, j.nrow) - 1) / p.G;
            if (!p.mask) f = FW_LIVE;
            else if (p.mne2 > 1) f = FW_LIVE | FW_MIXED;
            else if (p.map) {
                for (int tb = t_lo / FW_TB; tb <= t_hi / FW_TB; ++tb)
                    f |= p.map[((size_t) (j.seq % p.mne3) * p.n_tb + tb) * p.n_tiles + tile];
            } else if (j.nl <= 2) f = FW_LIVE | FW_MIXED;
            else {
                for (int t = t_lo; t <= t_hi; ++t) {
                    const char * mr = j.mask_row(p, t, 0) + 2 * (size_t) tile * FW_KT;
                    const int n = p.n_kv - tile * FW_KT;
                    if (n >= FW_KT) {
#pragma unroll
                        for (int c = 0; c < FW_KT / 8; ++c) {
                            const uint4 v = ldu16(mr + 16 * c);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) f |= ((w[i] & 0xFFFF) != 0xFC00 || (w[i] >> 16) != 0xFC00 ? FW_LIVE : 0) | (w[i] & 0x7FFF7FFF ? FW_MIXED : 0);
                        }
                    } else {
                        for (int i = 0; i < n; ++i) {
                            const uint32_t w = ((const uint16_t *) mr)[i];
                            f |= (w != 0xFC00 ? FW_LIVE : 0) | (w & 0x7FFF ? FW_MIXED : 0);
                        }
                    }
                }
            }
            if ((tile + 1) * FW_KT > p.n_kv) f |= FW_MIXED;     // the row's end lies inside
        }
        live = __ballot(f & FW_LIVE);
        mixed = __ballot(f & FW_MIXED);
    }
    // the next tile's number (bit 30: mixed), or -1
    template <int ROWS> __device__ __forceinline__ int next(const FwArgs & p, const FwJob & j) {
        while (!live) {
            w0 += 64;
            if (w0 >= j.nl) return -1;
            window<ROWS>(p, j);
        }
        const int b = __builtin_ctzll(live);
        live &= live - 1;
        return (j.split + (w0 + b) * p.nsplit) | ((mixed >> b & 1) ? 1 << 30 : 0);
    }
};

// this lane's query row r, channels 32 (s0 + s) + 8 g4 .. + 7 of step s: fetched first, ...
template <int NS>
__device__ __forceinline__ void fw_query(const FwArgs & p, const FwJob & j, int r, int s0, float (&x)[NS][8]) {
    const int g4 = (threadIdx.x & 63) >> 4;
    const char * qp = p.q + (size_t) (r / p.G) * p.q1 + (size_t) j.head(p, r) * p.q2 + (size_t) j.seq * p.q3 + 128 * s0 + 32 * g4;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const uint4 a = ldu16(qp + 128 * s), b = ldu16(qp + 128 * s + 16);
        __builtin_memcpy(&x[s][0], &a, 16);
        __builtin_memcpy(&x[s][4], &b, 16);
    }
}
// ... then taken as two f16 terms, scaled by a power of two that takes the largest magnitude of these channels to
// 2^13 .. 2^14 (what the low term then loses is below 2^-38 of it). Returns the scale of their scores
template <int NS>
__device__ __forceinline__ float fw_terms(const FwArgs & p, const float (&x)[NS][8], wh8 (&qh)[NS], wh8 (&ql)[NS]) {
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[s][i]));
    top = fw_row4<false>(top);
    const int e = top > 0.f && top < INFINITY ? max(-100, min(100, 14 - __builtin_amdgcn_frexp_expf(top))) : 0;
    const float f = __builtin_amdgcn_ldexpf(1.f, e);            // (exact: a product that leaves f32's normal range is below the bound)
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[s][i] * f;
        split8(y, qh[s], ql[s]);
    }
    return p.scale * __builtin_amdgcn_ldexpf(1.f, -e);
}

// a tile that the mask or the row's end cuts: s + slope mask, -inf where hidden (whatever the score: a
// hidden key's K may be anything) and beyond the end. Keys 16 u + 4 g4 + 0..3 of a lane
__device__ __forceinline__ void fw_mask(const FwArgs & p, const FwJob & j, int r, int tile, wf4 (&s)[2]) {
    const int h = j.head(p, r), g4 = (threadIdx.x & 63) >> 4;
    const float slope = fw_slope(p, (uint32_t) h);
    const char * mr = j.mask_row(p, r / p.G, h);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int key = tile * FW_KT + 16 * u + 4 * g4;
        uint64_t w = 0;
        if (p.mask) {
            if (key + 4 <= p.n_kv) __builtin_memcpy(&w, mr + 2 * (size_t) key, 8);
            else
                for (int i = 0; key + i < p.n_kv; ++i) w |= (uint64_t) ((const uint16_t *) mr)[key + i] << (16 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float mv = h2f((uint16_t) (w >> (16 * i)));
            s[u][i] = mv == -INFINITY || key + i >= p.n_kv ? -INFINITY : s[u][i] + slope * mv;
        }
    }
}

// Online softmax of a lane's row over its 8 keys of the tile and the other three lanes' (the row lies in
// four). First the reference: FW_LOW below the maximum that it was taken from, so weights use f16's whole range and a small
// one keeps its bits down to 2^-32 of the largest; raised only when a score exceeds that maximum by 8 (weights up to
// 2^15), so O is rescaled on the first tiles only. Returns -m for the weights 2^(s - m).
constexpr float FW_LOW = 7.f;
template <int ND>
__device__ __forceinline__ float fw_raise(const wf4 (&s)[2], float & m, float & l, wf4 (&o)[ND]) {
    float mt = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mt = fw_row4<false>(mt);
    const bool raise = mt > m + (FW_LOW + 8.f);                 // false while nothing was visible
    if (__any(raise)) {
        mt -= FW_LOW;
        const float al = raise ? __builtin_amdgcn_exp2f(m - mt) : 1.f;
        if (raise) m = mt;
        l *= al;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= al;
    }
    return m == -INFINITY ? 0.f : -m;
}
__device__ __forceinline__ float fw_weight(const wf4 (&s)[2], int i, float ms) {
    return __builtin_amdgcn_exp2f(s[i >> 2][i & 3] + ms);
}

// a sink's part of the denominator; one of -inf beside a row that sees nothing is no NaN
__device__ __forceinline__ float fw_sink(float sink, float m) { return sink == m ? 1.f : __builtin_amdgcn_exp2f(sink - m); }

// A row key by key, leaving masked keys out: an infinity or a NaN in V times a weight of 0 is a NaN, and
// what lies in the rows of hidden keys may not reach the result, so a row that shows one is computed
// again by its wave. acc[c]: channel d0 + 64 c + lane
template <int DK, int KV, int NC>
__device__ __forceinline__ void fw_again(const FwArgs & p, const FwJob & j, const char * vb, size_t v1, int r, int d0, float & m_, float & l_, float (&acc)[NC]) {
    const int lane = threadIdx.x & 63, tk = r / p.G, hd = j.head(p, r);
    const float sl = fw_slope(p, (uint32_t) hd);
    const float * qp = (const float *) (p.q + (size_t) tk * p.q1 + (size_t) hd * p.q2 + (size_t) j.seq * p.q3);
    const char * mr = j.mask_row(p, tk, hd);
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = 0.f;
    for (int i = 0; i < j.nl; ++i) {
        const int k0 = (j.split + i * p.nsplit) * FW_KT, key = k0 + lane;
        float mv = -INFINITY, x = -INFINITY;
        if (lane < FW_KT && key < p.n_kv) mv = p.mask ? sl * h2f(((const uint16_t *) mr)[key]) : 0.f;
        uint64_t seen = __ballot(mv != -INFINITY);
        if (!seen) continue;
        if (mv != -INFINITY) {
            const char * kr = j.kb + (size_t) key * p.k1;
            float dot = 0.f;
#pragma unroll 1
            for (int c = 0; c < DK; ++c) dot += qp[c] * fw_get<KV>(kr, c);
            x = dot * p.scale;
            if (p.softcap != 0.0f) x = p.softcap * tanhf(x);
            x += mv;
        }
        const float mn = fmaxf(m, wave_max<64>(x));
        const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float e = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - mn);
        m = mn;
        l = l * al + wave_sum<64>(e);
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] *= al;
        for (; seen; seen &= seen - 1) {
            const int s = __builtin_ctzll(seen);
            const float w = __shfl(e, s, 64);
            const char * vr = vb + (size_t) (k0 + s) * v1;
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[c] += w * fw_get<KV>(vr, d0 + 64 * c + lane);
        }
    }
    m_ = m;
    l_ = l;
}

// The end of a row group of 16: the lanes' sums joined, rows with a NaN computed again, the result (or
// the split's part of it) stored. o[d]: channels d0 + 16 d + 4 g4 + 0..3 of row r; D0: d0 == 0 stores m, l.
// Where two waves hold a row's channels, one of them may have to compute its half again and the other not. Both have the same
// m and l, so the half takes m as its reference (the sums of fw_again are relative to the keys' own maximum, other by up to
// what fw_raise lets pass), and both take the new m and l only where l itself is no number
template <int DK, int DV, int KV, int ND>
__device__ __forceinline__ void fw_store(const FwArgs & p, const FwJob & j, const char * vb, size_t v1, int vd0, int rg0, int d0, float m, float l, wf4 (&o)[ND]) {
    const int lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
    l = fw_row4<true>(l);
    float z = l * 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) z += o[d][i] * 0.f;
    const uint64_t b = __ballot(z != 0.f);                      // NaN compares unequal
    for (uint32_t bad = (uint32_t) ((b | b >> 16 | b >> 32 | b >> 48) & 0xFFFF); bad; bad &= bad - 1) {
        const int col = __builtin_ctz(bad);
        float m2, l2, acc[ND / 4];
        fw_again<DK, KV, ND / 4>(p, j, vb, v1, min(rg0 + col, j.nrow - 1), vd0 + d0, m2, l2, acc);
        if (n16 == col && l * 0.f != 0.f) { m = m2; l = l2; }
        const float f = m2 == m ? 1.f : __builtin_amdgcn_exp2f(m2 - m);     // (of the lanes of that row)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = __shfl(acc[d >> 2], 16 * (d & 3) + 4 * g4 + i, 64);
                if (n16 == col) o[d][i] = v * f;
            }
    }
    const int r = rg0 + n16;
    if (r >= j.nrow) return;
    const int tk = r / p.G, hd = j.head(p, r);
    if (p.nsplit == 1) {
        float a = 1.f;
        if (p.sinks) {
            const float sk = p.sinks[hd] * FW_L2E, mm = fmaxf(m, sk);
            a = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
            l = l * a + fw_sink(sk, mm);
        }
        const float inv = l == 0.f ? 0.f : a / l;
        char * out = p.dst + (size_t) hd * p.d1 + (size_t) tk * p.d2 + (size_t) j.seq * p.d3 + 4 * (d0 + 4 * g4);
#pragma unroll
        for (int d = 0; d < ND; ++d) *(wf4 *) (out + 64 * d) = o[d] * inv;
    } else {
        const size_t id = ((size_t) j.split * p.S + j.seq) * p.n_q * p.H + (size_t) tk * p.H + hd;
        if (d0 == 0 && g4 == 0) { p.mpart[id] = m; p.lpart[id] = l; }
        if (m != -INFINITY || l != 0.f) {                       // nothing visible in this split: the join skips it
            float * out = p.opart + id * DV + d0 + 4 * g4;
#pragma unroll
            for (int d = 0; d < ND; ++d) *(wf4 *) (out + 16 * d) = o[d];
        }
    }
}

// ---- absorbed: K rows of 576, V in them --------------------------------------------------------------
// Many rows, f16: four groups of 16, two waves each. O of 16 rows is 128 registers a lane and Q (two terms) 144, too
// much for one wave beside the rest of it, so the pair shares: wave dh multiplies channels [288 dh, + 288)
// of the keys, the halves of the scores are exchanged through LDS (the only barrier of a tile), both do
// the softmax, and each keeps half of the output channels.
// The matrix unit and its power bound it. 512 tokens, 32 heads, 4096 keys: 250 us warm, 1.08 PFLOP/s of f16 products (a
// large library product 1.18); a build of 14 % fewer busy cycles took the same time at a clock lower by as much. The form
// of 32 rows below takes 278
__global__ __launch_bounds__(512, 2) void k_fattn_latent64(FwArgs p) {
    constexpr int NS = 9, ND = 16, ROWS = 64, NW = 8, BUF = 9 * FW_PIECE, DMA = 5;         // LDS-DMA instructions of a wave and tile
    // the ring's tiles as objects of their own: reads of one need not wait for the DMA that fills another
    __shared__ __align__(128) char t0[BUF];
    __shared__ __align__(128) char t1[BUF];
    __shared__ __align__(128) char t2[BUF];
    __shared__ __align__(16) wf4 exch[2][NW][2][64];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;
    const int rg = wave >> 1, dh = wave & 1;
    const FwJob j = fw_job<ROWS, false>(p);
    const int r = min(j.r0 + 16 * rg + n16, j.nrow - 1);        // this lane's row

    float qx[NS][8];
    fw_query<NS>(p, j, r, NS * dh, qx);                         // (on its way while the tiles are listed)
    // ---- staging: instruction x of a tile fills rows 8 (x & 3) .. + 7 of piece x >> 2; lane l brings
    // the chunk that belongs at its place, (l % 8) ^ swz(row) of row l / 8
    const int srow = 8 * (wave & 3) + (lane >> 3), ssrc = 16 * ((lane & 7) ^ fw_swz(srow));
    auto dma_off = [&](int tile) { return min(srow, p.n_kv - 1 - (tile & FW_TILE) * FW_KT) * (int) p.k1 + ssrc; };
    auto dma_src = [&](int tile) { return fw_src(j.kb + (size_t) ((tile & FW_TILE) * FW_KT) * p.k1); };
    // instruction i of a wave: it keeps to one row group (wave & 3); two waves share one and halve its pieces
    auto dma = [&](const FwSrc & src, int off, char * buf, int i) __attribute__((always_inline)) {
        const int piece = min(2 * i + (wave >> 2), 8);          // (piece 8 is brought twice)
        fw_dma(src, off, 128 * piece, buf + piece * FW_PIECE + 1024 * (wave & 3));
    };
    // ---- the split's first tiles on their way while the tiles are listed; as a rule they are the list's.
    // id[c]: the tile in slot c of the ring (-1: none)
    char * const ring[3] = {t0, t1, t2};
    int id[3];
    auto dma_tile = [&](int tile, char * buf) __attribute__((always_inline)) {
        const FwSrc src = dma_src(tile);
        const int off = dma_off(tile);
#pragma unroll
        for (int i = 0; i < DMA; ++i) dma(src, off, buf, i);
    };
#pragma unroll
    for (int c = 0; c < 2; ++c) if (c < j.nl) dma_tile(j.tile(p, c), ring[c]);
    FwTiles tiles;
    tiles.w0 = 0;
    tiles.window<ROWS>(p, j);
    bool listed = true;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        id[c] = c == 0 || id[c - 1] >= 0 ? tiles.next<ROWS>(p, j) : -1;
        listed &= id[c] < 0 || (id[c] & FW_TILE) == j.tile(p, c);
    }
    if (!listed) {
        fw_vmcnt<0>();                                          // (behind the ones under way to the same places)
#pragma unroll
        for (int c = 0; c < 2; ++c) if (id[c] >= 0) dma_tile(id[c], ring[c]);
    }
    id[2] = id[1] >= 0 ? tiles.next<ROWS>(p, j) : -1;           // fetched by the first body
    wh8 qh[NS], ql[NS];
    const float qsc = fw_terms<NS>(p, qx, qh, ql);              // of this half's part of the scores

    wf4 o[ND];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = wf4{0.f, 0.f, 0.f, 0.f};
    // per-lane LDS offsets: step i of this wave's half is step gs = 9 dh + i of the row, chunk g4 of half gs & 1 of piece gs >> 1
    const int kx0 = 128 * n16 + 16 * (g4 ^ fw_swz(n16)), kx1 = 128 * n16 + 16 * ((4 + g4) ^ fw_swz(n16));
    const int ka0 = dh ? kx1 + 4 * FW_PIECE : kx0, ka1 = dh ? kx0 + 5 * FW_PIECE : kx1;
    const int iq = (lane >> 2) & 3, ip = lane & 3, vrow = 4 * g4 + iq, vsw = fw_swz(vrow);
    int va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) va[i] = (4 * dh + p.vpiece) * FW_PIECE + 128 * vrow + 16 * ((2 * i + (ip >> 1)) ^ vsw) + 8 * (ip & 1);

    int par = 0;
    wf4 s[2], t[2];                                             // the scores of the tile in hand, this half's of the next
    float ms = 0.f;
    wh8 ph, pl;
    float e[8];
    // fragments from LDS are read AK (AV) steps ahead: with eight waves at it a read takes some 250 cycles, a step's
    // matrix instructions 64. The first ones before the barrier's other business, and before the end of the scores
    constexpr int AK = 4, AV = 3;
    wh8 a[AK + 1][2], v[AV + 1][2];
    auto lda = [&](const char * buf, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) a[i % (AK + 1)][u] = *(const wh8 *) (buf + (i & 1 ? ka1 : ka0) + (i >> 1) * FW_PIECE + 2048 * u);
    };
    auto ldv = [&](const char * buf, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const char * a_ = buf + va[2 * (b & 1) + c] + (b >> 1) * FW_PIECE;
            const wh4 v0 = lds_tr4(a_), v1 = lds_tr4(a_ + 2048);
            v[b % (AV + 1)][c] = wh8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        }
    };
    auto ahead = [&](const char * buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AK; ++i) lda(buf, i);
    };
    // this half's part of the scores of the tile in `buf` to the exchange; meanwhile (W) the weights of the tile in
    // hand, whose values lie in `vbuf`
    // and a further tile goes to `fbuf`: instruction by instruction here, where the matrix unit hides them (all at once
    // behind the barrier they took 800 cycles). They run on past the last tile, into places no longer read
    auto scores = [&](const char * buf, const char * vbuf, char * fbuf, const FwSrc & fsrc, int foff, auto with) __attribute__((always_inline)) {
        constexpr bool W = decltype(with)::value;
        t[0] = t[1] = wf4{0.f, 0.f, 0.f, 0.f};
        wf4 tl[2] = {t[0], t[0]};                               // a chain of its own for the low term
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if constexpr (W) { if (i < DMA) dma(fsrc, foff, fbuf, i); }
            if (i + AK < NS) lda(buf, i + AK);
            if (W && i >= NS - AV) ldv(vbuf, i - (NS - AV));
#pragma unroll
            for (int u = 0; u < 2; ++u) t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], qh[i], t[u], 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) tl[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], ql[i], tl[u], 0, 0, 0);
            if constexpr (W) {
                if (i < 8) {
                    e[i] = fw_weight(s, i, ms);
                    l += e[i];
                    if (i & 1) split2(e[i - 1], e[i], i - 1, ph, pl);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        t[0] = (t[0] + tl[0]) * qsc;
        t[1] = (t[1] + tl[1]) * qsc;
        exch[par][wave][0][lane] = t[0];
        exch[par][wave][1][lane] = t[1];
    };
    // behind the barrier: the scores of tile `tile` whole, the reference maximum; the first fragments of the
    // tile in `buf` meanwhile
    auto whole = [&](int tile, const char * buf) __attribute__((always_inline)) {
        const wf4 x0 = exch[par][wave ^ 1][0][lane], x1 = exch[par][wave ^ 1][1][lane];
        __builtin_amdgcn_sched_barrier(0);
        ahead(buf);
        s[0] = t[0] + x0;
        s[1] = t[1] + x1;
        par ^= 1;
        if (p.softcap != 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = p.softcap * tanhf(s[i >> 2][i & 3]);
        }
        if (tile >> 30) fw_mask(p, j, r, tile & FW_TILE, s);
        ms = fw_raise<ND>(s, m, l, o);
    };
    // O^T += V^T P^T: keys 4 g4 + 0..3 of the two 16-key blocks a lane, as the scores lie; 32 channels at a
    // time, so that a term's product does not wait for the other's
    auto values = [&](const char * buf) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < ND / 2; ++b) {
            if (b + AV < ND / 2) ldv(buf, b + AV);
            o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][0], ph, o[2 * b], 0, 0, 0);
            o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][1], ph, o[2 * b + 1], 0, 0, 0);
            o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][0], pl, o[2 * b], 0, 0, 0);
            o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][1], pl, o[2 * b + 1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // the tile in slot C, its scores in hand, with the next tile's scores on the way: the weights are taken among the
    // matrix instructions of the next tile's scores, the exchange passes under this tile's values. The barrier then
    // frees slot C (and tells that the tile after the next is whole)
    auto body = [&](auto slot_) __attribute__((always_inline)) {
        constexpr int C = decltype(slot_)::value, C1 = (C + 1) % 3, F = (C + 2) % 3;
        const int further = id[F] >= 0 ? id[F] : id[C];         // (behind the last tile: any, into a place no longer read)
        scores(ring[C1], ring[C], ring[F], dma_src(further), dma_off(further), std::true_type{});
        values(ring[C]);
        fw_vmcnt<0>();                                          // the tile after the next has landed
        fw_barrier();
        id[C] = id[F] >= 0 ? tiles.next<ROWS>(p, j) : -1;
        whole(id[C1], ring[F]);                                 // (fragments read for nothing where no such tile is left)
    };

    fw_vmcnt<0>();
    __syncthreads();
    if (id[0] >= 0) {
        ahead(t0);
        scores(t0, t0, nullptr, dma_src(id[0]), 0, std::false_type{});
        fw_barrier();
        whole(id[0], t1);
        const char * last;
        for (;;) {
            last = t0;
            if (id[1] < 0) break;
            body(std::integral_constant<int, 0>{});
            last = t1;
            if (id[2] < 0) break;
            body(std::integral_constant<int, 1>{});
            last = t2;
            if (id[0] < 0) break;
            body(std::integral_constant<int, 2>{});
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = fw_weight(s, i, ms);
            l += e[i];
            if (i & 1) split2(e[i - 1], e[i], i - 1, ph, pl);
        }
        fw_vmcnt<0>();                                          // no DMA outlives the workgroup's LDS
#pragma unroll
        for (int b = 0; b < AV; ++b) ldv(last, b);
        values(last);
    }
    fw_store<576, 512, GGML_TYPE_F16, ND>(p, j, j.kb, p.k1, 64 * p.vpiece, j.r0 + 16 * rg, 256 * dh, m, l, o);
}

// ---- absorbed, few rows, and quantised -----------------------------------------------------------------
// 32 rows, and the work of a tile dealt out by kind, one wave of each kind a SIMD, so that one's waits are filled by the
// others' instructions:
//   4 waves   scores of the next tile (a pair of waves a row group, as above), its softmax; the weights go through LDS
//   4 waves   values of this tile, half of the channels of a row group each
//   4 waves   the tile after the next: f16 fetched by LDS-DMA into a ring of four (all 160 KB, with what is exchanged);
//             quantised, blocks turned into f16 integers, a ring of three
// Two barriers a tile: behind the halves of the scores, and behind the weights.
// f16: the cache bounds it. 4 sequences of up to 32768 tokens, 32 heads: 33 us for 123.5 MB (a large copy takes 24), the
// join 5.4 more; one wave doing scores and values in turn took 38, and alone on the chip 1.33 us a
// tile instead of 1.0. 200 tokens on 512 keys 26.9 us, 32.2 then.
// Quantised, a tile on every CU at once, 4 bits: 2.6 us with all of it in one wave a SIMD, 2.2 with the last kind apart, 1.9
// so; alone on the chip 2.6, 1.8 and 1.5 (8 bits 1.65). 4 x 32768 tokens at 4 bits: 39 us for 34.7 MB. What is left is the
// chain of one tile and the vector unit (a block's step enters its products, and V's steps the weights, in 32 bits): 500
// vector instructions and 68 matrix instructions a SIMD, 2000 and 1100 of some 3800 cycles
constexpr int FQ_BUF = 9 * FW_PIECE + 18 * FW_KT * 2;           // a tile and its blocks' steps, [block][key] f16, ...
constexpr int FQ_STEP = 10;                                     // ... times 2^10, out of the range where f16 keeps few bits

// the last kind, quantised: blocks through registers, two tiles ahead of the store
template <int KV, int ROWS>
__device__ __forceinline__ void fw_produce(const FwArgs & p, const FwJob & j, char * ring, uint16_t (&vtop)[3][FW_KT]) {
    // eight threads a row take two whole 32-blocks each, x and x + 8, and eight values of the last two blocks. A block
    // goes to LDS in four chunks of 8 values, thread x starting with the rot-th: the same chunk of all eight blocks
    // would lie in the same banks (1160 of a tile's 2700 LDS cycles were conflicts)
    constexpr int QB = qsize_of<KV>(), NL = KV == GGML_TYPE_Q8_0 ? 4 : 2;      // 8-byte loads of a block
    const int tid = threadIdx.x & 255;
    const int row = tid >> 3, x8 = tid & 7, sw = fw_swz(row), pblk = 16 + (x8 >> 2), pval = 8 * (x8 & 3), rot = x8 >> 1;
    int at[4], from[NL];                                        // places of the chunks, sources of the loads
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = rot * FW_PIECE + 128 * row + 16 * ((4 * (x8 & 1) + ((c + rot) & 3)) ^ sw);
#pragma unroll
    for (int c = 0; c < NL; ++c) from[c] = x8 * QB + 2 + 8 * ((c + rot) & (NL - 1));
    // integers to f16 exactly: 1024 + b has the byte b in its low bits, two at a time. 8 bits: b is n + 128; 4 bits: n + 8,
    // or 16 times that, from the high nibbles, so a chunk's nibble is a mask, a factor and an offset
    struct Nib { uint32_t mask; wh2 mul, off; };
    auto nibble = [](bool high) {
        const _Float16 m = high ? 0.0625f : 1.f, o = high ? -72.f : -1032.f;
        return Nib{high ? 0xF0F0F0F0u : 0x0F0F0F0Fu, wh2{m, m}, wh2{o, o}};
    };
    const Nib n0 = nibble(rot & 2), n1 = nibble((rot + 1) & 2), n2 = nibble(!(rot & 2)), n3 = nibble(!((rot + 1) & 2)), pnib = nibble(pval & 16);
    struct Regs { uint2 a[2][NL], w; _Float16 d[3]; } set[2];
    const uint32_t m0 = p.vpiece && x8 < 2 ? 0 : 0x7FFF, m2 = p.vpiece ? 0x7FFF : 0;
    auto load = [&](int tile, Regs & q) __attribute__((always_inline)) {
        const int key0 = (tile & FW_TILE) * FW_KT;
        const char * kb = j.kb + (size_t) key0 * p.k1;          // (uniform; a lane's offset has 32 bits)
        const uint32_t kr = (uint32_t) min(row, p.n_kv - 1 - key0) * (uint32_t) p.k1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            __builtin_memcpy(&q.d[i], kb + (kr + x8 * QB) + 8 * i * QB, 2);
#pragma unroll
            for (int c = 0; c < NL; ++c) __builtin_memcpy(&q.a[i][c], kb + (kr + from[c]) + 8 * i * QB, 8);
        }
        __builtin_memcpy(&q.d[2], kb + (kr + pblk * QB), 2);
        __builtin_memcpy(&q.w, kb + (kr + pblk * QB + (KV == GGML_TYPE_Q8_0 ? pval : pval & 15)) + 2, 8);
    };
    auto pair = [](uint32_t u, int t, const Nib & k) __attribute__((always_inline)) {      // bytes 2t, 2t + 1 of u
        const wh2 x = __builtin_bit_cast(wh2, __builtin_amdgcn_perm(0x64646464u, u, t ? 0x04030402u : 0x04010400u));
        return __builtin_bit_cast(uint32_t, KV == GGML_TYPE_Q8_0 ? x - wh2{(_Float16) 1152.f, (_Float16) 1152.f} : __builtin_elementwise_fma(x, k.mul, k.off));
    };
    auto chunk = [&](uint2 u, const Nib & k) __attribute__((always_inline)) {              // 8 values
        const uint32_t x = KV == GGML_TYPE_Q8_0 ? u.x ^ 0x80808080u : u.x & k.mask, y = KV == GGML_TYPE_Q8_0 ? u.y ^ 0x80808080u : u.y & k.mask;
        return make_uint4(pair(x, 0, k), pair(x, 1, k), pair(y, 0, k), pair(y, 1, k));
    };
    // a step past f16's range (64, or no number) becomes a NaN: as an infinity in a block that only K has, it would take a
    // visible key's score to -inf as soon as to +inf, and nothing would tell
    auto scaled = [](_Float16 d) __attribute__((always_inline)) {
        return __builtin_fabsf((float) d) < 65536.f / (1 << FQ_STEP) ? d * (_Float16) (1 << FQ_STEP) : (_Float16) __builtin_nanf("");
    };
    auto store = [&](const Regs & q, int slot, int half) __attribute__((always_inline)) {
        char * const buf = ring + slot * FQ_BUF;
        _Float16 * const steps = (_Float16 *) (buf + 9 * FW_PIECE);
        steps[(x8 + 8 * half) * FW_KT + row] = scaled(q.d[half]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *(uint4 *) (buf + at[c] + 4 * half * FW_PIECE) = chunk(q.a[half][c & (NL - 1)], c == 0 ? n0 : c == 1 ? n1 : c == 2 ? n2 : n3);
        if (half == 0) {
            // the largest step of each key's values: all blocks but the last two or, vpiece, but the first two
            const uint32_t b0 = __builtin_bit_cast(uint16_t, q.d[0]), b1 = __builtin_bit_cast(uint16_t, q.d[1]), b2 = __builtin_bit_cast(uint16_t, q.d[2]);
            int top = max(max(b0 & m0, b1 & 0x7FFF), b2 & m2);
            top = max(top, dpp_i<0xB1>(0, top));
            top = max(top, dpp_i<0x4E>(0, top));
            top = max(top, dpp_i<0x141>(0, top));
            if (x8 == 0) vtop[slot][row] = (uint16_t) top;
            return;
        }
        steps[pblk * FW_KT + row] = scaled(q.d[2]);
        *(uint4 *) (buf + 8 * FW_PIECE + 128 * row + 16 * (x8 ^ sw)) = chunk(q.w, pnib);
    };

    // the split's first two tiles on their way while the tiles are listed; as a rule they are the list's
    const int s0 = j.tile(p, 0), s1 = j.tile(p, 1);
    load(s0, set[0]);
    if (j.nl > 1) load(s1, set[1]);
    FwTiles tiles;
    tiles.w0 = 0;
    tiles.window<ROWS>(p, j);
    // tile 0 stored, 1 and 2 in registers
    int t0 = tiles.next<ROWS>(p, j), t1 = t0 >= 0 ? tiles.next<ROWS>(p, j) : -1, t2 = t1 >= 0 ? tiles.next<ROWS>(p, j) : -1;
    if (t0 >= 0) {
        if ((t0 & FW_TILE) != s0) load(t0, set[0]);
        if (t1 >= 0 && (t1 & FW_TILE) != s1) load(t1, set[1]);
        store(set[0], 0, 0);
        store(set[0], 0, 1);
        if (t2 >= 0) load(t2, set[0]);
    }
    fw_barrier();
    // beside tile i's scores: tile i + 1 to its slot, tile i + 3 on its way
    int slot = 1;
    auto body = [&](Regs & q) __attribute__((always_inline)) {
        if (t0 < 0) return false;
        if (t1 >= 0) store(q, slot, 0);
        fw_barrier();
        int t3 = -1;
        if (t1 >= 0) {
            store(q, slot, 1);
            if (t2 >= 0) t3 = tiles.next<ROWS>(p, j);
            if (t3 >= 0) load(t3, q);
        }
        t0 = t1; t1 = t2; t2 = t3;
        slot = slot == 2 ? 0 : slot + 1;
        fw_barrier();
        return true;
    };
    while (body(set[1]) && body(set[0])) {}
    fw_barrier();
}

// the last kind for f16: LDS-DMA, a wave eight rows of each piece; tile i + 2 beside tile i's scores
template <int ROWS>
__device__ __forceinline__ void fw_fetch(const FwArgs & p, const FwJob & j, char * ring) {
    constexpr int BUF = 9 * FW_PIECE;
    const int lane = threadIdx.x & 63, rowg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int srow = 8 * rowg + (lane >> 3), ssrc = 16 * ((lane & 7) ^ fw_swz(srow));
    auto dma = [&](int tile, int slot) __attribute__((always_inline)) {
        const int key0 = (tile & FW_TILE) * FW_KT, off = min(srow, p.n_kv - 1 - key0) * (int) p.k1 + ssrc;
        const FwSrc src = fw_src(j.kb + (size_t) key0 * p.k1);
        char * const to = ring + slot * BUF + 1024 * rowg;
#pragma unroll
        for (int i = 0; i < 9; ++i) fw_dma(src, off, 128 * i, to + i * FW_PIECE);
    };
    // the split's first two tiles on their way while the tiles are listed; as a rule they are the list's
    const int s0 = j.tile(p, 0), s1 = j.tile(p, 1);
    dma(s0, 0);
    dma(s1, 1);
    FwTiles tiles;
    tiles.w0 = 0;
    tiles.window<ROWS>(p, j);
    int t0 = tiles.next<ROWS>(p, j), t1 = t0 >= 0 ? tiles.next<ROWS>(p, j) : -1, t2 = t1 >= 0 ? tiles.next<ROWS>(p, j) : -1;
    if ((t0 >= 0 && (t0 & FW_TILE) != s0) || (t1 >= 0 && (t1 & FW_TILE) != s1)) {
        fw_vmcnt<0>();                                          // (behind the ones under way to the same places)
        dma(t0, 0);
        dma(t1 >= 0 ? t1 : t0, 1);
    }
    fw_vmcnt<9>();
    fw_barrier();
    for (int slot = 2; t0 >= 0; slot = (slot + 1) & 3) {
        if (t2 >= 0) dma(t2, slot);
        fw_barrier();
        if (t2 >= 0) fw_vmcnt<9>(); else fw_vmcnt<0>();         // the next tile has landed
        t0 = t1;
        t1 = t2;
        if (t2 >= 0) t2 = tiles.next<ROWS>(p, j);
        fw_barrier();
    }
    fw_vmcnt<0>();                                              // no DMA outlives the workgroup's LDS
    fw_barrier();
}

template <int KV>
__global__ __launch_bounds__(768, 3) void k_fattn_latent32(FwArgs p) {
    constexpr bool QUANT = KV != GGML_TYPE_F16;
    constexpr int NS = 9, ND = 16, ROWS = 32, AK = QUANT ? 2 : 3, AV = 2;      // fragments from LDS are read AK (AV) steps ahead
    constexpr int RING = QUANT ? 3 : 4, BUF = QUANT ? FQ_BUF : 9 * FW_PIECE;
    __shared__ __align__(128) char ring[RING * BUF];
    __shared__ __align__(16) wf4 exch[4][2][64];                // halves of scores
    __shared__ __align__(16) wf4 wgt[2][2][64];                 // weights: row group, 16 keys, the scores' lane
    __shared__ float scl[2][16];                                // a row's O takes this factor before them
    __shared__ __align__(16) uint16_t vtop[3][FW_KT];           // the largest step of each key's values, as f16's bits
    __shared__ float endm[2][64], endl[2][2][64];
    __shared__ int endq[2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, g4 = lane >> 4, rg = wave >> 1 & 1, dh = wave & 1;
    const FwJob j = fw_job<ROWS, false>(p);
    if (wave >= 8) {
        __builtin_amdgcn_s_setprio(2);                          // (the longest of the three; without it 49 us instead of 47)
        if constexpr (QUANT) fw_produce<KV, ROWS>(p, j, ring, vtop);
        else fw_fetch<ROWS>(p, j, ring);
        return;
    }
    const int r = min(j.r0 + 16 * rg + n16, j.nrow - 1);        // this lane's row
    FwTiles tiles;
    tiles.w0 = 0;
    int id0, id1;                                               // this tile, the next (-1: none)
    if (wave < 4) {
        float qx[NS][8];
        fw_query<NS>(p, j, r, NS * dh, qx);
        tiles.window<ROWS>(p, j);
        id0 = tiles.next<ROWS>(p, j);
        id1 = id0 >= 0 ? tiles.next<ROWS>(p, j) : -1;
        wh8 qh[NS], ql[NS];
        const float qsc = fw_terms<NS>(p, qx, qh, ql) * (QUANT ? 1.f / (1 << FQ_STEP) : 1.f);        // of this half's part of the scores
        const int kx0 = 128 * n16 + 16 * (g4 ^ fw_swz(n16)), kx1 = 128 * n16 + 16 * ((4 + g4) ^ fw_swz(n16));
        const int ka0 = dh ? kx1 + 4 * FW_PIECE : kx0, ka1 = dh ? kx0 + 5 * FW_PIECE : kx1;
        float m = -INFINITY, l = 0.f;
        // the weights take V's steps before they are split, so they and O are held in units of 2^qe, the largest (scaled)
        // step in the values of a key that the row sees, 1 at least: weights, up to 2^15, and their products with steps stay
        // in f16's range. (What other keys hold, and the channels that only K has, would cost the weights their last bits.)
        // A step of 64 or more is a NaN here: rows that see one are computed again
        int qe = 0;
        wf4 t[2];
        auto scores = [&](const char * buf) __attribute__((always_inline)) {
            wh8 a[AK + 1][2];
            wh4 d[QUANT ? AK + 2 : 1][2];                       // the blocks' steps of the lane's keys
            wf4 x[2][2];                                        // (f16: the low terms' products)
            auto lda = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    a[i % (AK + 1)][u] = *(const wh8 *) (buf + (i & 1 ? ka1 : ka0) + (i >> 1) * FW_PIECE + 2048 * u);
                    if constexpr (QUANT) d[i % (AK + 2)][u] = *(const wh4 *) (buf + 9 * FW_PIECE + 2 * ((NS * dh + i) * FW_KT + 16 * u + 4 * g4));
                }
            };
            auto step = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < 4; ++c) t[u][c] = __builtin_fmaf((float) d[QUANT ? i % (AK + 2) : 0][u][c], x[i & 1][u][c], t[u][c]);
            };
            t[0] = t[1] = wf4{0.f, 0.f, 0.f, 0.f};
            if constexpr (!QUANT) x[0][0] = x[0][1] = t[0];
#pragma unroll
            for (int i = 0; i < AK; ++i) lda(i);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (i + AK < NS) lda(i + AK);
                if constexpr (!QUANT) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], qh[i], t[u], 0, 0, 0);
#pragma unroll
                    for (int u = 0; u < 2; ++u) x[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], ql[i], x[0][u], 0, 0, 0);
                } else {
                    // one 32-block a step: its products are whole, then, a step later, take the block's step
#pragma unroll
                    for (int u = 0; u < 2; ++u) x[i & 1][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], qh[i], wf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int u = 0; u < 2; ++u) x[i & 1][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (AK + 1)][u], ql[i], x[i & 1][u], 0, 0, 0);
                    if (i) step(i - 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (QUANT) step(NS - 1);
            else { t[0] += x[0][0]; t[1] += x[0][1]; }
            t[0] *= qsc;
            t[1] *= qsc;
            exch[wave][0][lane] = t[0];
            exch[wave][1][lane] = t[1];
        };
        // the scores whole, the reference maximum, this wave's 16 keys' weights
        auto softmax = [&](int tile, int slot) __attribute__((always_inline)) {
            wf4 s[2] = {t[0] + exch[wave ^ 1][0][lane], t[1] + exch[wave ^ 1][1][lane]};
            if (p.softcap != 0.0f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = p.softcap * tanhf(s[i >> 2][i & 3]);
            }
            if (tile >> 30) fw_mask(p, j, r, tile & FW_TILE, s);
            float f = 1.f;
            if constexpr (QUANT) {
                const wu4 d[2] = {*(const wu4 *) &vtop[slot][4 * g4], *(const wu4 *) &vtop[slot][16 + 4 * g4]};
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, s[i >> 2][i & 3] == -INFINITY ? 0u : (uint32_t) d[i >> 2][i & 3]);
                // an exponent as frexp has it; below f16's normal range (0) it raises nothing, and rows that see a NaN start again
                const int x = max((int) (fw_row4_max(top) >> 10) - 14 + FQ_STEP, qe);
                f = __builtin_amdgcn_ldexpf(1.f, qe - x);       // the same in both waves of the row; 1 but on its first tiles
                qe = x;
            }
            wf4 one[1] = {wf4{f, 0.f, 0.f, 0.f}};               // O's factor
            const float ms = fw_raise<1>(s, m, l, one);
            const float qf = QUANT ? __builtin_amdgcn_ldexpf(1.f, -qe) : 1.f;
            const wf4 sv = dh ? s[1] : s[0];
            wf4 e;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = __builtin_amdgcn_exp2f(sv[i] + ms);
                l += e[i];
            }
            wgt[rg][dh][lane] = e * qf;
            if (dh == 0 && g4 == 0) scl[rg][n16] = one[0][0];
        };
        fw_barrier();
        for (int slot = 0; id0 >= 0; slot = slot == RING - 1 ? 0 : slot + 1) {
            scores(ring + slot * BUF);
            fw_barrier();
            softmax(id0, slot);
            id0 = id1;
            id1 = id1 >= 0 ? tiles.next<ROWS>(p, j) : -1;
            fw_barrier();
        }
        endl[rg][dh][lane] = l;
        if (dh == 0) endm[rg][lane] = m;
        if (dh == 0 && g4 == 0) endq[rg][n16] = qe;
        fw_barrier();
        return;
    }
    tiles.window<ROWS>(p, j);
    id0 = tiles.next<ROWS>(p, j);
    id1 = id0 >= 0 ? tiles.next<ROWS>(p, j) : -1;
    wf4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = wf4{0.f, 0.f, 0.f, 0.f};
    const int iq = (lane >> 2) & 3, ip = lane & 3, vrow = 4 * g4 + iq, vsw = fw_swz(vrow);
    int va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) va[i] = (4 * dh + p.vpiece) * FW_PIECE + 128 * vrow + 16 * ((2 * i + (ip >> 1)) ^ vsw) + 8 * (ip & 1);
    const int vstep = 9 * FW_PIECE + 2 * ((8 * dh + 2 * p.vpiece) * FW_KT + 4 * g4);
    wh8 v[AV + 1][2], ph[QUANT ? 2 : 1], pl[QUANT ? 2 : 1];     // (quantised: terms of a block's weights, and of the next one's)
    wh4 vd[QUANT ? AV + 1 : 1][2];
    float e[8];
    wh2 eh[4];
    auto ldv = [&](const char * buf, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) if constexpr (QUANT) vd[b % (AV + 1)][u] = *(const wh4 *) (buf + vstep + 2 * (b * FW_KT + 16 * u));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const char * a_ = buf + va[2 * (b & 1) + c] + (b >> 1) * FW_PIECE;
            const wh4 v0 = lds_tr4(a_), v1 = lds_tr4(a_ + 2048);
            v[b % (AV + 1)][c] = wh8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        }
    };
    auto ahead = [&](const char * buf) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < AV; ++b) ldv(buf, b);
    };
    // the weights times V's steps of 32-block b, as two terms
    auto terms = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const wh4 d = vd[QUANT ? b % (AV + 1) : 0][i >> 2];
            split2p(e[i], e[i + 1], eh[i >> 1], wh2{d[i & 3], d[(i & 3) + 1]}, i, ph[QUANT ? b & 1 : 0], pl[QUANT ? b & 1 : 0]);
        }
    };
    // O^T += V^T P^T, 32-blocks b0 .. b1 - 1 of this wave's channels
    auto values = [&](const char * buf, const int b0, const int b1) __attribute__((always_inline)) {
#pragma unroll
        for (int b = b0; b < b1; ++b) {
            if (b + AV < ND / 2) ldv(buf, b + AV);
            if constexpr (QUANT) { if (b + 1 < ND / 2) terms(b + 1); }
            const int w = QUANT ? b & 1 : 0;
            o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][0], ph[w], o[2 * b], 0, 0, 0);
            o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][1], ph[w], o[2 * b + 1], 0, 0, 0);
            o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][0], pl[w], o[2 * b], 0, 0, 0);
            o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b % (AV + 1)][1], pl[w], o[2 * b + 1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto weights = [&]() __attribute__((always_inline)) {
        const wf4 e0 = wgt[rg][0][lane], e1 = wgt[rg][1][lane];
        const float f = scl[rg][n16];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < 4 ? e0[i & 3] : e1[i & 3];
#pragma unroll
        for (int i = 0; i < 4; ++i) eh[i] = __builtin_bit_cast(wh2, __builtin_amdgcn_cvt_pkrtz(e[2 * i], e[2 * i + 1]));
        if (__any(f != 1.f)) {
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= f;
        }
        if constexpr (QUANT) terms(0);
        else split8(e, ph[0], pl[0]);
    };
    fw_barrier();
    if (id0 >= 0) {
        fw_barrier();
        ahead(ring);
        fw_barrier();
        for (int slot = 0;;) {                                  // the tile in `slot`; beside it the next one's scores
            const char * buf = ring + slot * BUF;
            weights();
            values(buf, 0, ND / 4);
            if (id1 >= 0) fw_barrier();
            values(buf, ND / 4, ND / 2);
            if (id1 < 0) break;
            id1 = tiles.next<ROWS>(p, j);
            slot = slot == RING - 1 ? 0 : slot + 1;
            ahead(ring + slot * BUF);
            fw_barrier();
        }
    }
    fw_barrier();
    if constexpr (QUANT) {
        const float f = __builtin_amdgcn_ldexpf(1.f, endq[rg][n16] - FQ_STEP);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= f;
    }
    fw_store<576, 512, KV, ND>(p, j, j.kb, p.k1, 64 * p.vpiece, j.r0 + 16 * rg, 256 * dh, endm[rg][lane], endl[rg][0][lane] + endl[rg][1][lane], o);
}

// ---- expanded: K rows of 192, V rows of 128 ----------------------------------------------------------
// W waves of NT row groups of 16 each, two workgroups a CU: a K or V fragment from LDS serves NT groups (and both terms),
// so with NT = 2 the LDS moves half of what the matrix instructions could take. 2048 tokens, 32 heads, 4096 keys: 260 us
// warm, 0.98 PFLOP/s, bounded as above; 499 tokens on 512: 23 us, the 16 tiles of the longest rows one after another, 1 us
// each (a tile's scores under the last one's weights, as above: 0.85, but 5 % lost on 2048 tokens, where NT = 2 did not fit)
template <int NT, int W>
__global__ __launch_bounds__(64 * W, W / 2) void k_fattn_expanded(FwArgs p) {
    constexpr int NS = 6, ND = 8, ROWS = 16 * NT * W, BUF = 5 * FW_PIECE, DMA = 20 / W;
    __shared__ __align__(128) char t0[BUF];
    __shared__ __align__(128) char t1[BUF];
    __shared__ __align__(128) char t2[BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;
    const FwJob j = fw_job<ROWS, true>(p);
    const char * const vb = p.v + (size_t) j.hk * p.v2 + (size_t) j.seq * p.v3;
    const int rg0 = j.r0 + 16 * NT * wave;

    float qx[NT][NS][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) fw_query<NS>(p, j, min(rg0 + 16 * nt + n16, j.nrow - 1), 0, qx[nt]);
    FwTiles tiles;
    tiles.w0 = 0;
    tiles.window<ROWS>(p, j);
    const int srow = lane >> 3, ssrc = 16 * ((lane & 7) ^ fw_swz(8 * wave + srow));   // (W is even: the same for rb below)
    struct Src { FwSrc k, v; int ko[4 / W], vo[4 / W]; };
    auto source = [&](int tile) __attribute__((always_inline)) {
        const int key0 = (tile & FW_TILE) * FW_KT;
        Src q{fw_src(j.kb + (size_t) key0 * p.k1), fw_src(vb + (size_t) key0 * p.v1)};
#pragma unroll
        for (int b = 0; b < 4 / W; ++b) {
            const int row = min(8 * (wave + W * b) + srow, p.n_kv - 1 - key0);  // eight rows
            q.ko[b] = row * (int) p.k1 + ssrc;
            q.vo[b] = row * (int) p.v1 + ssrc;
        }
        return q;
    };
    auto dma = [&](const Src & q, char * buf, int i) __attribute__((always_inline)) {      // piece i
#pragma unroll
        for (int b = 0; b < 4 / W; ++b)
            fw_dma(i < 3 ? q.k : q.v, i < 3 ? q.ko[b] : q.vo[b], 128 * (i < 3 ? i : i - 3), buf + i * FW_PIECE + 1024 * (wave + W * b));
    };
    char * const ring[3] = {t0, t1, t2};
    int id[3];
    id[0] = tiles.next<ROWS>(p, j);
    id[1] = id[0] >= 0 ? tiles.next<ROWS>(p, j) : -1;
    id[2] = -1;
    if (id[0] >= 0) {
        const Src q0 = source(id[0]), q1 = source(id[1] >= 0 ? id[1] : id[0]);
#pragma unroll
        for (int i = 0; i < 5; ++i) dma(q0, t0, i);
#pragma unroll
        for (int i = 0; i < 5; ++i) dma(q1, t1, i);
    }

    wh8 qh[NT][NS], ql[NT][NS];
    float qsc[NT], m[NT], l[NT];
    wf4 o[NT][ND];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        qsc[nt] = fw_terms<NS>(p, qx[nt], qh[nt], ql[nt]);
        m[nt] = -INFINITY; l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[nt][d] = wf4{0.f, 0.f, 0.f, 0.f};
    }
    const int ka0 = 128 * n16 + 16 * (g4 ^ fw_swz(n16)), ka1 = 128 * n16 + 16 * ((4 + g4) ^ fw_swz(n16));
    const int iq = (lane >> 2) & 3, ip = lane & 3, vrow = 4 * g4 + iq, vsw = fw_swz(vrow);
    int va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) va[i] = 3 * FW_PIECE + 128 * vrow + 16 * ((2 * i + (ip >> 1)) ^ vsw) + 8 * (ip & 1);

    auto body = [&](auto slot_) __attribute__((always_inline)) {
        constexpr int C = decltype(slot_)::value, F = (C + 2) % 3, N = (C + 1) % 3;
        char * const buf = ring[C];
        fw_vmcnt<DMA>();                                        // this wave's part of the tile
        fw_barrier();                                           // the tile is whole; the one before it is free
        // the tile after the next on its way, a piece a step below (all at once they hold the wave up); behind the last
        // one any, into a place no longer read
        id[F] = id[N] >= 0 ? tiles.next<ROWS>(p, j) : -1;
        const Src q = source(id[F] >= 0 ? id[F] : id[C]);
        wf4 s[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = wf4{0.f, 0.f, 0.f, 0.f};
        wh8 a[3][2];
        auto lda = [&](int i) {
#pragma unroll
            for (int u = 0; u < 2; ++u) a[i % 3][u] = *(const wh8 *) (buf + (i & 1 ? ka1 : ka0) + (i >> 1) * FW_PIECE + 2048 * u);
        };
        lda(0);
        lda(1);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i + 2 < NS) lda(i + 2);
            if (i < 5) dma(q, ring[F], i);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int u = 0; u < 2; ++u) s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % 3][u], t ? ql[nt][i] : qh[nt][i], s[nt][u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        wh8 ph[NT], pl[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            s[nt][0] *= qsc[nt];
            s[nt][1] *= qsc[nt];
        }
        if (p.softcap != 0.0f) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[nt][i >> 2][i & 3] = p.softcap * tanhf(s[nt][i >> 2][i & 3]);
        }
        if (id[C] >> 30) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) fw_mask(p, j, min(rg0 + 16 * nt + n16, j.nrow - 1), id[C] & FW_TILE, s[nt]);
        }
        wh4 v[3][2];
        auto ldv = [&](int d) {
            const char * a_ = buf + va[d & 3] + (d >> 2) * FW_PIECE;
            v[d % 3][0] = lds_tr4(a_);
            v[d % 3][1] = lds_tr4(a_ + 2048);
        };
        ldv(0);
        ldv(1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float ms = fw_raise<ND>(s[nt], m[nt], l[nt], o[nt]);
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = fw_weight(s[nt], i, ms);
                l[nt] += e[i];
            }
            split8(e, ph[nt], pl[nt]);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (d + 2 < ND) ldv(d + 2);
            const wh4 v0 = v[d % 3][0], v1 = v[d % 3][1];
            const wh8 vf = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, t ? pl[nt] : ph[nt], o[nt][d], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (;;) {
        if (id[0] < 0) break;
        body(std::integral_constant<int, 0>{});
        if (id[1] < 0) break;
        body(std::integral_constant<int, 1>{});
        if (id[2] < 0) break;
        body(std::integral_constant<int, 2>{});
    }
    fw_vmcnt<0>();                                              // no DMA outlives the workgroup's LDS
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) fw_store<192, 128, GGML_TYPE_F16, ND>(p, j, vb, p.v1, 0, rg0 + 16 * nt, 0, m[nt], l[nt], o[nt]);
}

// Joins the splits of one row. A workgroup takes 128 channels, four of them a lane; its eight half waves take every eighth
// split, so eight loads of 16 bytes a lane are in flight, on their way while every wave computes the weights for itself.
// The partials come from L2 / Infinity Cache: 128 rows, 64 splits, 16.8 MB in 5.4 us (with 256 channels and the weights
// by the workgroup 6.0).
template <int DV>
__global__ __launch_bounds__(256) void k_fattn_wide_join(FwArgs p) {
    constexpr int CH = 128, LG = CH / 4, GR = 256 / LG;         // channels, lanes and groups of them
    __shared__ __align__(16) wf4 part[GR][LG];
    const int tid = threadIdx.x, lane = tid & 63, c = tid % LG, g = tid / LG;
    const size_t rows = (size_t) p.S * p.n_q * p.H, id = blockIdx.x;
    const int h = (int) (id % p.H);
    const float * src = p.opart + id * DV + blockIdx.y * CH + 4 * c;
    wf4 v[8];
    auto fetch = [&](int s0) __attribute__((always_inline)) {   // (a split that saw nothing left nothing: read and not used)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *(const wf4 *) (src + (size_t) min(s0 + i * GR, p.nsplit - 1) * rows * DV);
    };
    fetch(g);
    constexpr int NQ = FW_MAX_SPLIT / 64;                       // split 64 q + lane
    float ms[NQ], ls[NQ], w[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int s = 64 * q + lane;
        ms[q] = s < p.nsplit ? p.mpart[s * rows + id] : -INFINITY;
        ls[q] = s < p.nsplit ? p.lpart[s * rows + id] : 0.f;
    }
    const float sink = p.sinks ? p.sinks[h] * FW_L2E : -INFINITY;
    const float m = fmaxf(wave_max<64>(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]))), sink);
    float l = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const bool none = ms[q] == -INFINITY && ls[q] == 0.f;
        w[q] = none ? -1.f : ms[q] == m ? 1.f : __builtin_amdgcn_exp2f(ms[q] - m);
        if (!none) l += ls[q] * w[q];
    }
    l = wave_sum<64>(l);
    if (p.sinks) l += fw_sink(sink, m);
    wf4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        if (64 * q >= p.nsplit) break;
        if (q) fetch(64 * q + g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = __shfl(w[q], g + i * GR, 64);       // (splits past the last have none)
            if (!(a < 0.f)) o += v[i] * a;
        }
    }
    part[g][c] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < GR; ++i) o += part[i][c];
    const size_t t = id / p.H % p.n_q, seq = id / ((size_t) p.H * p.n_q);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *(wf4 *) (p.dst + (size_t) h * p.d1 + t * p.d2 + seq * p.d3 + 4 * (blockIdx.y * CH + 4 * c)) = o * inv;
}

// The same for many rows: a wave a row and CH channels (of 128 channels, each half of it every other split). A workgroup
// a row took 44 us for 6400 rows of 512 channels and two splits
template <int DV>
__global__ __launch_bounds__(256) void k_fattn_wide_join_rows(FwArgs p) {
    constexpr int CH = DV < 256 ? DV : 256, LG = CH / 4, GR = 64 / LG;      // lanes of a split's part, splits at a time
    const int lane = threadIdx.x & 63;
    const size_t rows = (size_t) p.S * p.n_q * p.H, id = (size_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= rows) return;
    const int h = (int) (id % p.H);
    const float sink = p.sinks ? p.sinks[h] * FW_L2E : -INFINITY;
    float m = sink;
    for (int s = lane; s < p.nsplit; s += 64) m = fmaxf(m, p.mpart[s * rows + id]);
    m = wave_max<64>(m);
    const int c = lane % LG, g = lane / LG;
    const float * src = p.opart + id * DV + blockIdx.y * CH + 4 * c;
    wf4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int s0 = g; s0 < p.nsplit; s0 += 4 * GR) {
        wf4 v[4];
        float ms[4], ls[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * GR;
            const bool in = s < p.nsplit;
            ms[i] = in ? p.mpart[s * rows + id] : -INFINITY;
            ls[i] = in ? p.lpart[s * rows + id] : 0.f;
            v[i] = ms[i] == -INFINITY && ls[i] == 0.f ? wf4{0.f, 0.f, 0.f, 0.f} : *(const wf4 *) (src + (size_t) s * rows * DV);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!(ms[i] == -INFINITY && ls[i] == 0.f)) {        // a split that saw nothing left nothing to read
                const float w = ms[i] == m ? 1.f : __builtin_amdgcn_exp2f(ms[i] - m);
                l += ls[i] * w;
                o += v[i] * w;
            }
    }
    if constexpr (GR == 2) {
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], 32, 64);
    }
    if (p.sinks) l += fw_sink(sink, m);
    if (g) return;
    const size_t t = id / p.H % p.n_q, seq = id / ((size_t) p.H * p.n_q);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *(wf4 *) (p.dst + (size_t) h * p.d1 + t * p.d2 + seq * p.d3 + 4 * (blockIdx.y * CH + 4 * c)) = o * inv;
}

// The mask's tile map: for 32 tokens x one key tile, whether some key is visible and whether some value
// is not 0. Every head reads the same mask, so it is read once here instead of once a head; tiles
// without a visible key are never loaded, tiles of zeros need no mask. One wave an entry.
__global__ __launch_bounds__(256) void k_mask_map(const char * __restrict__ mask, size_t m1, size_t m3, int n_q, int n_kv, int n_tiles, int n_tb,
                                                  uint8_t * __restrict__ map) {
    const int lane = threadIdx.x & 63;
    const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), tb = blockIdx.y, seq = blockIdx.z;
    if (tile >= n_tiles) return;
    constexpr int PER = FW_KT / 8, TOK = 64 / PER;                 // lanes of a token's row, tokens a pass
    uint32_t f = 0;
#pragma unroll
    for (int t0 = 0; t0 < FW_TB; t0 += TOK) {
        const int t = tb * FW_TB + t0 + lane / PER, key = tile * FW_KT + 8 * (lane % PER);
        if (t >= n_q) continue;
        const char * mr = mask + (size_t) t * m1 + (size_t) seq * m3;
        if (key + 8 <= n_kv) {
            const uint4 v = ldu16(mr + 2 * (size_t) key);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) f |= ((w[i] & 0xFFFF) != 0xFC00 || (w[i] >> 16) != 0xFC00 ? FW_LIVE : 0) | (w[i] & 0x7FFF7FFF ? FW_MIXED : 0);
        } else {
            for (int i = 0; key + i < n_kv; ++i) {
                const uint32_t w = ((const uint16_t *) mr)[key + i];
                f |= (w != 0xFC00 ? FW_LIVE : 0) | (w & 0x7FFF ? FW_MIXED : 0);
            }
        }
    }
    const bool live = __any(f & FW_LIVE), mixed = __any(f & FW_MIXED);
    if (lane == 0) map[((size_t) seq * n_tb + tb) * n_tiles + tile] = (live ? FW_LIVE : 0) | (mixed ? FW_MIXED : 0);
}

// ---- host ------------------------------------------------------------------------------------------
struct FwPlan { bool wide; int rows, nsplit, n_tiles, n_tb; size_t part, map; };
constexpr size_t FW_JOIN_ROWS = 2048;   // from so many rows (times chunks) on the join takes a wave each: 4096 and four splits
                                        // 35 against 40 us in all, 1024 and sixteen 30 against 27
// From so many tokens of a workgroup on the tile map is built by a launch of its own, where a split has more than two tiles
// (expanded, 16 heads, 16 tokens on 8192: 25 us with the map, 30 listing from the mask's rows; 32 on 4096: 22 and 36). Fewer
// tokens are listed by every wave for itself (latent, 32 heads, 128 tokens on 1024 at 4 bits: 47.5, with the map 49.6), two
// tiles are not listed at all (expanded, 20 tokens on 2048: 13.8, with the map 16.1)
constexpr int FW_MAP_TOK = 5;

// Rows of a workgroup and splits: those that end soonest by the times below, measured (us). A tile of a workgroup takes
// t1 alone on its CU, t2 beside another (the absorbed form's tiles fill the LDS); its begin and end 6, the join 4 and
// 1 for 8 MB of partial results. Absorbed, f16, 32 heads: 64 tokens, 1024 keys 29.6 with 32 rows and 4 splits (64 rows, 8
// splits: 35); 512 tokens, 4096 keys 257 with 64 rows (32: 278)
// Expanded: 128 rows where they fill every CU twice (2048 tokens and keys, 32 heads: 118 against 134 with 64), else 64
// (499 tokens: 26 against 39); 32 for no more rows than that (16 tokens, 1024 keys 14.6 against 15.8)
struct FwRows { int rows; double t1, t2; };
static FwPlan fw_plan(const ggml_tensor * dst) {
    const ggml_tensor * q = dst->src[0], * k = dst->src[1], * v = dst->src[2], * m = dst->src[3];
    static const FwRows latent[2] = {{32, 1.0, 0}, {64, 1.63, 0}}, quant[1] = {{32, 1.55, 0}}, expanded[3] = {{32, 1.03, 1.27}, {64, 0.93, 1.46}, {128, 1.45, 2.8}};
    FwPlan p{};
    p.wide = k->ne[0] == 576;
    const int64_t G = q->ne[2] / k->ne[2], nrow = q->ne[1] * G, units = k->ne[2] * q->ne[3];
    const size_t rows = (size_t) q->ne[1] * q->ne[2] * q->ne[3];
    p.n_tiles = (int) mx_ceil_div(k->ne[1], FW_KT);
    const FwRows * cand = p.wide ? (k->type == GGML_TYPE_F16 ? latent : quant) : &expanded[nrow <= 32 ? 0 : units * mx_ceil_div(nrow, 128) >= 512 ? 2 : 1];
    const int n_cand = p.wide && k->type == GGML_TYPE_F16 && nrow > 32 ? 2 : 1;
    double best = 0;
    for (int c = 0; c < n_cand; ++c) {
        const int64_t blocks = units * mx_ceil_div(nrow, cand[c].rows);
        for (int ns = 1; ns <= FW_MAX_SPLIT && ns <= p.n_tiles; ++ns) {
            const int64_t n = blocks * ns, per = mx_ceil_div(p.n_tiles, ns);
            const bool pair = !p.wide && n > 256;
            const double us = (double) mx_ceil_div(n, pair ? 512 : 256) * ((double) per * (pair ? cand[c].t2 : cand[c].t1) + 6) +
                              (ns > 1 ? 4 + (double) rows * ns * v->ne[0] * 1e-6 : 0);
            if (p.nsplit == 0 || us < best) { best = us; p.nsplit = ns; p.rows = cand[c].rows; }
        }
    }
    p.part = p.nsplit > 1 ? (size_t) p.nsplit * rows : 0;
    p.n_tb = (int) mx_ceil_div(q->ne[1], FW_TB);
    if (m && m->ne[2] == 1 && std::min<int64_t>(q->ne[1], (p.rows + G - 2) / G + 1) >= FW_MAP_TOK && mx_ceil_div(p.n_tiles, p.nsplit) > 2) p.map = (size_t) m->ne[3] * p.n_tb * p.n_tiles;
    return p;
}

bool fa_wide_supported(const ggml_tensor * dst) {
    const ggml_tensor * q = dst->src[0], * k = dst->src[1], * v = dst->src[2], * m = dst->src[3], * sk = dst->src[4];
    if (q->type != GGML_TYPE_F32 || dst->type != GGML_TYPE_F32 || q->nb[0] != 4 || dst->nb[0] != 4 || q->ne[0] != k->ne[0]) return false;
    const bool wide = k->ne[0] == 576 && v->ne[0] == 512;
    if (!wide && !(k->ne[0] == 192 && v->ne[0] == 128)) return false;
    if (k->type != v->type || !(k->type == GGML_TYPE_F16 || (wide && (k->type == GGML_TYPE_Q8_0 || k->type == GGML_TYPE_Q4_0)))) return false;
    const size_t es = mx_type(k->type).size;
    if (k->nb[0] != es || v->nb[0] != es || v->ne[1] != k->ne[1] || v->ne[2] != k->ne[2] || v->ne[3] != k->ne[3]) return false;
    if (k->ne[1] < 1 || k->ne[2] < 1 || q->ne[2] % k->ne[2] || (q->ne[3] != k->ne[3] && k->ne[3] != 1)) return false;
    if (wide) {
        // the values are channels of the key's own row, from its start or behind 64 others
        const ggml_tensor * kr = k->view_src ? k->view_src : k, * vr = v->view_src ? v->view_src : v;
        const size_t ko = k->view_src ? k->view_offs : 0, vo = v->view_src ? v->view_offs : 0;
        if (kr != vr || (vo != ko && vo != ko + mx_row_size(k->type, 64))) return false;
        for (int i = 1; i < 4; ++i) if (k->nb[i] != v->nb[i] && k->ne[i] > 1) return false;
    }
    // f16 rows go to LDS 16 bytes at a time; blocks are 2-byte aligned
    const size_t al = k->type == GGML_TYPE_F16 ? 16 : 2;
    for (int i = 1; i < 4; ++i) if (q->nb[i] % 4 || dst->nb[i] % 16 || k->nb[i] % al || v->nb[i] % al) return false;
    for (const ggml_tensor * t : {k, v}) if (t->view_offs % al || (uintptr_t) t->data % al) return false;
    if ((uintptr_t) q->data % 4 || (uintptr_t) dst->data % 16) return false;
    if (dst->ne[0] != v->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3]) return false;
    if (m && (m->type != GGML_TYPE_F16 || m->nb[0] != 2 || m->ne[0] < k->ne[1] || m->ne[1] < q->ne[1] || m->ne[2] < 1 || m->ne[3] < 1 ||
              q->ne[2] % m->ne[2] || q->ne[3] % m->ne[3] || m->nb[1] % 2 || m->nb[2] % 2 || m->nb[3] % 2)) return false;
    if (sk && (sk->type != GGML_TYPE_F32 || sk->nb[0] != 4 || sk->ne[0] < q->ne[2])) return false;
    if (mx_op_param<float>(dst, 1) > 0.0f && !m) return false;
    // grid and index ranges of the kernels; a tile's rows are addressed in 31 bits
    if (k->nb[1] > INT32_MAX / 64 || v->nb[1] > INT32_MAX / 64) return false;
    const int64_t G = q->ne[2] / k->ne[2];
    return k->ne[1] <= INT32_MAX / 2 - 64 && q->ne[1] * G < INT32_MAX / 2 && q->ne[1] * q->ne[2] * q->ne[3] < INT32_MAX / 2 &&
           mx_ceil_div(q->ne[1], FW_TB) < 65536 && q->ne[3] < 65536;
}

size_t fa_wide_scratch(const ggml_tensor * dst) {
    if (!fa_wide_supported(dst)) return 0;
    const FwPlan p = fw_plan(dst);
    return p.part * (dst->ne[0] + 2) * sizeof(float) + p.map + 5 * 256;
}

void fa_wide_run(OpCtx & c, ggml_tensor * dst) {
    const ggml_tensor * q = dst->src[0], * k = dst->src[1], * v = dst->src[2], * m = dst->src[3], * sk = dst->src[4];
    const FwPlan pl = fw_plan(dst);
    FwArgs a{};
    a.q = (const char *) q->data; a.q1 = q->nb[1]; a.q2 = q->nb[2]; a.q3 = q->nb[3];
    a.k = (const char *) k->data; a.k1 = k->nb[1]; a.k2 = k->nb[2]; a.k3 = k->ne[3] == 1 ? 0 : k->nb[3];
    a.v = (const char *) v->data; a.v1 = v->nb[1]; a.v2 = v->nb[2]; a.v3 = v->ne[3] == 1 ? 0 : v->nb[3];
    if (m) { a.mask = (const char *) m->data; a.m1 = m->nb[1]; a.m2 = m->nb[2]; a.m3 = m->nb[3]; a.mne2 = (int) m->ne[2]; a.mne3 = (int) m->ne[3]; }
    else a.mne2 = a.mne3 = 1;
    a.sinks = sk ? (const float *) sk->data : nullptr;
    a.dst = (char *) dst->data; a.d1 = dst->nb[1]; a.d2 = dst->nb[2]; a.d3 = dst->nb[3];
    a.n_q = (int) q->ne[1]; a.n_kv = (int) k->ne[1]; a.H = (int) q->ne[2]; a.Hkv = (int) k->ne[2]; a.G = a.H / a.Hkv; a.S = (int) q->ne[3];
    a.nsplit = pl.nsplit; a.n_tiles = pl.n_tiles;
    if (pl.wide && v->data != k->data) a.vpiece = 1;
    a.scale = mx_op_param<float>(dst, 0);
    a.max_bias = mx_op_param<float>(dst, 1);
    a.softcap = mx_op_param<float>(dst, 2);
    if (a.softcap != 0.0f) { a.scale /= a.softcap; a.softcap *= FW_L2E; }
    else a.scale *= FW_L2E;
    a.n_head_log2 = 1u << (uint32_t) floor(log2((double) a.H));
    a.m0 = powf(2.0f, -(a.max_bias) / a.n_head_log2);
    a.m1f = powf(2.0f, -(a.max_bias / 2.0f) / a.n_head_log2);
    const int DV = (int) v->ne[0];
    if (pl.part) {
        a.opart = (float *) c.scratch->take(pl.part * DV * sizeof(float));
        a.mpart = (float *) c.scratch->take(pl.part * sizeof(float));
        a.lpart = (float *) c.scratch->take(pl.part * sizeof(float));
    }
    if (pl.map) {
        uint8_t * map = (uint8_t *) c.scratch->take(pl.map);
        const dim3 grid((unsigned) mx_ceil_div(pl.n_tiles, 4), (unsigned) pl.n_tb, (unsigned) a.mne3);
        k_mask_map<<<grid, 256, 0, c.st>>>(a.mask, a.m1, a.m3, a.n_q, a.n_kv, pl.n_tiles, pl.n_tb, map);
        a.map = map;
        a.n_tb = pl.n_tb;
    }
    MX_KLOG("fattn_wide DK=%d type=%d rows=%d nsplit=%d map=%d", (int) k->ne[0], (int) k->type, pl.rows, pl.nsplit, pl.map != 0);
    const dim3 grid((unsigned) (mx_ceil_div((int64_t) a.n_q * a.G, pl.rows) * a.Hkv * a.S), (unsigned) pl.nsplit);
    if (!pl.wide) {
        if (pl.rows == 32) k_fattn_expanded<1, 2><<<grid, 128, 0, c.st>>>(a);
        else if (pl.rows == 64) k_fattn_expanded<1, 4><<<grid, 256, 0, c.st>>>(a);
        else        k_fattn_expanded<2, 4><<<grid, 256, 0, c.st>>>(a);
    } else if (k->type == GGML_TYPE_Q8_0) k_fattn_latent32<GGML_TYPE_Q8_0><<<grid, 768, 0, c.st>>>(a);
    else if (k->type == GGML_TYPE_Q4_0) k_fattn_latent32<GGML_TYPE_Q4_0><<<grid, 768, 0, c.st>>>(a);
    else if (pl.rows == 32) k_fattn_latent32<GGML_TYPE_F16><<<grid, 768, 0, c.st>>>(a);
    else k_fattn_latent64<<<grid, 512, 0, c.st>>>(a);
    if (pl.nsplit > 1) {
        const unsigned rows = (unsigned) (a.S * a.n_q * a.H), chunks = (unsigned) (DV / std::min(DV, 256));
        if (rows * (size_t) chunks >= FW_JOIN_ROWS) {
            const dim3 grid((rows + 3) / 4, chunks);
            if (pl.wide) k_fattn_wide_join_rows<512><<<grid, 256, 0, c.st>>>(a);
            else         k_fattn_wide_join_rows<128><<<grid, 256, 0, c.st>>>(a);
        } else {
            const dim3 grid(rows, (unsigned) (DV / 128));
            if (pl.wide) k_fattn_wide_join<512><<<grid, 256, 0, c.st>>>(a);
            else         k_fattn_wide_join<128><<<grid, 256, 0, c.st>>>(a);
        }
    }
}

}  // namespace mx
