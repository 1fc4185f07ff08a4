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
// units as two terms, high + low (22 bits), each product twice; K and V are exact in f16, quantised
// ones as their integers with the block's step applied in f32 (to the products of K, to the weights of
// V). The rate that bounds the large cases is therefore half the f16 rate.
//
// Split: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_16x16x32_f16, so a lane holds scores and
// outputs of one query row (lane & 15): softmax state and rescaling are lane-local, and P^T goes from
// the score registers straight into the second product (its k index runs over the keys the lane has;
// V's rows follow by transposing LDS reads). A workgroup's four waves share one K/V tile in LDS; they
// are RG groups of 16 NT query rows (any mix of heads and tokens of one KV head: rows are flattened
// token-major), and 4 / RG key groups whose results are merged at the end. Tiles are double-buffered,
// the next tile in flight in registers meanwhile. With few rows the tiles are dealt out over `nsplit`
// workgroups and joined by a second launch.
#include "backend.h"
#include "quants.cuh"

#include <algorithm>
#include <type_traits>

namespace mx {

typedef _Float16 wh8 __attribute__((ext_vector_type(8)));
typedef _Float16 wh4 __attribute__((ext_vector_type(4)));
typedef _Float16 wh2 __attribute__((ext_vector_type(2)));
typedef float wf4 __attribute__((ext_vector_type(4)));
typedef __fp16 w16x4 __attribute__((vector_size(8)));
typedef __attribute__((address_space(3))) w16x4 * lds_w4;

constexpr int FW_WIN = 1024;                 // tiles a workgroup lists at a time
constexpr int FW_TB = 32;                    // tokens of one entry of the mask's tile map
constexpr float FW_L2E = 1.4426950408889634f;
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
    int n_q, n_kv, H, G, Hkv, S, nsplit, n_tiles, vchunk;   // vchunk: V's first 16-byte chunk (or 32-block) of a K row
    float scale, softcap, max_bias, m0, m1f;
    uint32_t n_head_log2;
};

__device__ __forceinline__ uint4 ldu16(const char * p) { uint4 v; __builtin_memcpy(&v, p, 16); return v; }

// hi + lo = x to 22 bits: the high term truncated, the remainder (exact in f32) truncated again
__device__ __forceinline__ void split8(const float (&x)[8], wh8 & hi, wh8 & lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const wh2 h = __builtin_bit_cast(wh2, __builtin_amdgcn_cvt_pkrtz(x[j], x[j + 1]));
        const wh2 l = __builtin_bit_cast(wh2, __builtin_amdgcn_cvt_pkrtz(x[j] - (float) h[0], x[j + 1] - (float) h[1]));
        hi[j] = h[0]; hi[j + 1] = h[1];
        lo[j] = l[0]; lo[j + 1] = l[1];
    }
}

// element i of a cache row, for the plain loop below
template <int KV> __device__ __forceinline__ float fw_get(const char * row, int i) {
    if constexpr (KV == GGML_TYPE_F16) return h2f(*(const uint16_t *) (row + 2 * (size_t) i));
    else return dequant_one<KV>(row + (size_t) (i >> 5) * qsize_of<KV>(), i & 31);
}

__device__ __forceinline__ float fw_slope(const FwArgs & p, uint32_t h) {
    return p.max_bias > 0.0f ? (h < p.n_head_log2 ? powf(p.m0, h + 1) : powf(p.m1f, 2 * (h - p.n_head_log2) + 1)) : 1.0f;
}

// 16-byte chunk `ch` of LDS row `row`: chunks are XORed within groups of eight so that eight
// consecutive rows' reads at one chunk, and the transposing reads of four rows x two chunks, fall on
// different banks (rows are multiples of 128 B)
__device__ __forceinline__ int fw_swz(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

template <int DK, int DV, int KV, bool VSEP, int NT, int RG, int KT>
struct FwGeo {
    static constexpr int KB = 2 * DK, VB = 2 * DV;              // LDS row bytes (f16 values)
    static constexpr int KTILE = KT * KB, VTILE = VSEP ? KT * VB : 0;
    static constexpr int NBLK = DK / 32;                        // quantised blocks of a row
    static constexpr int STILE = KV == GGML_TYPE_F16 ? 0 : NBLK * KT * 4;   // their steps, [block][key] f32
    static constexpr int BUF = KTILE + VTILE + STILE;
    static constexpr int LDS = 2 * BUF + FW_WIN * 2 + 16 + 32;  // + the tile list, the buffers' largest steps [2][4 waves]
    static constexpr int ROWS = 16 * NT * RG;
};

template <int DK, int DV, int KV, bool VSEP, int NT, int RG, int KT, int OCC>
__global__ __launch_bounds__(256, OCC) void k_fattn_wide(FwArgs p) {
    using geo = FwGeo<DK, DV, KV, VSEP, NT, RG, KT>;
    constexpr bool QUANT = KV != GGML_TYPE_F16;
    constexpr int KG = 4 / RG;                                  // key groups
    constexpr int KW = KT / KG, NSUB = KW / 16, NKH = NSUB / 2; // keys of a wave, in 16s and 32s
    constexpr int NS = DK / 32, ND = DV / 16;
    static_assert(KW % 32 == 0 && DK % 64 == 0 && DV % 64 == 0, "tiles");
    extern __shared__ __align__(16) char lds[];
    uint16_t * const list = (uint16_t *) (lds + 2 * geo::BUF);
    int * const list_n = (int *) (list + FW_WIN);
    float * const dtop = (float *) (list_n + 4);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n16 = lane & 15, g4 = lane >> 4;
    const int rg = wave % RG, kg = wave / RG;
    const int split = blockIdx.y;
    // (KV head, sequence) units: with a multiple of eight the workgroups of one unit stay on one XCD
    // and share its L2; the last rows (most keys, under a causal mask) go first
    const int nrb = (p.n_q * p.G + geo::ROWS - 1) / geo::ROWS, units = p.Hkv * p.S;
    int unit, rb;
    if (units % 8 == 0) { unit = blockIdx.x % 8 + 8 * (blockIdx.x / 8 / nrb); rb = nrb - 1 - blockIdx.x / 8 % nrb; }
    else { unit = blockIdx.x / nrb; rb = nrb - 1 - blockIdx.x % nrb; }
    const int hk = unit % p.Hkv, seq = unit / p.Hkv;
    const int nrow = p.n_q * p.G;
    const char * const kb = p.k + (size_t) hk * p.k2 + (size_t) seq * p.k3;
    const char * const vb = VSEP ? p.v + (size_t) hk * p.v2 + (size_t) seq * p.v3 : kb;

    // ---- this lane's query rows
    int tok[NT], head[NT];
    const char * mrow[NT];
    float slope[NT], qsc[NT];
    wh8 qh[NT][NS], ql[NT][NS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = min(rb * geo::ROWS + (rg * NT + nt) * 16 + n16, nrow - 1);
        tok[nt] = r / p.G;
        head[nt] = hk * p.G + r % p.G;
        slope[nt] = fw_slope(p, (uint32_t) head[nt]);
        mrow[nt] = p.mask ? p.mask + (size_t) tok[nt] * p.m1 + (size_t) (head[nt] % p.mne2) * p.m2 + (size_t) (seq % p.mne3) * p.m3 : nullptr;
        const char * qp = p.q + (size_t) tok[nt] * p.q1 + (size_t) head[nt] * p.q2 + (size_t) seq * p.q3;
        float x[NS][8], top = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const uint4 a = ldu16(qp + 4 * (32 * s + 8 * g4)), b = ldu16(qp + 4 * (32 * s + 8 * g4 + 4));
            __builtin_memcpy(&x[s][0], &a, 16);
            __builtin_memcpy(&x[s][4], &b, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[s][j]));
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // the row's largest magnitude to 2^13 .. 2^14: what the low term then loses is below 2^-38 of it
        const int e = top > 0.f && top < INFINITY ? max(-100, min(100, 14 - __builtin_amdgcn_frexp_expf(top))) : 0;
        qsc[nt] = p.scale * __builtin_amdgcn_ldexpf(1.f, -e);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = __builtin_amdgcn_ldexpf(x[s][j], e);
            split8(x[s], qh[nt][s], ql[nt][s]);
        }
    }

    wf4 o[NT][ND];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt] = -INFINITY; l_run[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[nt][d] = wf4{0.f, 0.f, 0.f, 0.f};
    }

    // quantised: the weights take V's steps before they are split, so they and O are held in units of
    // 2^(qe - 7), 2^qe the largest step seen: neither term of a weight falls out of f16's range
    int qe = -1000;
    // ---- tile staging. f16: eight threads read 128 B of a row at a time, rows tid / 8 and + 32;
    // chunk c of LDS row r holds the source's c ^ swz(r), so the LDS writes are linear
    constexpr int KI = DK / 64, VI = DV / 64, RP = KT / 32;     // 128-byte pieces of a row, row passes
    const int srow = tid >> 3, sch = tid & 7;
    const int ssrc = 16 * (sch ^ fw_swz(srow));
    uint4 kst[QUANT ? 1 : RP * KI], vst[VSEP ? RP * VI : 1];
    // quantised: a thread takes blocks tid % 4 + 4 i of row tid / 4
    constexpr int QB = qsize_of<QUANT ? KV : GGML_TYPE_Q8_0>(), QI = (geo::NBLK + 3) / 4;
    uint4 qa[QUANT ? QI : 1], qb[KV == GGML_TYPE_Q8_0 ? QI : 1];
    uint16_t qd[QUANT ? QI : 1];
    auto load_tile = [&](int tile) {
        if constexpr (!QUANT) {
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                const size_t key = (size_t) min(tile * KT + 32 * r + srow, p.n_kv - 1);
                const char * kr = kb + key * p.k1 + ssrc;
#pragma unroll
                for (int i = 0; i < KI; ++i) kst[r * KI + i] = ldu16(kr + 128 * i);
                if constexpr (VSEP) {
                    const char * vr = vb + key * p.v1 + ssrc;
#pragma unroll
                    for (int i = 0; i < VI; ++i) vst[r * VI + i] = ldu16(vr + 128 * i);
                }
            }
        } else {
            const char * kr = kb + (size_t) min(tile * KT + (tid >> 2), p.n_kv - 1) * p.k1;
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const char * b = kr + (size_t) min((tid & 3) + 4 * i, geo::NBLK - 1) * QB;
                qd[i] = ld_u16(b);
                qa[i] = ldu16(b + 2);
                if constexpr (KV == GGML_TYPE_Q8_0) qb[i] = ldu16(b + 18);
            }
        }
    };
    auto store_tile = [&](char * buf) {
        if constexpr (!QUANT) {
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                char * kd = buf + (32 * r + srow) * geo::KB + 16 * sch;
#pragma unroll
                for (int i = 0; i < KI; ++i) *(uint4 *) (kd + 128 * i) = kst[r * KI + i];
                if constexpr (VSEP) {
                    char * vd = buf + geo::KTILE + (32 * r + srow) * geo::VB + 16 * sch;
#pragma unroll
                    for (int i = 0; i < VI; ++i) *(uint4 *) (vd + 128 * i) = vst[r * VI + i];
                }
            }
        } else {
            // integers to f16 exactly: 1024 + n has n in its low bits, two at a time
            const int row = tid >> 2, sw = fw_swz(row);
            float * steps = (float *) (buf + geo::KTILE);
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const int b = (tid & 3) + 4 * i;
                if (b < geo::NBLK) {
                    steps[b * KT + row] = h2f(qd[i]);
                    top = fmaxf(top, fabsf(h2f(qd[i])));
                    uint32_t w[16];                             // 32 values in order, as f16 pairs
                    if constexpr (KV == GGML_TYPE_Q8_0) {
                        const uint32_t src[8] = {qa[i].x, qa[i].y, qa[i].z, qa[i].w, qb[i].x, qb[i].y, qb[i].z, qb[i].w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t u = src[j] ^ 0x80808080u;            // n + 128
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const uint32_t pr = __builtin_amdgcn_perm(0x64646464u, u, t ? 0x04030402u : 0x04010400u);
                                w[2 * j + t] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(wh2, pr) - wh2{(_Float16) 1152.f, (_Float16) 1152.f});
                            }
                        }
                    } else {
                        const uint32_t src[4] = {qa[i].x, qa[i].y, qa[i].z, qa[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int t = 0; t < 4; ++t) {       // bytes 4j + 2(t&1), + 1; low nibbles are values 0..15, high 16..31
                                const uint32_t nib = (t & 2 ? src[j] >> 4 : src[j]) & 0x0F0F0F0Fu;
                                const uint32_t pr = __builtin_amdgcn_perm(0x64646464u, nib, t & 1 ? 0x04030402u : 0x04010400u);
                                w[2 * j + (t & 1) + (t & 2 ? 8 : 0)] =
                                    __builtin_bit_cast(uint32_t, __builtin_bit_cast(wh2, pr) - wh2{(_Float16) 1032.f, (_Float16) 1032.f});
                            }
                    }
                    char * kd = buf + row * geo::KB;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *(uint4 *) (kd + 16 * ((4 * b + j) ^ sw)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
            }
            top = wave_max<64>(top);
            if (lane == 0) dtop[(buf == lds ? 0 : 4) + wave] = top;
        }
    };
    // mask words of a tile for this lane: keys 16 sub + 4 g4 + 0..3; beyond the row's end -inf
    uint2 mk[NT][NSUB], mkn[NT][NSUB];
    auto load_mask = [&](int tile, uint2 (&m)[NT][NSUB]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int s = 0; s < NSUB; ++s) {
                const int key = tile * KT + kg * KW + 16 * s + 4 * g4;
                uint32_t v[4];
                if (key + 4 <= p.n_kv) {
                    uint2 u = make_uint2(0, 0);
                    if (mrow[nt]) __builtin_memcpy(&u, mrow[nt] + 2 * (size_t) key, 8);
                    m[nt][s] = u;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = key + j >= p.n_kv ? 0xFC00u : mrow[nt] ? ((const uint16_t *) mrow[nt])[key + j] : 0u;
                    m[nt][s] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
                }
            }
    };

    const int nl = (p.n_tiles - split + p.nsplit - 1) / p.nsplit;   // this split's tiles: split, split + nsplit, ...
    const int t_lo = min(rb * geo::ROWS, nrow - 1) / p.G, t_hi = min(rb * geo::ROWS + geo::ROWS - 1, nrow - 1) / p.G;

    // per-lane LDS offsets, constant over tiles
    const int krow = kg * KW + n16;
    const int ka0 = krow * geo::KB + 16 * (g4 ^ fw_swz(n16)), ka1 = krow * geo::KB + 16 * ((4 + g4) ^ fw_swz(n16));
    const int iq = (lane >> 2) & 3, ip = lane & 3;
    const int vrow = kg * KW + 4 * g4 + iq, vsw = fw_swz(4 * g4 + iq);
    int va[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        va[j] = (VSEP ? geo::KTILE : 16 * (QUANT ? 4 : 1) * p.vchunk) + vrow * (VSEP ? geo::VB : geo::KB) + 16 * ((2 * j + (ip >> 1)) ^ vsw) + 8 * (ip & 1);
    constexpr int VROW = VSEP ? geo::VB : geo::KB;

    for (int w0 = 0; w0 < nl; w0 += FW_WIN) {
        // ---- list the window's tiles that some row of the workgroup looks at
        const int nw = min(FW_WIN, nl - w0);
        const bool per_head = p.mask && p.mne2 > 1;
        uint32_t * flag = (uint32_t *) lds;                     // (the tile buffers are free here)
        for (int j = tid; j < nw; j += 256) {
            const int tile = split + (w0 + j) * p.nsplit;
            uint32_t f = 0;
            if (p.mask && !per_head && p.map) {
                bool live = false, mixed = false;
                for (int tb = t_lo / FW_TB; tb <= t_hi / FW_TB; ++tb) {
                    const uint32_t u = p.map[((size_t) (seq % p.mne3) * p.n_tb + tb) * p.n_tiles + tile];
                    live |= u & FW_LIVE; mixed |= u & FW_MIXED;
                }
                f = (live ? FW_LIVE : 0) | (mixed ? FW_MIXED : 0);
            } else if (!p.mask) f = FW_LIVE;
            else if (per_head || nl <= 2) f = FW_LIVE | FW_MIXED;
            if ((tile + 1) * KT > p.n_kv) f |= FW_MIXED;        // the row's end lies inside
            flag[j] = f;
        }
        __syncthreads();
        if (p.mask && !per_head && !p.map && nl > 2) {
            // few tokens: read their mask rows here, a thread (8 keys) at a time
            const int nt_ = t_hi - t_lo + 1, per = KT / 8;
            for (int u = tid; u < nw * nt_ * per; u += 256) {
                const int c = u % per, j = u / per % nw, t = t_lo + u / per / nw;
                const int key = (split + (w0 + j) * p.nsplit) * KT + 8 * c;
                const char * mr = p.mask + (size_t) t * p.m1 + (size_t) (seq % p.mne3) * p.m3;
                uint32_t f = 0;
                if (key + 8 <= p.n_kv) {
                    const uint4 v = ldu16(mr + 2 * (size_t) key);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) f |= ((w[i] & 0xFFFF) != 0xFC00 || (w[i] >> 16) != 0xFC00 ? FW_LIVE : 0) | (w[i] & 0x7FFF7FFF ? FW_MIXED : 0);
                } else {
                    for (int i = 0; key + i < p.n_kv; ++i) {
                        const uint32_t w = ((const uint16_t *) mr)[key + i];
                        f |= (w != 0xFC00 ? FW_LIVE : 0) | (w & 0x7FFF ? FW_MIXED : 0);
                    }
                }
                if (f) atomicOr(&flag[j], f);
            }
            __syncthreads();
        }
        if (wave == 0) {
            int n = 0;
            for (int j0 = 0; j0 < nw; j0 += 64) {
                const uint32_t f = j0 + lane < nw ? flag[j0 + lane] : 0;
                const uint64_t b = __ballot(f & FW_LIVE);
                if (f & FW_LIVE) list[n + __popcll(b & ((1ull << lane) - 1))] = (uint16_t) (j0 + lane) | (f & FW_MIXED ? 0x8000 : 0);
                n += __popcll(b);
            }
            if (lane == 0) *list_n = n;
        }
        __syncthreads();
        const int cnt = *list_n;
        auto entry = [&](int i) { return __builtin_amdgcn_readfirstlane((int) list[i]); };
        auto tile_of = [&](int e) { return split + (w0 + (e & 0x7FFF)) * p.nsplit; };
        int cur = 0, ent = 0;
        if (cnt > 0) {
            ent = entry(0);
            load_tile(tile_of(ent));
            if (ent & 0x8000) load_mask(tile_of(ent), mk);
            store_tile(lds);
        }
        __syncthreads();
        for (int i = 0; i < cnt; ++i) {
            char * const buf = lds + cur * geo::BUF;
            const bool more = i + 1 < cnt, mixed = ent & 0x8000;
            int next = 0;
            if (more) {
                next = entry(i + 1);
                load_tile(tile_of(next));
                if (next & 0x8000) load_mask(tile_of(next), mkn);
            }
            // ---- S^T: keys x rows
            wf4 s[NT][NSUB];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < NSUB; ++u) s[nt][u] = wf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                wh8 a[NSUB];
#pragma unroll
                for (int u = 0; u < NSUB; ++u) a[u] = *(const wh8 *) (buf + (st & 1 ? ka1 : ka0) + 128 * (st >> 1) + u * 16 * geo::KB);
                if constexpr (!QUANT) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int u = 0; u < NSUB; ++u) s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], qh[nt][st], s[nt][u], 0, 0, 0);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int u = 0; u < NSUB; ++u) s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], ql[nt][st], s[nt][u], 0, 0, 0);
                } else {
                    // one 32-block a step: its products are whole, then take the block's step
                    wf4 t[NT][NSUB];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int u = 0; u < NSUB; ++u) t[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], qh[nt][st], wf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int u = 0; u < NSUB; ++u) t[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], ql[nt][st], t[nt][u], 0, 0, 0);
#pragma unroll
                    for (int u = 0; u < NSUB; ++u) {
                        const wf4 d = *(const wf4 *) (buf + geo::KTILE + 4 * (st * KT + kg * KW + 16 * u + 4 * g4));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) s[nt][u][j] += d[j] * t[nt][u][j];
                    }
                }
            }
            float qf = 1.f;
            if constexpr (QUANT) {
                const wf4 dm = *(const wf4 *) (dtop + 4 * cur);
                const float top = fmaxf(fmaxf(dm[0], dm[1]), fmaxf(dm[2], dm[3]));
                const int e = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : -1000;
                if (e > qe) {                                   // the same in every wave; on the first tiles only
                    const float f = __builtin_amdgcn_ldexpf(1.f, max(qe - e, -200));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int d = 0; d < ND; ++d) o[nt][d] *= f;
                    qe = e;
                }
                qf = qe == -1000 ? 1.f : __builtin_amdgcn_ldexpf(1.f, 7 - qe);
            }
            // ---- softmax of this lane's rows, its keys; the reference maximum is raised only when
            // a score exceeds it by 5.5 (weights up to 2^8), so O is rescaled on the first tiles only
            wh8 ph[NT][NKH], pl[NT][NKH];
            float pw[QUANT ? NT : 1][QUANT ? NKH : 1][8];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float mt = -INFINITY;
#pragma unroll
                for (int u = 0; u < NSUB; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float x = s[nt][u][j] * qsc[nt];
                        if (p.softcap != 0.0f) x = p.softcap * tanhf(x);
                        if (mixed) {
                            const uint32_t w = j & 2 ? mk[nt][u].y : mk[nt][u].x;
                            const float mv = h2f((uint16_t) (j & 1 ? w >> 16 : w & 0xFFFF));
                            x = mv == -INFINITY ? -INFINITY : x + slope[nt] * mv;   // (a masked key's K may be anything)
                        }
                        s[nt][u][j] = x;
                        mt = fmaxf(mt, x);
                    }
                mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
                mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
                const bool raise = mt > m_run[nt] + 5.5f;       // false while nothing was visible
                if (__any(raise)) {
                    const float al = raise ? __builtin_amdgcn_exp2f((m_run[nt] - mt) * FW_L2E) : 1.f;
                    if (raise) m_run[nt] = mt;
                    l_run[nt] *= al;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[nt][d][j] *= al;
                }
                const float ms = m_run[nt] == -INFINITY ? 0.f : -m_run[nt] * FW_L2E;
#pragma unroll
                for (int h = 0; h < NKH; ++h) {
                    float e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][2 * h + (j >> 2)][j & 3], FW_L2E, ms));
                        l_run[nt] += e[j];
                        if constexpr (QUANT) pw[nt][h][j] = e[j] * qf;
                    }
                    if constexpr (!QUANT) split8(e, ph[nt][h], pl[nt][h]);
                }
            }
            // ---- O^T += V^T P^T: keys 4 g4 + 0..3 of two 16-key blocks a lane, as the scores lie
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                if constexpr (QUANT) {
                    if (d % 2 == 0) {                           // a 32-block of V: its steps enter the weights
                        const int b = p.vchunk + d / 2;
#pragma unroll
                        for (int h = 0; h < NKH; ++h) {
                            const float * sp = (const float *) (buf + geo::KTILE) + b * KT + kg * KW + 32 * h + 4 * g4;
                            const wf4 d0 = *(const wf4 *) sp, d1 = *(const wf4 *) (sp + 16);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float e[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) e[j] = pw[nt][h][j] * (j < 4 ? d0[j & 3] : d1[j & 3]);
                                split8(e, ph[nt][h], pl[nt][h]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < NKH; ++h) {
                    const char * va_ = buf + va[d & 3] + 128 * (d >> 2) + 32 * h * VROW;
                    const wh4 v0 = __builtin_bit_cast(wh4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_w4) va_));
                    const wh4 v1 = __builtin_bit_cast(wh4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_w4) (va_ + 16 * VROW)));
                    const wh8 vf = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[nt][h], o[nt][d], 0, 0, 0);
                        o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[nt][h], o[nt][d], 0, 0, 0);
                    }
                }
            }
            if (more) store_tile(lds + (cur ^ 1) * geo::BUF);
            __syncthreads();                                    // the next tile is whole, this one is free
            if (next & 0x8000) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int u = 0; u < NSUB; ++u) mk[nt][u] = mkn[nt][u];
            }
            cur ^= 1;
            ent = next;
        }
    }

    if constexpr (QUANT) {
        const float f = qe == -1000 ? 1.f : __builtin_amdgcn_ldexpf(1.f, qe - 7);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < ND; ++d) o[nt][d] *= f;
    }
    // ---- a row's sum lies in four lanes
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        l_run[nt] += __shfl_xor(l_run[nt], 16, 64);
        l_run[nt] += __shfl_xor(l_run[nt], 32, 64);
    }
    // ---- key groups: the second's results go through LDS into the first's
    if constexpr (KG == 2) {
        float * xo = (float *) lds + rg * (NT * ND * 4 + 2 * NT) * 64 + lane;
        if (kg == 1) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                xo[(2 * nt) * 64] = m_run[nt];
                xo[(2 * nt + 1) * 64] = l_run[nt];
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) xo[(2 * NT + (nt * ND + d) * 4 + j) * 64] = o[nt][d][j];
            }
        }
        __syncthreads();
        if (kg == 1) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float m1 = xo[(2 * nt) * 64], l1 = xo[(2 * nt + 1) * 64], m = fmaxf(m_run[nt], m1);
            const float a0 = m_run[nt] == m ? 1.f : __builtin_amdgcn_exp2f((m_run[nt] - m) * FW_L2E);
            const float a1 = m1 == m ? 1.f : __builtin_amdgcn_exp2f((m1 - m) * FW_L2E);
            m_run[nt] = m;
            l_run[nt] = l_run[nt] * a0 + l1 * a1;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[nt][d][j] = o[nt][d][j] * a0 + xo[(2 * NT + (nt * ND + d) * 4 + j) * 64] * a1;
        }
    }
    // ---- store
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = rb * geo::ROWS + (rg * NT + nt) * 16 + n16;
        // An infinity or a NaN in V times a weight of 0 is a NaN: a row that shows one is computed
        // again, key by key, leaving masked keys out (what lies in their rows may not reach the result)
        float z = l_run[nt] * 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) z += o[nt][d][j] * 0.f;
        uint32_t bad = 0;
        {
            const uint64_t b = __ballot(z != 0.f);              // NaN compares unequal
            bad = (uint32_t) ((b | b >> 16 | b >> 32 | b >> 48) & 0xFFFF);
        }
        while (bad) {
            const int col = __builtin_ctz(bad);
            bad &= bad - 1;
            const int tk = __shfl(tok[nt], col, 64), hd = __shfl(head[nt], col, 64);
            const float sl = __shfl(slope[nt], col, 64);
            const float * qp = (const float *) (p.q + (size_t) tk * p.q1 + (size_t) hd * p.q2 + (size_t) seq * p.q3);
            const char * mr = p.mask ? p.mask + (size_t) tk * p.m1 + (size_t) (hd % p.mne2) * p.m2 + (size_t) (seq % p.mne3) * p.m3 : nullptr;
            float m = -INFINITY, l = 0.f, acc[DV / 64];
#pragma unroll
            for (int c = 0; c < DV / 64; ++c) acc[c] = 0.f;
            for (int j = 0; j < nl; ++j) {
                for (int k0 = (split + j * p.nsplit) * KT, k1 = min(k0 + KT, p.n_kv); k0 < k1; k0 += 64) {
                    const int key = k0 + lane;
                    float mv = -INFINITY, x = -INFINITY;
                    if (key < k1) mv = mr ? sl * h2f(((const uint16_t *) mr)[key]) : 0.f;
                    if (mv != -INFINITY) {
                        const char * kr = kb + (size_t) key * p.k1;
                        float dot = 0.f;
                        for (int c = 0; c < DK; ++c) dot += qp[c] * fw_get<KV>(kr, c);
                        x = dot * p.scale;
                        if (p.softcap != 0.0f) x = p.softcap * tanhf(x);
                        x += mv;
                    }
                    uint64_t seen = __ballot(mv != -INFINITY);
                    if (!seen) continue;
                    const float mn = fmaxf(m, wave_max<64>(x));
                    const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * FW_L2E);
                    const float e = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x - mn) * FW_L2E);
                    m = mn;
                    l = l * al + wave_sum<64>(e);
#pragma unroll
                    for (int c = 0; c < DV / 64; ++c) acc[c] *= al;
                    for (; seen; seen &= seen - 1) {
                        const int s_ = __builtin_ctzll(seen);
                        const float w = __shfl(e, s_, 64);
                        const char * vr = vb + (size_t) (k0 + s_) * (VSEP ? p.v1 : p.k1);
#pragma unroll
                        for (int c = 0; c < DV / 64; ++c) {
                            const int d = lane + 64 * c;
                            acc[c] += w * fw_get<KV>(vr, VSEP ? d : d + (QUANT ? 32 : 8) * p.vchunk);
                        }
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = __shfl(acc[d >> 2], 16 * (d & 3) + 4 * g4 + j, 64);
                    if (n16 == col) o[nt][d][j] = v;
                }
            if (n16 == col) { m_run[nt] = m; l_run[nt] = l; }
        }
        if (r >= nrow) continue;
        if (p.nsplit == 1) {
            float a = 1.f, l = l_run[nt];
            if (p.sinks) {
                const float sk = p.sinks[head[nt]], m = fmaxf(m_run[nt], sk);
                a = m_run[nt] == m ? 1.f : __builtin_amdgcn_exp2f((m_run[nt] - m) * FW_L2E);
                l = l * a + __builtin_amdgcn_exp2f((sk - m) * FW_L2E);
            }
            const float inv = l == 0.f ? 0.f : a / l;
            char * out = p.dst + (size_t) head[nt] * p.d1 + (size_t) tok[nt] * p.d2 + (size_t) seq * p.d3;
#pragma unroll
            for (int d = 0; d < ND; ++d) *(wf4 *) (out + 4 * (16 * d + 4 * g4)) = o[nt][d] * inv;
        } else {
            const size_t id = ((size_t) split * p.S + seq) * p.n_q * p.H + (size_t) tok[nt] * p.H + head[nt];
            if (g4 == 0) { p.mpart[id] = m_run[nt]; p.lpart[id] = l_run[nt]; }
            if (m_run[nt] != -INFINITY || l_run[nt] != 0.f) {   // nothing visible in this split: the join skips it
                float * out = p.opart + id * DV;
#pragma unroll
                for (int d = 0; d < ND; ++d) *(wf4 *) (out + 16 * d + 4 * g4) = o[nt][d];
            }
        }
    }
}

// Joins the splits of one row: a workgroup takes 64 output channels of a row, four waves every fourth
// split. The partials come from L2 / Infinity Cache; the launch is a few microseconds of latency.
template <int DV>
__global__ __launch_bounds__(256) void k_fattn_wide_join(FwArgs p) {
    __shared__ float wgt[FW_WIN];
    __shared__ float red[16], part[4][64];
    const int tid = threadIdx.x;
    const size_t rows = (size_t) p.S * p.n_q * p.H, id = blockIdx.x;
    const int h = (int) (id % p.H);
    float m = -INFINITY;
    for (int s = tid; s < p.nsplit; s += 256) m = fmaxf(m, p.mpart[s * rows + id]);
    m = block_max(m, red);
    if (p.sinks) m = fmaxf(m, p.sinks[h]);
    float l = 0.f;
    for (int s = tid; s < p.nsplit; s += 256) {
        const float ms = p.mpart[s * rows + id], ls = p.lpart[s * rows + id];
        const bool none = ms == -INFINITY && ls == 0.f;
        const float a = none ? 0.f : ms == m ? 1.f : __builtin_amdgcn_exp2f((ms - m) * FW_L2E);
        wgt[s] = none ? -1.f : a;
        l += ls * a;
    }
    __syncthreads();
    l = block_sum(l, red);
    if (p.sinks) l += __builtin_amdgcn_exp2f((p.sinks[h] - m) * FW_L2E);
    const int c = blockIdx.y * 64 + (tid & 63), w = tid >> 6;
    float o = 0.f;
#pragma unroll 4
    for (int s = w; s < p.nsplit; s += 4) {
        const float a = wgt[s];
        if (!(a < 0.f)) o += a * p.opart[(s * rows + id) * DV + c];
    }
    part[w][tid & 63] = o;
    __syncthreads();
    if (w) return;
    o = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    const size_t t = id / p.H % p.n_q, seq = id / ((size_t) p.H * p.n_q);
    ((float *) (p.dst + (size_t) h * p.d1 + t * p.d2 + seq * p.d3))[c] = l == 0.f ? 0.f : o / l;
}

// The mask's tile map: for 32 tokens x one key tile, whether some key is visible and whether some value
// is not 0. Every head reads the same mask, so it is read once here instead of once a head; tiles
// without a visible key are never loaded, tiles of zeros need no mask. One wave an entry.
template <int KT>
__global__ __launch_bounds__(256) void k_mask_map(const char * __restrict__ mask, size_t m1, size_t m3, int n_q, int n_kv, int n_tiles, int n_tb,
                                                  uint8_t * __restrict__ map) {
    const int lane = threadIdx.x & 63;
    const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), tb = blockIdx.y, seq = blockIdx.z;
    if (tile >= n_tiles) return;
    constexpr int PER = KT / 8, TOK = 64 / PER;                 // lanes of a token's row, tokens a pass
    uint32_t f = 0;
#pragma unroll
    for (int t0 = 0; t0 < FW_TB; t0 += TOK) {
        const int t = tb * FW_TB + t0 + lane / PER, key = tile * KT + 8 * (lane % PER);
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
struct FwPlan { bool wide, few; int rows, kt, nsplit, n_tiles, n_tb; size_t part, map; };
constexpr int FW_MAP_TOK = 17;   // from so many tokens on the tile map is built by a launch of its own

static FwPlan fw_plan(const ggml_tensor * dst) {
    const ggml_tensor * q = dst->src[0], * k = dst->src[1], * v = dst->src[2], * m = dst->src[3];
    FwPlan p{};
    p.wide = k->ne[0] == 576;
    const int64_t G = q->ne[2] / k->ne[2], nrow = q->ne[1] * G, units = k->ne[2] * q->ne[3];
    p.few = nrow <= 32;
    p.rows = p.wide ? (p.few ? 32 : 64) : (p.few ? 32 : 128);
    p.kt = p.wide || p.few ? 64 : 32;
    p.n_tiles = (int) mx_ceil_div(k->ne[1], p.kt);
    // splits: the number that ends soonest, counted in tile times on 256 CUs (one workgroup a CU: its
    // tiles fill the LDS; two for the expanded form's 128-row workgroups), against the join
    const int64_t blocks = units * mx_ceil_div(nrow, p.rows), slots = !p.wide && !p.few ? 512 : 256;
    int64_t best = INT64_MAX;
    p.nsplit = 1;
    for (int ns = 1; ns <= 256 && ns <= p.n_tiles; ++ns) {
        const int64_t cost = mx_ceil_div(blocks * ns, slots) * (mx_ceil_div(p.n_tiles, ns) * 2 + 1) + (ns > 1 ? 3 : 0);
        if (cost < best) { best = cost; p.nsplit = ns; }
    }
    const size_t rows = (size_t) q->ne[1] * q->ne[2] * q->ne[3];
    p.part = p.nsplit > 1 ? (size_t) p.nsplit * rows : 0;
    p.n_tb = (int) mx_ceil_div(q->ne[1], FW_TB);
    if (m && m->ne[2] == 1 && q->ne[1] >= FW_MAP_TOK && p.n_tiles > 2) p.map = (size_t) m->ne[3] * p.n_tb * p.n_tiles;
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
    for (int i = 1; i < 4; ++i) if (q->nb[i] % 4 || dst->nb[i] % 4 || k->nb[i] % 2 || v->nb[i] % 2) return false;
    if (dst->ne[0] != v->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3]) return false;
    if (m && (m->type != GGML_TYPE_F16 || m->nb[0] != 2 || m->ne[0] < k->ne[1] || m->ne[1] < q->ne[1] || m->ne[2] < 1 || m->ne[3] < 1 ||
              q->ne[2] % m->ne[2] || q->ne[3] % m->ne[3] || m->nb[1] % 2 || m->nb[2] % 2 || m->nb[3] % 2)) return false;
    if (sk && (sk->type != GGML_TYPE_F32 || sk->nb[0] != 4 || sk->ne[0] < q->ne[2])) return false;
    if (mx_op_param<float>(dst, 1) > 0.0f && !m) return false;
    // grid and index ranges of the kernels
    const int64_t G = q->ne[2] / k->ne[2];
    return k->ne[1] <= INT32_MAX / 2 - 64 && q->ne[1] * G < INT32_MAX / 2 && q->ne[1] * q->ne[2] * q->ne[3] < INT32_MAX / 2 &&
           mx_ceil_div(q->ne[1], FW_TB) < 65536 && q->ne[3] < 65536;
}

size_t fa_wide_scratch(const ggml_tensor * dst) {
    if (!fa_wide_supported(dst)) return 0;
    const FwPlan p = fw_plan(dst);
    return p.part * (dst->ne[0] + 2) * sizeof(float) + p.map + 5 * 256;
}

template <int DK, int DV, int KV, bool VSEP, int NT, int RG, int KT, int OCC>
static void fw_launch(OpCtx & c, const FwPlan & pl, const FwArgs & a) {
    using geo = FwGeo<DK, DV, KV, VSEP, NT, RG, KT>;
    static_assert(geo::LDS <= 160 * 1024, "LDS");
    const dim3 grid((unsigned) (mx_ceil_div((int64_t) a.n_q * a.G, geo::ROWS) * a.Hkv * a.S), (unsigned) pl.nsplit);
    auto kern = k_fattn_wide<DK, DV, KV, VSEP, NT, RG, KT, OCC>;
    MX_LDS_OPTIN(kern, geo::LDS);
    kern<<<grid, 256, geo::LDS, c.st>>>(a);
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
    if (pl.wide && v->data != k->data) a.vchunk = k->type == GGML_TYPE_F16 ? 8 : 2;    // 64 channels on
    a.scale = mx_op_param<float>(dst, 0);
    a.max_bias = mx_op_param<float>(dst, 1);
    a.softcap = mx_op_param<float>(dst, 2);
    if (a.softcap != 0.0f) a.scale /= a.softcap;
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
        if (pl.kt == 64) k_mask_map<64><<<grid, 256, 0, c.st>>>(a.mask, a.m1, a.m3, a.n_q, a.n_kv, pl.n_tiles, pl.n_tb, map);
        else             k_mask_map<32><<<grid, 256, 0, c.st>>>(a.mask, a.m1, a.m3, a.n_q, a.n_kv, pl.n_tiles, pl.n_tb, map);
        a.map = map;
        a.n_tb = pl.n_tb;
    }
    MX_KLOG("fattn_wide DK=%d type=%d rows=%d kt=%d nsplit=%d map=%d", (int) k->ne[0], (int) k->type, pl.rows, pl.kt, pl.nsplit, pl.map != 0);
    if (pl.wide) {
        switch (k->type) {
            case GGML_TYPE_F16:
                if (pl.few) fw_launch<576, 512, GGML_TYPE_F16, false, 1, 2, 64, 1>(c, pl, a);
                else        fw_launch<576, 512, GGML_TYPE_F16, false, 1, 4, 64, 1>(c, pl, a);
                break;
            case GGML_TYPE_Q8_0:
                if (pl.few) fw_launch<576, 512, GGML_TYPE_Q8_0, false, 1, 2, 64, 1>(c, pl, a);
                else        fw_launch<576, 512, GGML_TYPE_Q8_0, false, 1, 4, 64, 1>(c, pl, a);
                break;
            default:
                if (pl.few) fw_launch<576, 512, GGML_TYPE_Q4_0, false, 1, 2, 64, 1>(c, pl, a);
                else        fw_launch<576, 512, GGML_TYPE_Q4_0, false, 1, 4, 64, 1>(c, pl, a);
                break;
        }
    } else if (pl.few) fw_launch<192, 128, GGML_TYPE_F16, true, 1, 2, 64, 1>(c, pl, a);
    else               fw_launch<192, 128, GGML_TYPE_F16, true, 2, 4, 32, 2>(c, pl, a);
    if (pl.nsplit > 1) {
        const dim3 grid((unsigned) (a.S * a.n_q * a.H), (unsigned) (DV / 64));
        if (pl.wide) k_fattn_wide_join<512><<<grid, 256, 0, c.st>>>(a);
        else         k_fattn_wide_join<128><<<grid, 256, 0, c.st>>>(a);
    }
}

}  // namespace mx
