// ops_append.hip — rotary positions with several axes, their gradient, and cache rows appended with
// the rotation on the way.
//
// Semantics: ggml_rope_multi / ggml_rope_multi_back / ggml_rope_ext_back and ggml_concat
// (ggml/include/ggml.h); SET_ROWS as ops_misc.hip. All of it moves bytes: one launch reads its input
// once and writes its result once, and a token's cos / sin are computed once for all its heads.
#include "backend.h"
#include "quants.cuh"
#include "rope.cuh"

#include <type_traits>

namespace mx {

struct G4 { int64_t ne[4]; size_t nb[4]; };
static G4 g4(const ggml_tensor * t) {
    G4 g;
    for (int i = 0; i < 4; ++i) { g.ne[i] = t->ne[i]; g.nb[i] = t->nb[i]; }
    return g;
}

template <typename T> __device__ __forceinline__ float rd(T v);
template <> __device__ __forceinline__ float rd<float>(float v) { return v; }
template <> __device__ __forceinline__ float rd<uint16_t>(uint16_t v) { return h2f(v); }
template <typename T> __device__ __forceinline__ T wr(float v);
template <> __device__ __forceinline__ float wr<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t wr<uint16_t>(float v) { return f2h(v); }

// V elements at once (V * sizeof(T) = 16 bytes, aligned: checked by the host), or one
template <typename T, int V> struct Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> ldv(const T * p) {
    Pack<T, V> r;
    if constexpr (V == 1) r.v[0] = *p;
    else { const uint4 u = *(const uint4 *) p; __builtin_memcpy(r.v, &u, 16); }
    return r;
}
template <typename T, int V> __device__ __forceinline__ void stv(T * p, const Pack<T, V> & r) {
    if constexpr (V == 1) *p = r.v[0];
    else { uint4 u; __builtin_memcpy(&u, r.v, 16); *(uint4 *) p = u; }
}

// One workgroup = one token and `hper` of its heads. y = (a cos - b sin, a sin + b cos) for every
// channel pair (a, b) of a head: a at i and b at i + np, or (ADJ) neighbours. V pairs a step: 16-byte
// loads and stores when rows and pair counts allow them. In place is safe: a thread reads the pair it
// writes. 64-bit angle arithmetic costs ~100 instructions a pair and is spent once a token, not once a head.
// Memory bounds the long ones: 4096 tokens of 32 heads of 128 in f16, 67 MB in 13.5 us (5.0 TB/s; a large copy 5.2); 1521
// tokens of 16 heads of 80 in f32 5.4 us; one token 2.5 us, a launch.
template <typename T, bool ADJ, int V>
__global__ __launch_bounds__(256) void k_rope_axes(const char * __restrict__ x, const int32_t * __restrict__ pos, const float * __restrict__ ff,
                                                   char * __restrict__ y, G4 gx, G4 gy, RopeP p, int np, int hper) {
    __shared__ float2 tab[MX_ROPE_MAXP];
    const int64_t i2 = blockIdx.x % gx.ne[2], i3 = blockIdx.x / gx.ne[2];
    const char * px = x + i2 * gx.nb[2] + i3 * gx.nb[3];
    char * py = y + i2 * gy.nb[2] + i3 * gy.nb[3];
    const int h0 = blockIdx.y * hper, nh = min(hper, (int) gx.ne[1] - h0);
    const int steps = np / V, n = nh * steps;                   // a head's pairs, V at a time
    Pack<T, V> lo, hi;
    auto fetch = [&](int u) {                                   // on its way while the table, or the step before, is computed
        const T * rx = (const T *) (px + (h0 + u / steps) * gx.nb[1]);
        const int i = u % steps * V;
        lo = ldv<T, V>(rx + (ADJ ? 2 * i : i));
        hi = ldv<T, V>(rx + (ADJ ? 2 * i + V : i + np));
    };
    if (threadIdx.x < n) fetch(threadIdx.x);
    for (int i = threadIdx.x; i < np; i += blockDim.x) tab[i] = rope_pair(p, i, pos, i2, gx.ne[2], ff);
    __syncthreads();
    for (int u = threadIdx.x; u < n; u += blockDim.x) {
        const int h = h0 + u / steps, i = u % steps * V;
        T * ry = (T *) (py + h * gy.nb[1]);
        Pack<T, V> alo = lo, ahi = hi;
        if (u + (int) blockDim.x < n) fetch(u + blockDim.x);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            // (ADJ: pair j is elements 2j and 2j + 1 of the 2V that lo and hi hold; V = 1: lo and hi)
            T & a = !ADJ ? alo.v[j] : (2 * j < V ? alo.v[(2 * j) % V] : ahi.v[(2 * j) % V]);
            T & b = !ADJ || V == 1 ? ahi.v[j] : (2 * j < V ? alo.v[(2 * j + 1) % V] : ahi.v[(2 * j + 1) % V]);
            const float2 t = tab[i + j];
            const float x0 = rd<T>(a), x1 = rd<T>(b);
            if constexpr (std::is_same<T, float>::value) {      // (rows in f32 are the ones that an append turns as well)
                const float2 v = rope_turn<true>(x0, x1, t);
                a = v.x;
                b = v.y;
            } else {
                a = wr<T>(x0 * t.x - x1 * t.y);
                b = wr<T>(x0 * t.y + x1 * t.x);
            }
        }
        stv<T, V>(ry + (ADJ ? 2 * i : i), alo);
        stv<T, V>(ry + (ADJ ? 2 * i + V : i + np), ahi);
    }
    const int rest = (int) gx.ne[0] - 2 * np;                   // channels that do not turn
    for (int u = threadIdx.x; u < nh * rest; u += blockDim.x) {
        const int h = h0 + u / rest, i = 2 * np + u % rest;
        ((T *) (py + h * gy.nb[1]))[i] = ((const T *) (px + h * gx.nb[1]))[i];
    }
}

constexpr int64_t MX_MAX_TOKENS = UINT32_MAX / 256;            // a launch counts its threads in 32 bits: workgroups of 256, one a token

static bool rope_pos_ok(const ggml_tensor * dst) {
    const ggml_tensor * x = dst->src[0], * pos = dst->src[1], * ff = dst->src[2];
    const int mode = mx_op_param<int32_t>(dst, 2), n_dims = mx_op_param<int32_t>(dst, 1);
    const int np = rope_pairs(mode, n_dims);
    if (!pos || pos->type != GGML_TYPE_I32 || pos->nb[0] != 4 || pos->ne[0] < x->ne[2] * (rope_has_axes(mode) ? 4 : 1)) return false;
    if (ff && (ff->type != GGML_TYPE_F32 || ff->nb[0] != 4 || ff->ne[0] < np)) return false;
    return true;
}

// ROPE with several axes, and ROPE_BACK of every mode
bool rope_axes_supported(const ggml_tensor * dst) {
    const ggml_tensor * x = dst->src[0];
    const int mode = mx_op_param<int32_t>(dst, 2), n_dims = mx_op_param<int32_t>(dst, 1);
    if (!x || !dst->src[1]) return false;
    if ((x->type != GGML_TYPE_F32 && x->type != GGML_TYPE_F16) || dst->type != x->type || !mx_are_same_shape(x, dst)) return false;
    const size_t e = mx_type(x->type).size;
    if (x->nb[0] != e || dst->nb[0] != e) return false;
    for (int i = 1; i < 4; ++i) if (x->nb[i] % e || dst->nb[i] % e) return false;
    if (n_dims <= 0 || n_dims % 2 || n_dims > x->ne[0]) return false;
    switch (mode) {
        case GGML_ROPE_TYPE_NORMAL: case GGML_ROPE_TYPE_NEOX: break;
        case GGML_ROPE_TYPE_VISION: if (2 * n_dims != x->ne[0]) return false;   // (fallthrough) // ggml.c asserts it too
        case GGML_ROPE_TYPE_MROPE: case GGML_ROPE_TYPE_IMROPE: {
            int64_t n = 0;
            for (int i = 0; i < 4; ++i) { const int s = mx_op_param<int32_t>(dst, 11 + i); if (s < 0) return false; n += s; }
            if (n <= 0 || n > INT32_MAX) return false;
            break;
        }
        default: return false;
    }
    if (rope_pairs(mode, n_dims) > MX_ROPE_MAXP || x->ne[0] * x->ne[1] > INT32_MAX / 2 || x->ne[2] * x->ne[3] > MX_MAX_TOKENS) return false;
    return rope_pos_ok(dst);
}

void op_rope_axes(OpCtx & c, ggml_tensor * dst) {
    const ggml_tensor * x = dst->src[0], * ff = dst->src[2];
    const RopeP p = rope_params(dst);
    const int np = rope_pairs(p.mode, p.n_dims);
    const bool adj = p.mode == GGML_ROPE_TYPE_NORMAL;
    const int v = x->type == GGML_TYPE_F32 ? 4 : 8;
    size_t bits = (uintptr_t) x->data | (uintptr_t) dst->data;
    for (int i = 1; i < 4; ++i) bits |= x->nb[i] | dst->nb[i];
    const bool wide = bits % 16 == 0 && np % v == 0;            // 16-byte accesses stay aligned and inside the pairs
    // heads a workgroup: all of a token's, or, when the tokens alone leave CUs idle, so many that
    // 256 threads still have a step each
    const int steps = np / (wide ? v : 1);
    int hper = (int) x->ne[1];
    const int64_t toks = x->ne[2] * x->ne[3];
    if (toks < 1024) hper = std::min<int64_t>(hper, std::max<int64_t>(mx_ceil_div(256, std::max(1, steps)), mx_ceil_div(x->ne[1] * toks, 1024)));
    const dim3 grid((unsigned) toks, (unsigned) mx_ceil_div(x->ne[1], hper));
    MX_KLOG("rope_axes mode=%d back=%d type=%d wide=%d hper=%d", p.mode, dst->op == GGML_OP_ROPE_BACK, (int) x->type, (int) wide, hper);
#define RA(T, A, V) k_rope_axes<T, A, V><<<grid, 256, 0, c.st>>>((const char *) x->data, (const int32_t *) dst->src[1]->data, \
                        ff ? (const float *) ff->data : nullptr, (char *) dst->data, g4(x), g4(dst), p, np, hper)
    if (x->type == GGML_TYPE_F32) {
        if (wide) { if (adj) RA(float, true, 4); else RA(float, false, 4); }
        else      { if (adj) RA(float, true, 1); else RA(float, false, 1); }
    } else {
        if (wide) { if (adj) RA(uint16_t, true, 8); else RA(uint16_t, false, 8); }
        else      { if (adj) RA(uint16_t, true, 1); else RA(uint16_t, false, 1); }
    }
#undef RA
}

// ---------------------------------------------------------------------------
// CONCAT along one dimension: every element (or 16 bytes of a row) of the result is read from the
// operand that owns its index. Two halves of 8.4 MB along dimension 2 7.0 us (4.8 TB/s), 2011 rows of 512 and 64 in f32 3.9; element
// by element the index arithmetic bounds it: rows of 512 and 63 7.0 us
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_concat(const char * __restrict__ a, const char * __restrict__ b, char * __restrict__ y, G4 ga, G4 gb, G4 gy,
                                                int dim, int64_t n) {
    for (int64_t u = blockIdx.x * (int64_t) blockDim.x + threadIdx.x; u < n; u += (int64_t) gridDim.x * blockDim.x) {
        int64_t i[4], r = u;
        for (int d = 0; d < 3; ++d) { i[d] = r % gy.ne[d]; r /= gy.ne[d]; }
        i[3] = r;
        T * o = (T *) (y + i[0] * gy.nb[0] + i[1] * gy.nb[1] + i[2] * gy.nb[2] + i[3] * gy.nb[3]);
        const bool second = i[dim] >= ga.ne[dim];
        if (second) i[dim] -= ga.ne[dim];
        const G4 & g = second ? gb : ga;
        *o = *(const T *) ((second ? b : a) + i[0] * g.nb[0] + i[1] * g.nb[1] + i[2] * g.nb[2] + i[3] * g.nb[3]);
    }
}

bool concat_supported(const ggml_tensor * dst) {
    const ggml_tensor * a = dst->src[0], * b = dst->src[1];
    const int dim = mx_op_param<int32_t>(dst, 0);
    if (!a || !b || dim < 0 || dim > 3 || a->type != b->type || dst->type != a->type) return false;
    const mx_type_info ti = mx_type(dst->type);
    if (ti.blck != 1) return false;                             // (blocks would have to end at the seam)
    for (int i = 0; i < 4; ++i) {
        if (i == dim ? dst->ne[i] != a->ne[i] + b->ne[i] : (dst->ne[i] != a->ne[i] || a->ne[i] != b->ne[i])) return false;
        if ((a->nb[i] | b->nb[i] | dst->nb[i]) % ti.size) return false;
    }
    return true;
}

void op_concat(OpCtx & c, ggml_tensor * dst) {
    const ggml_tensor * a = dst->src[0], * b = dst->src[1];
    const int dim = mx_op_param<int32_t>(dst, 0);
    G4 ga = g4(a), gb = g4(b), gy = g4(dst);
    int e = mx_type(dst->type).size;
    // 16 bytes at a time where rows are dense, aligned, and whole on both sides of the seam
    size_t bits = (uintptr_t) a->data | (uintptr_t) b->data | (uintptr_t) dst->data | (size_t) a->ne[0] * e | (size_t) b->ne[0] * e;
    for (int i = 1; i < 4; ++i) bits |= a->nb[i] | b->nb[i] | dst->nb[i];
    if (bits % 16 == 0 && a->nb[0] == (size_t) e && b->nb[0] == (size_t) e && dst->nb[0] == (size_t) e) {
        for (G4 * g : {&ga, &gb, &gy}) { g->ne[0] = g->ne[0] * e / 16; g->nb[0] = 16; }
        e = 16;
    }
    const int64_t n = gy.ne[0] * gy.ne[1] * gy.ne[2] * gy.ne[3];
    const unsigned grid = (unsigned) std::min<int64_t>(mx_ceil_div(n, 256), 65536);
    MX_KLOG("concat dim=%d bytes=%d", dim, e);
#define CC(T) k_concat<T><<<grid, 256, 0, c.st>>>((const char *) a->data, (const char *) b->data, (char *) dst->data, ga, gb, gy, dim, n)
    switch (e) {
        case 1: CC(uint8_t); break;
        case 2: CC(uint16_t); break;
        case 4: CC(uint32_t); break;
        case 8: CC(uint2); break;
        default: CC(uint4); break;
    }
#undef CC
}

// ---------------------------------------------------------------------------
// Cache rows appended with the rotation on the way: one launch, one workgroup a token.
// A row is [normalised part | rotated heads] or the reverse (a latent cache), or rotated heads alone
// (keys); a second, unturned row (values) may go to a cache of its own. The row is assembled in LDS in
// 32 bits and rounded once into the cache's type. Against the separate launches (RMS_NORM + MUL, ROPE,
// CONCAT, SET_ROWS) it saves their round trips through memory, and at a token or two the launches. The chain fetch, sum,
// rotate, store of a row bounds it: 8 latent rows 4.7 us, 2011 6.3 us (7 MB), 512 rows of keys and of values 5.4 us; 1800 rows of
// 16 heads of keys and of values in f32, 59 MB, 14.6 us. With one axis a table's recurrence adds 0.6 us. Rows in 8 and 4 bits are
// rounded by a thread a block (18 of a latent row's 192): 0.7 and 0.5 us more than f16.
// ---------------------------------------------------------------------------
struct RowDst {
    char * base; size_t nb1; int64_t ne1; int type;             // a cache
    const char * idx; size_t idx_nb; int i64;                   // its row of each token
    int width;                                                  // elements of a row; 0: none
};
struct AppendP {
    const char * nx; size_t n_tok; const float * nw; char * nout; size_t nout_tok; int n_norm, norm_at; float eps;   // n_norm = 0: none
    const char * rx; size_t r_head, r_tok; const int32_t * pos; const float * ff; int heads, dim, rot_at, np, adj, by_token; int64_t ntok;
    RopeP rope;
    const char * vx; size_t v_tok; int v4;                      // v4: rows of whole 16 bytes, aligned
    RowDst k, v;
};
constexpr int APPEND_MAX_ROW = 8192;                            // elements of both rows in LDS: 32 KB

// the cell of token t, -1 when it is none of the cache's
__device__ __forceinline__ int64_t cell_of(const RowDst & d, int64_t t) {
    const int64_t c = d.i64 ? *(const int64_t *) (d.idx + t * d.idx_nb) : (int64_t) *(const int32_t *) (d.idx + t * d.idx_nb);
    return c < 0 || c >= d.ne1 ? -1 : c;
}
// `row` (LDS, width values) -> that cell; none takes nothing
__device__ __forceinline__ void store_row(const RowDst & d, const float * row, int64_t cell) {
    if (cell < 0) return;
    char * o = d.base + cell * d.nb1;
    const int nt = blockDim.x;
    switch (d.type) {                                           // uniform
        case GGML_TYPE_F32:
            if ((((uintptr_t) o) & 15) == 0 && d.width % 4 == 0) {
                for (int i = 4 * threadIdx.x; i < d.width; i += 4 * nt) *(float4 *) (o + 4 * i) = *(const float4 *) (row + i);
            } else {
                for (int i = threadIdx.x; i < d.width; i += nt) ((float *) o)[i] = row[i];
            }
            break;
        case GGML_TYPE_F16:
        case GGML_TYPE_BF16: {
            const bool h = d.type == GGML_TYPE_F16;
            if ((((uintptr_t) o) & 7) == 0 && d.width % 4 == 0) {
                for (int i = 4 * threadIdx.x; i < d.width; i += 4 * nt) {
                    const float4 f = *(const float4 *) (row + i);
                    uint2 w;
                    w.x = (h ? f2h(f.x) : f2bf(f.x)) | (uint32_t) (h ? f2h(f.y) : f2bf(f.y)) << 16;
                    w.y = (h ? f2h(f.z) : f2bf(f.z)) | (uint32_t) (h ? f2h(f.w) : f2bf(f.w)) << 16;
                    *(uint2 *) (o + 2 * i) = w;
                }
            } else {
                for (int i = threadIdx.x; i < d.width; i += nt) ((uint16_t *) o)[i] = h ? f2h(row[i]) : f2bf(row[i]);
            }
            break;
        }
        case GGML_TYPE_Q8_0:
            for (int b = threadIdx.x; b < d.width / 32; b += nt) quantize_block_q8_0(row + 32 * b, o + 34 * b);
            break;
        default:   // GGML_TYPE_Q4_0
            for (int b = threadIdx.x; b < d.width / 32; b += nt) quantize_block_q4_0(row + 32 * b, o + 18 * b);
            break;
    }
}

// LATENT: the normalised part, no second row
template <bool LATENT>
__global__ __launch_bounds__(256) void k_append_rows(AppendP p) {
    extern __shared__ __align__(16) float row[];                // [k.width, to a multiple of 4][v.width]
    const int v0 = (p.k.width + 3) & ~3;
    __shared__ float2 tab[MX_ROPE_MAXP];
    __shared__ float red[16];
    const int64_t t = blockIdx.x;
    const int nt = blockDim.x, tid = threadIdx.x;
    // everything the row needs is fetched first, up to AHEAD elements (pairs) a thread; a chain of table, sum and
    // rotation that fetched its own spent 9 us on 2011 latent rows, 7 of them waiting (and one kernel for both kinds of row 7.2: registers)
    constexpr int AHEAD = 4;
    float nv[LATENT ? AHEAD : 1], wv[LATENT ? AHEAD : 1], r0[AHEAD], r1[AHEAD];
    float4 vv[LATENT ? 1 : AHEAD];                              // (four elements each where p.v4 says so, else .x)
    const float * xn = (const float *) (p.nx + t * p.n_tok), * xv = (const float *) (p.vx + t * p.v_tok);
    const int pairs = p.heads * p.np;
    auto pair = [&](int u, float & x0, float & x1) {
        const int h = u / p.np, i = u % p.np;
        const float * x = (const float *) (p.rx + t * p.r_tok + h * p.r_head);
        x0 = x[p.adj ? 2 * i : i];
        x1 = x[p.adj ? 2 * i + 1 : i + p.np];
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
        const int i = tid + a * nt;
        if constexpr (LATENT) {
            nv[a] = i < p.n_norm ? xn[i] : 0.f;
            wv[a] = i < p.n_norm ? p.nw[i] : 0.f;
        } else {
            vv[a] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.v4) { if (4 * i < p.v.width) vv[a] = ((const float4 *) xv)[i]; }
            else if (i < p.v.width) vv[a].x = xv[i];
        }
        if (i < pairs) pair(i, r0[a], r1[a]);
    }
    const int64_t kcell = cell_of(p.k, t), vcell = !LATENT && p.v.width ? cell_of(p.v, t) : -1;
    for (int i = tid; i < p.np; i += nt) tab[i] = rope_pair(p.rope, i, p.pos, t, p.ntok, p.ff);
    if constexpr (LATENT) {
        float s = 0.f;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) s += nv[a] * nv[a];
        for (int i = tid + AHEAD * nt; i < p.n_norm; i += nt) s += xn[i] * xn[i];
        s = block_sum(s, red);
        const float inv = 1.0f / sqrtf(s / p.n_norm + p.eps);
        float * out = p.nout ? (float *) (p.nout + t * p.nout_tok) : nullptr;
        auto put = [&](int i, float x, float w) {
            const float v = x * inv * w;
            row[p.norm_at + i] = v;
            if (out) out[i] = v;
        };
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) if (tid + a * nt < p.n_norm) put(tid + a * nt, nv[a], wv[a]);
        for (int i = tid + AHEAD * nt; i < p.n_norm; i += nt) put(i, xn[i], p.nw[i]);
    } else if (p.v4) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) if (4 * (tid + a * nt) < p.v.width) *(float4 *) (row + v0 + 4 * (tid + a * nt)) = vv[a];
        for (int i = tid + AHEAD * nt; 4 * i < p.v.width; i += nt) *(float4 *) (row + v0 + 4 * i) = ((const float4 *) xv)[i];
    } else {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) if (tid + a * nt < p.v.width) row[v0 + tid + a * nt] = vv[a].x;
        for (int i = tid + AHEAD * nt; i < p.v.width; i += nt) row[v0 + i] = xv[i];
    }
    __syncthreads();                                            // the table
    auto turn = [&](int u, float x0, float x1) {
        const int h = u / p.np, i = u % p.np;
        const float2 v = p.by_token ? rope_turn<true>(x0, x1, tab[i]) : rope_turn<false>(x0, x1, tab[i]);
        float * r = row + p.rot_at + h * p.dim;
        r[p.adj ? 2 * i : i] = v.x;
        r[p.adj ? 2 * i + 1 : i + p.np] = v.y;
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) if (tid + a * nt < pairs) turn(tid + a * nt, r0[a], r1[a]);
    for (int u = tid + AHEAD * nt; u < pairs; u += nt) {
        float x0, x1;
        pair(u, x0, x1);
        turn(u, x0, x1);
    }
    const int rest = p.dim - 2 * p.np;
    for (int u = tid; u < p.heads * rest; u += nt) {
        const int h = u / rest, i = 2 * p.np + u % rest;
        row[p.rot_at + h * p.dim + i] = ((const float *) (p.rx + t * p.r_tok + h * p.r_head))[i];
    }
    __syncthreads();
    store_row(p.k, row, kcell);
    if constexpr (!LATENT) store_row(p.v, row + v0, vcell);
}

static const ggml_tensor * through_views(const ggml_tensor * t) {
    while (t && (t->op == GGML_OP_RESHAPE || t->op == GGML_OP_VIEW) && t->src[0]) t = t->src[0];
    return t;
}
static bool is_view(const ggml_tensor * t) {
    return t->op == GGML_OP_NONE || t->op == GGML_OP_RESHAPE || t->op == GGML_OP_VIEW || t->op == GGML_OP_PERMUTE || t->op == GGML_OP_TRANSPOSE;
}

// SET_ROWS of `n` dense rows into a cache that the kernel can write
static bool row_dst(const ggml_tensor * sr, int64_t n, RowDst * d) {
    const ggml_tensor * s = sr->src[0], * ix = sr->src[1];
    if (s->type != GGML_TYPE_F32 || s->nb[0] != 4 || s->ne[1] != n || s->ne[2] != 1 || s->ne[3] != 1 || sr->ne[2] != 1 || sr->ne[3] != 1) return false;
    if (ix->ne[0] != n || mx_nelements(ix) != n || (ix->type != GGML_TYPE_I64 && ix->type != GGML_TYPE_I32)) return false;
    const bool q = sr->type == GGML_TYPE_Q8_0 || sr->type == GGML_TYPE_Q4_0;
    if (!q && sr->type != GGML_TYPE_F32 && sr->type != GGML_TYPE_F16 && sr->type != GGML_TYPE_BF16) return false;
    if (q && s->ne[0] % 32) return false;
    if (sr->nb[0] != (size_t) mx_type(sr->type).size || s->ne[0] > APPEND_MAX_ROW) return false;
    *d = RowDst{(char *) sr->data, sr->nb[1], sr->ne[1], (int) sr->type, (const char *) ix->data, ix->nb[0], ix->type == GGML_TYPE_I64, (int) s->ne[0]};
    return true;
}

// Matched at node i: ROPE -> SET_ROWS [-> SET_ROWS of as many rows of something else], or
// RMS_NORM -> MUL, ROPE -> CONCAT -> SET_ROWS (the pair and ROPE in either order, CONCAT either way
// round); views between them. Nothing else may read the members' results, except the MUL's, which is
// written as well then. Positions enter by the same functions as the unfused ROPE, so fusing changes
// no angle. Tokens of one cell are written by workgroups that know nothing of each other, as by SET_ROWS: the cell
// holds values of any of them.
int fuse_append_rows(OpCtx & c, ggml_cgraph * g, int i, const UseCount & use_map) {
    static const bool off = getenv("GGML_MI355X_NO_APPEND_FUSION") != nullptr;   // A/B
    if (off) return 0;
    auto uses = [&](const ggml_tensor * t) { auto it = use_map.find(t); return it == use_map.end() ? 0 : it->second; };
    ggml_tensor * node[5] = {};
    int at[5], n = 0;
    for (int j = i; j < g->n_nodes && n < 5 && j < i + 16; ++j) {
        ggml_tensor * t = g->nodes[j];
        if (is_view(t)) continue;
        if (n == 0 || t->op == GGML_OP_RMS_NORM || t->op == GGML_OP_MUL || t->op == GGML_OP_ROPE || t->op == GGML_OP_CONCAT || t->op == GGML_OP_SET_ROWS) {
            node[n] = t;
            at[n++] = j;
        } else break;
    }
    if (n < 2) return 0;
    // the value of t, through views that keep its elements in place, has one reader
    auto single = [&](const ggml_tensor * t, const ggml_tensor * from) {
        for (const ggml_tensor * s = from; ; s = s->src[0]) {
            if (!s || uses(s) != 1 || (s->flags & GGML_TENSOR_FLAG_OUTPUT)) return false;
            if (s == t) break;
            if (s->data != t->data || !mx_is_contiguous(s) || mx_nelements(s) != mx_nelements(t)) return false;
        }
        return mx_is_contiguous(t);
    };
    ggml_tensor * norm = nullptr, * mul = nullptr, * rope = nullptr, * cat = nullptr, * sk = nullptr, * sv = nullptr;
    int last;
    if (node[0]->op == GGML_OP_ROPE && node[1]->op == GGML_OP_SET_ROWS) {
        rope = node[0]; sk = node[1]; last = at[1];
        if (through_views(sk->src[0]) != rope || !single(rope, sk->src[0])) return 0;
        if (n > 2 && node[2]->op == GGML_OP_SET_ROWS && through_views(node[2]->src[0]) != rope && node[2]->src[2] != sk) { sv = node[2]; }
    } else if (n == 5 && node[3]->op == GGML_OP_CONCAT && node[4]->op == GGML_OP_SET_ROWS) {
        const int r = node[0]->op == GGML_OP_ROPE ? 0 : 2;
        rope = node[r]; norm = node[r == 0 ? 1 : 0]; mul = node[r == 0 ? 2 : 1]; cat = node[3]; sk = node[4]; last = at[4];
        if (rope->op != GGML_OP_ROPE || norm->op != GGML_OP_RMS_NORM || mul->op != GGML_OP_MUL) return 0;
        if (through_views(sk->src[0]) != cat || !single(cat, sk->src[0])) return 0;
    } else return 0;

    // a member in place (a view of its input) leaves its result there, which the one launch would not
    for (const ggml_tensor * t : {rope, norm, mul, cat}) if (t && t->view_src) return 0;
    AppendP p{};
    const ggml_tensor * x = rope->src[0];
    const int64_t ntok = x->ne[2];
    if (rope->type != GGML_TYPE_F32 || x->type != GGML_TYPE_F32 || x->nb[0] != 4 || x->ne[3] != 1 || !rope_pos_ok(rope)) return 0;
    p.rope = rope_params(rope);
    if (p.rope.mode != GGML_ROPE_TYPE_NORMAL && p.rope.mode != GGML_ROPE_TYPE_NEOX && !rope_axes_supported(rope)) return 0;
    p.np = rope_pairs(p.rope.mode, p.rope.n_dims);
    if (p.np < 1 || p.np > MX_ROPE_MAXP || 2 * p.np > x->ne[0]) return 0;
    p.rx = (const char *) x->data; p.r_head = x->nb[1]; p.r_tok = x->nb[2];
    p.pos = (const int32_t *) rope->src[1]->data; p.ff = rope->src[2] ? (const float *) rope->src[2]->data : nullptr;
    p.dim = (int) x->ne[0]; p.adj = p.rope.mode == GGML_ROPE_TYPE_NORMAL; p.by_token = rope_has_axes(p.rope.mode) || rope_by_token(rope); p.ntok = ntok;
    if (x->ne[0] * x->ne[1] > APPEND_MAX_ROW) return 0;
    p.heads = (int) x->ne[1];
    const int turned = p.heads * p.dim;
    if (!row_dst(sk, ntok, &p.k)) return 0;
    const ggml_tensor * w = nullptr, * nx = nullptr;
    bool keep_mul = false;
    if (cat) {
        if (mx_op_param<int32_t>(cat, 0) != 0 || cat->type != GGML_TYPE_F32) return 0;
        const bool first = through_views(cat->src[0]) == mul;
        const ggml_tensor * ms = cat->src[first ? 0 : 1], * rs = cat->src[first ? 1 : 0];
        if (through_views(ms) != mul || through_views(rs) != rope || !single(rope, rs)) return 0;
        w = mul->src[0] == norm ? mul->src[1] : mul->src[1] == norm ? mul->src[0] : nullptr;
        nx = norm->src[0];
        if (!w || w == norm || uses(norm) != 1 || (norm->flags & GGML_TENSOR_FLAG_OUTPUT) || !mx_is_contiguous(mul) || ms->data != mul->data ||
            !mx_is_contiguous(ms)) return 0;
        keep_mul = !single(mul, ms);
        const int64_t d = nx->ne[0];
        if (nx->type != GGML_TYPE_F32 || norm->type != GGML_TYPE_F32 || mul->type != GGML_TYPE_F32 || nx->nb[0] != 4 || mx_nrows(nx) != ntok ||
            !mx_are_same_shape(mul, norm) || w->type != GGML_TYPE_F32 || w->ne[0] != d || mx_nelements(w) != d || w->nb[0] != 4 || d > APPEND_MAX_ROW) return 0;
        // tokens along dimension 1 or 2 of the norm's input, rows of one head
        if (!((nx->ne[1] == ntok && nx->ne[2] == 1) || (nx->ne[1] == 1 && nx->ne[2] == ntok)) || nx->ne[3] != 1) return 0;
        if (cat->ne[0] != d + turned || cat->ne[1] != 1 || ms->ne[0] != d || rs->ne[0] != p.dim || p.heads != 1 || p.k.width != d + turned) return 0;
        p.nx = (const char *) nx->data; p.n_tok = nx->ne[1] == ntok && ntok > 1 ? nx->nb[1] : nx->nb[2];
        p.nw = (const float *) w->data; p.n_norm = (int) d; p.eps = mx_op_param<float>(norm, 0);
        p.norm_at = first ? 0 : turned; p.rot_at = first ? (int) d : 0;
        if (keep_mul) { p.nout = (char *) mul->data; p.nout_tok = d * 4; }
    } else if (p.k.width != turned) return 0;
    if (sv && row_dst(sv, ntok, &p.v) && p.k.width + p.v.width <= APPEND_MAX_ROW &&
        fused_io_ok({sk, sv}, {x, rope->src[1], rope->src[2], sk->src[1], sv->src[0], sv->src[1]})) {
        const ggml_tensor * vx = sv->src[0];
        p.vx = (const char *) vx->data; p.v_tok = vx->nb[1];
        p.v4 = p.v.width % 4 == 0 && ((uintptr_t) vx->data | vx->nb[1]) % 16 == 0;
        last = at[2];
    } else { sv = nullptr; p.v.width = 0; }
    if (!sv && !fused_io_ok({sk, keep_mul ? mul : nullptr}, {x, rope->src[1], rope->src[2], sk->src[1], nx, w})) return 0;
    if (p.k.width > APPEND_MAX_ROW || ntok > MX_MAX_TOKENS) return 0;
    kv_new_row_flush(c);                                        // (its cache may be the one written here)
    for (int j = i; j <= last; ++j) {
        deferred_guard_node_ext(c, g->nodes[j]);
        act_cache_invalidate(c.s, g->nodes[j]);
    }
    const size_t lds = (size_t) (p.k.width + 3 + p.v.width) * sizeof(float);
    const int threads = p.k.width + p.v.width >= 1024 ? 256 : p.k.width + p.v.width >= 512 ? 192 : 64;
    MX_KLOG("append_rows norm=%d heads=%d dim=%d mode=%d type=%d v=%d keep=%d", p.n_norm, p.heads, p.dim, p.rope.mode, p.k.type, p.v.width, (int) keep_mul);
    if (cat) k_append_rows<true><<<(unsigned) ntok, threads, lds, c.st>>>(p);
    else     k_append_rows<false><<<(unsigned) ntok, threads, lds, c.st>>>(p);
    return last - i + 1;
}

}  // namespace mx
