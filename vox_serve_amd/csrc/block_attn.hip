// Long contexts: rows rotated into a paged cache, the bounds of its blocks, the blocks that a row reads, and attention over them
// (voxhip.h: vox_rope_append, vox_block_bounds, vox_block_select, vox_block_attention).
#include "vox_internal.h"

typedef _Float16 half_t;

// one element of either 16-bit type, as its bits <-> fp32
template <int F16>
__device__ __forceinline__ float elem_f(bf16_t b) {
    if constexpr (F16) { union { uint16_t u; half_t h; } c; c.u = b; return (float)c.h; }
    else return bf2f(b);
}
// (fp16: f is rounded to 32 bits first, as everywhere - left to itself the compiler joins a multiply-add and the conversion to one instruction that rounds
// once, and a value in 20000 comes out one fp16 step from the other order's)
template <int F16>
__device__ __forceinline__ bf16_t f_elem(float f) {
    if constexpr (F16) { asm("" : "+v"(f)); union { uint16_t u; half_t h; } c; c.h = (half_t)f; return c.u; }
    else return f2bf(f);
}

// The step of values whose largest finite magnitude is amax: the smallest power of two of which 127 reach it, at least 2^-100.
__device__ __forceinline__ float step_of(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 126;        // amax = f 2^e, f in [0.5, 1); (subnormal amax: e = -126, the floor below)
    const int m = e - 7 < -100 ? -100 : e - 7;
    float s = __uint_as_float((u32)(m + 127) << 23);
    if (amax > 127.0f * s) s *= 2.0f;                               // (not at the floor: there 127 s is far above)
    return s;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __uint_as_float(0x7f800000u) ? a : 0.0f;             // NaN and infinities: 0
}

static int check_cache(const char* who, const vox_block_cache& c, bool bounds) {
    if (!c.kv) return vox_fail(VOX_ERR_INVALID, "%s: no cache", who);
    if (c.n_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return vox_fail(VOX_ERR_INVALID, "%s: %d pages of %d tokens, %d kv heads", who, c.n_pages, c.page_size, c.kv_heads);
    if (c.dtype != VOX_DTYPE_BF16 && c.dtype != VOX_DTYPE_F16) return vox_fail(VOX_ERR_INVALID, "%s: dtype %d", who, c.dtype);
    if ((size_t)c.kv & 15) return vox_fail(VOX_ERR_INVALID, "%s: the cache does not lie on 16 bytes", who);
    if (!bounds) return VOX_OK;
    if (c.block != 16 && c.block != 32 && c.block != 64 && c.block != 128) return vox_fail(VOX_ERR_INVALID, "%s: blocks of %d tokens (16, 32, 64 or 128)", who, c.block);
    if (c.page_size % c.block) return vox_fail(VOX_ERR_INVALID, "%s: pages of %d tokens are not whole blocks of %d", who, c.page_size, c.block);
    if (c.head_dim != 64 && c.head_dim != 128) return vox_fail(VOX_ERR_INVALID, "%s: head_dim %d (64 or 128)", who, c.head_dim);
    return VOX_OK;
}
static int check_bounds(const char* who, const vox_block_cache& c) {
    if (!c.bounds || !c.steps) return vox_fail(VOX_ERR_INVALID, "%s: no bounds or no steps", who);
    if ((size_t)c.bounds & 15 || (size_t)c.steps & 3) return vox_fail(VOX_ERR_INVALID, "%s: bounds on 16 bytes, steps on 4", who);
    return VOX_OK;
}
static int check_rows(const char* who, const vox_block_cache& c, const vox_block_rows& r) {
    if (r.n_rows < 0 || r.n_req < 0 || r.n_own < 0 || r.max_kvlen < 0) return vox_fail(VOX_ERR_INVALID, "%s: %d rows of %d requests, max_kvlen %d", who, r.n_rows, r.n_req, r.max_kvlen);
    if (r.heads <= 0 || r.heads % c.kv_heads || r.heads / c.kv_heads > 64) return vox_fail(VOX_ERR_INVALID, "%s: %d heads on %d kv heads (1 to 64 on each)", who, r.heads, c.kv_heads);
    if (r.n_rows && (!r.q_req || !r.q_kvlen || !r.kv_indptr || !r.kv_indices)) return vox_fail(VOX_ERR_INVALID, "%s: a plan array is NULL", who);
    return VOX_OK;
}
template <class A>
static int launch(const void* kern, dim3 grid, int threads, size_t lds, hipStream_t st, A& a) {
    void* args[] = {&a};
    if (lds > 64 * 1024) VOX_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    VOX_HIP(hipLaunchKernel(kern, grid, dim3(threads), args, lds, st));
    return VOX_OK;
}

// ================================================================================================
// rotate and append
// ================================================================================================
struct RopeAppendArgs {
    const bf16_t *q, *k, *v;
    bf16_t *q_out, *kv;
    const int *pos, *page, *slot;
    const float* cs;
    long q_stride, k_stride, v_stride;
    int n_rows, Hq, Hkv, D, rot, interleave, max_pos, page_size, n_pages;
};
// one thread a pair of channels that turn together (or two that do not)
template <int F16>
__global__ __launch_bounds__(256) void k_rope_append(RopeAppendArgs a) {
    const int n = blockIdx.y, half_d = a.D >> 1, half = a.rot >> 1, heads = a.Hq + 2 * a.Hkv;
    const int pg = a.page[n], slot = a.slot[n];
    if (pg < 0 || pg >= a.n_pages || slot < 0 || slot >= a.page_size) return;
    int p = a.rot ? a.pos[n] : 0;
    p = p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
    for (int i = blockIdx.x * 256 + threadIdx.x; i < heads * half_d; i += gridDim.x * 256) {
        const int head = i / half_d, c = i % half_d;
        const int kind = head < a.Hq ? 0 : head < a.Hq + a.Hkv ? 1 : 2, h = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - a.Hkv;
        const bf16_t* const src = (kind == 0 ? a.q + n * a.q_stride : kind == 1 ? a.k + n * a.k_stride : a.v + n * a.v_stride) + (size_t)h * a.D;
        bf16_t* const dst = kind == 0 ? a.q_out + ((size_t)n * a.Hq + h) * a.D
                                      : a.kv + (((size_t)pg * 2 + (kind == 2)) * a.page_size + slot) * a.Hkv * a.D + (size_t)h * a.D;
        const bool turns = kind < 2 && c < half;
        const int i0 = turns && !a.interleave ? c : turns || kind == 2 ? 2 * c : a.rot + 2 * (c - half), i1 = turns && !a.interleave ? c + half : i0 + 1;
        bf16_t x = src[i0], y = src[i1];
        if (turns) {
            const float fx = elem_f<F16>(x), fy = elem_f<F16>(y), cc = a.cs[((size_t)p * half + c) * 2], ss = a.cs[((size_t)p * half + c) * 2 + 1];
            x = f_elem<F16>(__fmaf_rn(-fy, ss, fx * cc));
            y = f_elem<F16>(__fmaf_rn(fx, ss, fy * cc));
        }
        dst[i0] = x;
        dst[i1] = y;
    }
}

struct BoundsArgs {
    const bf16_t* kv;
    int8_t* bounds;
    float* steps;
    const int *page, *slot;
    int n_rows, n_pages, page_size, block, Hkv;
};
// one wave a row that completes its block, and kv head: D / 8 lanes hold a key, 512 / D keys at once
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_bounds(BoundsArgs a) {
    constexpr int LPT = D / 8, TPI = 64 / LPT;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, lane = threadIdx.x & 63, l = lane % LPT;
    if (n >= a.n_rows) return;
    const int pg = a.page[n], slot = a.slot[n];
    if (pg < 0 || pg >= a.n_pages || slot < 0 || slot >= a.page_size || (slot + 1) % a.block) return;
    const bf16_t* const k = a.kv + ((size_t)pg * 2 * a.page_size + slot + 1 - a.block) * a.Hkv * D + (size_t)h * D;
    const float inf = __uint_as_float(0x7f800000u);
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { hi[i] = -inf; lo[i] = inf; }
    for (int t = lane / LPT; t < a.block; t += TPI) {
        const uint4 v = reinterpret_cast<const uint4*>(k + (size_t)t * a.Hkv * D)[l];
        const u32 w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = elem_f<F16>((bf16_t)(w[i / 2] >> (16 * (i % 2))));
            hi[i] = x > hi[i] ? x : hi[i];                          // (false for NaN)
            lo[i] = x < lo[i] ? x : lo[i];
        }
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        for (int o = LPT; o < 64; o <<= 1) {
            hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], o, 64));
            lo[i] = fminf(lo[i], __shfl_xor(lo[i], o, 64));
        }
    }
    // the largest finite magnitude: of all keys, not of the bounds, where infinities stand in front of it
    for (int t = lane / LPT; t < a.block; t += TPI) {
        const uint4 v = reinterpret_cast<const uint4*>(k + (size_t)t * a.Hkv * D)[l];
        const u32 w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(elem_f<F16>((bf16_t)(w[i / 2] >> (16 * (i % 2))))));
    }
    for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    const float step = step_of(amax), inv = 1.0f / step;
    if (lane < LPT) {
        const int per = a.page_size / a.block;
        const size_t at = ((size_t)pg * a.Hkv + h) * per + slot / a.block;
        u32 wh[2] = {0, 0}, wl[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool any = hi[i] >= lo[i];                        // (a channel of NaN: no)
            const int H = any ? (int)fminf(fmaxf(ceilf(hi[i] * inv), -127.0f), 127.0f) : 0, L = any ? (int)fminf(fmaxf(floorf(lo[i] * inv), -127.0f), 127.0f) : 0;
            wh[i / 4] |= (u32)(H & 255) << (8 * (i % 4));
            wl[i / 4] |= (u32)(L & 255) << (8 * (i % 4));
        }
        *reinterpret_cast<uint2*>(a.bounds + at * 2 * D + 8 * l) = make_uint2(wh[0], wh[1]);
        *reinterpret_cast<uint2*>(a.bounds + at * 2 * D + D + 8 * l) = make_uint2(wl[0], wl[1]);
        if (lane == 0) a.steps[at] = step;
    }
}

// ================================================================================================
// choose
// ================================================================================================
struct SelectArgs {
    const bf16_t* q;
    const int8_t* bounds;
    const float* steps;
    const int *q_req, *q_kvlen, *indptr, *indices;
    int* blocks;
    long q_stride;
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top, first, last;
};
// order of the scores as unsigned numbers; 0 is below all of them
__device__ __forceinline__ u32 score_key(float s) {
    const u32 b = __float_as_uint(s);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ int q_steps(float x, float inv) {
    const float t = fminf(fmaxf(__builtin_rintf(x * inv), -127.0f), 127.0f);
    return x == x ? (int)t : 0;
}
// one block of threads a row and kv head
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_select(SelectArgs a) {
    extern __shared__ u32 key[];                                    // of every candidate
    __shared__ int sum_pos[D], sum_neg[D], red[4];
    __shared__ float redf[4];
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, G = a.Hq / a.Hkv;
    int n = a.q_kvlen[i];
    const int r = a.q_req[i];
    if (n <= 0 || r < 0 || r >= a.n_req) return;
    n = min(n, a.max_kvlen);
    int* const out = a.blocks + ((size_t)i * a.Hkv + h) * a.top;
    const int have = (n + a.block - 1) / a.block;
    if (have <= a.top) {
        for (int j = tid; j < a.top; j += 256) out[j] = j < have ? j : -1;
        return;
    }
    const bf16_t* const q = a.q + (size_t)i * a.q_stride + (size_t)h * G * D;
    float amax = 0.0f;
    for (int e = tid; e < G * D; e += 256) amax = fmaxf(amax, finite_abs(elem_f<F16>(q[e])));
    for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    if (lane == 0) redf[wave] = amax;
    __syncthreads();
    const float inv = 1.0f / step_of(fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3])));
    for (int d = tid; d < D; d += 256) {
        int p = 0, m = 0;
        for (int g = 0; g < G; ++g) {
            const int s = q_steps(elem_f<F16>(q[g * D + d]), inv);
            p += max(s, 0); m += min(s, 0);
        }
        sum_pos[d] = p; sum_neg[d] = m;
    }
    __syncthreads();
    const int per = a.page_size / a.block, lo = a.first, cand = have - a.last - a.first, need = a.top - a.first - a.last;
    const int p0 = a.indptr[r], np = a.indptr[r + 1] - p0;
    for (int c = tid; c < cand; c += 256) {
        const int j = lo + c, pj = j / per;
        const int pg = pj < np ? a.indices[p0 + pj] : -1;
        u32 k = 0;                                                  // a block without a page: behind all others
        if (pg >= 0 && pg < a.n_pages) {
            const size_t at = ((size_t)pg * a.Hkv + h) * per + j % per;
            const int8_t* const b = a.bounds + at * 2 * D;
            int s = 0;
            for (int d = 0; d < D; ++d) s += sum_pos[d] * b[d] + sum_neg[d] * b[D + d];
            k = score_key((float)s * a.steps[at]);
        }
        key[c] = k;
    }
    __syncthreads();
    // the need-th largest key, bit by bit: the largest t that at least `need` keys reach
    u32 t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const u32 at = t | (1u << bit);
        int count = 0;
        for (int c = tid; c < cand; c += 256) count += key[c] >= at;
        for (int o = 1; o < 64; o <<= 1) count += __shfl_xor(count, o, 64);
        if (lane == 0) red[wave] = count;
        __syncthreads();
        if (red[0] + red[1] + red[2] + red[3] >= need) t = at;
        __syncthreads();
    }
    if (wave) return;
    // in order of their index: larger keys, and as many equal ones as are left
    int above = 0;
    for (int c = lane; c < cand; c += 64) above += key[c] > t;
    for (int o = 1; o < 64; o <<= 1) above += __shfl_xor(above, o, 64);
    int ties = need - above, at = a.first;
    for (int j = lane; j < a.first; j += 64) out[j] = j;
    const unsigned long long below = lane ? ~0ull >> (64 - lane) : 0ull;
    for (int c0 = 0; c0 < cand; c0 += 64) {
        const int c = c0 + lane;
        const u32 k = c < cand ? key[c] : 0;
        const bool eq = c < cand && k == t, gt = c < cand && k > t;
        const unsigned long long be = __ballot(eq);
        const bool take = gt || (eq && __popcll(be & below) < ties);
        const unsigned long long bt = __ballot(take);
        if (take) out[at + __popcll(bt & below)] = lo + c;
        at += __popcll(bt);
        ties -= min(ties, (int)__popcll(be));
    }
    for (int j = lane; j < a.last; j += 64) out[at + j] = have - a.last + j;
}

// ================================================================================================
// attend
// ================================================================================================
struct BlockAttnArgs {
    const bf16_t *q, *kv;
    const int *q_req, *q_kvlen, *indptr, *indices, *blocks;
    bf16_t* out;
    long q_stride;
    float scale;
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top;
};
// one wave a row and query head: 64 tokens at a time, a token a lane for the scores, D / 64 channels a lane for the values
template <int F16, int D>
__global__ __launch_bounds__(64) void k_block_attention(BlockAttnArgs a) {
    __shared__ float q[D];
    const int i = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x, h = hq / (a.Hq / a.Hkv);
    int n = a.q_kvlen[i];
    const int r = a.q_req[i];
    if (n <= 0 || r < 0 || r >= a.n_req) return;
    n = min(n, a.max_kvlen);
    const float inf = __uint_as_float(0x7f800000u);
    for (int d = lane; d < D; d += 64) q[d] = elem_f<F16>(a.q[(size_t)i * a.q_stride + (size_t)hq * D + d]);
    __syncthreads();
    const int* const list = a.blocks + ((size_t)i * a.Hkv + h) * a.top;
    const int per = a.page_size / a.block, p0 = a.indptr[r], np = a.indptr[r + 1] - p0, have = (n + a.block - 1) / a.block;
    float m = -inf, l = 0.0f, o[D / 64] = {};
    int seen = -1;
    for (int e = 0; e < a.top; ++e) {
        const int j = list[e];
        if (j <= seen) continue;
        seen = j;
        if (j >= have || j / per >= np) continue;
        const int pg = a.indices[p0 + j / per];
        if (pg < 0 || pg >= a.n_pages) continue;
        const size_t base = ((size_t)pg * 2 * a.page_size + (size_t)(j % per) * a.block) * a.Hkv * D + (size_t)h * D;
        const int len = min(a.block, n - j * a.block);
        for (int t0 = 0; t0 < len; t0 += 64) {
            const int t = t0 + lane;
            float s = -inf;
            if (t < len) {
                const bf16_t* const k = a.kv + base + (size_t)t * a.Hkv * D;
                float z = 0.0f;
                for (int d = 0; d < D; ++d) z = __fmaf_rn(q[d], elem_f<F16>(k[d]), z);
                s = z * a.scale;
            }
            float top = s;
            for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
            const float now = fmaxf(m, top);
            const float keep = m == -inf ? 0.0f : expf(m - now), p = t < len ? expf(s - now) : 0.0f;
            float all = p;
            for (int x = 1; x < 64; x <<= 1) all += __shfl_xor(all, x, 64);
            l = l * keep + all;
            m = now;
            for (int x = 0; x < D / 64; ++x) o[x] *= keep;
            const bf16_t* const v = a.kv + base + (size_t)a.page_size * a.Hkv * D;
            for (int t1 = 0; t1 < min(64, len - t0); ++t1) {
                const float w = __shfl(p, t1, 64);
                for (int x = 0; x < D / 64; ++x) o[x] = __fmaf_rn(w, elem_f<F16>(v[(size_t)(t0 + t1) * a.Hkv * D + lane + 64 * x]), o[x]);
            }
        }
    }
    for (int x = 0; x < D / 64; ++x) a.out[((size_t)i * a.Hq + hq) * D + lane + 64 * x] = f_elem<F16>(seen >= 0 && l != 0.0f ? o[x] / l : 0.0f);
}

// ================================================================================================
// entry points
// ================================================================================================
#define BY_TYPE_AND_DIM(KERN, c) \
    ((c).dtype == VOX_DTYPE_F16 ? ((c).head_dim == 128 ? (const void*)KERN<1, 128> : (const void*)KERN<1, 64>) \
                                : ((c).head_dim == 128 ? (const void*)KERN<0, 128> : (const void*)KERN<0, 64>))

static int launch_bounds(hipStream_t st, const vox_block_cache& c, const int* page, const int* slot, int n_rows) {
    if (n_rows == 0) return VOX_OK;
    BoundsArgs b{(const bf16_t*)c.kv, c.bounds, c.steps, page, slot, n_rows, c.n_pages, c.page_size, c.block, c.kv_heads};
    return launch(BY_TYPE_AND_DIM(k_block_bounds, c), dim3((n_rows + 3) / 4, c.kv_heads), 256, 0, st, b);
}

extern "C" {

int vox_block_bounds(vox_ctx* ctx, void* stream, const vox_block_cache* c, const int32_t* page, const int32_t* slot, int n_rows) {
    (void)ctx;
    if (!c) return vox_fail(VOX_ERR_INVALID, "block_bounds: no cache");
    VOX_TRY(check_cache("block_bounds", *c, true));
    VOX_TRY(check_bounds("block_bounds", *c));
    if (n_rows < 0 || (n_rows && (!page || !slot))) return vox_fail(VOX_ERR_INVALID, "block_bounds: %d rows, or no page or slot", n_rows);
    return launch_bounds((hipStream_t)stream, *c, page, slot, n_rows);
}

int vox_rope_append(vox_ctx* ctx, void* stream, const vox_rope_append_args* a) {
    (void)ctx;
    if (!a) return vox_fail(VOX_ERR_INVALID, "rope_append: no arguments");
    const vox_block_cache& c = a->cache;
    VOX_TRY(check_cache("rope_append", c, c.bounds != nullptr));
    if (c.bounds) VOX_TRY(check_bounds("rope_append", c));
    const int D = c.head_dim;
    if (D < 2 || D % 2 || D > 512) return vox_fail(VOX_ERR_INVALID, "rope_append: head_dim %d (even, 2 to 512)", D);
    if (a->n_rows < 0 || a->n_own < 0 || a->heads <= 0) return vox_fail(VOX_ERR_INVALID, "rope_append: %d rows of %d requests, %d heads", a->n_rows, a->n_own, a->heads);
    if (a->rot < 0 || a->rot % 2 || a->rot > D) return vox_fail(VOX_ERR_INVALID, "rope_append: %d of %d channels turn", a->rot, D);
    if (a->n_rows == 0) return VOX_OK;
    if (!a->q || !a->k || !a->v || !a->q_out || !a->page || !a->slot) return vox_fail(VOX_ERR_INVALID, "rope_append: an operand is NULL");
    if (a->rot && (!a->pos || !a->table || a->table_max_pos <= 0)) return vox_fail(VOX_ERR_INVALID, "rope_append: no positions or no table");
    if (((size_t)a->q | (size_t)a->k | (size_t)a->v | (size_t)a->q_out) & 1 || (a->rot && (size_t)a->table & 3)) return vox_fail(VOX_ERR_INVALID, "rope_append: an operand does not lie on its type");
    if (a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0) return vox_fail(VOX_ERR_INVALID, "rope_append: a stride is negative");
    RopeAppendArgs r{(const bf16_t*)a->q, (const bf16_t*)a->k, (const bf16_t*)a->v, (bf16_t*)a->q_out, (bf16_t*)c.kv, a->pos, a->page, a->slot, a->table,
                     (long)a->q_stride, (long)a->k_stride, (long)a->v_stride, a->n_rows, a->heads, c.kv_heads, D, a->rot, a->interleave, a->table_max_pos, c.page_size, c.n_pages};
    const int pairs = (a->heads + 2 * c.kv_heads) * (D / 2);
    for (int at = 0; at < a->n_rows; at += 65535) {                 // (grid.y)
        RopeAppendArgs p = r;
        p.n_rows = a->n_rows - at < 65535 ? a->n_rows - at : 65535;
        p.q += (size_t)at * r.q_stride; p.k += (size_t)at * r.k_stride; p.v += (size_t)at * r.v_stride; p.q_out += (size_t)at * r.Hq * D;
        p.pos = p.pos ? p.pos + at : nullptr; p.page += at; p.slot += at;
        VOX_TRY(launch(c.dtype == VOX_DTYPE_F16 ? (const void*)k_rope_append<1> : (const void*)k_rope_append<0>, dim3((pairs + 255) / 256, p.n_rows), 256, 0, (hipStream_t)stream, p));
    }
    return c.bounds ? launch_bounds((hipStream_t)stream, c, a->page, a->slot, a->n_rows) : VOX_OK;
}

static int check_select(const vox_block_select_args* a) {
    if (!a) return vox_fail(VOX_ERR_INVALID, "block_select: no arguments");
    const vox_block_cache& c = a->cache;
    if (c.n_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return vox_fail(VOX_ERR_INVALID, "block_select: %d pages of %d tokens, %d kv heads", c.n_pages, c.page_size, c.kv_heads);
    vox_block_cache k = c;
    k.kv = c.bounds;                                                // the keys are not read: the bounds stand for them
    VOX_TRY(check_cache("block_select", k, true));
    VOX_TRY(check_bounds("block_select", c));
    VOX_TRY(check_rows("block_select", c, a->rows));
    if (a->first < 0 || a->last < 1 || a->top > VOX_BLOCK_TOP_MAX || (int64_t)a->first + a->last > a->top) return vox_fail(VOX_ERR_INVALID, "block_select: top %d (up to %d), first %d, last %d (1 at least)", a->top, VOX_BLOCK_TOP_MAX, a->first, a->last);
    if ((a->rows.max_kvlen + (int64_t)c.block - 1) / c.block > VOX_BLOCK_SELECT_MAX) return vox_fail(VOX_ERR_INVALID, "block_select: %d tokens are more than %d blocks of %d", a->rows.max_kvlen, VOX_BLOCK_SELECT_MAX, c.block);
    if (a->q_stride < 0) return vox_fail(VOX_ERR_INVALID, "block_select: a stride is negative");
    return VOX_OK;
}
int64_t vox_block_select_workspace_bytes(const vox_block_select_args* a) {
    if (check_select(a) != VOX_OK) return -1;
    return 0;
}
int vox_block_select(vox_ctx* ctx, void* stream, const vox_block_select_args* a) {
    (void)ctx;
    VOX_TRY(check_select(a));
    const vox_block_cache& c = a->cache;
    const vox_block_rows& r = a->rows;
    if (r.n_rows == 0) return VOX_OK;
    if (!a->q || !a->blocks || (size_t)a->q & 1) return vox_fail(VOX_ERR_INVALID, "block_select: an operand is NULL, or does not lie on its type");
    SelectArgs s{(const bf16_t*)a->q, c.bounds, c.steps, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (long)a->q_stride,
                 r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages, c.page_size, c.block, a->top, a->first, a->last};
    const int most = (r.max_kvlen + c.block - 1) / c.block;
    return launch(BY_TYPE_AND_DIM(k_block_select, c), dim3(r.n_rows, c.kv_heads), 256, (size_t)most * 4, (hipStream_t)stream, s);
}

static int check_attention(const vox_block_attention_args* a) {
    if (!a) return vox_fail(VOX_ERR_INVALID, "block_attention: no arguments");
    VOX_TRY(check_cache("block_attention", a->cache, true));
    VOX_TRY(check_rows("block_attention", a->cache, a->rows));
    if (a->top < 0 || a->top > VOX_BLOCK_TOP_MAX) return vox_fail(VOX_ERR_INVALID, "block_attention: lists of %d blocks (up to %d)", a->top, VOX_BLOCK_TOP_MAX);
    if (a->q_stride < 0) return vox_fail(VOX_ERR_INVALID, "block_attention: a stride is negative");
    return VOX_OK;
}
int64_t vox_block_attention_workspace_bytes(const vox_block_attention_args* a) {
    if (check_attention(a) != VOX_OK) return -1;
    return 0;
}
int vox_block_attention(vox_ctx* ctx, void* stream, const vox_block_attention_args* a) {
    (void)ctx;
    VOX_TRY(check_attention(a));
    const vox_block_cache& c = a->cache;
    const vox_block_rows& r = a->rows;
    if (r.n_rows == 0) return VOX_OK;
    if (!a->q || (!a->blocks && a->top) || !a->out || ((size_t)a->q | (size_t)a->out) & 1) return vox_fail(VOX_ERR_INVALID, "block_attention: an operand is NULL, or does not lie on its type");
    BlockAttnArgs s{(const bf16_t*)a->q, (const bf16_t*)c.kv, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (bf16_t*)a->out, (long)a->q_stride, a->scale,
                    r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages, c.page_size, c.block, a->top};
    return launch(BY_TYPE_AND_DIM(k_block_attention, c), dim3(r.n_rows, r.heads), 64, 0, (hipStream_t)stream, s);
}

}  // extern "C"
