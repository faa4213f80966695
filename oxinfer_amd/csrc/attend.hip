// Attention of a ragged batch of query rows over the 8-bit key / value cache:
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s),   s_j = cap tanh(scale q k_j / cap) - slope |position - j|
// over the keys that the row sees. One pass over the cache; the maximum and the sum run along.
//
// A tile is 16 query rows of one key head: row i of the tile's sequence and query head h of the group are entry i g + h, so that all heads
// of a group share what is read. A wave takes a block of 32 keys at a time:
//   S^T = K Q^T   2 x d / 32 matrix instructions (16 keys x 16 entries x 32 channels); a lane gets 8 scores of one entry
//   O^T += V^T P^T   d / 16 of them (16 channels x 16 entries x 32 keys), the P^T operand being the lane's 8 weights where they are
// The codes become f16 exactly (1024 + u by a byte permute, less 1152). The key scale joins the score's own factor. The value scale joins
// the weight's exponent, p' = 2^(s + log2 v_scale - m), at no cost, m being the running maximum of s + log2 v_scale; the sum of weights
// is formed of p' / v_scale. p' is at most 2^15 (2^11 when the maximum is set, and the maximum is set anew only when a weight would pass 2^15:
// hardly ever behind a wave's first blocks): of weights rounded to f16, small ones keep as many bits as there are.
// f32 rows: q and p' go in as two f16 values each (value and residual, 22 bits), twice the matrix instructions, which the reads hide.
// bf16 rows: as one (11 bits, where the rows and results have 8); the rows are scaled by a power of two each, so that nothing overflows.
#include "kv.hpp"

namespace oxhip {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttendArgs {
    KvView kv;
    KvBatchView b;
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    const float* slopes;
    const int32_t *prefix, *first;
    float* partial;
    uint32_t* counters;
    float scale, cap;
    uint32_t n_q, g, window, splits, cols, vec;  // cols: entries of a tile that may be in use; vec: q by 16 bytes, out by 16 bytes
};

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NO_MAX = -1.7e38f;      // below any score, and far enough from it that 2^(NO_MAX - score) is 0
constexpr float HEAD_ROOM = 11.0f, MOST_ROOM = 15.0f;  // log2 of a weight when the maximum is set, and before it is set anew

// Eight codes as f16 values, exactly.
__device__ __forceinline__ half8 code_values(uint32_t a, uint32_t b) {
    const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    union { half2v h[4]; half8 v; } o;
    o.h[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u)) + off;
    o.h[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u)) + off;
    o.h[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)) + off;
    o.h[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)) + off;
    return o.v;
}
__device__ __forceinline__ f32x4 mma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// The largest over the four lanes that hold an entry's scores.
__device__ __forceinline__ float entry_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float entry_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// tanh: by its series below 1/4 (the next term is 2^-27 of the value), where 1 - 2 / (e^2x + 1) cancels, and by that above.
__device__ __forceinline__ float tanh_of(float x) {
    const float a = fabsf(x), z = x * x;
    const float series = x + x * z * (-0.333333333f + z * (0.133333333f + z * (-0.0539682540f + z * (0.0218694885f - z * 0.00886323553f))));
    const float e = __builtin_amdgcn_exp2f(2.0f * LOG2E * a);
    return a < 0.25f ? series : copysignf(1.0f - 2.0f / (e + 1.0f), x);
}

// KD = d / 32; F32: f32 rows; RULES: capped or biased scores, or a factor outside the range that the plain path takes.
template <int KD, bool F32, bool RULES>
__global__ __launch_bounds__(512) void attend_split_kernel(AttendArgs a) {
    constexpr int NW = 8, PLANES = F32 ? 2 : 1, CHUNK = KD >= 2 ? 64 : 32;  // channels whose sums the waves exchange at a time
    __shared__ float red[NW][16][CHUNK + 1];
    __shared__ float m_s[NW][16], l_s[NW][16];
    __shared__ uint32_t last_s;
    constexpr uint32_t d = KD * 32;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, grp = lane >> 4;
    const uint32_t split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits, kvh = pair % a.kv.n_kv, place = pair / a.kv.n_kv, g = a.g;

    int32_t s, tile;
    if (a.b.row_start) {
        s = kv_find(a.b, place, g, 16, 1);
        tile = (int32_t)(place - (uint32_t)kv_first_place((uint64_t)(uint32_t)max(a.b.row_start[s], 0) * g, s, 16, 1));
    } else {
        const uint32_t per = (g + 15) / 16;
        s = (int32_t)(place / per);
        tile = (int32_t)(place % per);
    }
    const KvSeq seq = kv_seq(a.b, s, a.kv.shift);
    const int64_t entries = (int64_t)seq.n * g;
    if (tile < 0 || (int64_t)tile * 16 >= entries) return;
    const uint32_t e = (uint32_t)tile * 16 + n, cols = (uint32_t)min((int64_t)16, entries - (int64_t)tile * 16);
    const bool live = n < cols;
    const uint32_t i = live ? e / g : 0u, head = kvh * g + (live ? e % g : 0u);
    const size_t row = (size_t)seq.row0 + i;
    const int32_t pos = seq.len - seq.n + (int32_t)i;

    // what the entry sees: keys below `pre`, and [lo, hi)
    int32_t lo = 0, hi = 0, pre = 0;
    if (live) {
        hi = max(pos + 1, 0);
        if (a.window && pos >= (int32_t)a.window) lo = pos - (int32_t)a.window + 1;
        if (a.first) lo = max(lo, a.first[row]);
        if (hi <= lo) lo = hi = 0;
        if (a.prefix) pre = min(max(a.prefix[s], 0), seq.len);
    }
    int32_t lo_min = hi > lo ? lo : INT32_MAX, hi_max = hi, lo_max = live ? lo : 0, hi_min = live ? hi : INT32_MAX, pre_max = pre;
#pragma unroll
    for (int m = 8; m; m >>= 1) {
        lo_min = min(lo_min, __shfl_xor(lo_min, m));
        hi_max = max(hi_max, __shfl_xor(hi_max, m));
        lo_max = max(lo_max, __shfl_xor(lo_max, m));
        hi_min = min(hi_min, __shfl_xor(hi_min, m));
        pre_max = max(pre_max, __shfl_xor(pre_max, m));
    }
    lo_min = __builtin_amdgcn_readfirstlane(lo_min);
    hi_max = __builtin_amdgcn_readfirstlane(hi_max);
    lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    hi_min = __builtin_amdgcn_readfirstlane(hi_min);
    pre_max = __builtin_amdgcn_readfirstlane(pre_max);
    const KvSpan span = kv_span(pre_max, lo_min, hi_max);
    // the splits' shares: equal, and at least a block for each wave
    const uint32_t share = max((uint32_t)NW, (span.count + a.splits - 1) / a.splits), active = max(1u, (span.count + share - 1) / share);
    if (split >= active) return;
    const uint32_t b0 = split * share, b1 = min(b0 + share, span.count);

    // the entry's query as operands, scaled to 2^14 at most
    half8 qh[KD], ql[PLANES == 2 ? KD : 1];
    float factor;  // of a score, with the key scale: natural units where RULES, else times log2 e
    {
        float v[KD][8], top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KD; ks++) {
            const size_t at = row * a.q_stride + (size_t)head * d + ks * 32 + grp * 8;
            if (!live) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[ks][j] = 0.0f;
            } else if constexpr (F32) {
                const float* p = static_cast<const float*>(a.q) + at;
                if (a.vec & 1) {
                    const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
                    v[ks][0] = x.x; v[ks][1] = x.y; v[ks][2] = x.z; v[ks][3] = x.w;
                    v[ks][4] = y.x; v[ks][5] = y.y; v[ks][6] = y.z; v[ks][7] = y.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[ks][j] = p[j];
                }
            } else {
                const uint16_t* p = static_cast<const uint16_t*>(a.q) + at;
                if (a.vec & 1) {
                    const uint4 u = *reinterpret_cast<const uint4*>(p);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 8; j++) v[ks][j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[ks][j] = bf16_bits_to_f32(p[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[ks][j]));
        }
        top = entry_max(top);
        const int ex = max(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 0, -40);
        const float up = ldexpf(1.0f, 14 - ex);
#pragma unroll
        for (int ks = 0; ks < KD; ks++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = v[ks][j] * up;
                qh[ks][j] = (_Float16)x;
                if constexpr (F32) ql[ks][j] = (_Float16)(x - (float)qh[ks][j]);
            }
        factor = ldexpf(RULES ? a.scale : a.scale * LOG2E, ex - 14);
    }
    const float slope = RULES && a.slopes && live ? a.slopes[head] : 0.0f;

    f32x4 acc[2 * KD];
#pragma unroll
    for (int t = 0; t < 2 * KD; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = NO_MAX, l = 0.0f;
    const uint32_t steps = b1 > b0 + wave ? (b1 - b0 - wave + NW - 1) / NW : 0;  // of this wave: blocks b0 + wave, + NW, ...
    for (uint32_t t0 = 0; t0 < steps; t0 += 64) {
        // where the next 64 blocks lie, and their scales: one request each, a lane a block
        int64_t at = -1;
        float ksc = 0.0f, vsc = 0.0f;
        if (t0 + lane < steps) {
            const uint32_t blk = kv_span_block(span, b0 + wave + (t0 + lane) * NW);
            const int32_t page = kv_page(a.b, a.kv, s, blk);
            if (page >= 0) {
                at = (int64_t)kv_block_index(a.kv, page, kvh, blk);
                ksc = a.kv.k_scale[at];
                vsc = a.kv.v_scale[at];
            }
        }
        const float lvs = __builtin_amdgcn_logf(vsc);  // (log2)
        const uint32_t many = min(steps - t0, 64u);
        for (uint32_t t = 0; t < many; t++) {
            const uint32_t blk = kv_span_block(span, b0 + wave + (t0 + t) * NW);
            const int32_t k0 = (int32_t)(blk * KV_BLOCK);
            const int64_t where = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), t) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)at, t));
            if (where < 0) {  // no page of the cache: rows that would see it come out as NaN
                if ((k0 < hi && k0 + (int32_t)KV_BLOCK > lo) || k0 < pre) l = __builtin_nanf("");
                continue;
            }
            const float ks_b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc), t)), lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs), t));
            const gbytes kp = as_global(a.kv.k + (size_t)where * (KV_BLOCK * d)) + lane * 16, vp = as_global(a.kv.v + (size_t)where * (KV_BLOCK * d)) + lane * 16;
            uint4 kq[KD], vq[KD];
#pragma unroll
            for (int x = 0; x < KD; x++) kq[x] = gload<uint4>(kp + x * 1024);
#pragma unroll
            for (int x = 0; x < KD; x++) vq[x] = gload<uint4>(vp + x * 1024);
            f32x4 sc[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int x = 0; x < KD; x++) {
                const half8 k_lo = code_values(kq[x].x, kq[x].y), k_hi = code_values(kq[x].z, kq[x].w);
                sc[0] = mma(k_lo, qh[x], sc[0]);
                sc[1] = mma(k_hi, qh[x], sc[1]);
                if constexpr (F32) {
                    sc[0] = mma(k_lo, ql[x], sc[0]);
                    sc[1] = mma(k_hi, ql[x], sc[1]);
                }
            }
            // scores: of keys k0 + 4 grp + r and k0 + 16 + 4 grp + r
            const float f = factor * ks_b;
            float x[8];
            const int32_t own = k0 + 4 * (int32_t)grp;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                x[r] = sc[r >> 2][r & 3] * f;
                if constexpr (RULES) {
                    if (a.cap > 0.0f) x[r] = a.cap * tanh_of(x[r] / a.cap);
                    x[r] -= slope * fabsf((float)(pos - (own + 16 * (r >> 2) + (r & 3))));
                    x[r] *= LOG2E;
                }
            }
            const int32_t end = k0 + (int32_t)KV_BLOCK;
            if (!((k0 >= lo_max && end <= hi_min) || end <= pre_max)) {
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const int32_t j = own + 16 * (r >> 2) + (r & 3);
                    x[r] = (j >= lo && j < hi) || j < pre ? x[r] : -__builtin_inff();
                }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__builtin_amdgcn_ballot_w64(top + lv > m + (MOST_ROOM - HEAD_ROOM))) {
                const float to = fmaxf(m, entry_max(top) + lv), down = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= down;
#pragma unroll
                for (int c = 0; c < 2 * KD; c++) acc[c] *= down;
            }
            const float shift = lv + HEAD_ROOM - m;
            half8 ph, pl;
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const float p = __builtin_amdgcn_exp2f(x[r] + shift);
                sum += p;
                ph[r] = (_Float16)p;
                if constexpr (F32) pl[r] = (_Float16)(p - (float)ph[r]);
            }
            l += sum * __builtin_amdgcn_exp2f(-lv);
#pragma unroll
            for (int c = 0; c < KD; c++) {
                const half8 v_lo = code_values(vq[c].x, vq[c].y), v_hi = code_values(vq[c].z, vq[c].w);
                acc[2 * c] = mma(v_lo, ph, acc[2 * c]);
                acc[2 * c + 1] = mma(v_hi, ph, acc[2 * c + 1]);
                if constexpr (F32) {
                    acc[2 * c] = mma(v_lo, pl, acc[2 * c]);
                    acc[2 * c + 1] = mma(v_hi, pl, acc[2 * c + 1]);
                }
            }
        }
    }
    // the waves' parts meet
    l = entry_sum(l);
    if (lane < 16) {
        m_s[wave][lane] = m;
        l_s[wave][lane] = l;
    }
    __syncthreads();
    auto meet = [&](uint32_t entry, float& top, float& sum) {
        top = m_s[0][entry];
        for (int w = 1; w < NW; w++) top = fmaxf(top, m_s[w][entry]);
        sum = 0.0f;
        for (int w = 0; w < NW; w++) sum += l_s[w][entry] * __builtin_amdgcn_exp2f(m_s[w][entry] - top);
    };
    auto store = [&](uint32_t entry, uint32_t c, float x) {
        const uint32_t at = (uint32_t)tile * 16 + entry;
        const size_t to = ((size_t)seq.row0 + at / g) * a.out_stride + (size_t)(kvh * g + at % g) * d + c;
        if constexpr (F32) static_cast<float*>(a.out)[to] = x;
        else static_cast<uint16_t*>(a.out)[to] = f32_to_bf16_bits(x);
    };
    const size_t stride = (size_t)a.cols * (d + 2);
    float* mine = a.partial + ((size_t)pair * a.splits + split) * stride;  // [cols][d], then the maxima, then the sums
    {
        float top, sum;
        meet(n, top, sum);
        const float down = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int c = 0; c < 2 * KD; c++) acc[c] *= down;
        if (active > 1 && wave == 0 && lane < cols) {
            __hip_atomic_store(mine + (size_t)a.cols * d + lane, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(mine + (size_t)a.cols * (d + 1) + lane, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
#pragma unroll
    for (uint32_t c0 = 0; c0 < d; c0 += CHUNK) {
#pragma unroll
        for (uint32_t c = 0; c < CHUNK / 16; c++)
            if (c0 / 16 + c < 2 * KD)
#pragma unroll
                for (int r = 0; r < 4; r++) red[wave][n][c * 16 + grp * 4 + r] = acc[c0 / 16 + c < 2 * KD ? c0 / 16 + c : 0][r];
        __syncthreads();
        for (uint32_t idx = tid; idx < cols * CHUNK; idx += NW * 64) {
            const uint32_t entry = idx / CHUNK, c = idx % CHUNK;
            if (c0 + c < d) {
                float x = 0.0f;
                for (int w = 0; w < NW; w++) x += red[w][entry][c];
                if (active > 1) {
                    __hip_atomic_store(mine + (size_t)entry * d + c0 + c, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                } else {
                    float top, sum;
                    meet(entry, top, sum);
                    store(entry, c0 + c, sum == 0.0f ? 0.0f : x / sum);  // (a row that sees nothing: zeros)
                }
            }
        }
        __syncthreads();
    }
    if (active == 1) return;
    // The splits' parts meet through memory: the last workgroup to arrive adds them, in their order; the counter returns to zero for the next
    // launch. (Device-scope accesses throughout and a wait for this thread's stores before the arrival: no cache is written back or emptied.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const uint32_t seen = __hip_atomic_fetch_add(&a.counters[(size_t)pair * CTR_STRIDE], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = seen == active - 1;
        if (seen == active - 1) __hip_atomic_store(&a.counters[(size_t)pair * CTR_STRIDE], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_s) return;
    const float* all = a.partial + (size_t)pair * a.splits * stride;
    auto get = [&](size_t at) { return __hip_atomic_load(all + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    for (uint32_t idx = tid; idx < cols * d; idx += NW * 64) {
        const uint32_t entry = idx / d;
        float top = NO_MAX;
        for (uint32_t z = 0; z < active; z++) top = fmaxf(top, get(z * stride + (size_t)a.cols * d + entry));
        float x = 0.0f, sum = 0.0f;
        for (uint32_t z = 0; z < active; z++) {
            const float w = __builtin_amdgcn_exp2f(get(z * stride + (size_t)a.cols * d + entry) - top);
            sum += w * get(z * stride + (size_t)a.cols * (d + 1) + entry);
            x += w * get(z * stride + idx);
        }
        store(entry, idx % d, sum == 0.0f ? 0.0f : x / sum);
    }
}

template <bool F32, bool RULES>
static hipError_t launch_split(const AttendArgs& a, dim3 grid, hipStream_t s) {
    switch (a.kv.d / 32) {
        case 1: attend_split_kernel<1, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 2: attend_split_kernel<2, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 3: attend_split_kernel<3, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 4: attend_split_kernel<4, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 5: attend_split_kernel<5, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 6: attend_split_kernel<6, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        case 7: attend_split_kernel<7, F32, RULES><<<grid, 512, 0, s>>>(a); break;
        default: attend_split_kernel<8, F32, RULES><<<grid, 512, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

hipError_t launch_attend(const KvView& kv, const KvBatchView& b, const AttendCall& call, const DecodeScratch& sc, hipStream_t s) {
    AttendArgs a{};
    a.kv = kv;
    a.b = b;
    a.q = call.q;
    a.out = call.out;
    a.q_stride = call.q_stride;
    a.out_stride = call.out_stride;
    a.slopes = call.slopes;
    a.prefix = call.prefix;
    a.first = call.first;
    a.partial = sc.partial;
    a.counters = sc.counters;
    a.scale = call.scale;
    a.cap = call.cap;
    a.n_q = call.n_q;
    a.g = call.n_q / kv.n_kv;
    a.window = call.window;
    const size_t size = call.bf16 ? 2 : 4;
    a.vec = reinterpret_cast<uintptr_t>(call.q) % 16 == 0 && call.q_stride * size % 16 == 0 ? 1u : 0u;
    const uint64_t tiles = b.row_start ? kv_places((uint64_t)b.rows * a.g, b.n_seqs, 16, 1) : (uint64_t)b.n_seqs * ((a.g + 15) / 16);
    a.cols = b.row_start ? 16u : min(16u, a.g);
    // splits of a tile's keys: enough workgroups for the chip, as far as a table's longest sequence gives each wave a block and the scratch
    // holds their parts
    const uint64_t pairs = tiles * kv.n_kv, most = ((uint64_t)b.max_pages << kv.shift) / 8;
    uint64_t splits = 1024 / pairs;
    splits = splits < most ? splits : most;
    const uint64_t room = sc.partial_floats / (pairs * a.cols * (kv.d + 2));
    splits = splits < room ? splits : room;
    if (pairs * CTR_STRIDE > sc.ncounters || splits < 1) splits = 1;
    a.splits = (uint32_t)splits;
    if (pairs * splits > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(pairs * splits));
    const bool rules = call.cap > 0.0f || call.slopes || !(call.scale >= 0x1p-10f && call.scale <= 0x1p40f);
    if (call.bf16) return rules ? launch_split<false, true>(a, grid, s) : launch_split<false, false>(a, grid, s);
    return rules ? launch_split<true, true>(a, grid, s) : launch_split<true, false>(a, grid, s);
}

}  // namespace oxhip
