// Causal grouped-query attention of ragged rows over pages of keys and values, or over packed prompts; softmax in f32.
//   * f32, and heads beyond 256 dimensions: tiles of 16 or 64 packed rows against tiles of keys, plain multiply-adds;
//   * where a request's keys are cut into ranges, the ranges meet in a second small kernel.
#include "paged_common.cuh"
#include "tile_common.cuh"

namespace zq {
namespace {

struct RaggedCall {
    RaggedArgs a;
    RaggedPlan p;
};

constexpr uint32_t kPlainThreads = 256;

__device__ __forceinline__ void store4(float* o, float4 v) { *reinterpret_cast<float4*>(o) = v; }

// Four values of a key or value row -> shared memory, zeros where there is no row.
__device__ __forceinline__ void stage4(float* dst, const float* src, bool ok) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(ok ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void stage4(float* dst, const bf16* src, bool ok) {
    const uint2 v = ok ? *reinterpret_cast<const uint2*>(src) : make_uint2(0, 0);
    store4(dst, make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16),
                            __uint_as_float(v.y & 0xFFFF0000u)));
}

// M rows x N keys at a time, 16 x 16 threads: thread (ty, tx) has rows ty * RPT ... of the scores and of the output, keys tx + 16 j of
// the scores, values tx * 4 + 64 c ... of the output. S = Q K^T from shared memory, the online softmax in registers (a row's 16
// threads are half a warp), P through shared memory, O += P V. The next keys travel under the values' product, the values under the
// scores.
template <typename T, int M, int N, int VC>
__global__ void __launch_bounds__(kPlainThreads)
ragged_plain_kernel(const __grid_constant__ RaggedCall call) {
    constexpr int RPT = M / 16, CPT = N / 16;
    extern __shared__ __align__(16) float smf[];
    pdl_launch_dependents();
    pdl_wait();
    const RaggedArgs& a = call.a;
    const RaggedPlan& p = call.p;
    const GqaShape& s = a.s;
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, qp = s.dimp + 4, vp = s.vdimp;
    float *Q = smf, *K = Q + M * qp, *V = K + N * qp, *P = V + N * vp;
    const T *q = static_cast<const T*>(a.q), *kc = static_cast<const T*>(a.k), *vc = static_cast<const T*>(a.v);
    const float scale2 = a.scale * kLog2e;
    for_items<kPlainThreads>(a, p, [&](const Item& it) {
        const uint32_t k_first = it.k_begin;
        uint32_t k_end = it.k_end;
        {   // nothing behind what the tile's last token sees
            const uint32_t last = min(it.tile * p.tokens + p.tokens, it.n_rows) - 1;
            const int32_t see = seen_by(it, last);
            k_end = see <= 0 ? k_first : min(k_end, (uint32_t)see);
        }
        __syncthreads();  // the item before has been read
        for (uint32_t i = tid; i < M * (s.dimp / 4); i += kPlainThreads) {
            const uint32_t m = i / (s.dimp / 4), c = i % (s.dimp / 4) * 4;
            uint32_t token, head;
            const bool ok = row_of(p, it, m, M, token, head);
            stage4(Q + m * qp + c, q + (ok ? (size_t)(it.row0 + token) * a.q_ld + (size_t)(it.g * p.R + head) * s.dimp + c : 0), ok);
        }
        auto stage = [&](float* dst, const T* base, size_t ld, uint32_t pitch, uint32_t dp, uint32_t k0) {
            for (uint32_t i = tid; i < N * (dp / 4); i += kPlainThreads) {
                const uint32_t n = i / (dp / 4), c = i % (dp / 4) * 4, key = k0 + n;
                const T* row = key < k_end ? token_row(a, it, base, ld, key) : nullptr;
                stage4(dst + n * pitch + c, row ? row + (size_t)it.g * dp + c : base, row != nullptr);
            }
            copy_commit();
        };
        float o[RPT][VC][4], m[RPT], l[RPT];
        int32_t see[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            uint32_t token, head;
            see[r] = row_of(p, it, ty * RPT + r, M, token, head) ? min(seen_by(it, token), (int32_t)k_end) : 0;
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][c][e] = 0.0f;
        }
        if (k_first < k_end) stage(K, kc, a.k_ld, qp, s.dimp, k_first);
        for (uint32_t k0 = k_first; k0 < k_end; k0 += N) {
            stage(V, vc, a.v_ld, vp, s.vdimp, k0);
            copy_wait<1>();
            __syncthreads();
            float z[RPT][CPT];
#pragma unroll
            for (int r = 0; r < RPT; ++r)
#pragma unroll
                for (int j = 0; j < CPT; ++j) z[r][j] = 0.0f;
            for (uint32_t d = 0; d < s.dimp; d += 4) {
                float4 x[RPT], y[CPT];
#pragma unroll
                for (int r = 0; r < RPT; ++r) x[r] = *reinterpret_cast<const float4*>(Q + (ty * RPT + r) * qp + d);
#pragma unroll
                for (int j = 0; j < CPT; ++j) y[j] = *reinterpret_cast<const float4*>(K + (tx + 16 * j) * qp + d);
#pragma unroll
                for (int r = 0; r < RPT; ++r)
#pragma unroll
                    for (int j = 0; j < CPT; ++j)
                        z[r][j] = fmaf(x[r].x, y[j].x, fmaf(x[r].y, y[j].y, fmaf(x[r].z, y[j].z, fmaf(x[r].w, y[j].w, z[r][j]))));
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < CPT; ++j) {
                    z[r][j] = (int32_t)(k0 + tx + 16 * j) < see[r] ? z[r][j] * scale2 : -INFINITY;
                    mx = fmaxf(mx, z[r][j]);
                }
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
                mx = fmaxf(mx, m[r]);
                const float shift = mx == -INFINITY ? 0.0f : mx, f = exp2f(m[r] - shift);
                m[r] = mx;
                l[r] *= f;
#pragma unroll
                for (int j = 0; j < CPT; ++j) {
                    const float w = exp2f(z[r][j] - shift);
                    l[r] += w;
                    P[(ty * RPT + r) * (N + 4) + tx + 16 * j] = w;
                }
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[r][c][e] *= f;
            }
            copy_wait<0>();
            __syncthreads();
            if (k0 + N < k_end) stage(K, kc, a.k_ld, qp, s.dimp, k0 + N);
            for (uint32_t n = 0; n < N; n += 4) {
                float4 w[RPT];
#pragma unroll
                for (int r = 0; r < RPT; ++r) w[r] = *reinterpret_cast<const float4*>(P + (ty * RPT + r) * (N + 4) + n);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        const uint32_t col = tx * 4 + 64 * c;
                        if (col >= s.vdimp) continue;
                        const float4 x = *reinterpret_cast<const float4*>(V + (n + e) * vp + col);
#pragma unroll
                        for (int r = 0; r < RPT; ++r) {
                            const float y = e == 0 ? w[r].x : e == 1 ? w[r].y : e == 2 ? w[r].z : w[r].w;
                            o[r][c][0] = fmaf(y, x.x, o[r][c][0]);
                            o[r][c][1] = fmaf(y, x.y, o[r][c][1]);
                            o[r][c][2] = fmaf(y, x.z, o[r][c][2]);
                            o[r][c][3] = fmaf(y, x.w, o[r][c][3]);
                        }
                    }
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            float sum = l[r];
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
            uint32_t token, head;
            if (!row_of(p, it, ty * RPT + r, M, token, head)) continue;
            const uint32_t row = it.row0 + token, h = it.g * p.R + head;
            if (it.ranges == 1) {
                T* out = static_cast<T*>(a.out) + (size_t)row * a.out_pitch;
                const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t col = tx * 4 + 64 * c + e;
                        if (col < s.vdim) out[(size_t)h * s.vdim + col] = to_act<T>(o[r][c][e] * inv);
                    }
                if (h == 0)
                    for (uint32_t i = s.heads * s.vdim + tx; i < a.out_pitch; i += 16) out[i] = to_act<T>(0.0f);
            } else {
                const size_t at = ((size_t)row * s.heads + h) * p.max_ranges + it.range;
#pragma unroll
                for (int c = 0; c < VC; ++c)
                    if (tx * 4 + 64 * c < s.vdimp)
                        store4(p.part + at * s.vdimp + tx * 4 + 64 * c, make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]));
                if (tx == 0) {
                    float* ml = p.part + (size_t)a.rows * s.heads * p.max_ranges * s.vdimp + at * 2;
                    ml[0] = m[r];
                    ml[1] = sum;
                }
            }
            if (p.max_ranges > 1 && h == 0 && it.range == 0 && tx == 0) p.n_ranges[row] = it.ranges;
        }
    });
}

// The ranges of a row and head, a warp each: out = sum of their values, each brought to the common maximum, over their sums. Rows of
// one range are written already; rows behind the last request have none.
template <typename T>
__global__ void __launch_bounds__(128)
ragged_combine_kernel(const __grid_constant__ RaggedCall call) {
    pdl_launch_dependents();
    pdl_wait();
    const RaggedArgs& a = call.a;
    const RaggedPlan& p = call.p;
    const GqaShape& s = a.s;
    const uint32_t lane = threadIdx.x & 31, unit = blockIdx.x * 4 + (threadIdx.x >> 5), row = unit / s.heads, h = unit % s.heads;
    if (row >= a.rows || (int32_t)row >= a.row_start[a.requests] || (int32_t)row < a.row_start[0]) return;
    const uint32_t n = p.n_ranges[row];
    if (n < 2) return;
    const size_t at = (size_t)unit * p.max_ranges;
    const float* part = p.part + at * s.vdimp;
    const float2* ml = reinterpret_cast<const float2*>(p.part + (size_t)a.rows * s.heads * p.max_ranges * s.vdimp) + at;
    float mx = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32) mx = fmaxf(mx, ml[i].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
    const float shift = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    for (uint32_t i = lane; i < n; i += 32) sum += exp2f(ml[i].x - shift) * ml[i].y;
    sum = warp_sum_f(sum);
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    T* out = static_cast<T*>(a.out) + (size_t)row * a.out_pitch;
    for (uint32_t c = lane * 4; c < s.vdimp; c += 128) {
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t i = 0; i < n; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(part + (size_t)i * s.vdimp + c);
            const float f = exp2f(ml[i].x - shift);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
        }
        const float o[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < s.vdim) out[(size_t)h * s.vdim + c + e] = to_act<T>(o[e]);
    }
    if (h == 0)
        for (uint32_t i = s.heads * s.vdim + lane; i < a.out_pitch; i += 32) out[i] = to_act<T>(0.0f);
}

int done(cudaError_t e) { return e == cudaSuccess ? ZQ_OK : cuda_fail(e); }

// Rows of a tile: 64 where requests bring more packed rows than the small tile has, on the mean.
uint32_t tile_rows(const RaggedArgs& a) {
    const uint32_t R = a.s.heads / a.s.kv_heads;
    return (a.s.dimp > 256 || a.s.vdimp > 256 || (uint64_t)a.rows * R <= (uint64_t)16 * a.requests) ? 16 : 64;
}

// Ranges: as many as fill the SMs twice while the host sees too few units of work; beyond that no range longer than 512 keys, so that
// requests of different lengths share the SMs evenly, or as much longer as keeps the sums of the ranges within 2^19 rows.
RaggedPlan plan_of(const RaggedArgs& a, uint32_t M) {
    RaggedPlan p{};
    p.R = a.s.heads / a.s.kv_heads;
    p.tokens = p.R <= M ? M / p.R : 1;
    p.head_tiles = p.R <= M ? 1 : (p.R + M - 1) / M;
    const uint64_t tiles = (uint64_t)a.rows / p.tokens + (a.requests < a.rows ? a.requests : a.rows);
    const uint64_t units = (tiles ? tiles : 1) * a.s.kv_heads * p.head_tiles;
    const uint64_t fill = 2ull * sm_count() / units;
    p.fill = fill < 1 ? 1 : (uint32_t)fill;
    uint64_t most = 512;
    while (most < a.capacity && units * ((a.capacity + most - 1) / most) * M > (1ull << 19)) most *= 2;
    p.most_keys = (uint32_t)most;
    const uint32_t blocks = (a.capacity + kRangeKeys - 1) / kRangeKeys, least = (a.capacity + p.most_keys - 1) / p.most_keys;
    p.max_ranges = blocks < p.fill ? blocks : p.fill;
    if (p.max_ranges < least) p.max_ranges = least;
    if (p.max_ranges < 1) p.max_ranges = 1;
    p.part = static_cast<float*>(a.work);
    p.n_ranges = reinterpret_cast<uint32_t*>(p.part + (size_t)a.rows * a.s.heads * p.max_ranges * (a.s.vdimp + 2));
    return p;
}
size_t plan_bytes(const RaggedArgs& a, const RaggedPlan& p) {
    return p.max_ranges < 2 ? 0 : (size_t)a.rows * a.s.heads * p.max_ranges * (a.s.vdimp + 2) * 4 + (size_t)a.rows * 4;
}

template <typename T, int M, int N, int VC>
int plain(const RaggedCall& c, cudaStream_t st) {
    const GqaShape& s = c.a.s;
    const size_t smem = ((size_t)(M + N) * (s.dimp + 4) + (size_t)N * s.vdimp + (size_t)M * (N + 4)) * 4;
    ZQ_CUDA(cudaFuncSetAttribute(ragged_plain_kernel<T, M, N, VC>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
    const uint32_t per_sm = smem <= 72 * 1024 ? 3 : smem <= 110 * 1024 ? 2 : 1;
    return done(launch_pdl(ragged_plain_kernel<T, M, N, VC>, dim3(per_sm * sm_count()), dim3(kPlainThreads), smem, st, c));
}
template <typename T>
int plain_any(const RaggedCall& c, uint32_t M, cudaStream_t st) {
    const uint32_t v = c.a.s.vdimp;
    if (c.a.s.dimp > 256 || v > 256) return plain<T, 16, 32, 8>(c, st);
    if (M == 16) return v <= 64 ? plain<T, 16, 64, 1>(c, st) : v <= 128 ? plain<T, 16, 64, 2>(c, st) : plain<T, 16, 64, 4>(c, st);
    return v <= 64 ? plain<T, 64, 64, 1>(c, st) : v <= 128 ? plain<T, 64, 64, 2>(c, st) : plain<T, 64, 64, 4>(c, st);
}

}  // namespace

size_t ragged_work_bytes(const RaggedArgs& a, bool f32) {
    const uint32_t M = tile_rows(a);
    return !f32 && M == 64 && ragged_tc_takes(a) ? ragged_tc_work_bytes(a) : plan_bytes(a, plan_of(a, M));
}

int launch_ragged_attention(const RaggedArgs& a, bool f32, cudaStream_t st) {
    if (a.rows == 0 || a.requests == 0) return ZQ_OK;
    const uint32_t M = tile_rows(a);
    if (!f32 && M == 64 && ragged_tc_takes(a)) return launch_ragged_tc(a, st);
    const RaggedCall c{a, plan_of(a, M)};
    int rc = f32 ? plain_any<float>(c, M, st) : plain_any<bf16>(c, M, st);
    if (rc != ZQ_OK || c.p.max_ranges < 2) return rc;
    const dim3 grid(((uint64_t)a.rows * a.s.heads + 3) / 4);
    return done(f32 ? launch_pdl(ragged_combine_kernel<float>, grid, dim3(128), 0, st, c)
                    : launch_pdl(ragged_combine_kernel<bf16>, grid, dim3(128), 0, st, c));
}

}  // namespace zq
