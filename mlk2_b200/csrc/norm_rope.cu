// Head norms and position rotation of queries and keys in one pass: for each
// head row x of d elements
//   x <- x * rsqrt(mean(x^2) + eps) * w                  (with weights)
//   (x_a, x_b) <- (x_a cos - x_b sin, x_b cos + x_a sin)   for rot/2 pairs
// in f32, rounded once to the element type. The angles' cosines and sines are
// table rows chosen by the token's position on the pair's axis.
//
// HBM-bound: 2 B read and 2 B written per element, about 7 flops. A head row
// belongs to L lanes (a power of two, >= d/16), each holding two 8-element
// vectors: the two halves of the same 8 pairs, so a rotation never leaves the
// lane and only the norm's sum crosses lanes (log2 L shuffles). Elements past
// `rot` pass through as further vector pairs. A lane's cosines and sines
// depend on the token alone, so a warp loads them once and applies them to
// several of the token's head rows.
#include "heads.cuh"

namespace mlkb {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kThreads = 256;
constexpr int kSteps = 2;   // head-row steps a warp has in flight
constexpr int kBlocks = 4;  // blocks of an SM

struct RopeParams {
    mlkb_heads q, k, qo, ko;
    const void* qw;
    const void* kw;
    const float* table;
    const int32_t* positions;
    int64_t table_rows, pos_stride;
    int32_t ends[kMaxAxes];  // first pair past each axis' section
    int32_t tokens, heads, rows, d, rot, axes;  // rows: head rows of a token, q's then k's
    int32_t spw;                                // steps a warp does (each 32 / L head rows)
    int32_t chunks;                             // warps per token
    float eps, inv_d;
    int* status;
};

template <typename T, int L, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_rope_kernel(const RopeParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const unsigned warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t tok = warp / static_cast<unsigned>(p.chunks);
    if (tok >= p.tokens) return;
    const int step0 = static_cast<int>(warp - static_cast<unsigned>(tok) * p.chunks) * p.spw;
    const int c = lane % L, sub = lane / L;
    const int half = p.rot >> 1, nrot = p.rot >> 4;
    const bool live = c < p.d / 16, turned = c < nrot;
    // element offsets of the lane's two vectors
    const int e0 = turned ? 8 * c : p.rot + 16 * (c - nrot);
    const int e1 = turned ? half + 8 * c : e0 + 8;
    constexpr int kRowsPerStep = 32 / L;

    uint4 va[kSteps], vb[kSteps];
    int row[kSteps];
    auto load = [&](int st) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            row[u] = (st + u < step0 + p.spw) ? (st + u) * kRowsPerStep + sub : p.rows;
            va[u] = vb[u] = make_uint4(0, 0, 0, 0);
            if (live && row[u] < p.rows) {
                const bool isq = row[u] < p.heads;
                const mlkb_heads& v = isq ? p.q : p.k;
                const T* x = static_cast<const T*>(v.data) + tok * v.row_stride +
                             (isq ? row[u] : row[u] - p.heads) * v.head_stride;
                va[u] = *reinterpret_cast<const uint4*>(x + e0);
                vb[u] = *reinterpret_cast<const uint4*>(x + e1);
            }
        }
    };
    load(step0);  // in flight under the position and the table row below

    // The lane's cosines and sines: for split pairs (i, i + half), pairs 8c..8c+7
    // serve both vectors; for neighbours (2i, 2i + 1), vector 0 holds pairs
    // 4c..4c+3 and vector 1 pairs rot/4 + 4c...
    float cs[8], sn[8];
    bool bad = false;
    if (p.axes == 1) {
        const int64_t pos = p.positions[tok];
        bad = pos < 0 || pos >= p.table_rows;
        if (turned && !bad) {
            const float* row = p.table + pos * p.rot;
            const int i0 = kInterleaved ? 4 * c : 8 * c, i1 = kInterleaved ? half / 2 + 4 * c : i0 + 4;
            const float4 a = *reinterpret_cast<const float4*>(row + i0);
            const float4 b = *reinterpret_cast<const float4*>(row + i1);
            const float4 s = *reinterpret_cast<const float4*>(row + half + i0);
            const float4 t = *reinterpret_cast<const float4*>(row + half + i1);
            cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w;
            cs[4] = b.x; cs[5] = b.y; cs[6] = b.z; cs[7] = b.w;
            sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
            sn[4] = t.x; sn[5] = t.y; sn[6] = t.z; sn[7] = t.w;
        }
    } else {
        int64_t pos[kMaxAxes];
#pragma unroll
        for (int a = 0; a < kMaxAxes; ++a) {
            pos[a] = a < p.axes ? p.positions[a * p.pos_stride + tok] : 0;
            bad = bad || pos[a] < 0 || pos[a] >= p.table_rows;
        }
        if (turned && !bad) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pair = kInterleaved ? (i < 4 ? 4 * c + i : half / 2 + 4 * c + i - 4) : 8 * c + i;
                int64_t at = pos[0];
#pragma unroll
                for (int a = 1; a < kMaxAxes; ++a) {
                    if (pair >= p.ends[a - 1]) at = pos[a];
                }
                cs[i] = p.table[at * p.rot + pair];
                sn[i] = p.table[at * p.rot + half + pair];
            }
        }
    }
    if (bad) {  // a position outside the table: the token's rows are left as they are
        if (lane == 0 && p.status != nullptr) atomicExch(p.status, MLKB_ERR_INVALID);
        return;
    }

    for (int st = step0; st < step0 + p.spw; st += kSteps) {
        if (st > step0) load(st);
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            const bool isq = row[u] < p.heads;
            const T* w = static_cast<const T*>(isq ? p.qw : p.kw);
            float a[8], b[8];
            unpack8<T>(va[u], a);
            unpack8<T>(vb[u], b);
            if (p.qw != nullptr) {  // uniform
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                float r = rsqrtf(fmaf(ss, p.inv_d, p.eps));
                if (__any_sync(0xffffffffu, ss > 3.0e38f)) {
                    // The squares left the f32 range (bf16 values past 2^63): once
                    // more on values scaled by 2^-70, exact in f32. (eps has no
                    // weight there.)
                    float s2 = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = a[i] * 0x1p-70f, y = b[i] * 0x1p-70f;
                        s2 = fmaf(x, x, fmaf(y, y, s2));
                    }
#pragma unroll
                    for (int o = L / 2; o > 0; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
                    if (ss > 3.0e38f) r = rsqrtf(s2 * p.inv_d) * 0x1p-70f;
                }
                if (live && row[u] < p.rows) {
                    float wa[8], wb[8];
                    unpack8<T>(*reinterpret_cast<const uint4*>(w + e0), wa);
                    unpack8<T>(*reinterpret_cast<const uint4*>(w + e1), wb);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        a[i] = a[i] * r * wa[i];
                        b[i] = b[i] * r * wb[i];
                    }
                }
            }
            if (!live || row[u] >= p.rows) continue;
            if (turned) {
                if constexpr (kInterleaved) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], t = b[2 * i + 1];
                        a[2 * i] = x * cs[i] - y * sn[i];
                        a[2 * i + 1] = y * cs[i] + x * sn[i];
                        b[2 * i] = z * cs[4 + i] - t * sn[4 + i];
                        b[2 * i + 1] = t * cs[4 + i] + z * sn[4 + i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = a[i], y = b[i];
                        a[i] = x * cs[i] - y * sn[i];
                        b[i] = y * cs[i] + x * sn[i];
                    }
                }
            }
            const mlkb_heads& v = isq ? p.qo : p.ko;
            T* y = static_cast<T*>(v.data) + tok * v.row_stride +
                   (isq ? row[u] : row[u] - p.heads) * v.head_stride;
            *reinterpret_cast<uint4*>(y + e0) = pack8<T>(a);
            *reinterpret_cast<uint4*>(y + e1) = pack8<T>(b);
        }
    }
}

template <typename T, int L>
int launchNormRope(RopeParams& p, bool interleaved, cudaStream_t s) {
    const int steps = (p.rows + 32 / L - 1) / (32 / L);
    // Few tokens: a warp takes one step, so that they spread over the SMs. Many:
    // kSteps, whose loads are in flight together and share the table row.
    const int64_t all = static_cast<int64_t>(p.tokens) * steps;
    p.chunks = all <= static_cast<int64_t>(smCount()) * 32 ? steps : (steps + kSteps - 1) / kSteps;
    p.spw = (steps + p.chunks - 1) / p.chunks;
    const int64_t blocks = (static_cast<int64_t>(p.tokens) * p.chunks + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff / (kThreads / 32)) return setError(MLKB_ERR_INVALID, "norm_rope: too many head rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const cudaError_t e = interleaved ? cudaLaunchKernelEx(&cfg, norm_rope_kernel<T, L, true>, p)
                                      : cudaLaunchKernelEx(&cfg, norm_rope_kernel<T, L, false>, p);
    return e == cudaSuccess ? okStatus() : setCudaError(MLKB_ERR_LAUNCH, e, "norm_rope launch");
}

template <typename T>
int launchNormRope(RopeParams& p, bool interleaved, cudaStream_t s) {
    const int units = p.d / 16;
    return units <= 1    ? launchNormRope<T, 1>(p, interleaved, s)
           : units <= 2  ? launchNormRope<T, 2>(p, interleaved, s)
           : units <= 4  ? launchNormRope<T, 4>(p, interleaved, s)
           : units <= 8  ? launchNormRope<T, 8>(p, interleaved, s)
           : units <= 16 ? launchNormRope<T, 16>(p, interleaved, s)
                         : launchNormRope<T, 32>(p, interleaved, s);
}

}  // namespace
}  // namespace mlkb

extern "C" int mlkb_norm_rope(const mlkb_heads* q, const mlkb_heads* k, const mlkb_heads* q_out,
                              const mlkb_heads* k_out, int64_t heads, int64_t kv_heads, int64_t d,
                              int64_t rot, const void* q_weight, const void* k_weight, double eps,
                              const float* table, int64_t table_rows, const int32_t* positions,
                              int64_t position_stride, const int32_t* sections, int32_t n_axes,
                              int32_t interleaved, int32_t elem_dtype, void* stream) {
    using namespace mlkb;
    if (elem_dtype != MLKB_F16 && elem_dtype != MLKB_BF16) {
        return setError(MLKB_ERR_INVALID, "norm_rope: dtype must be f16 or bf16");
    }
    if (heads < 1 || kv_heads < 0 || heads > 65536 || kv_heads > 65536) {
        return setError(MLKB_ERR_INVALID, "norm_rope: 1 to 65536 heads, 0 to 65536 kv heads");
    }
    if (d < 16 || d > 512 || d % 16 != 0 || rot < 16 || rot > d || rot % 16 != 0) {
        return setError(MLKB_ERR_INVALID,
                        "norm_rope: d and rot must be multiples of 16, rot <= d <= 512");
    }
    if (!std::isfinite(eps) || eps < 0) return setError(MLKB_ERR_INVALID, "norm_rope: bad eps");
    if ((q_weight == nullptr) != (k_weight == nullptr) && kv_heads > 0) {
        return setError(MLKB_ERR_INVALID, "norm_rope: weights of both q and k, or of neither");
    }
    if (!aligned16(q_weight) || !aligned16(k_weight)) {
        return setError(MLKB_ERR_INVALID, "norm_rope: weights must be 16-byte aligned");
    }
    RopeParams p = {};
    if (int st = checkHeads(q, heads, d, false, "norm_rope q", &p.q)) return st;
    if (int st = checkHeads(q_out, heads, d, true, "norm_rope q_out", &p.qo)) return st;
    if (kv_heads > 0) {
        if (int st = checkHeads(k, kv_heads, d, false, "norm_rope k", &p.k)) return st;
        if (int st = checkHeads(k_out, kv_heads, d, true, "norm_rope k_out", &p.ko)) return st;
    }
    const int64_t tokens = p.q.rows;
    if (p.qo.rows != tokens || (kv_heads > 0 && (p.k.rows != tokens || p.ko.rows != tokens))) {
        return setError(MLKB_ERR_INVALID, "norm_rope: q, k and their outputs must have equal rows");
    }
    if (n_axes < 1 || n_axes > kMaxAxes || (n_axes > 1 && sections == nullptr)) {
        return setError(MLKB_ERR_INVALID, "norm_rope: 1 to 4 position axes, with their sections");
    }
    int64_t pairs = 0;
    for (int a = 0; a < n_axes; ++a) {
        const int64_t n = sections != nullptr ? sections[a] : rot / 2;
        if (n < 0) return setError(MLKB_ERR_INVALID, "norm_rope: negative section");
        pairs += n;
        p.ends[a] = static_cast<int32_t>(pairs < rot ? pairs : rot);
    }
    for (int a = n_axes; a < kMaxAxes; ++a) p.ends[a] = 0x7fffffff;
    if (n_axes < kMaxAxes) p.ends[n_axes - 1] = 0x7fffffff;
    if (pairs != rot / 2) {
        return setError(MLKB_ERR_INVALID, "norm_rope: the sections must add up to rot / 2");
    }
    if (tokens == 0) return okStatus();
    if (table == nullptr || positions == nullptr || table_rows < 1 || !aligned16(table) ||
        (reinterpret_cast<uintptr_t>(positions) & 3u) != 0) {
        return setError(MLKB_ERR_INVALID, "norm_rope: table (16-byte aligned) and positions needed");
    }
    if (n_axes > 1 && position_stride < 0) {
        return setError(MLKB_ERR_INVALID, "norm_rope: negative position stride");
    }
    if (int st = needDevice()) return st;
    p.qw = q_weight;
    p.kw = k_weight;
    p.table = table;
    p.positions = positions;
    p.table_rows = table_rows;
    p.pos_stride = position_stride;
    p.tokens = static_cast<int32_t>(tokens);
    p.heads = static_cast<int32_t>(heads);
    p.rows = static_cast<int32_t>(heads + kv_heads);
    p.d = static_cast<int32_t>(d);
    p.rot = static_cast<int32_t>(rot);
    p.axes = n_axes;
    p.eps = static_cast<float>(eps);
    p.inv_d = 1.0f / static_cast<float>(d);
    p.status = deviceStatusPtr();
    return elem_dtype == MLKB_F16 ? launchNormRope<__half>(p, interleaved != 0, asStream(stream))
                                  : launchNormRope<__nv_bfloat16>(p, interleaved != 0, asStream(stream));
}
