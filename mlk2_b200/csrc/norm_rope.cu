// Head norms and position rotation of queries and keys in one pass: for each
// head row x of d elements
//   x <- x * rsqrt(mean(x^2) + eps) * w                  (with weights)
//   (x_a, x_b) <- (x_a cos - x_b sin, x_b cos + x_a sin)   for rot/2 pairs
// in f32, rounded once to the element type. The angles' cosines and sines are
// table rows chosen by the token's position on the pair's axis.
//
// HBM-bound: 2 B read and 2 B written per element, about 7 flops. A head row
// belongs to d/16 lanes, each holding two 8-element vectors: the two halves of
// the same 8 pairs, so a rotation never leaves the lane and only the norm's sum
// crosses lanes. Elements past `rot` pass through as further vector pairs. A
// lane's cosines and sines depend on the token alone, so a warp loads them once
// and applies them to several of the token's head rows.
//
// bf16, d 128, 32 + 8 heads: 16384 tokens 57 us, 6.0 TB/s (93 % of the measured
// copy rate); 5003 tokens 21.9 us, 74 %, of which 3 us are the launch and the
// first loads; 65536 tokens of 16 + 2 heads 121 us, 79 %. The last has few rows to
// share a token's table row and weights. What was tried around kSteps (5 to 20),
// kDepth (2 to 6) and kBlocks (5 to 8) is within 4 % of these or slower.
#include "heads.cuh"
#include "tc_common.cuh"

namespace mlkb {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kThreads = 128;
constexpr int kSteps = 10; // most steps of a warp (each 32 / (d / 16) head rows)
constexpr int kDepth = 3;  // steps in flight
constexpr int kBlocks = 6; // blocks of an SM

// One of q and k.
struct RopeSide {
    mlkb_heads in, out;
    const void* weight;
    int32_t rows, steps;  // head rows of a token, and the steps that do them
};

struct RopeParams {
    RopeSide side[2];
    const float* table;
    const int32_t* positions;
    int64_t table_rows, pos_stride;
    int32_t ends[kMaxAxes];  // first pair past each axis' section
    int32_t tokens, d, rot, axes;
    int32_t steps, chunks;   // steps a warp does; warps that share a token
    float eps, inv_d;
    float eps_up, eps_down;  // eps scaled by 2^140 and by 2^-140, from 64 bits
    int* status;
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ void copy16(void* smem, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::smem_u32(smem)), "l"(global)
                 : "memory");
}

// 8 elements as 4 pairs of f32.
template <typename T>
__device__ __forceinline__ void widen(const uint4& u, uint64_t (&x)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        x[i] = tc::pair(f.x, f.y);
    }
}

template <typename T>
__device__ __forceinline__ uint4 narrow(const uint64_t (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = tc::unpair(x[i]);
        w[i] = pack2<T>(f.x, f.y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kBlocks)
norm_rope_kernel(const __grid_constant__ RopeParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const unsigned warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t tok = warp / static_cast<unsigned>(p.chunks);
    if (tok >= p.tokens) return;
    // The warp's steps of the token: q's come first, then k's.
    const int first = static_cast<int>(warp - static_cast<unsigned>(tok) * p.chunks) * p.steps;
    const int last = min(first + p.steps, p.side[0].steps + p.side[1].steps);
    const int units = p.d >> 4, rows = 32 / units;  // lanes of a head row, head rows of a step
    const int sub = lane / units, c = lane - sub * units;
    const int half = p.rot >> 1, nrot = p.rot >> 4;
    const bool live = sub < rows, turned = c < nrot;
    // element offsets of the lane's two vectors
    const int e0 = turned ? 8 * c : p.rot + 16 * (c - nrot);
    const int e1 = turned ? half + 8 * c : e0 + 8;

    // A lane's vectors arrive through shared memory, kDepth steps ahead: in
    // registers so many would cost the warps that keep HBM busy. Each lane reads
    // what it fetched itself.
    __shared__ uint4 ring[kDepth][2][kThreads];
    int ahead = first;
    auto fetch = [&]() {
        const RopeSide& side = p.side[ahead >= p.side[0].steps ? 1 : 0];
        const int row = (ahead >= p.side[0].steps ? ahead - p.side[0].steps : ahead) * rows + sub;
        if (ahead < last && live && row < side.rows) {
            const T* x = static_cast<const T*>(side.in.data) + tok * side.in.row_stride +
                         row * side.in.head_stride;
            const int at = ahead % kDepth;
            copy16(&ring[at][0][threadIdx.x], x + e0);
            copy16(&ring[at][1][threadIdx.x], x + e1);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++ahead;
    };
#pragma unroll 1
    for (int u = 0; u < kDepth - 1; ++u) fetch();  // under the position and the table row below

    // The lane's cosines and sines: for split pairs (i, i + half), pairs 8c..8c+7
    // serve both vectors; for neighbours (2i, 2i + 1), vector 0 holds pairs
    // 4c..4c+3 and vector 1 pairs rot/4 + 4c...
    float cs[8], sn[8];
    bool bad = false;
    if (p.axes == 1) {
        const int64_t pos = p.positions[tok];
        bad = pos < 0 || pos >= p.table_rows;
        if (turned && !bad) {
            const float* t = p.table + pos * p.rot;
            const int i0 = kInterleaved ? 4 * c : 8 * c, i1 = kInterleaved ? half / 2 + 4 * c : i0 + 4;
            *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(t + i0);
            *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(t + i1);
            *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(t + half + i0);
            *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(t + half + i1);
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
        asm volatile("cp.async.wait_all;" ::: "memory");  // the block's memory may go to another
        return;
    }
    // As pairs: for split pairs those of two neighbours, else one value twice
    // (the sine with the signs of the two sums).
    constexpr int kPairs = kInterleaved ? 8 : 4;
    uint64_t cs2[kPairs], sn2[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        cs2[i] = kInterleaved ? tc::pair(cs[i], cs[i]) : tc::pair(cs[2 * i], cs[2 * i + 1]);
        sn2[i] = kInterleaved ? tc::pair(-sn[i], sn[i]) : tc::pair(sn[2 * i], sn[2 * i + 1]);
    }
    uint64_t wa[4] = {}, wb[4] = {};
    const bool norm = p.side[0].weight != nullptr;
    const bool butterfly = (units & (units - 1)) == 0;
    auto sum = [&](float v) {  // over the lanes of a head row
        if (butterfly) {
            for (int o = units >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            return v;
        }
        float t = v;
        for (int o = 1, at = c + 1; o < units; ++o, ++at) {
            if (at == units) at = 0;
            t += __shfl_sync(0xffffffffu, v, sub * units + at);
        }
        return t;
    };

    for (int step = first; step < last; ++step) {
        const bool second = step >= p.side[0].steps;
        const RopeSide& side = p.side[second ? 1 : 0];
        const int row = (second ? step - p.side[0].steps : step) * rows + sub;
        const bool mine = live && row < side.rows;
        if (norm && live && (step == first || step == p.side[0].steps)) {
            const T* w = static_cast<const T*>(side.weight);
            widen<T>(*reinterpret_cast<const uint4*>(w + e0), wa);
            widen<T>(*reinterpret_cast<const uint4*>(w + e1), wb);
        }
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
        uint64_t a[4], b[4];
        widen<T>(ring[step % kDepth][0][threadIdx.x], a);
        widen<T>(ring[step % kDepth][1][threadIdx.x], b);
        if (norm) {  // uniform
            uint64_t s2[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s2[0] = tc::fma2(a[i], a[i], s2[0]);
                s2[1] = tc::fma2(b[i], b[i], s2[1]);
            }
            const float2 sa = tc::unpair(tc::add2(s2[0], s2[1]));
            const float ss = sum(mine ? sa.x + sa.y : 0.0f);
            float r = rsqrtf(fmaf(ss, p.inv_d, p.eps));
            const bool large = ss > 3.0e38f, small = ss < 0x1p-80f && p.eps < 0x1p-60f;
            if (__any_sync(0xffffffffu, large || small)) {
                // The squares left the f32 range (bf16 values past 2^63, or below 2^-63
                // with an eps that does not hide them): once more on values scaled by
                // 2^-70 or 2^70, exact in f32.
                const float f = large ? 0x1p-70f : 0x1p70f;
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 u = tc::unpair(a[i]), v = tc::unpair(b[i]);
                    const float u0 = u.x * f, u1 = u.y * f, v0 = v.x * f, v1 = v.y * f;
                    t += fmaf(u0, u0, u1 * u1) + fmaf(v0, v0, v1 * v1);
                }
                t = sum(mine ? t : 0.0f);
                if (large) r = rsqrtf(fmaf(t, p.inv_d, p.eps_down)) * 0x1p-70f;
                if (small) r = rsqrtf(fmaf(t, p.inv_d, p.eps_up));
                const uint64_t keep = small ? tc::pair(f, f) : tc::pair(1.0f, 1.0f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = mul2(a[i], keep);
                    b[i] = mul2(b[i], keep);
                }
            }
            const uint64_t r2 = tc::pair(r, r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = mul2(mul2(a[i], r2), wa[i]);
                b[i] = mul2(mul2(b[i], r2), wb[i]);
            }
        }
        if (!mine) continue;
        if (turned) {
            if constexpr (kInterleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = tc::unpair(a[i]), g = tc::unpair(b[i]);
                    a[i] = tc::fma2(a[i], cs2[i], mul2(tc::pair(f.y, f.x), sn2[i]));
                    b[i] = tc::fma2(b[i], cs2[4 + i], mul2(tc::pair(g.y, g.x), sn2[4 + i]));
                }
            } else {
                const uint64_t minus = tc::pair(-1.0f, -1.0f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t f = a[i], g = b[i];
                    a[i] = tc::fma2(mul2(g, minus), sn2[i], mul2(f, cs2[i]));
                    b[i] = tc::fma2(f, sn2[i], mul2(g, cs2[i]));
                }
            }
        }
        T* y = static_cast<T*>(side.out.data) + tok * side.out.row_stride +
               row * side.out.head_stride;
        *reinterpret_cast<uint4*>(y + e0) = narrow<T>(a);
        *reinterpret_cast<uint4*>(y + e1) = narrow<T>(b);
    }
}

template <typename T>
int launchNormRope(RopeParams& p, bool interleaved, cudaStream_t s) {
    const int rows = 32 / (p.d / 16);
    int total = 0;
    for (RopeSide& side : p.side) {
        side.steps = (side.rows + rows - 1) / rows;
        total += side.steps;
    }
    // A warp's steps share the token's position, table row and weights: up to
    // kSteps of them where that leaves 32 warps to an SM.
    const int64_t most = static_cast<int64_t>(p.tokens) * total / (static_cast<int64_t>(smCount()) * 32);
    const int steps = most < 1 ? 1 : most < kSteps ? static_cast<int>(most) : kSteps;
    p.chunks = (total + steps - 1) / steps;
    p.steps = (total + p.chunks - 1) / p.chunks;
    const int64_t warps = static_cast<int64_t>(p.tokens) * p.chunks;
    if (warps > 0x7fffff00) return setError(MLKB_ERR_INVALID, "norm_rope: too many head rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((warps + kThreads / 32 - 1) / (kThreads / 32)));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const cudaError_t e = interleaved ? cudaLaunchKernelEx(&cfg, norm_rope_kernel<T, true>, p)
                                      : cudaLaunchKernelEx(&cfg, norm_rope_kernel<T, false>, p);
    return e == cudaSuccess ? okStatus() : setCudaError(MLKB_ERR_LAUNCH, e, "norm_rope launch");
}

// Whether an output starts where its own input does but runs on otherwise, or
// starts where the other side's input does.
bool overlaps(const mlkb_heads& in, const mlkb_heads& out, const RopeSide& other) {
    if (sameStart(in, out)) return in.row_stride != out.row_stride || in.head_stride != out.head_stride;
    return sameStart(out, other.in);
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
    if (!(eps >= 0 && eps <= 3e38)) return setError(MLKB_ERR_INVALID, "norm_rope: eps must be 0 to 3e38");
    if ((q_weight == nullptr) != (k_weight == nullptr) && kv_heads > 0) {
        return setError(MLKB_ERR_INVALID, "norm_rope: weights of both q and k, or of neither");
    }
    if (!aligned16(q_weight) || !aligned16(k_weight)) {
        return setError(MLKB_ERR_INVALID, "norm_rope: weights must be 16-byte aligned");
    }
    RopeParams p = {};
    RopeSide &qs = p.side[0], &ks = p.side[1];
    if (int st = checkHeads(q, heads, d, false, "norm_rope q", &qs.in)) return st;
    if (int st = checkHeads(q_out, heads, d, true, "norm_rope q_out", &qs.out)) return st;
    if (kv_heads > 0) {
        if (int st = checkHeads(k, kv_heads, d, false, "norm_rope k", &ks.in)) return st;
        if (int st = checkHeads(k_out, kv_heads, d, true, "norm_rope k_out", &ks.out)) return st;
    }
    const int64_t tokens = qs.in.rows;
    if (qs.out.rows != tokens || (kv_heads > 0 && (ks.in.rows != tokens || ks.out.rows != tokens))) {
        return setError(MLKB_ERR_INVALID, "norm_rope: q, k and their outputs must have equal rows");
    }
    if (overlaps(qs.in, qs.out, ks) || (kv_heads > 0 && overlaps(ks.in, ks.out, qs)) ||
        (sameStart(qs.out, ks.out) && !sameStart(qs.in, ks.in))) {
        return setError(MLKB_ERR_INVALID, "norm_rope: outputs may be their own inputs, and overlap nothing else");
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
    qs.weight = q_weight;
    ks.weight = k_weight;
    qs.rows = static_cast<int32_t>(heads);
    ks.rows = static_cast<int32_t>(kv_heads);
    p.table = table;
    p.positions = positions;
    p.table_rows = table_rows;
    p.pos_stride = position_stride;
    p.tokens = static_cast<int32_t>(tokens);
    p.d = static_cast<int32_t>(d);
    p.rot = static_cast<int32_t>(rot);
    p.axes = n_axes;
    p.eps = static_cast<float>(eps);
    // An eps above 0 stays above it, so that rows of zeros stay zeros (nothing else is
    // as small: the least square of a bf16 value is 2^-266).
    const double up = std::ldexp(eps, 140);
    p.eps_up = eps > 0 && up < 1.5e-45 ? 1.5e-45f : static_cast<float>(up < 3e38 ? up : 3e38);
    p.eps_down = static_cast<float>(std::ldexp(eps, -140));
    p.inv_d = 1.0f / static_cast<float>(d);
    p.status = deviceStatusPtr();
    return elem_dtype == MLKB_F16 ? launchNormRope<__half>(p, interleaved != 0, asStream(stream))
                                  : launchNormRope<__nv_bfloat16>(p, interleaved != 0, asStream(stream));
}
