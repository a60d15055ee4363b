// kvq_chunk.hip -- gfx950 kernels of chunk attention: new tokens over int8 pages.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "kvq_chunk.hpp"
#include "kvq_device.hpp"

namespace kvq {
namespace {

// Sequence b's new tokens: rows [row0, row0 + n) of the packed batch, of a
// sequence of len tokens.
struct ChunkSeq {
    int row0, n, len;
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkArgs& a, int b) {
    ChunkSeq s;
    s.row0 = min(max(a.offsets[b], 0), a.T);
    s.n = max(min(max(a.offsets[b + 1], 0), a.T) - s.row0, 0);
    s.len = min(max(a.lengths[b], 0), a.max_len);
    if (a.granted && a.granted[b] <= 0) s.len = 0;
    return s;
}
// Tokens that new token i attends.
__device__ __forceinline__ int chunk_keys(const ChunkArgs& a, const ChunkSeq& s, int i) {
    return a.causal ? max(min(s.len, s.len - s.n + i + 1), 0) : s.len;
}

__device__ __forceinline__ float chunk_load(const ChunkArgs& a, int64_t i) {
    if (a.bf16) return __uint_as_float(static_cast<unsigned>(static_cast<const uint16_t*>(a.q)[i]) << 16);
    return static_cast<const float*>(a.q)[i];
}
__device__ __forceinline__ void chunk_store(const ChunkArgs& a, int64_t i, float x) {
    if (a.bf16) static_cast<uint16_t*>(a.out)[i] = bf16_of(x);
    else static_cast<float*>(a.out)[i] = x;
}

// Any head dim, page size or alignment: a wave a (token, query head), 64 keys at
// a time.  Lane k has the dot product of key k; the outputs are spread over the
// lanes.  q and the accumulator are in LDS.  Codes are read once per row, from L2 where
// neighbouring rows read them too: 2048 tokens over 32,768 keys (d = 128) take 932 ms,
// the matrix-core kernel 1.2, so it is for shapes that one does not take.
__global__ __launch_bounds__(kWave) void chunk_generic(const ChunkArgs a) {
    extern __shared__ float s_chunk[];
    float* s_q = s_chunk;
    float* s_acc = s_q + a.d;
    float* s_w = s_acc + a.d;
    size_t* s_row = reinterpret_cast<size_t*>(s_w + kWave);  // behind an even number of floats
    const int lane = threadIdx.x;
    const unsigned rows = static_cast<unsigned>(a.T) * a.Hq;
    for (unsigned r = blockIdx.x; r < rows; r += gridDim.x) {
        const int t = static_cast<int>(r / a.Hq), h = static_cast<int>(r % a.Hq);
        // The last sequence that begins at or before t.
        int b = 0;
        for (int step = 1 << (31 - __clz(a.B)); step > 0; step >>= 1)
            if (b + step < a.B && a.offsets[b + step] <= t) b += step;
        const ChunkSeq s = chunk_seq(a, b);
        if (t < s.row0 || t >= s.row0 + s.n) continue;
        const int keys = chunk_keys(a, s, t - s.row0);
        const int kvh = h / a.G;
        __syncthreads();
        for (int i = lane; i < a.d; i += kWave) {
            s_q[i] = chunk_load(a, t * a.q_stride + static_cast<int64_t>(h) * a.d + i);
            s_acc[i] = 0.0f;
        }
        float m = -INFINITY, l = 0.0f;
        for (int k0 = 0; k0 < keys; k0 += kWave) {
            __syncthreads();
            float x = -INFINITY;
            size_t row = 0;
            if (k0 + lane < keys) {
                row = cache_row(a.pages, a.Hkv, 0, b, kvh, k0 + lane);
                float dot = 0.0f;
                for (int i = 0; i < a.d; i++) dot = fmaf(s_q[i], static_cast<float>(a.k[row * a.d + i]), dot);
                x = dot * a.ks[row] * a.scale_log2;
            }
            const float mn = fmaxf(m, wave_max(x));
            const float ms = mn == -INFINITY ? 0.0f : mn;
            const float alpha = fast_exp2(m - ms);
            const float p = fast_exp2(x - ms);
            m = mn;
            l = l * alpha + (k0 + lane < keys ? p : 0.0f);
            s_w[lane] = k0 + lane < keys ? p * a.vs[row] : 0.0f;
            s_row[lane] = row;
            __syncthreads();
            const int n = min(kWave, keys - k0);
            for (int i = lane; i < a.d; i += kWave) {
                float acc = s_acc[i] * alpha;
                for (int k = 0; k < n; k++) acc = fmaf(s_w[k], static_cast<float>(a.v[s_row[k] * a.d + i]), acc);
                s_acc[i] = acc;
            }
        }
        l = wave_sum(l);
        for (int i = lane; i < a.d; i += kWave)
            chunk_store(a, t * a.out_stride + static_cast<int64_t>(h) * a.d + i, keys > 0 ? s_acc[i] / l : 0.0f);
    }
}

}  // namespace
}  // namespace kvq

#include "kvq_chunk_mfma.hpp"

namespace kvq {
namespace {

template <int D, int LIMBS>
hipError_t launch_mfma(const ChunkArgs& a, unsigned items, hipStream_t stream) {
    hipLaunchKernelGGL((chunk_mfma<D, LIMBS>), dim3(items), dim3(chunk_waves(D, LIMBS) * kWave), 0, stream, a);
    return hipGetLastError();
}

int chunk_dim(int d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

constexpr size_t kChunkCounters = 256 * 1024;
constexpr long long kChunkMaxUnits = 1 << 22;  // workgroups of 512 threads along x (2^32 threads are not launched)

}  // namespace

ChunkPlan chunk_plan(const ChunkArgs& a, bool vec_ok) {
    ChunkPlan p{};
    p.mfma = vec_ok && a.d <= 256 && a.d % 8 == 0 && a.G <= 128;
    if (!p.mfma || a.T == 0) return p;
    p.D = chunk_dim(a.d);
    const int waves = chunk_waves(p.D, a.bf16 ? 1 : 2);
    p.rows = 32 * waves;
    p.tile_tokens = p.rows / a.G;
    const long long tiles = std::min<long long>(a.T, a.T / p.tile_tokens + a.B);
    const long long units = tiles * a.Hkv;
    if (units > kChunkMaxUnits) p.mfma = false;
    if (!p.mfma) return ChunkPlan{};
    const int blocks = (a.max_len + kChunkKeys - 1) / kChunkKeys;
    p.max_tiles = static_cast<int>(tiles);
    p.slots = 256;  // a workgroup a CU
    p.max_splits = units < p.slots && a.B <= waves * kWave ? std::min(p.slots, (blocks + 1) / 2) : 1;
    p.items = static_cast<unsigned>(p.max_splits > 1 ? std::max<long long>(units, std::min<long long>(p.slots, units * p.max_splits)) : units);
    p.records = p.max_splits > 1 ? p.items : 0;
    if (p.records) p.bytes = kChunkCounters + p.records * p.rows * (p.D + 2) * sizeof(float);
    return p;
}

hipError_t launch_chunk(ChunkArgs a, const ChunkPlan& p, void* workspace, hipStream_t stream) {
    if (a.T == 0) return hipSuccess;
    if (p.mfma) {
        a.tile_tokens = p.tile_tokens;
        a.slots = p.slots;
        a.max_splits = p.max_splits;
        a.max_tiles = p.max_tiles;
        a.heads = make_fastdiv(static_cast<uint32_t>(a.Hkv));
        a.group = make_fastdiv(static_cast<uint32_t>(a.G));
        a.counters = static_cast<int*>(workspace);
        a.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + (p.records ? kChunkCounters : 0));
        a.part_ml = a.part_acc + p.records * p.rows * p.D;
#define KVQ_CHUNK_CASE(DIM) \
    case DIM: return a.bf16 ? launch_mfma<DIM, 1>(a, p.items, stream) : launch_mfma<DIM, 2>(a, p.items, stream);
        switch (p.D) {
            KVQ_CHUNK_CASE(64)
            KVQ_CHUNK_CASE(96)
            KVQ_CHUNK_CASE(128)
            KVQ_CHUNK_CASE(192)
            KVQ_CHUNK_CASE(256)
        }
#undef KVQ_CHUNK_CASE
    }
    const long long rows = static_cast<long long>(a.T) * a.Hq;
    const unsigned groups = static_cast<unsigned>(rows < (1 << 20) ? rows : (1 << 20));
    const size_t lds = sizeof(float) * (2 * static_cast<size_t>(a.d) + kWave) + sizeof(size_t) * kWave;
    hipLaunchKernelGGL(chunk_generic, dim3(groups), dim3(kWave), lds, stream, a);
    return hipGetLastError();
}

}  // namespace kvq
