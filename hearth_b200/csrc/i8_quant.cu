// Rows of the 8-bit linear path: f32 rows -> int8 values with ONE f32 scale per row, in the tiled plane the product
// kernels (i8_gemm.cu) read, plus the moves between that plane and row-major tensors.
//
//   quantize       v = x
//   silu_mul       v = g / (1 + exp(-g)) * u
//   add_rms_norm   h = x + r (written out), v = weight * h, and the row's factor f = 1 / sqrt(mean(h^2) + eps)
//   then           a = max |v|,  q = rint(v * (127 / a)),  scale = a / 127 (* f)
//
// The norm's factor multiplies every value of its row, so it cancels out of q and only the scale carries it: one pass
// over the row computes h, the maximum and the sum of squares together, and the int8 values do not depend on the order
// of that sum.  All steps are f32 with IEEE rounding (h, v, 127 / a and the product each rounded once), so for quantize and
// the norm q is determined to the last bit; silu_mul's v is within five half units of the exact value, since expf is within
// one unit.  Never compile this file with fast-math.  A row whose maximum is below I8_MIN_MAX (2^-100,
// where 127 / a would leave the range of f32) is stored as zeros with scale 0.  A row with an infinity or a NaN in it (or
// whose sum of squares overflows) is stored as zeros with scale NaN, so whatever is computed from it is NaN, too.
//
// HBM-bound: 4 B (quantize, + 4 silu_mul, + 8 add_rms_norm) read or written per element and 1 B written.  One CTA per
// row (a cluster of eight for a few long rows) keeps the row in registers between the reduction and the rounding, up to
// 32 values a thread; many rows of more than 32768 columns are read twice.  Measured: quantize of 4096 x 4096 13.7 us
// (6.1 TB/s), add_rms_norm 36 us (6.1 TB/s), silu_mul 26 us (5.8 TB/s), of 512 x 17408 19.5 us (4.1 TB/s: two rows are all
// that fit an SM's registers, and they load and compute in step; 56 registers with 36 bytes of spills a thread), one row of 4096 columns 1.5 / 2.3 / 1.9 us behind its
// predecessor in a graph.
//
// Reference counterparts with a scale per 32 columns: ops::rms_norm_q8 and ops::silu_mul_q8
// (hearth-llm/src/ops.rs:273-306, :442-504), quantize_q8_0 (hearth-quant/src/q8_0.rs:20-51).
#include "common.cuh"

namespace hb200 {

namespace {

constexpr float I8_MIN_MAX = 7.888609052210118e-31f;  // 2^-100

// Programmatic dependent launch: the next kernel of the stream may start its prologue now; this one touches nothing a
// predecessor wrote (or reads) before the wait.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16-byte chunk of (row, column): column c's byte is at chunk_addr + (c & 15).
__device__ __forceinline__ size_t plane_off(const I8Plane& p, int row, int c) {
    const size_t tile = (size_t)(row >> p.row_shift) * p.tile_stride + (size_t)(c >> 7) * p.kb_stride;
    const int r = row & ((1 << p.row_shift) - 1);
    return tile + (size_t)r * 128 + (size_t)((((c >> 4) & 7) ^ (r & 7)) << 4) + (c & 15);
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    const uint32_t lo = __byte_perm((uint32_t)a, (uint32_t)b, 0x0040);
    const uint32_t hi = __byte_perm((uint32_t)c, (uint32_t)d, 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// A thread's next four columns of a row, zero past column n; a warp takes 128 columns together.  VEC (rows aligned to 16 bytes):
// c .. c + 3.  Otherwise c, c + 32, c + 64 and c + 96, so that a warp's reads are neighbours all the same (norm of 1385 x 6202
// 24.6 us, with c .. c + 3 29.6; of 2238 x 873 and its values 10.8 and 15.3; quantize alone 11.9 and 10.0).
template <bool VEC>
__device__ __forceinline__ float4 read4(const float* row, int c, int n) {
    if (VEC) return c < n ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v;
    v.x = c < n ? row[c] : 0.f;
    v.y = c + 32 < n ? row[c + 32] : 0.f;
    v.z = c + 64 < n ? row[c + 64] : 0.f;
    v.w = c + 96 < n ? row[c + 96] : 0.f;
    return v;
}
template <bool VEC>
__device__ __forceinline__ int first_column() {
    return VEC ? threadIdx.x * 4 : (threadIdx.x & ~31) * 4 + (threadIdx.x & 31);
}
// STREAM: the lines are the first to leave L2 (see i8_stream_bytes).
template <bool VEC, bool STREAM>
__device__ __forceinline__ float4 read4(const float* row, int c, int n) {
    if (VEC && STREAM) return c < n ? __ldcs(reinterpret_cast<const float4*>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
    return read4<VEC>(row, c, n);
}
template <bool VEC, bool STREAM>
__device__ __forceinline__ void write4(float* row, int c, int n, float4 v) {
    if (VEC) {
        if (c >= n) return;
        if (STREAM) __stcs(reinterpret_cast<float4*>(row + c), v);
        else *reinterpret_cast<float4*>(row + c) = v;
        return;
    }
    if (c < n) row[c] = v.x;
    if (c + 32 < n) row[c + 32] = v.y;
    if (c + 64 < n) row[c + 64] = v.z;
    if (c + 96 < n) row[c + 96] = v.w;
}

__device__ __forceinline__ float silu_mul1(float g, float u) { return __fmul_rn(__fdiv_rn(g, __fadd_rn(1.0f, expf(-g))), u); }

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
    return make_float4(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y), __fadd_rn(a.z, b.z), __fadd_rn(a.w, b.w));
}
__device__ __forceinline__ float4 mul4(float4 a, float4 b) {
    return make_float4(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y), __fmul_rn(a.z, b.z), __fmul_rn(a.w, b.w));
}

// The values v of N float4s of a row, `step` columns apart from column c (zero past the row's end or `limit`); the norm adds h * h to `sq`
// and writes h.  All reads of the inputs come before the first write: the compiler may not move a read over a write
// that could be to the same memory (the sum may overwrite an input), and reads one behind the other would leave HBM idle.
template <int OP, bool VEC, bool STREAM, int N>
__device__ __forceinline__ void values(const I8Rows& p, size_t row, int c, int step, int limit, float4 (&v)[N], float& sq) {
    const int n = min(p.n_cols, limit);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = read4<VEC, STREAM>(p.x + row * p.ld, c + i * step, n);
    if constexpr (OP != I8_QUANTIZE) if (OP == I8_SILU_MUL || p.y) {
        float4 y[N];
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = read4<VEC, STREAM>(p.y + row * p.ld, c + i * step, n);
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (OP == I8_SILU_MUL)
                v[i] = make_float4(silu_mul1(v[i].x, y[i].x), silu_mul1(v[i].y, y[i].y), silu_mul1(v[i].z, y[i].z), silu_mul1(v[i].w, y[i].w));
            else
                v[i] = add4(v[i], y[i]);
        }
    }
    if constexpr (OP == I8_ADD_RMS_NORM) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (p.sum) write4<VEC, false>(p.sum + row * p.ld_sum, c + i * step, n, v[i]);
            sq = fmaf(v[i].x, v[i].x, sq);
            sq = fmaf(v[i].y, v[i].y, sq);
            sq = fmaf(v[i].z, v[i].z, sq);
            sq = fmaf(v[i].w, v[i].w, sq);
        }
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = mul4(read4<VEC>(p.weight, c + i * step, n), v[i]);
    }
}

// One float4 a second time, for rows that do not fit the registers: the norm reads h back where it was written (x or r
// may be the same memory as the sum).
template <int OP, bool VEC>
__device__ __forceinline__ float4 value_again(const I8Rows& p, size_t row, int c, int limit) {
    if (OP == I8_ADD_RMS_NORM && p.sum)
        return mul4(read4<VEC>(p.weight, c, p.n_cols), read4<VEC>(p.sum + row * p.ld_sum, c, p.n_cols));
    float unused = 0.f;
    float4 v[1];
    values<OP, VEC, false, 1>(p, row, c, 0, limit, v, unused);
    return v[0];
}

__device__ __forceinline__ uint32_t absmax4(uint32_t m, float4 v) {
    // as integers the bits of |v| order like the numbers, and a NaN is above infinity: nothing gets lost
    m = max(m, __float_as_uint(v.x) & 0x7FFFFFFFu);
    m = max(m, __float_as_uint(v.y) & 0x7FFFFFFFu);
    m = max(m, __float_as_uint(v.z) & 0x7FFFFFFFu);
    return max(m, __float_as_uint(v.w) & 0x7FFFFFFFu);
}

__device__ __forceinline__ uint32_t round4(float4 v, float inv) {
    return pack4(__float2int_rn(__fmul_rn(v.x, inv)), __float2int_rn(__fmul_rn(v.y, inv)), __float2int_rn(__fmul_rn(v.z, inv)),
                 __float2int_rn(__fmul_rn(v.w, inv)));
}

// The int8 values of read4's four columns into the plane, a word a lane either way (whole blocks of 128 columns are written, so
// the lanes of a warp agree on c < padded).  Columns 32 apart: the four lanes of a quad put their bytes of each 32-column run
// together, and each stores the word of one run (single bytes stored took twice the time of everything else).
template <bool VEC>
__device__ __forceinline__ void store4(const I8Plane& p, int row, int c, int padded, uint32_t q) {
    if (c >= padded) return;
    if (!VEC) {
        const int at = threadIdx.x & 3;
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t w = (q >> (8 * j) & 0xFFu) << (8 * at);
            w |= __shfl_xor_sync(0xffffffffu, w, 1);
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
            if (at == j) mine = w;
        }
        q = mine;
        c += 31 * at;  // from base + lane to base + 32 * at + (lane - at)
    }
    *reinterpret_cast<uint32_t*>(p.q + plane_off(p, row, c)) = q;
}

__device__ __forceinline__ uint32_t peer_smem(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}

// One CTA per row, or (CLUSTER) the CTAs of a cluster, each with a run of `quads` float4s of it.  NV = float4s of the row a
// thread keeps (0: the row is read twice).
template <int OP, int NV, bool VEC, bool STREAM, bool CLUSTER, int MAX_THREADS, int MIN_CTAS>
__global__ void __launch_bounds__(MAX_THREADS, MIN_CTAS) i8_rows_kernel(const I8Rows p, int quads) {
    __shared__ uint32_t s_max[32];
    __shared__ float s_sq[32];
    __shared__ uint2 s_part[CLUSTER ? 8 : 1];  // maximum and sum of squares of every CTA of the row
    const int row = CLUSTER ? blockIdx.y : blockIdx.x, rank = CLUSTER ? blockIdx.x : 0;
    const int step = blockDim.x * 4;
    const int first = rank * quads * 4;                             // this CTA's columns: [first, padded)
    const int padded = min((p.n_cols + 127) & ~127, first + quads * 4);
    const int c0 = first + first_column<VEC>();
    pdl_trigger();
    if (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA's memory is there
    pdl_wait();
    constexpr int BATCH = NV == 8 && OP == I8_ADD_RMS_NORM ? 2 : NV >= 4 ? 4 : (NV > 0 ? NV : 1), BATCHES = NV > 0 ? NV / BATCH : 1;
    float4 v[BATCHES][BATCH];
    uint32_t m = 0;
    float sq = 0.f;
    if (NV > 0) {
#pragma unroll
        for (int b = 0; b < BATCHES; b++) values<OP, VEC, STREAM, BATCH>(p, row, c0 + b * BATCH * step, step, padded, v[b], sq);
#pragma unroll
        for (int i = 0; i < NV; i++) m = absmax4(m, v[i / BATCH][i % BATCH]);
    } else {
        for (int c = c0; c < padded; c += step) {
            values<OP, VEC, STREAM, BATCH>(p, row, c, 0, padded, v[0], sq);
            m = absmax4(m, v[0][0]);
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (OP == I8_ADD_RMS_NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    }
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
        if (lane == 0) {
            s_max[threadIdx.x >> 5] = m;
            if (OP == I8_ADD_RMS_NORM) s_sq[threadIdx.x >> 5] = sq;
        }
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, lane < warps ? s_max[lane] : 0u);
        if (OP == I8_ADD_RMS_NORM) {
            sq = lane < warps ? s_sq[lane] : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        }
    }
    if (CLUSTER) {
        const uint32_t n = gridDim.x;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (threadIdx.x < n)
            asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(peer_smem(&s_part[rank], threadIdx.x)), "r"(m), "r"(__float_as_uint(sq)) : "memory");
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        sq = 0.f;
#pragma unroll
        for (int r = 0; r < 8; r++)
            if (r < n) {
                m = max(m, s_part[r].x);
                sq += __uint_as_float(s_part[r].y);
            }
    }
    const float a = __uint_as_float(m);
    const bool bad = m >= 0x7F800000u || (OP == I8_ADD_RMS_NORM && !(sq <= 3.4028234e38f));
    const float inv = (!bad && a >= I8_MIN_MAX) ? __fdiv_rn(127.0f, a) : 0.0f;
    if (threadIdx.x == 0 && rank == 0) {
        float scale = (a >= I8_MIN_MAX) ? __fdiv_rn(a, 127.0f) : 0.0f;
        if (OP == I8_ADD_RMS_NORM) scale = __fmul_rn(scale, __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sq, (float)p.n_cols), p.eps))));
        p.scales[row] = bad ? __uint_as_float(0x7FC00000u) : scale;
    }
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = c0 + i * step;
            store4<VEC>(p.plane, row, c, padded, bad ? 0u : round4(v[i / BATCH][i % BATCH], inv));
        }
    } else {
        for (int c = c0; c < padded; c += step) store4<VEC>(p.plane, row, c, padded, bad ? 0u : round4(value_again<OP, VEC>(p, row, c, padded), inv));
    }
}

// Row-major int8 rows (`ld` bytes apart) <-> plane, a 16-byte piece of four rows a thread.  grid (columns / 2048, rows / 4 at
// most 65535).
constexpr int MOVE_ROWS = 4;

// -> plane; columns past n_cols become zero.
__global__ void __launch_bounds__(128) i8_load_kernel(const int8_t* q, size_t ld, const float* scales_in, int n_rows, int n_cols, I8Plane plane,
                                                      float* scales) {
    pdl_trigger();
    pdl_wait();
    const int c = (blockIdx.x * 128 + threadIdx.x) * 16;
    if (c >= ((n_cols + 127) & ~127)) return;
    const bool whole = c + 16 <= n_cols && ((reinterpret_cast<uintptr_t>(q) | ld) & 15) == 0;
    for (size_t row0 = (size_t)blockIdx.y * MOVE_ROWS; row0 < (size_t)n_rows; row0 += (size_t)gridDim.y * MOVE_ROWS) {
        uint4 v[MOVE_ROWS];
#pragma unroll
        for (int i = 0; i < MOVE_ROWS; i++) {
            v[i] = make_uint4(0, 0, 0, 0);
            if (row0 + i >= (size_t)n_rows) continue;
            const int8_t* src = q + (row0 + i) * ld + c;
            if (whole) {
                v[i] = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (c + j < n_cols) w[j / 4] |= (uint32_t)(uint8_t)src[j] << (8 * (j % 4));
                v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < MOVE_ROWS; i++) {
            if (row0 + i >= (size_t)n_rows) continue;
            *reinterpret_cast<uint4*>(plane.q + plane_off(plane, (int)row0 + i, c)) = v[i];
            if (c == 0) scales[row0 + i] = scales_in[row0 + i];
        }
    }
}

// Plane -> row-major rows and / or scales.
__global__ void __launch_bounds__(128) i8_store_kernel(I8Plane plane, const float* scales, int n_rows, int n_cols, int8_t* q, size_t ld,
                                                       float* scales_out) {
    pdl_trigger();
    pdl_wait();
    const int c = (blockIdx.x * 128 + threadIdx.x) * 16;
    if (c >= n_cols) return;
    const bool whole = c + 16 <= n_cols && ((reinterpret_cast<uintptr_t>(q) | ld) & 15) == 0;
    for (size_t row0 = (size_t)blockIdx.y * MOVE_ROWS; row0 < (size_t)n_rows; row0 += (size_t)gridDim.y * MOVE_ROWS) {
#pragma unroll
        for (int i = 0; i < MOVE_ROWS; i++) {
            if (row0 + i >= (size_t)n_rows) continue;
            if (q) {
                const uint4 v = *reinterpret_cast<const uint4*>(plane.q + plane_off(plane, (int)row0 + i, c));
                int8_t* dst = q + (row0 + i) * ld + c;
                if (whole) {
                    *reinterpret_cast<uint4*>(dst) = v;
                } else {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c + j < n_cols) dst[j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
                }
            }
            if (scales_out && c == 0) scales_out[row0 + i] = scales[row0 + i];
        }
    }
}

// Plane -> the f32 values it stands for, q * scale.  A thread takes four columns of a group of eight rows: its eight loads
// are in flight together (one row a thread ran at 2.4 TB/s).
template <bool VEC, bool STREAM>
__global__ void __launch_bounds__(128) i8_dequantize_kernel(I8Plane plane, const float* scales, int n_rows, int n_cols, float* out, size_t ld) {
    pdl_trigger();
    pdl_wait();
    const int c = blockIdx.x * 512 + first_column<VEC>(), word = blockIdx.x * 512 + threadIdx.x * 4;
    if ((word & ~127) >= n_cols) return;  // (a warp's 128 columns together)
    const int row0 = blockIdx.y * 8, rows = min(8, n_rows - row0);
    uint32_t v[8];
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = row0 + min(i, rows - 1);
        v[i] = *reinterpret_cast<const uint32_t*>(plane.q + plane_off(plane, r, word));
        if (!VEC) {  // the bytes of columns c, c + 32, c + 64, c + 96 from the words that hold them
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t from = __shfl_sync(0xffffffffu, v[i], (threadIdx.x >> 2 & 7) + 8 * j);
                w |= (from >> (8 * (threadIdx.x & 3)) & 0xFFu) << (8 * j);
            }
            v[i] = w;
        }
        s[i] = scales[r];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (i >= rows) break;
        const float4 f = make_float4(__fmul_rn((float)(int8_t)(v[i]), s[i]), __fmul_rn((float)(int8_t)(v[i] >> 8), s[i]),
                                     __fmul_rn((float)(int8_t)(v[i] >> 16), s[i]), __fmul_rn((float)(int8_t)(v[i] >> 24), s[i]));
        write4<VEC, STREAM>(out + (size_t)(row0 + i) * ld, c, n_cols, f);
    }
}

// From this many bytes of row-major input (or output) on, the lines a call touches are marked as the first to leave L2: they
// would push out the 8-bit rows that the next kernel reads, and each other before anybody reads them again.  Measured with
// the values read back behind it, us without and with: silu_mul of 4096 x 4096 40.1 / 37.6, of 512 x 17408 28.9 / 27.6, of 2048 x
// 2048 14.4 / 13.9, norm of 4096 x 4096 48.3 / 47.2 (the norm alone 35.1 / 36.0).  Below, a set that stays in L2 between calls
// would lose by it: silu_mul of 512 x 4096 9.4 / 10.8.
constexpr size_t i8_stream_bytes = 32u << 20;

bool vec_rows(const void* p, size_t ld) { return ((reinterpret_cast<uintptr_t>(p) & 15) == 0) && (ld % 4 == 0); }

// A launch that may start its prologue under the end of the kernel before it.
template <typename... P, typename... A>
int launch_pdl(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    HB_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    return 0;
}

template <int OP, int NV, int MAX_THREADS, int MIN_CTAS>
int launch_rows_nv(const I8Rows& p, int n_rows, int threads, bool vec, bool stream, cudaStream_t st) {
    constexpr bool CAN = NV >= 4;  // so many bytes come with at least four float4s a thread, or with rows that are read twice
    return launch_pdl(!vec     ? i8_rows_kernel<OP, NV, false, false, false, MAX_THREADS, MIN_CTAS>
                      : stream ? i8_rows_kernel<OP, NV, true, CAN, false, MAX_THREADS, MIN_CTAS>
                               : i8_rows_kernel<OP, NV, true, false, false, MAX_THREADS, MIN_CTAS>,
                      dim3(n_rows), threads, st, 1, p, I8_MAX_COLS / 4);
}
template <int OP, int NV, int MAX_THREADS, int MIN_CTAS>
int launch_rows_cluster(const I8Rows& p, int n_rows, int ctas, int quads, bool vec, cudaStream_t st) {
    const int threads = ((quads + NV - 1) / NV + 31) / 32 * 32;
    return launch_pdl(vec ? i8_rows_kernel<OP, NV, true, false, true, MAX_THREADS, MIN_CTAS> : i8_rows_kernel<OP, NV, false, false, true, MAX_THREADS, MIN_CTAS>,
                      dim3(ctas, n_rows), threads, st, ctas, p, quads);
}

template <int OP>
int launch_rows_op(const I8Rows& p, int n_rows, bool vec, bool stream, cudaStream_t st) {
    const int quads = ((p.n_cols + 127) & ~127) / 4;  // float4s of a padded row
    const auto threads = [&](int nv) { return ((quads + nv - 1) / nv + 31) / 32 * 32; };
    // Few rows: as few float4s a thread as still leave all rows resident at once (latency).  Many rows: four or eight, so
    // that the loads of a row are in flight together and several rows share an SM, one computing while others load.
    // Measured, us: silu_mul of 512 x 4096 4.7 with two, 7.7 with four; of 512 x 17408 20.4 with eight and two CTAs per SM,
    // 35.3 with eight and one.
    const auto resident = [&](int nv) { return threads(nv) <= 1024 && n_rows <= (long long)slot_sm_count() * (2048 / threads(nv)); };
    // A few long rows: eight CTAs of a cluster per row (silu_mul of 32 x 17408 5.8 -> 3.3, norm of 1 x 12288 3.8 -> 2.4; from
    // about a hundred rows on one CTA per row is ahead again, 128 x 12288 4.2 against 5.6, and so it is at 5120 columns).
    if (quads > 1536 && n_rows <= 64) {
        const int part = ((quads + 7) / 8 + 31) / 32 * 32;
        if (part <= 1024) return launch_rows_cluster<OP, 1, 1024, 1>(p, n_rows, 8, part, vec, st);
        return launch_rows_cluster<OP, 2, 1024, 1>(p, n_rows, 8, part, vec, st);
    }
    if (resident(1)) return launch_rows_nv<OP, 1, 1024, 1>(p, n_rows, threads(1), vec, stream, st);
    if (resident(2)) return launch_rows_nv<OP, 2, 1024, 1>(p, n_rows, threads(2), vec, stream, st);
    // (48 registers: five CTAs of 256 threads or four of 320 per SM; silu_mul of 4096 x 4096 26.2 us, with 56 and four 30.9)
    if (threads(4) <= 256) return launch_rows_nv<OP, 4, 256, 5>(p, n_rows, threads(4), vec, stream, st);
    if (threads(4) <= 320) return launch_rows_nv<OP, 4, 320, 4>(p, n_rows, threads(4), vec, stream, st);
    if (threads(4) <= 512) return launch_rows_nv<OP, 4, 512, 2>(p, n_rows, threads(4), vec, stream, st);
    if (threads(4) <= 1024 && resident(4)) return launch_rows_nv<OP, 4, 1024, 1>(p, n_rows, threads(4), vec, stream, st);
    if (threads(8) <= 576) return launch_rows_nv<OP, 8, 576, 2>(p, n_rows, threads(8), vec, stream, st);
    if (threads(8) <= 1024) return launch_rows_nv<OP, 8, 1024, 1>(p, n_rows, threads(8), vec, stream, st);
    return launch_rows_nv<OP, 0, 1024, 1>(p, n_rows, 1024, vec, stream, st);
}

dim3 move_grid(int n_rows, int n_cols) {
    const int rows = (n_rows + MOVE_ROWS - 1) / MOVE_ROWS;
    return dim3((n_cols + 2047) / 2048, rows < 65535 ? rows : 65535);
}

}  // namespace

int launch_i8_rows(int op, const I8Rows& p, int n_rows, cudaStream_t st) {
    if (n_rows <= 0) return 0;
    const bool stream = (size_t)n_rows * p.n_cols * sizeof(float) * (p.y ? 2 : 1) >= i8_stream_bytes;
    bool vec = (p.n_cols % 4 == 0) && vec_rows(p.x, p.ld);
    if (p.y) vec = vec && vec_rows(p.y, p.ld);
    if (p.weight) vec = vec && vec_rows(p.weight, 0);
    if (p.sum) vec = vec && vec_rows(p.sum, p.ld_sum);
    switch (op) {
        case I8_QUANTIZE: return launch_rows_op<I8_QUANTIZE>(p, n_rows, vec, stream, st);
        case I8_SILU_MUL: return launch_rows_op<I8_SILU_MUL>(p, n_rows, vec, stream, st);
        default: return launch_rows_op<I8_ADD_RMS_NORM>(p, n_rows, vec, stream, st);
    }
}

int launch_i8_load(const int8_t* q, size_t ld, const float* scales_in, int n_rows, int n_cols, const I8Plane& plane, float* scales, cudaStream_t st) {
    if (n_rows <= 0) return 0;
    return launch_pdl(i8_load_kernel, move_grid(n_rows, n_cols), 128, st, 1, q, ld, scales_in, n_rows, n_cols, plane, scales);
}

int launch_i8_store(const I8Plane& plane, const float* scales, int n_rows, int n_cols, int8_t* q, size_t ld, float* scales_out, cudaStream_t st) {
    if (n_rows <= 0) return 0;
    return launch_pdl(i8_store_kernel, move_grid(n_rows, n_cols), 128, st, 1, plane, scales, n_rows, n_cols, q, ld, scales_out);
}

int launch_i8_dequantize(const I8Plane& plane, const float* scales, int n_rows, int n_cols, float* out, size_t ld, cudaStream_t st) {
    if (n_rows <= 0) return 0;
    const dim3 grid((n_cols + 511) / 512, (n_rows + 7) / 8);
    const bool vec = (n_cols % 4 == 0) && vec_rows(out, ld), stream = (size_t)n_rows * n_cols * sizeof(float) >= i8_stream_bytes;
    return launch_pdl(!vec ? i8_dequantize_kernel<false, false> : stream ? i8_dequantize_kernel<true, true> : i8_dequantize_kernel<true, false>, grid, 128, st,
                      1, plane, scales, n_rows, n_cols, out, ld);
}

}  // namespace hb200
