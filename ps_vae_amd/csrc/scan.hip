// Selective state space scan along packed sequences: forward, backward and the form for single tokens.
//
//   delta = softplus(dt + dt_bias)                          (or dt + dt_bias)
//   h[t, d, n] = exp(delta[t, d] A[d, n]) h[t-1, d, n] + delta[t, d] x[t, d] B[t, g, n]          g = the group of d
//   ypre[t, d] = sum_n C[t, g, n] h[t, d, n] + D[d] x[t, d]            y = ypre silu(z)   (or ypre)
//
// with G[t] = dL/dh[t] = C[t] dyp[t] + a[t+1] G[t+1], a = exp(delta A), dyp = dL/dypre = dy silu(z):
//   dC[t, n] = sum_d h dyp      dB[t, n] = sum_d G delta x      dA[d, n] = sum_t G a h[t-1] delta
//   dx = delta sum_n G B + D dyp      ddelta = x sum_n G B + sum_n G a h[t-1] A      dh0 = a[0] G[0]
//
// What bounds it: one exponential for every (row, channel, state) at a quarter of the vector rate, i.e. 16 cycles of a
// SIMD for 64 of them, beside 4 cycles for each multiply-add: about 36 cycles forward and 90 backward for 64 cells, against
// the 10 (22) bytes a channel and row that a 16-bit forward (backward) pass moves for 16 states.  No matrix instruction
// helps: every channel and state has a decay of its own.
//
// Layout: P lanes side by side share a channel and hold K states each (P K = the states rounded up: 4 x 1, 4 x 2, 4 x 4,
// 8 x 4, 16 x 4), a workgroup of 256 lanes takes 256 / P channels of one group and one sequence and walks the time axis in
// tiles of 16 rows: rows are read as vectors, brought to (delta, delta x, dyp) once, and passed to the lanes through LDS.
// With the states of a channel spread over P lanes, the sum over the states costs log2 P steps inside the lanes' own row
// (data-parallel moves, no LDS), and four times the workgroups of a lane-per-channel layout fill the chip at S x D = 8 k.
// Few sequences: the time axis is cut into chunks (every sequence into as many), a first pass finds each chunk's end
// state from zero, and the second, which makes the outputs, starts from the join of the chunks in front of it.
#include "seq_device.h"

namespace {

constexpr int TILE = 16;         // rows a tile; also the distance of the states kept for the backward pass
constexpr int PITCH = 20;        // floats of LDS a channel's tile of rows takes: 16-byte rows that 16 channels spread over all banks
constexpr int MAX_CHUNKS = 64;
constexpr float LOG2E = 1.44269504088896340736f;

// Device pointers and sizes of one call; `T` rows, `S` sequences, `D` channels in `G` groups, `N` states.
struct Scan {
    const void *x, *dt, *B, *C, *z, *dy;
    int64_t ldx, lddt, ldb, ldc, ldz, lddy;
    const float *A, *D, *bias, *h0;
    void *y, *dx, *ddt, *dz;
    int64_t ldy, lddx, ldddt, lddz;
    float *hT, *kept;
    const float* dhT;
    float* dh0;
    float *part_bc, *part_a, *part_d;      // dB/dC [tiles of a group][T][G][2 NP], dA [slots * chunks][D][NP], dD/dbias [slots * chunks][2][D]
    float *chunk_h, *chunk_s;              // [chunks][S][D][NP] end state (or carry) of a chunk from zero, [chunks][S][D] its sum of delta
    const int32_t* off;
    int T, S, Dn, G, N, chunks, softplus, zero_outside, vec;
};

__device__ __forceinline__ float softplusf(float v) {
    if (v > 20.f) return v;                // exp(-20) is below half a step of 20
    // log(1 + e) = e log(u) / (u - 1) with u = 1 + e as rounded: the rounding of u cancels (Kahan's form, in Goldberg 1991)
    const float e = expf(v), u = 1.f + e;
    return u == 1.f ? e : logf(u) * (e / (u - 1.f));
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Sum over P neighbouring lanes (all get it).  quad_perm swaps neighbours, then pairs; the half mirror and the mirror
// bring the other quad and the other eight lanes, whose members are equal by then.
template <int P> __device__ __forceinline__ float lanes_add(float v) {
    v += dpp<0xb1>(v);                     // quad_perm [1,0,3,2]
    v += dpp<0x4e>(v);                     // quad_perm [2,3,0,1]
    if constexpr (P >= 8) v += dpp<0x141>(v);   // row_half_mirror
    if constexpr (P >= 16) v += dpp<0x140>(v);  // row_mirror
    return v;
}
// Sum over the lanes of a row of 16 that are a multiple of P apart.
template <int P> __device__ __forceinline__ float stride_add(float v) {
    if constexpr (P <= 8) v += dpp<0x128>(v);   // row_ror:8
    if constexpr (P <= 4) v += dpp<0x124>(v);   // row_ror:4
    return v;
}
// a + b folded over the halves of the wave (rows of 32, or of 16): lanes of even rows hold a's sum, those of odd rows b's.
__device__ __forceinline__ float fold32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned u = r[0], v = r[1];     // copies: a bit cast straight from r[1] is compiled as one from r[0]
    return __builtin_bit_cast(float, u) + __builtin_bit_cast(float, v);
}
__device__ __forceinline__ float fold16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned u = r[0], v = r[1];     // copies: a bit cast straight from r[1] is compiled as one from r[0]
    return __builtin_bit_cast(float, u) + __builtin_bit_cast(float, v);
}

template <int K> __device__ __forceinline__ void lds_load(const float* p, float (&v)[K]) {
    if constexpr (K == 4) { const float4 q = *(const float4*)p; v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
    else if constexpr (K == 2) { const float2 q = *(const float2*)p; v[0] = q.x; v[1] = q.y; }
    else v[0] = p[0];
}

// What a lane and a workgroup are: sizes that follow from (P, K).
template <int P, int K> struct Shape {
    static constexpr int NP = P * K;                  // states, rounded up
    static constexpr int CB = 256 / P;                // channels a workgroup
    static constexpr int VE = CB >= 64 ? 4 : CB / 16; // channels of a lane when rows are staged
    static constexpr int TPR = CB / VE;               // lanes a row: 16
    static constexpr int NBC = (TILE * NP + 255) / 256;
};

// The workgroup's place: its channels [c0, c0 + nc) of the whole, their group.
struct Place { int g, c0, nc, blk; };
template <int P, int K> __device__ __forceinline__ Place place(const Scan& q) {
    const int per = q.Dn / q.G, tiles = (per + Shape<P, K>::CB - 1) / Shape<P, K>::CB;
    const int g = blockIdx.x / tiles, blk = blockIdx.x - g * tiles, c = blk * Shape<P, K>::CB;
    return {g, g * per + c, min(Shape<P, K>::CB, per - c), blk};
}

// Tiles [first, last) of chunk c of a sequence of `len` rows.
struct Range { int first, last; };
__device__ __forceinline__ Range chunk_tiles(int len, int chunks, int c) {
    const int n = (len + TILE - 1) / TILE, per = (n + chunks - 1) / chunks;
    return {min(c * per, n), min((c + 1) * per, n)};
}

// Row of `kept` for tile i of a sequence that begins at row `begin`: sequences that share a row of 16 are kept apart by
// their number, and the last index is below T / 16 + S.
__device__ __forceinline__ int64_t kept_row(int begin, int s, int tile) { return (int64_t)(begin >> 4) + s + tile; }

// A tile's B or C, element by element (fewer than the rows' own elements by the channels over the states).
template <class T, int P, int K>
__device__ __forceinline__ void fetch_bc(const void* src, int64_t ld, const Scan& q, const Place& w, int row0, int rows, float (&v)[Shape<P, K>::NBC]) {
    constexpr int NP = Shape<P, K>::NP;
#pragma unroll
    for (int j = 0; j < Shape<P, K>::NBC; ++j) {
        const int e = j * 256 + threadIdx.x, r = e / NP, n = e - r * NP;
        v[j] = r < rows && n < q.N ? (float)((const T*)src)[(int64_t)(row0 + r) * ld + w.g * q.N + n] : 0.f;
    }
}
template <int P, int K> __device__ __forceinline__ void put_bc(float* lds, const float (&v)[Shape<P, K>::NBC]) {
#pragma unroll
    for (int j = 0; j < Shape<P, K>::NBC; ++j) {
        const int e = j * 256 + threadIdx.x;
        if (e < TILE * Shape<P, K>::NP) lds[e] = v[j];
    }
}

// State of (channel d, states p K ..) in an array [rows][D][N]; lanes past the states read 0 and write nothing.
template <int K> __device__ __forceinline__ void load_state(const float* base, int64_t row, const Scan& q, int d, int n0, float (&h)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) h[k] = base && n0 + k < q.N ? base[(row * q.Dn + d) * q.N + n0 + k] : 0.f;
}
template <int K> __device__ __forceinline__ void save_state(float* base, int64_t row, const Scan& q, int d, int n0, const float (&h)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (n0 + k < q.N) base[(row * q.Dn + d) * q.N + n0 + k] = h[k];
}
// The same in this file's own arrays, whose states are rounded up to NP.
template <int K> __device__ __forceinline__ float* own_state(float* base, int64_t row, const Scan& q, int NP, int d, int n0) {
    return base + (row * q.Dn + d) * NP + n0;
}
template <int K> __device__ __forceinline__ void put_state(float* p, const float (&h)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) p[k] = h[k];
}

// Rows that no sequence holds become zero (one more z-slice of the grid does it, where the caller asks for it).
template <class T> __device__ __forceinline__ void zero_rows(void* out, int64_t ld, const Scan& q, const Place& w, int slots) {
    if (!out) return;
    const int first = q.S ? min(max(q.off[0], 0), q.T) : q.T;
    const int last = q.S ? min(max(q.off[q.S], first), q.T) : q.T;
    for (int t = blockIdx.y; t < q.T - (last - first); t += slots) {
        const int row = t < first ? t : t - first + last;
        for (int c = threadIdx.x; c < w.nc; c += 256) ((T*)out)[(int64_t)row * ld + w.c0 + c] = (T)0.f;
    }
}

// Forward.  ENDS: only each chunk's end state from zero and its sum of delta, for all chunks but the last.
template <class T, int P, int K, bool ENDS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(Scan q) {
    using Sh = Shape<P, K>;
    constexpr int NP = Sh::NP, VE = Sh::VE;
    __shared__ __attribute__((aligned(16))) float s_delta[Sh::CB * PITCH], s_dx[Sh::CB * PITCH], s_y[ENDS ? 4 : Sh::CB * PITCH];
    __shared__ __attribute__((aligned(16))) float s_b[TILE * NP], s_c[ENDS ? 4 : TILE * NP];
    const Place w = place<P, K>(q);
    const int chunk = blockIdx.z;
    if (!ENDS && chunk == q.chunks) { zero_rows<T>(q.y, q.ldy, q, w, gridDim.y); return; }
    const int r = threadIdx.x / Sh::TPR, c = threadIdx.x % Sh::TPR * VE;       // staging: row and first channel of this lane
    const int ch = threadIdx.x / P, n0 = threadIdx.x % P * K;                   // scanning: channel and first state
    const int left = w.nc - c, d = w.c0 + min(ch, w.nc - 1);
    const bool live = ch < w.nc;
    float A2[K], bias[VE], skip[VE];
    load_state<K>(q.A, 0, q, d, n0, A2);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] *= LOG2E;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
        bias[i] = q.bias && i < left ? q.bias[w.c0 + c + i] : 0.f;
        skip[i] = q.D && i < left ? q.D[w.c0 + c + i] : 0.f;
    }
    for (int s = blockIdx.y; s < q.S; s += gridDim.y) {
        const SeqBounds sq = seq_bounds(q.off, s, q.S, q.T);
        const int len = sq.end - sq.begin;
        const Range tiles = chunk_tiles(len, q.chunks, chunk);
        float h[K], sum = 0.f;
        if (ENDS) {
#pragma unroll
            for (int k = 0; k < K; ++k) h[k] = 0.f;
        } else {
            load_state<K>(q.h0, s, q, d, n0, h);
            for (int i = 0; i < chunk; ++i) {          // join the chunks in front: h = exp(A sum) h + end
                const int64_t row = (int64_t)i * q.S + s;
                const float ds = q.chunk_s[row * q.Dn + d];
                const float* e = own_state<K>(q.chunk_h, row, q, NP, d, n0);
#pragma unroll
                for (int k = 0; k < K; ++k) h[k] = fmaf(__builtin_amdgcn_exp2f(ds * A2[k]), h[k], e[k]);
            }
        }
        float nx[VE], nt[VE], nz[VE], nb[Sh::NBC], nc[Sh::NBC];
        auto fetch = [&](int tile) {
            const int row0 = sq.begin + tile * TILE, rows = min(TILE, sq.end - row0), n = r < rows ? left : 0;
            const int64_t row = row0 + min(r, rows - 1);
            load_some<VE>((const T*)q.x + row * q.ldx + w.c0 + c, n, q.vec, nx);
            load_some<VE>((const T*)q.dt + row * q.lddt + w.c0 + c, n, q.vec, nt);
            if (!ENDS && q.z) load_some<VE>((const T*)q.z + row * q.ldz + w.c0 + c, n, q.vec, nz);
            fetch_bc<T, P, K>(q.B, q.ldb, q, w, row0, rows, nb);
            if (!ENDS) fetch_bc<T, P, K>(q.C, q.ldc, q, w, row0, rows, nc);
        };
        if (tiles.first < tiles.last) fetch(tiles.first);
        for (int tile = tiles.first; tile < tiles.last; ++tile) {
            const int row0 = sq.begin + tile * TILE, rows = min(TILE, sq.end - row0);
            float cx[VE], cz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float v = nt[i] + bias[i];
                const float delta = r < rows && i < left ? (q.softplus ? softplusf(v) : v) : 0.f;   // rows behind the end change nothing
                cx[i] = nx[i];
                cz[i] = nz[i];
                s_delta[(c + i) * PITCH + r] = delta;
                s_dx[(c + i) * PITCH + r] = delta * nx[i];
            }
            put_bc<P, K>(s_b, nb);
            if (!ENDS) put_bc<P, K>(s_c, nc);
            __syncthreads();
            if (tile + 1 < tiles.last) fetch(tile + 1);
            if (!ENDS && q.kept && live) put_state<K>(own_state<K>(q.kept, kept_row(sq.begin, s, tile), q, NP, d, n0), h);
#pragma unroll
            for (int t4 = 0; t4 < TILE; t4 += 4) {
                if (t4 < rows) {
                    float dl[4], dx[4], yv[4];
                    lds_load<4>(s_delta + ch * PITCH + t4, dl);
                    lds_load<4>(s_dx + ch * PITCH + t4, dx);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float b[K], cc[K];
                        lds_load<K>(s_b + (t4 + j) * NP + n0, b);
                        if (!ENDS) lds_load<K>(s_c + (t4 + j) * NP + n0, cc);
                        yv[j] = 0.f;
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            h[k] = fmaf(__builtin_amdgcn_exp2f(dl[j] * A2[k]), h[k], dx[j] * b[k]);
                            if (!ENDS) yv[j] = fmaf(h[k], cc[k], yv[j]);
                        }
                        if (ENDS) sum += dl[j];
                        else yv[j] = lanes_add<P>(yv[j]);
                    }
                    if (!ENDS && n0 == 0) *(float4*)(s_y + ch * PITCH + t4) = make_float4(yv[0], yv[1], yv[2], yv[3]);
                }
            }
            __syncthreads();
            if (!ENDS && r < rows) {
                float o[VE];
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    o[i] = fmaf(skip[i], cx[i], s_y[(c + i) * PITCH + r]);
                    if (q.z) o[i] *= cz[i] * sigmoidf(cz[i]);
                }
                store_some<VE>((T*)q.y + (int64_t)(row0 + r) * q.ldy + w.c0 + c, left, q.vec, o);
            }
        }
        if (ENDS) {
            const int64_t row = (int64_t)chunk * q.S + s;
            if (live) {
                put_state<K>(own_state<K>(q.chunk_h, row, q, NP, d, n0), h);
                if (n0 == 0) q.chunk_s[row * q.Dn + d] = sum;
            }
        } else if (q.hT && chunk == q.chunks - 1 && live) {
            save_state<K>(q.hT, s, q, d, n0, h);
        }
        __syncthreads();                               // the last tile's s_y is read before the next sequence writes it
    }
}

// Backward.  CARRY: only what each chunk passes to the one in front of it, from a zero carry, and its sum of delta.
template <class T, int P, int K, bool CARRY>
__global__ __launch_bounds__(256) void scan_bwd_kernel(Scan q) {
    using Sh = Shape<P, K>;
    constexpr int NP = Sh::NP, VE = Sh::VE;
    // the lanes of a channel overwrite their rows of the first three with sum_n G B, sum_n G a h' A and sum_n h C
    __shared__ __attribute__((aligned(16))) float s_delta[Sh::CB * PITCH], s_dx[CARRY ? 4 : Sh::CB * PITCH], s_dy[Sh::CB * PITCH];
    __shared__ __attribute__((aligned(16))) float s_b[CARRY ? 4 : TILE * NP], s_c[TILE * NP];
    __shared__ float s_bc[CARRY ? 4 : 4 * TILE * 2 * NP];
    const Place w = place<P, K>(q);
    const int chunk = blockIdx.z + (CARRY ? 1 : 0);
    if (!CARRY && chunk == q.chunks) {
        zero_rows<T>(q.dx, q.lddx, q, w, gridDim.y);
        zero_rows<T>(q.ddt, q.ldddt, q, w, gridDim.y);
        if (q.z) zero_rows<T>(q.dz, q.lddz, q, w, gridDim.y);
        return;
    }
    const int r = threadIdx.x / Sh::TPR, c = threadIdx.x % Sh::TPR * VE;
    const int ch = threadIdx.x / P, n0 = threadIdx.x % P * K, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int left = w.nc - c, d = w.c0 + min(ch, w.nc - 1);
    const bool live = ch < w.nc;
    float A[K], A2[K], dA[K], bias[VE], skip[VE], dD[VE], dbias[VE];
    load_state<K>(q.A, 0, q, d, n0, A);
#pragma unroll
    for (int k = 0; k < K; ++k) { A2[k] = A[k] * LOG2E; dA[k] = 0.f; }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
        bias[i] = q.bias && i < left ? q.bias[w.c0 + c + i] : 0.f;
        skip[i] = q.D && i < left ? q.D[w.c0 + c + i] : 0.f;
        dD[i] = dbias[i] = 0.f;
    }
    for (int s = blockIdx.y; s < q.S; s += gridDim.y) {
        const SeqBounds sq = seq_bounds(q.off, s, q.S, q.T);
        const int len = sq.end - sq.begin;
        const Range tiles = chunk_tiles(len, q.chunks, chunk);
        float ag[K], sum = 0.f;                        // ag = a[t+1] G[t+1], the carry from the rows behind
        if (CARRY) {
#pragma unroll
            for (int k = 0; k < K; ++k) ag[k] = 0.f;
        } else {
            load_state<K>(q.dhT, s, q, d, n0, ag);
            for (int i = q.chunks - 1; i > chunk; --i) {
                const int64_t row = (int64_t)(i - 1) * q.S + s;
                const float ds = q.chunk_s[row * q.Dn + d];
                const float* e = own_state<K>(q.chunk_h, row, q, NP, d, n0);
#pragma unroll
                for (int k = 0; k < K; ++k) ag[k] = fmaf(__builtin_amdgcn_exp2f(ds * A2[k]), ag[k], e[k]);
            }
        }
        float nx[VE], nt[VE], nz[VE], ng[VE], nb[Sh::NBC], nc[Sh::NBC], nh[K];
        auto fetch = [&](int tile) {
            const int row0 = sq.begin + tile * TILE, rows = min(TILE, sq.end - row0), n = r < rows ? left : 0;
            const int64_t row = row0 + min(r, rows - 1);
            load_some<VE>((const T*)q.dt + row * q.lddt + w.c0 + c, n, q.vec, nt);
            load_some<VE>((const T*)q.dy + row * q.lddy + w.c0 + c, n, q.vec, ng);
            if (q.z) load_some<VE>((const T*)q.z + row * q.ldz + w.c0 + c, n, q.vec, nz);
            fetch_bc<T, P, K>(q.C, q.ldc, q, w, row0, rows, nc);
            if (!CARRY) {
                load_some<VE>((const T*)q.x + row * q.ldx + w.c0 + c, n, q.vec, nx);
                fetch_bc<T, P, K>(q.B, q.ldb, q, w, row0, rows, nb);
                const float* k0 = own_state<K>(q.kept, kept_row(sq.begin, s, tile), q, NP, d, n0);
#pragma unroll
                for (int k = 0; k < K; ++k) nh[k] = k0[k];
            }
        };
        if (tiles.first < tiles.last) fetch(tiles.last - 1);
        for (int tile = tiles.last - 1; tile >= tiles.first; --tile) {
            const int row0 = sq.begin + tile * TILE, rows = min(TILE, sq.end - row0);
            float cx[VE], cz[VE], cg[VE], cv[VE], cd[VE], h[K];
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                cv[i] = nt[i] + bias[i];
                cd[i] = r < rows && i < left ? (q.softplus ? softplusf(cv[i]) : cv[i]) : 0.f;
                cx[i] = nx[i]; cz[i] = nz[i]; cg[i] = ng[i];
                s_delta[(c + i) * PITCH + r] = cd[i];
                if (!CARRY) s_dx[(c + i) * PITCH + r] = cd[i] * cx[i];
                s_dy[(c + i) * PITCH + r] = q.z ? cg[i] * cz[i] * sigmoidf(cz[i]) : cg[i];
            }
            if (!CARRY) put_bc<P, K>(s_b, nb);
            put_bc<P, K>(s_c, nc);
#pragma unroll
            for (int k = 0; k < K; ++k) h[k] = nh[k];
            __syncthreads();
            if (tile > tiles.first) fetch(tile - 1);
            if constexpr (CARRY) {
#pragma unroll
                for (int t4 = TILE - 4; t4 >= 0; t4 -= 4) {
                    if (t4 >= rows) continue;
                    float dl[4], dy[4];
                    lds_load<4>(s_delta + ch * PITCH + t4, dl);
                    lds_load<4>(s_dy + ch * PITCH + t4, dy);
#pragma unroll
                    for (int j = 3; j >= 0; --j) {
                        float cc[K];
                        lds_load<K>(s_c + (t4 + j) * NP + n0, cc);
                        sum += dl[j];
#pragma unroll
                        for (int k = 0; k < K; ++k) ag[k] = __builtin_amdgcn_exp2f(dl[j] * A2[k]) * fmaf(dy[j], cc[k], ag[k]);
                    }
                }
                __syncthreads();
            } else {
            // forward over the tile: the decays a and the decayed states a h[t-1] stay in registers
            float a[TILE][K], p[TILE][K], dAt[K];
#pragma unroll
            for (int k = 0; k < K; ++k) dAt[k] = 0.f;
#pragma unroll
            for (int t4 = 0; t4 < TILE; t4 += 4) {
                if (t4 >= rows) continue;
                float dl[4], dx[4];
                lds_load<4>(s_delta + ch * PITCH + t4, dl);
                lds_load<4>(s_dx + ch * PITCH + t4, dx);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float b[K];
                    lds_load<K>(s_b + (t4 + j) * NP + n0, b);
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        a[t4 + j][k] = __builtin_amdgcn_exp2f(dl[j] * A2[k]);
                        p[t4 + j][k] = a[t4 + j][k] * h[k];
                        h[k] = fmaf(dx[j], b[k], p[t4 + j][k]);
                    }
                }
            }
#pragma unroll
            for (int t4 = TILE - 4; t4 >= 0; t4 -= 4) {
                if (t4 >= rows) continue;
                float dl[4], dx[4], dy[4], su[4], sv[4], sy[4];
                lds_load<4>(s_delta + ch * PITCH + t4, dl);
                lds_load<4>(s_dx + ch * PITCH + t4, dx);
                lds_load<4>(s_dy + ch * PITCH + t4, dy);
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    const int t = t4 + j;
                    float b[K], cc[K], db[K], dc[K];
                    lds_load<K>(s_b + t * NP + n0, b);
                    lds_load<K>(s_c + t * NP + n0, cc);
                    su[j] = sv[j] = sy[j] = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const float g = fmaf(dy[j], cc[k], ag[k]);
                        const float hk = fmaf(dx[j], b[k], p[t][k]);
                        const float v = g * p[t][k];
                        dc[k] = live ? dy[j] * hk : 0.f;
                        db[k] = live ? g * dx[j] : 0.f;
                        su[j] = fmaf(g, b[k], su[j]);
                        sv[j] = fmaf(v, A[k], sv[j]);
                        sy[j] = fmaf(hk, cc[k], sy[j]);
                        dAt[k] = fmaf(v, dl[j], dAt[k]);
                        ag[k] = a[t][k] * g;
                    }
                    su[j] = lanes_add<P>(su[j]);
                    sv[j] = lanes_add<P>(sv[j]);
                    sy[j] = lanes_add<P>(sy[j]);
                    // sums over this wave's channels: row of 16 lanes 0, 1: dB of even, odd k; rows 2, 3: dC
                    float* bc = s_bc + ((wave * TILE + t) * 2 + (lane >> 5)) * NP + n0;
                    float f[K];
#pragma unroll
                    for (int k = 0; k < K; ++k) f[k] = fold32(db[k], dc[k]);
                    const int odd = lane >> 4 & 1;
                    if constexpr (K == 1) {
                        const float e = stride_add<P>(f[0] + __shfl_xor(f[0], 16, 64));
                        if ((lane & 31) < P) bc[0] = e;
                    } else {
#pragma unroll
                        for (int k = 0; k < K; k += 2) {
                            const float e = stride_add<P>(fold16(f[k], f[k + 1]));
                            if ((lane & 15) < P) bc[k + odd] = e;
                        }
                    }
                }
                if (n0 == 0) {
                    *(float4*)(s_delta + ch * PITCH + t4) = make_float4(su[0], su[1], su[2], su[3]);
                    *(float4*)(s_dx + ch * PITCH + t4) = make_float4(sv[0], sv[1], sv[2], sv[3]);
                    *(float4*)(s_dy + ch * PITCH + t4) = make_float4(sy[0], sy[1], sy[2], sy[3]);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) dA[k] += dAt[k];     // tile sums first: a long sum of short ones rounds less
            __syncthreads();
            if (r < rows) {
                float odx[VE], odt[VE], odz[VE];
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const int at = (c + i) * PITCH + r;
                    const float su = s_delta[at], sv = s_dx[at], ypre = fmaf(skip[i], cx[i], s_dy[at]);
                    float dyp = cg[i];
                    if (q.z) {
                        const float sg = sigmoidf(cz[i]);
                        dyp = cg[i] * cz[i] * sg;
                        odz[i] = cg[i] * ypre * sg * (1.f + cz[i] * (1.f - sg));
                    }
                    odx[i] = fmaf(su, cd[i], skip[i] * dyp);
                    odt[i] = fmaf(su, cx[i], sv);
                    if (q.softplus) odt[i] *= cv[i] > 20.f ? 1.f : sigmoidf(cv[i]);
                    dD[i] = fmaf(dyp, cx[i], dD[i]);
                    dbias[i] += odt[i];
                }
                const int64_t row = row0 + r;
                store_some<VE>((T*)q.dx + row * q.lddx + w.c0 + c, left, q.vec, odx);
                store_some<VE>((T*)q.ddt + row * q.ldddt + w.c0 + c, left, q.vec, odt);
                if (q.z) store_some<VE>((T*)q.dz + row * q.lddz + w.c0 + c, left, q.vec, odz);
            }
            for (int e = threadIdx.x; e < rows * 2 * NP; e += 256) {
                const float v = (s_bc[e] + s_bc[TILE * 2 * NP + e]) + (s_bc[2 * TILE * 2 * NP + e] + s_bc[3 * TILE * 2 * NP + e]);
                const int row = e / (2 * NP), col = e - row * 2 * NP;
                q.part_bc[(((int64_t)w.blk * q.T + row0 + row) * q.G + w.g) * 2 * NP + col] = v;
            }
            __syncthreads();
            }
        }
        if (CARRY) {
            const int64_t row = (int64_t)(chunk - 1) * q.S + s;
            if (live) {
                put_state<K>(own_state<K>(q.chunk_h, row, q, NP, d, n0), ag);
                if (n0 == 0) q.chunk_s[row * q.Dn + d] = sum;
            }
        } else if (q.dh0 && chunk == 0 && live) {
            save_state<K>(q.dh0, s, q, d, n0, ag);
        }
    }
    if constexpr (!CARRY) {
        const int64_t slot = (int64_t)blockIdx.y * q.chunks + chunk;
        if (live) put_state<K>(own_state<K>(q.part_a, slot, q, NP, d, n0), dA);
        // dD and ddt_bias: join the 16 rows of lanes that hold the same channels
#pragma unroll
        for (int i = 0; i < VE; ++i) { s_delta[(c + i) * PITCH + r] = dD[i]; s_dy[(c + i) * PITCH + r] = dbias[i]; }
        __syncthreads();
        for (int i = threadIdx.x; i < w.nc; i += 256) {
            float u = 0.f, v = 0.f;
#pragma unroll
            for (int k = 0; k < TILE; ++k) { u += s_delta[i * PITCH + k]; v += s_dy[i * PITCH + k]; }
            q.part_d[slot * 2 * q.Dn + w.c0 + i] = u;
            q.part_d[slot * 2 * q.Dn + q.Dn + w.c0 + i] = v;
        }
    }
}

// The sums over workgroups: dB and dC over the channel tiles of a group, dA / dD / ddt_bias over slots and chunks.
struct ScanJoin {
    const float *part_bc, *part_a, *part_d;
    void *dB, *dC;
    int64_t lddb, lddc;
    float *dA, *dD, *dbias;
    const int32_t* off;
    int T, S, Dn, G, N, NP, tiles, parts, blocks_bc, blocks_a, zero_outside;
};
template <class T> __global__ __launch_bounds__(256) void scan_join_kernel(ScanJoin q) {
    int blk = blockIdx.x;
    if (blk < q.blocks_bc) {
        const int64_t cols = (int64_t)q.T * q.G * 2 * q.NP;
        int begin = 0, end = q.T;                       // rows that a sequence holds
        if (q.off) {
            begin = min(max(q.off[0], 0), q.T);
            end = min(max(q.off[q.S], begin), q.T);
        }
        for (int64_t i = (int64_t)blk * 256 + threadIdx.x; i < cols; i += (int64_t)q.blocks_bc * 256) {
            const int n = (int)(i % q.NP), isC = (int)(i / q.NP & 1), g = (int)(i / (2 * q.NP) % q.G);
            const int64_t row = i / (2 * q.NP) / q.G;
            if (n >= q.N) continue;
            float s = 0.f;
            if (row >= begin && row < end)
                for (int p = 0; p < q.tiles; ++p) s += q.part_bc[(int64_t)p * cols + i];
            else if (!q.zero_outside) continue;
            if (isC) ((T*)q.dC)[row * q.lddc + g * q.N + n] = (T)s;
            else ((T*)q.dB)[row * q.lddb + g * q.N + n] = (T)s;
        }
        return;
    }
    blk -= q.blocks_bc;
    if (blk < q.blocks_a) {
        const int64_t i = (int64_t)blk * 256 + threadIdx.x;
        if (i >= (int64_t)q.Dn * q.N) return;
        const int64_t at = i / q.N * q.NP + i % q.N, step = (int64_t)q.Dn * q.NP;
        float s = 0.f;
        for (int p = 0; p < q.parts; ++p) s += q.part_a[p * step + at];
        q.dA[i] = s;
        return;
    }
    blk -= q.blocks_a;
    const int i = blk * 256 + threadIdx.x;
    if (i >= q.Dn) return;
    float u = 0.f, v = 0.f;
    for (int p = 0; p < q.parts; ++p) {
        u += q.part_d[(int64_t)p * 2 * q.Dn + i];
        v += q.part_d[(int64_t)p * 2 * q.Dn + q.Dn + i];
    }
    if (q.dD) q.dD[i] = u;
    if (q.dbias) q.dbias[i] = v;
}

// One token for each of S sequences: bound by the states, read and written once.  P lanes a channel as above; a lane has
// its states to itself, so `hT` may be `h0`.
template <class T, int P, int K> __global__ __launch_bounds__(256) void scan_step_kernel(Scan q, int vec_state) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / P;
    const int n0 = threadIdx.x % P * K;
    if (i >= (int64_t)q.S * q.Dn) return;              // whole groups of P lanes
    const int64_t s = i / q.Dn;
    const int d = (int)(i - s * q.Dn), g = d / (q.Dn / q.G);
    float h[K], A[K];
    if (vec_state) {
        load_vec<K>(q.h0 + i * q.N + n0, h);
        load_vec<K>(q.A + (int64_t)d * q.N + n0, A);
    } else {
        load_state<K>(q.h0, s, q, d, n0, h);
        load_state<K>(q.A, 0, q, d, n0, A);
    }
    const float x = (float)((const T*)q.x)[s * q.ldx + d];
    const float v = (float)((const T*)q.dt)[s * q.lddt + d] + (q.bias ? q.bias[d] : 0.f);
    const float delta = q.softplus ? softplusf(v) : v;
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int n = n0 + k < q.N ? n0 + k : 0;
        const float b = (float)((const T*)q.B)[s * q.ldb + g * q.N + n], c = (float)((const T*)q.C)[s * q.ldc + g * q.N + n];
        h[k] = fmaf(__builtin_amdgcn_exp2f(delta * (A[k] * LOG2E)), h[k], delta * x * b);
        if (n0 + k < q.N) y = fmaf(h[k], c, y);
    }
    y = lanes_add<P>(y);
    if (vec_state) {
        store_vec<K>(q.hT + i * q.N + n0, h);
    } else {
        save_state<K>(q.hT, s, q, d, n0, h);
    }
    if (n0 == 0) {
        if (q.D) y = fmaf(q.D[d], x, y);
        if (q.z) {
            const float z = (float)((const T*)q.z)[s * q.ldz + d];
            y *= z * sigmoidf(z);
        }
        ((T*)q.y)[s * q.ldy + d] = (T)y;
    }
}

// ------------------------------------------------------------------ host side

struct Plan { int P, K, NP, CB, VE, tiles, blocks, chunks, slots; };

Plan scan_plan(int64_t T, int S, int D, int G, int N) {
    Plan p;
    p.P = N <= 16 ? 4 : (N <= 32 ? 8 : 16);
    p.K = N <= 4 ? 1 : (N <= 8 ? 2 : 4);
    p.NP = p.P * p.K;
    p.CB = 256 / p.P;
    p.VE = p.CB >= 64 ? 4 : p.CB / 16;
    p.tiles = (D / G + p.CB - 1) / p.CB;
    p.blocks = p.tiles * G;
    // Chunks: the two-pass form computes every exponential twice, so it is taken only where workgroups of whole sequences
    // leave more than half of the chip idle (fewer than two for every CU), and a chunk has four tiles at least on average.
    const int64_t whole = (int64_t)p.blocks * (S > 0 ? S : 1), tiles = (T + TILE - 1) / TILE;
    int64_t c = 1;
    if (whole < 512) c = (1024 + whole - 1) / whole;
    const int64_t most = tiles / (4 * (int64_t)(S > 0 ? S : 1));
    if (c > most) c = most;
    if (opt(OPT_SCAN_CHUNKS) >= 1) c = opt(OPT_SCAN_CHUNKS);
    p.chunks = (int)(c < 1 ? 1 : (c > MAX_CHUNKS ? MAX_CHUNKS : c));
    // Workgroups along the sequences: each leaves one partial sum of the parameters' gradients, so no more than fill the chip
    int64_t slots = (4096 + p.blocks * p.chunks - 1) / (p.blocks * p.chunks);
    if (slots > S) slots = S;
    p.slots = (int)(slots < 1 ? 1 : slots);
    return p;
}

size_t chunk_floats(const Plan& p, int S, int D) { return p.chunks > 1 ? (size_t)(p.chunks - 1) * S * D * (p.NP + 1) : 0; }
size_t floats16(size_t n) { return (n + 3) / 4 * 4; }

bool scan_sizes_ok(int64_t T, int S, int D, int G, int N, const void* off) {
    if (T < 0 || T > INT32_MAX - 64 || S < 0 || S > (1 << 24) || D < 1 || D > (1 << 21) || G < 1 || D % G || N < 1 || N > 64) return false;
    return off || S == 0 ? (S > 0 || T == 0) : T % S == 0;
}

int scan_operands(const psvae_scan* a) {
    if (!a) return PSVAE_E_NULL;
    if (!dtype_known(a->dtype) || !scan_sizes_ok(a->T, a->S, a->D, a->G, a->N, a->seq_off)) return PSVAE_E_SHAPE;
    if (a->flags & ~(PSVAE_SEQ_SOFTPLUS | PSVAE_SEQ_ZERO_OUTSIDE)) return PSVAE_E_SHAPE;
    if (a->T > 0 && (!a->x || !a->dt || !a->B || !a->C)) return PSVAE_E_NULL;
    if (!a->A) return PSVAE_E_NULL;
    if (a->ldx < a->D || a->lddt < a->D || a->ldb < (int64_t)a->G * a->N || a->ldc < (int64_t)a->G * a->N || (a->z && a->ldz < a->D)) return PSVAE_E_SHAPE;
    return 0;
}

Scan scan_args(const psvae_scan* a, const Plan& p) {
    Scan q{};
    q.x = a->x; q.dt = a->dt; q.B = a->B; q.C = a->C; q.z = a->z;
    q.ldx = a->ldx; q.lddt = a->lddt; q.ldb = a->ldb; q.ldc = a->ldc; q.ldz = a->ldz;
    q.A = a->A; q.D = a->skip; q.bias = a->dt_bias; q.h0 = a->h0; q.off = a->seq_off;
    q.T = (int)a->T; q.S = a->S; q.Dn = a->D; q.G = a->G; q.N = a->N; q.chunks = p.chunks;
    q.softplus = (a->flags & PSVAE_SEQ_SOFTPLUS) != 0;
    q.zero_outside = a->seq_off && (a->flags & PSVAE_SEQ_ZERO_OUTSIDE);
    q.vec = a->D / a->G % p.VE == 0 && rows_vec(a->x, a->ldx, p.VE, a->dtype) && rows_vec(a->dt, a->lddt, p.VE, a->dtype) &&
            rows_vec(a->z, a->ldz, p.VE, a->dtype);
    return q;
}

template <class T, int P, int K> int fwd_run(hipStream_t s, const Scan& q, const Plan& p) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<T, P, K, true>), dim3(p.blocks, p.slots, p.chunks - 1), dim3(256), 0, s, q);
        PSVAE_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, P, K, false>), dim3(p.blocks, p.slots, p.chunks + q.zero_outside), dim3(256), 0, s, q);
    PSVAE_LAUNCH_CHECK();
    return 0;
}
template <class T, int P, int K> int bwd_run(hipStream_t s, const Scan& q, const Plan& p) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_bwd_kernel<T, P, K, true>), dim3(p.blocks, p.slots, p.chunks - 1), dim3(256), 0, s, q);
        PSVAE_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, P, K, false>), dim3(p.blocks, p.slots, p.chunks + q.zero_outside), dim3(256), 0, s, q);
    PSVAE_LAUNCH_CHECK();
    return 0;
}
template <class T, int P, int K> int step_run(hipStream_t s, const Scan& q, const Plan&) {
    const int64_t lanes = (int64_t)q.S * q.Dn * P;
    const int vec = q.N == P * K && rows_vec(q.A, 0, K, PSVAE_F32) && rows_vec(q.h0, 0, K, PSVAE_F32) && rows_vec(q.hT, 0, K, PSVAE_F32);
    hipLaunchKernelGGL((scan_step_kernel<T, P, K>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, s, q, vec);
    PSVAE_LAUNCH_CHECK();
    return 0;
}
// Runs NAME<T, P, K> for the call's type and plan.
#define PSVAE_SCAN_RUN(NAME, dtype, s, q, p)                           \
    [&]() -> int {                                                     \
        PSVAE_BY_TYPE(dtype, T, {                                      \
            if ((p).P == 16) return NAME<T, 16, 4>(s, q, p);           \
            if ((p).P == 8) return NAME<T, 8, 4>(s, q, p);             \
            if ((p).K == 4) return NAME<T, 4, 4>(s, q, p);             \
            if ((p).K == 2) return NAME<T, 4, 2>(s, q, p);             \
            return NAME<T, 4, 1>(s, q, p);                             \
        });                                                            \
    }()

// Where the parts of a backward call's scratch lie (in floats).
struct BwdScratch { size_t bc, a, d, chunk, total; };
BwdScratch bwd_scratch(const Plan& p, int64_t T, int S, int D, int G) {
    BwdScratch o;
    const size_t parts = (size_t)p.slots * p.chunks;
    o.bc = 0;
    o.a = o.bc + floats16((size_t)p.tiles * T * G * 2 * p.NP);
    o.d = o.a + floats16(parts * D * p.NP);
    o.chunk = o.d + floats16(parts * 2 * D);
    o.total = o.chunk + chunk_floats(p, S, D);
    return o;
}

}  // namespace

extern "C" size_t psvae_selective_scan_scratch_bytes(int64_t T, int S, int D, int G, int N, int backward) {
    if (!scan_sizes_ok(T, S, D, G, N, &T)) return 0;
    const Plan p = scan_plan(T, S, D, G, N);
    return (backward ? bwd_scratch(p, T, S, D, G).total : chunk_floats(p, S, D)) * sizeof(float);
}

extern "C" size_t psvae_selective_scan_saved_bytes(int64_t T, int S, int D, int G, int N) {
    if (!scan_sizes_ok(T, S, D, G, N, &T)) return 0;
    return (size_t)(T / TILE + S) * D * scan_plan(T, S, D, G, N).NP * sizeof(float);
}

extern "C" int psvae_selective_scan_forward(const psvae_scan* a, void* y, int64_t ldy, float* hT, void* saved, void* scratch,
                                            size_t scratch_bytes, void* stream) {
    PSVAE_TRY(scan_operands(a));
    if (ldy < a->D) return PSVAE_E_SHAPE;
    if (a->T > 0 && !y) return PSVAE_E_NULL;
    if (a->S == 0) return 0;
    const Plan p = scan_plan(a->T, a->S, a->D, a->G, a->N);
    Scan q = scan_args(a, p);
    if (p.chunks > 1) {
        if (!scratch) return PSVAE_E_NULL;
        if (scratch_bytes < chunk_floats(p, a->S, a->D) * sizeof(float)) return PSVAE_E_WORKSPACE;
    }
    if ((saved && !aligned16(saved)) || (scratch && !aligned16(scratch))) return PSVAE_E_ALIGN;
    q.y = y; q.ldy = ldy; q.hT = hT; q.kept = (float*)saved;
    q.chunk_h = (float*)scratch;
    q.chunk_s = q.chunk_h + (size_t)(p.chunks - 1) * a->S * a->D * p.NP;
    q.vec = q.vec && rows_vec(y, ldy, p.VE, a->dtype);
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SCAN_FWD, (double)a->T * a->D * (a->z ? 4 : 3) * dtype_bytes(a->dtype));
    return PSVAE_SCAN_RUN(fwd_run, a->dtype, s, q, p);
}

extern "C" int psvae_selective_scan_backward(const psvae_scan* a, const void* saved, const void* dy, int64_t lddy, const float* dhT,
                                             const psvae_scan_grads* g, void* scratch, size_t scratch_bytes, void* stream) {
    PSVAE_TRY(scan_operands(a));
    if (!g) return PSVAE_E_NULL;
    if (a->T > 0 && (!saved || !dy || !g->dx || !g->ddt || !g->dB || !g->dC || (a->z && !g->dz))) return PSVAE_E_NULL;
    if (!g->dA || !scratch) return PSVAE_E_NULL;
    if (lddy < a->D || g->lddx < a->D || g->ldddt < a->D || (a->z && g->lddz < a->D) || g->lddb < (int64_t)a->G * a->N || g->lddc < (int64_t)a->G * a->N) return PSVAE_E_SHAPE;
    const Plan p = scan_plan(a->T, a->S, a->D, a->G, a->N);
    Scan q = scan_args(a, p);
    const BwdScratch o = bwd_scratch(p, a->T, a->S, a->D, a->G);
    if (!aligned16(scratch) || (saved && !aligned16(saved))) return PSVAE_E_ALIGN;
    if (scratch_bytes < o.total * sizeof(float)) return PSVAE_E_WORKSPACE;
    float* base = (float*)scratch;
    q.dy = dy; q.lddy = lddy; q.dhT = dhT; q.kept = (float*)saved;
    q.dx = g->dx; q.lddx = g->lddx; q.ddt = g->ddt; q.ldddt = g->ldddt; q.dz = g->dz; q.lddz = g->lddz; q.dh0 = g->dh0;
    q.part_bc = base + o.bc; q.part_a = base + o.a; q.part_d = base + o.d;
    q.chunk_h = base + o.chunk;
    q.chunk_s = q.chunk_h + (size_t)(p.chunks - 1) * a->S * a->D * p.NP;
    q.vec = q.vec && rows_vec(dy, lddy, p.VE, a->dtype) && rows_vec(g->dx, g->lddx, p.VE, a->dtype) &&
            rows_vec(g->ddt, g->ldddt, p.VE, a->dtype) && (!a->z || rows_vec(g->dz, g->lddz, p.VE, a->dtype));
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SCAN_BWD, (double)a->T * a->D * (a->z ? 7 : 5) * dtype_bytes(a->dtype));
    if (a->S > 0) {
        const int rc = PSVAE_SCAN_RUN(bwd_run, a->dtype, s, q, p);
        PSVAE_TRY(rc);
    }
    ScanJoin j{q.part_bc, q.part_a, q.part_d, g->dB, g->dC, g->lddb, g->lddc, g->dA, g->d_skip, g->d_dt_bias, a->seq_off,
               q.T, a->S, a->D, a->G, a->N, p.NP, p.tiles, a->S > 0 ? p.slots * p.chunks : 0, 0, 0, q.zero_outside};
    const int64_t cols = (int64_t)a->T * a->G * 2 * p.NP;
    j.blocks_bc = (int)((cols + 255) / 256 < 8192 ? (cols + 255) / 256 : 8192);
    j.blocks_a = (int)(((int64_t)a->D * a->N + 255) / 256);
    PSVAE_BY_TYPE(a->dtype, T, {
        hipLaunchKernelGGL((scan_join_kernel<T>), dim3(j.blocks_bc + j.blocks_a + (a->D + 255) / 256), dim3(256), 0, s, j);
    });
    PSVAE_LAUNCH_CHECK();
    return 0;
}

extern "C" int psvae_selective_scan_step(const psvae_scan* a, void* y, int64_t ldy, float* hT, void* stream) {
    PSVAE_TRY(scan_operands(a));
    if (ldy < a->D || a->T != a->S || a->seq_off || (a->flags & PSVAE_SEQ_ZERO_OUTSIDE)) return PSVAE_E_SHAPE;
    if (a->S == 0) return 0;
    if (!y || !a->h0 || !hT) return PSVAE_E_NULL;
    const Plan p = scan_plan(a->T, a->S, a->D, a->G, a->N);
    Scan q = scan_args(a, p);
    q.y = y; q.ldy = ldy; q.hT = hT;
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SCAN_FWD, (double)a->S * a->D * a->N * 8);
    return PSVAE_SCAN_RUN(step_run, a->dtype, s, q, p);
}
