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
// What bounds it: the vector units.  Every (row, channel, state) has a decay of its own, so no matrix product appears (and
// forming delta A with the 4 x 4 x 1 matrix instruction cost more in waits than it saved: 159 against 146 us): 3 vector
// operations and one exponential, which takes twice as long, for the state, one for y; backward 15 and one exponential.
// With the sums, softplus and gates a forward pass issues 8.3 vector instructions a cell, a backward pass 25, and counters
// show the vector units busy 94 % and 86 % of the time.  Measured at 16 states, bf16, 32 x 512 x 2048 (0.54 G cells): forward
// 142 us (1.9 TB/s of its 4 operands), backward 464 us.  HBM alone would take 54 us forward, 108 where the states are kept for
// a backward pass (268 MB more; the kernel takes 155 us then), and 162 us backward (805 MB: 4 operands, the kept states, 3
// gradients and the parts of dB and dC).
//
// Layout: P lanes side by side share a channel and hold K states each (P K = the states rounded up: 4 x 1, 4 x 2, 4 x 4,
// 8 x 4, 16 x 4), a workgroup of 256 lanes takes 256 / P channels of one group and one sequence and walks the time axis in
// tiles of 16 rows: rows are read as vectors one tile ahead, brought to (delta, delta x, dyp) once, and passed to the lanes
// through LDS.  With the states of a channel spread over P lanes, the sum over the states costs log2 P steps inside the
// lanes' own row (data-parallel moves, no LDS), and four times the workgroups of a lane-per-channel layout fill the chip.
// (8 x 2 and 16 x 1 for 16 states were slower wherever 4 x 4 was cut into pieces instead: 612 and 807 against 585 us for
// the backward pass of 8 x 2048 x 2048.)  dB and dC are sums over channels: a fold over the halves of the wave and of its
// halves (permlane swaps, which leave every lane half as many sums), then inside rows of 16 lanes, the waves through LDS and
// the workgroups through memory, in a fixed order.  (The second fold and the rest as 16 x 16 x 4 matrix products with columns
// of ones, whose results nothing waits for: 573 against 470 us for the backward pass of 32 x 512 x 2048, as the fp32 matrix
// instruction takes more than the vector operations it replaces.)
// Few sequences: the time axis is cut into pieces ("chunks", every sequence into as many), a first pass finds each one's end
// state from zero, and the second, which makes the outputs, starts from the join of the pieces in front of it.
#include "seq_device.h"

namespace {

constexpr int TILE = 16;         // rows a tile
constexpr int HALF = 8;          // rows the lanes work through at a time; the distance of the states kept for the backward pass
constexpr int PITCH = 20;        // floats of LDS a channel's tile of rows takes: 16-byte rows that 16 channels spread over all banks
constexpr int MAX_CHUNKS = 64;
constexpr float LOG2E = 1.44269504088896340736f, LOG2E_LOW = 1.92596299112661747e-8f, LN2 = 0.69314718055994530942f;

// Device pointers and sizes of one call; `T` rows, `S` sequences, `D` channels in `G` groups, `N` states.
struct Scan {
    const void *x, *dt, *B, *C, *z, *dy;
    int64_t ldx, lddt, ldb, ldc, ldz, lddy;
    const float *A, *D, *bias, *h0;
    void *y, *dx, *ddt, *dz;
    int64_t ldy;
    float *hT, *kept;
    const float* dhT;
    float* dh0;
    float *part_bc, *part_a, *part_d;      // dB/dC [tiles of a group][T][G][2 NP], dA [slots * chunks][D][NP], dD/dbias [slots * chunks][2][D]
    float *chunk_h, *chunk_s;              // [chunks][S][D][NP] end state (or carry) of a chunk from zero, [chunks][S][D] its sum of delta
    const int32_t* off;
    int T, S, Dn, G, N, chunks, softplus, zero_outside, vec;
};

// softplus and its slope, the sigmoid, without branches.  exp(v) = 2^t (1 + r ln 2) with t = v log2 e as rounded and r what
// the rounding (and the constant's) left out; log(1 + e) = log(u) + (e - (u - 1)) / u with u = 1 + e as rounded.  From 20
// on exp(-v) is below half a step of v (and a NaN goes the same way); exp(-100) is zero beside anything.
__device__ __forceinline__ float softplus_slope(float v, float& slope) {
    const float w = __builtin_amdgcn_fmed3f(v, -100.f, 100.f), t = w * LOG2E, r = fmaf(w, LOG2E_LOW, fmaf(w, LOG2E, -t));
    const float e0 = __builtin_amdgcn_exp2f(t), e = fmaf(e0, r * LN2, e0);
    const float u = 1.f + e, inv = __builtin_amdgcn_rcpf(u);
    slope = v > 20.f ? 1.f : e * inv;
    return v <= 20.f ? fmaf(e - (u - 1.f), inv, __builtin_amdgcn_logf(u) * LN2) : v;
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

// Row of `kept` for the first half of tile i of a sequence that begins at row `begin`: sequences that share eight rows are
// kept apart by their number, and the last index is below T / 8 + S.
__device__ __forceinline__ int64_t kept_row(int begin, int s, int tile) { return (int64_t)(begin / HALF) + s + tile * (TILE / HALF); }

// Where a channel's four rows 4 q .. lie in its PITCH floats of LDS: quarter q changes places by the channel's sixteenth, so
// that the 16 lanes that write one row of 64 (or 32) channels reach as many bank groups.
__device__ __forceinline__ int quarter(int q, int ch) { return 4 * (q ^ (ch >> 4 & 3)); }

// V elements of a row, zeros from the n-th on.
template <bool VEC, class T, int V> __device__ __forceinline__ void fetch_row(const T* p, int n, Raw<T, V>& out) {
#pragma unroll
    for (int i = 0; i < V; ++i) out.v[i] = (T)0.f;
    if constexpr (VEC) {
        if (n > 0) out.load(p);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) out.v[i] = p[i];
    }
}
template <bool VEC, class T, int V> __device__ __forceinline__ void store_row(T* p, int n, const float (&in)[V]) {
    if constexpr (VEC) {
        if (n > 0) store_vec<V>(p, in);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (T)in[i];
    }
}

// A tile's B or C: a lane has NBC states of one row (with 8 or 4 states some lanes have none).
template <class T, int P, int K, bool VEC> struct TileBC {
    static constexpr int NP = P * K, V = Shape<P, K>::NBC;
    Raw<T, V> v;
    static __device__ __forceinline__ int row() { return threadIdx.x * V / NP; }
    static __device__ __forceinline__ int state() { return threadIdx.x * V % NP; }
    __device__ __forceinline__ void fetch(const T* p, int N, int rows) { fetch_row<VEC>(p, row() < rows ? N - state() : 0, v); }   // p: the lane's place
    __device__ __forceinline__ void put(float* tile) const {
        if (TILE * NP < 256 && (int)threadIdx.x >= TILE * NP) return;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = v[i];
        store_vec<V>(tile + threadIdx.x * V, f);
    }
};

// A log2 e, kept finite: rows behind a sequence's end have delta = 0, and 0 x infinity would not leave their states alone.
template <int K> __device__ __forceinline__ void scale_rates(float (&A)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        A[k] *= LOG2E;
        A[k] = A[k] < -3e38f ? -3e38f : (A[k] > 3e38f ? 3e38f : A[k]);
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

// A state behind a piece: h 2^(2 v) + e, the decay in two halves as it may leave fp32's range where the product does not: h is
// zero in front of the first input whatever the rates and steps behind it sum up to (infinity times zero would be NaN), and
// what is left of a large h that fades below 2^-126 of itself is still a number.  From v = 127 on every normal h
// becomes infinite, and zero stays zero.
__device__ __forceinline__ float join(float h, float v, float e) {
    const float half = __builtin_amdgcn_exp2f(fminf(v, 127.f));
    return fmaf(half * h, half, e);
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
template <class T, int P, int K, bool VEC, bool ENDS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(Scan q) {
    using Sh = Shape<P, K>;
    constexpr int NP = Sh::NP, VE = Sh::VE, U = sizeof(T);
    // LDS, one block of constant parts (so that an address is a lane's base and an immediate): delta, delta x and y of the
    // tile by channel, B and C by row
    constexpr int AREA = Sh::CB * PITCH, DELTA = 0, DX = AREA, BT = 2 * AREA, CT = BT + TILE * NP, YT = CT + (ENDS ? 0 : TILE * NP);
    __shared__ __attribute__((aligned(16))) float lds[YT + (ENDS ? 0 : AREA)];
    const Place w = place<P, K>(q);
    const int chunk = blockIdx.z;
    if (!ENDS && chunk == q.chunks) { zero_rows<T>(q.y, q.ldy, q, w, gridDim.y); return; }
    const int r = threadIdx.x / Sh::TPR, c = threadIdx.x % Sh::TPR * VE;       // staging: row and first channel of this lane
    const int ch = threadIdx.x / P, n0 = threadIdx.x % P * K;                   // scanning: channel and first state
    const int left = w.nc - c, d = w.c0 + ch;
    float *const at_row = lds + c * PITCH + quarter(r >> 2, c) + (r & 3), *const at_n = lds + n0;
    float *const at_q[4] = {lds + ch * PITCH + quarter(0, ch), lds + ch * PITCH + quarter(1, ch), lds + ch * PITCH + quarter(2, ch),
                            lds + ch * PITCH + quarter(3, ch)};
    const bool live = ch < w.nc, gated = !ENDS && q.z;
    float A2[K], bias[VE], skip[VE];
    load_state<K>(live ? q.A : nullptr, 0, q, d, n0, A2);
    scale_rates<K>(A2);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
        bias[i] = q.bias && i < left ? q.bias[w.c0 + c + i] : 0.f;
        skip[i] = !ENDS && q.D && i < left ? q.D[w.c0 + c + i] : 0.f;
    }
    for (int s = blockIdx.y; s < q.S; s += gridDim.y) {
        const SeqBounds sq = seq_bounds(q.off, s, q.S, q.T);
        const Range tiles = chunk_tiles(sq.end - sq.begin, q.chunks, chunk);
        float h[K], sum = 0.f;
        load_state<K>(!ENDS && live ? q.h0 : nullptr, s, q, d, n0, h);
        if (!ENDS && live)
            for (int i = 0; i < chunk; ++i) {          // join the chunks in front: h = exp(A sum) h + end
                const int64_t row = (int64_t)i * q.S + s;
                const float half_ds = 0.5f * q.chunk_s[row * q.Dn + d];
                const float* e = own_state<K>(q.chunk_h, row, q, NP, d, n0);
#pragma unroll
                for (int k = 0; k < K; ++k) h[k] = join(h[k], half_ds * A2[k], e[k]);
            }
        const int64_t first = sq.begin + (int64_t)tiles.first * TILE, row = first + r, bc_row = first + TileBC<T, P, K, VEC>::row();
        const T *px = (const T*)q.x + row * q.ldx + w.c0 + c, *pt = (const T*)q.dt + row * q.lddt + w.c0 + c,
                *pz = (const T*)q.z + row * q.ldz + w.c0 + c, *pb = (const T*)q.B + bc_row * q.ldb + w.g * q.N + TileBC<T, P, K, VEC>::state(),
                *pc = (const T*)q.C + bc_row * q.ldc + w.g * q.N + TileBC<T, P, K, VEC>::state();
        T* py = (T*)q.y + row * q.ldy + w.c0 + c;
        float* keep = q.kept ? own_state<K>(q.kept, kept_row(sq.begin, s, tiles.first), q, NP, d, n0) : nullptr;
        Raw<T, VE> nx, nt, nz;
        TileBC<T, P, K, VEC> nb, nc;
        auto fetch = [&](int rows) {
            const int n = r < rows ? left : 0;
            fetch_row<VEC>(px, n, nx);
            fetch_row<VEC>(pt, n, nt);
            if (gated) fetch_row<VEC>(pz, n, nz);
            nb.fetch(pb, q.N, rows);
            if (!ENDS) nc.fetch(pc, q.N, rows);
            px += TILE * q.ldx; pt += TILE * q.lddt; pz += TILE * q.ldz; pb += TILE * q.ldb; pc += TILE * q.ldc;
        };
        int remain = sq.end - (int)first;               // rows from this tile's first to the sequence's end
        if (tiles.first < tiles.last) fetch(min(TILE, remain));
        for (int tile = tiles.first; tile < tiles.last; ++tile, remain -= TILE) {
            const int rows = min(TILE, remain), n = r < rows ? left : 0;
            float cx[VE], cz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                float v = (float)nt.v[i] + bias[i], slope;
                if (q.softplus) v = softplus_slope(v, slope);
                v = i < n ? v : 0.f;                     // rows behind the end change nothing
                cx[i] = (float)nx.v[i];
                if (gated) cz[i] = (float)nz.v[i];
                at_row[DELTA + i * PITCH] = v;
                at_row[DX + i * PITCH] = v * cx[i];
            }
            nb.put(lds + BT);
            if (!ENDS) nc.put(lds + CT);
            __syncthreads();
            if (tile + 1 < tiles.last) fetch(min(TILE, remain - TILE));
#pragma unroll
            for (int half = 0; half < TILE / HALF; ++half) {
                if (half * HALF >= rows) break;
                if (!ENDS && keep) {
                    if (live) put_state<K>(keep, h);
                    keep += (int64_t)q.Dn * NP;
                }
#pragma unroll
                for (int t4 = half * HALF; t4 < (half + 1) * HALF; t4 += 4) {
                    float dl[4], dx[4], yv[4];
                    lds_load<4>(at_q[t4 / 4] + DELTA, dl);
                    lds_load<4>(at_q[t4 / 4] + DX, dx);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float b[K], cc[K];
                        lds_load<K>(at_n + BT + (t4 + j) * NP, b);
                        if (!ENDS) lds_load<K>(at_n + CT + (t4 + j) * NP, cc);
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            h[k] = fmaf(__builtin_amdgcn_exp2f(dl[j] * A2[k]), h[k], dx[j] * b[k]);
                            if (!ENDS) yv[j] = k ? fmaf(h[k], cc[k], yv[j]) : h[k] * cc[k];
                        }
                        if (ENDS) sum += dl[j];
                        else yv[j] = lanes_add<P>(yv[j]);
                    }
                    if (!ENDS && n0 == 0) *(float4*)(at_q[t4 / 4] + YT) = make_float4(yv[0], yv[1], yv[2], yv[3]);
                }
            }
            __syncthreads();
            if (!ENDS) {
                float o[VE];
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    o[i] = fmaf(skip[i], cx[i], at_row[YT + i * PITCH]);
                    if (gated) o[i] *= cz[i] * sigmoidf(cz[i]);
                }
                store_row<VEC>(py, n, o);
                py += TILE * q.ldy;
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
    }
}

// Backward.  CARRY: only what each chunk passes to the one in front of it, from a zero carry, and its sum of delta.
template <class T, int P, int K, bool VEC, bool CARRY>
__global__ __launch_bounds__(256, CARRY ? 3 : 2) void scan_bwd_kernel(Scan q) {
    using Sh = Shape<P, K>;
    constexpr int NP = Sh::NP, VE = Sh::VE, U = sizeof(T);
    // LDS, one block of constant parts: by channel what its lanes need of the rows (delta, delta x, dyp), what they make of
    // them (sum_n G B, sum_n G a h' A2, sum_n h C) and the slope of softplus; by row B, C and the waves' sums for dB and dC
    constexpr int AREA = Sh::CB * PITCH, DELTA = 0, DY = AREA, CT = 2 * AREA, BT = CT + TILE * NP, DX = BT + TILE * NP, SU = DX + AREA,
                  SV = SU + AREA, SY = SV + AREA, SLOPE = SY + AREA, BC = SLOPE + AREA, BCW = TILE * 2 * NP;
    __shared__ __attribute__((aligned(16))) float lds[CARRY ? BT : BC + 4 * BCW];
    __shared__ float s_bias[Sh::CB], s_skip[Sh::CB];
    const Place w = place<P, K>(q);
    const int chunk = blockIdx.z + (CARRY ? 1 : 0);
    if (!CARRY && chunk == q.chunks) {
        zero_rows<T>(q.dx, q.Dn, q, w, gridDim.y);
        zero_rows<T>(q.ddt, q.Dn, q, w, gridDim.y);
        if (q.z) zero_rows<T>(q.dz, q.Dn, q, w, gridDim.y);
        return;
    }
    const int r = threadIdx.x / Sh::TPR, c = threadIdx.x % Sh::TPR * VE;
    const int ch = threadIdx.x / P, n0 = threadIdx.x % P * K, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int left = w.nc - c, d = w.c0 + ch;
    float *const at_row = lds + c * PITCH + quarter(r >> 2, c) + (r & 3), *const at_n = lds + n0;
    float *const at_q[4] = {lds + ch * PITCH + quarter(0, ch), lds + ch * PITCH + quarter(1, ch), lds + ch * PITCH + quarter(2, ch),
                            lds + ch * PITCH + quarter(3, ch)};
    const int odd = K == 1 ? 0 : lane >> 4 & 1, copy = (lane & 15) / P;       // of the sums for dB and dC, below
    float* const at_bc = lds + (wave * TILE * 2 + copy * 2 + (lane >> 5)) * NP + n0 + odd;
    const bool live = ch < w.nc, gated = q.z;          // lanes without a channel compute with zeros
    float A2[K], dA[K], dD[VE], dbias[VE];
    load_state<K>(live ? q.A : nullptr, 0, q, d, n0, A2);
    scale_rates<K>(A2);
#pragma unroll
    for (int k = 0; k < K; ++k) dA[k] = 0.f;
#pragma unroll
    for (int i = 0; i < VE; ++i) dD[i] = dbias[i] = 0.f;
    for (int i = threadIdx.x; i < Sh::CB; i += 256) {
        s_bias[i] = q.bias && i < w.nc ? q.bias[w.c0 + i] : 0.f;
        s_skip[i] = q.D && i < w.nc ? q.D[w.c0 + i] : 0.f;
    }
    __syncthreads();
    for (int s = blockIdx.y; s < q.S; s += gridDim.y) {
        const SeqBounds sq = seq_bounds(q.off, s, q.S, q.T);
        const Range tiles = chunk_tiles(sq.end - sq.begin, q.chunks, chunk);
        float ag[K], sum = 0.f;                        // ag = a[t+1] G[t+1], the carry from the rows behind
        load_state<K>(!CARRY && live ? q.dhT : nullptr, s, q, d, n0, ag);
        if (!CARRY && live)
            for (int i = q.chunks - 1; i > chunk; --i) {
                const int64_t row = (int64_t)(i - 1) * q.S + s;
                const float half_ds = 0.5f * q.chunk_s[row * q.Dn + d];
                const float* e = own_state<K>(q.chunk_h, row, q, NP, d, n0);
#pragma unroll
                for (int k = 0; k < K; ++k) ag[k] = join(ag[k], half_ds * A2[k], e[k]);
            }
        // Wait for every load (vmcnt 0), dhT's above all: a wait for it inside the tiles would be one for the rows fetched ahead,
        // too.  8 x 2048 x 2048 forward + backward 784 against 793 us without it, 32 x 512 x 2048 621 against 629.
        __builtin_amdgcn_s_waitcnt(0x0f70);
        const int64_t first = sq.begin + (int64_t)(tiles.last - 1) * TILE;     // the last tile's first row
        const int64_t row = first + r, bc_row = first + TileBC<T, P, K, VEC>::row();
        const T *px = (const T*)q.x + row * q.ldx + w.c0 + c, *pt = (const T*)q.dt + row * q.lddt + w.c0 + c,
                *pz = (const T*)q.z + row * q.ldz + w.c0 + c, *pg = (const T*)q.dy + row * q.lddy + w.c0 + c,
                *pb = (const T*)q.B + bc_row * q.ldb + w.g * q.N + TileBC<T, P, K, VEC>::state(),
                *pc = (const T*)q.C + bc_row * q.ldc + w.g * q.N + TileBC<T, P, K, VEC>::state();
        int64_t out = row * q.Dn + w.c0 + c;           // the gradients are contiguous
        const float* keep = CARRY ? nullptr : own_state<K>(q.kept, kept_row(sq.begin, s, tiles.last - 1), q, NP, d, n0);
        float* bc_out = CARRY ? nullptr : q.part_bc + (((int64_t)w.blk * q.T + first) * q.G + w.g) * 2 * NP;
        Raw<T, VE> nx, nt, nz, ng;
        TileBC<T, P, K, VEC> nb, nc;
        float nh[TILE / HALF][K];
        auto fetch = [&](int rows) {
            const int n = r < rows ? left : 0;
            fetch_row<VEC>(pt, n, nt);
            fetch_row<VEC>(pg, n, ng);
            if (gated) fetch_row<VEC>(pz, n, nz);
            nc.fetch(pc, q.N, rows);
            if constexpr (!CARRY) {
                fetch_row<VEC>(px, n, nx);
                nb.fetch(pb, q.N, rows);
#pragma unroll
                for (int half = 0; half < TILE / HALF; ++half) {
#pragma unroll
                    for (int k = 0; k < K; ++k) nh[half][k] = 0.f;
                    if (live && half * HALF < rows)
#pragma unroll
                        for (int k = 0; k < K; ++k) nh[half][k] = keep[(int64_t)half * q.Dn * NP + k];
                }
            }
            pt -= TILE * q.lddt; pg -= TILE * q.lddy; pz -= TILE * q.ldz; pc -= TILE * q.ldc;
            if constexpr (!CARRY) {
                px -= TILE * q.ldx;
                pb -= TILE * q.ldb;
                keep -= (int64_t)q.Dn * NP * (TILE / HALF);
            }
        };
        Raw<T, VE> cx, cz, cg;
        float h[TILE / HALF][K];
        auto stage = [&](int rows) {
            const int n = r < rows ? left : 0;
            cx = nx; cz = nz; cg = ng;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                float v = (float)nt.v[i] + s_bias[c + i], dy = (float)cg.v[i], slope = 1.f;
                if (q.softplus) v = softplus_slope(v, slope);
                v = i < n ? v : 0.f;                     // rows behind the end change nothing
                if (gated) dy *= (float)cz.v[i] * sigmoidf((float)cz.v[i]);
                at_row[DELTA + i * PITCH] = v;
                at_row[DY + i * PITCH] = dy;
                if constexpr (!CARRY) { at_row[DX + i * PITCH] = v * (float)cx.v[i]; at_row[SLOPE + i * PITCH] = slope; }
            }
            if constexpr (!CARRY) nb.put(lds + BT);
            nc.put(lds + CT);
#pragma unroll
            for (int half = 0; half < TILE / HALF; ++half)
#pragma unroll
                for (int k = 0; k < K; ++k) h[half][k] = nh[half][k];
        };
        int rows = sq.end - (int)first;                 // the last tile of the sequence may be short
        rows = min(rows, TILE);
        if (tiles.first < tiles.last) {
            fetch(rows);
            stage(rows);
        }
        for (int tile = tiles.last - 1; tile >= tiles.first; --tile, rows = TILE) {
            const int n = r < rows ? left : 0;
            __syncthreads();
            if (tile > tiles.first) fetch(TILE);
            if constexpr (CARRY) {
#pragma unroll
                for (int half = TILE / HALF - 1; half >= 0; --half) {
                    if (half * HALF >= rows) continue;
#pragma unroll
                    for (int t4 = (half + 1) * HALF - 4; t4 >= half * HALF; t4 -= 4) {
                        float dl[4], dy[4];
                        lds_load<4>(at_q[t4 / 4] + DELTA, dl);
                        lds_load<4>(at_q[t4 / 4] + DY, dy);
#pragma unroll
                        for (int j = 3; j >= 0; --j) {
                            float cc[K];
                            lds_load<K>(at_n + CT + (t4 + j) * NP, cc);
                            sum += dl[j];
#pragma unroll
                            for (int k = 0; k < K; ++k) ag[k] = __builtin_amdgcn_exp2f(dl[j] * A2[k]) * fmaf(dy[j], cc[k], ag[k]);
                        }
                    }
                }
                __syncthreads();
                if (tile > tiles.first) stage(TILE);
            } else {
                float dAt[K];
#pragma unroll
                for (int k = 0; k < K; ++k) dAt[k] = 0.f;
#pragma unroll
                for (int half = TILE / HALF - 1; half >= 0; --half) {
                    if (half * HALF >= rows) continue;
                    // forward over eight rows from the kept state: the decays a and the decayed states a h[t-1] stay in registers
                    float a[HALF][K], p[HALF][K];
#pragma unroll
                    for (int t4 = 0; t4 < HALF; t4 += 4) {
                        float dl[4], dx[4];
                        lds_load<4>(at_q[half * 2 + t4 / 4] + DELTA, dl);
                        lds_load<4>(at_q[half * 2 + t4 / 4] + DX, dx);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float b[K];
                            lds_load<K>(at_n + BT + (half * HALF + t4 + j) * NP, b);
#pragma unroll
                            for (int k = 0; k < K; ++k) {
                                a[t4 + j][k] = __builtin_amdgcn_exp2f(dl[j] * A2[k]);
                                p[t4 + j][k] = a[t4 + j][k] * h[half][k];
                                h[half][k] = fmaf(dx[j], b[k], p[t4 + j][k]);
                            }
                        }
                    }
#pragma unroll
                    for (int t4 = HALF - 4; t4 >= 0; t4 -= 4) {
                        float *const rows4 = at_q[half * 2 + t4 / 4];
                        float dl[4], dx[4], dy[4], su[4], sv[4], sy[4], e[4][K > 1 ? K / 2 : 1];
                        lds_load<4>(rows4 + DELTA, dl);
                        lds_load<4>(rows4 + DX, dx);
                        lds_load<4>(rows4 + DY, dy);
#pragma unroll
                        for (int j = 3; j >= 0; --j) {
                            const int t = half * HALF + t4 + j;
                            float b[K], cc[K], db[K], dc[K];
                            lds_load<K>(at_n + BT + t * NP, b);
                            lds_load<K>(at_n + CT + t * NP, cc);
#pragma unroll
                            for (int k = 0; k < K; ++k) {
                                const float g = fmaf(dy[j], cc[k], ag[k]);
                                const float hk = fmaf(dx[j], b[k], p[t4 + j][k]);
                                const float v = g * p[t4 + j][k];
                                dc[k] = dy[j] * hk;
                                db[k] = g * dx[j];
                                su[j] = k ? fmaf(g, b[k], su[j]) : g * b[k];
                                sv[j] = k ? fmaf(v, A2[k], sv[j]) : v * A2[k];
                                sy[j] = k ? fmaf(hk, cc[k], sy[j]) : hk * cc[k];
                                dAt[k] = fmaf(v, dl[j], dAt[k]);
                                ag[k] = a[t4 + j][k] * g;
                            }
                            su[j] = lanes_add<P>(su[j]);
                            sv[j] = lanes_add<P>(sv[j]);
                            sy[j] = lanes_add<P>(sy[j]);
                            // sums over this wave's channels: rows 0, 1 of 16 lanes get dB of even, odd k; rows 2, 3 dC
                            float f[K];
#pragma unroll
                            for (int k = 0; k < K; ++k) f[k] = fold32(db[k], dc[k]);
                            if constexpr (K == 1) e[j][0] = stride_add<P>(fold16(f[0], f[0]));
                            else
#pragma unroll
                                for (int k = 0; k < K; k += 2) e[j][k / 2] = stride_add<P>(fold16(f[k], f[k + 1]));
                        }
                        // the lanes of a row that hold the same states write one of the four steps each
                        constexpr int COPIES = P < 16 ? 16 / P : 1;
#pragma unroll
                        for (int k = 0; k < (K > 1 ? K / 2 : 1); ++k)
#pragma unroll
                            for (int j0 = 0; j0 < 4; j0 += COPIES) {
                                float v = e[j0][k];
#pragma unroll
                                for (int j = 1; j < COPIES; ++j) v = copy == j ? e[j0 + j][k] : v;
                                at_bc[BC + (half * HALF + t4 + j0) * 2 * NP + 2 * k] = v;
                            }
                        if (n0 == 0) {
                            *(float4*)(rows4 + SU) = make_float4(su[0], su[1], su[2], su[3]);
                            *(float4*)(rows4 + SV) = make_float4(sv[0], sv[1], sv[2], sv[3]);
                            *(float4*)(rows4 + SY) = make_float4(sy[0], sy[1], sy[2], sy[3]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < K; ++k) dA[k] += dAt[k];     // tile sums first: a long sum of short ones rounds less
                __syncthreads();
                float odx[VE], odt[VE], odz[VE];
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                        const float x = (float)cx.v[i], su = at_row[SU + i * PITCH], dyp = at_row[DY + i * PITCH], skip = s_skip[c + i];
                    if (gated) {
                        const float z = (float)cz.v[i], sg = sigmoidf(z);
                        odz[i] = (float)cg.v[i] * fmaf(skip, x, at_row[SY + i * PITCH]) * sg * fmaf(z, 1.f - sg, 1.f);
                    }
                    odx[i] = fmaf(su, at_row[DELTA + i * PITCH], skip * dyp);
                    odt[i] = i < n ? fmaf(su, x, at_row[SV + i * PITCH] * LN2) * at_row[SLOPE + i * PITCH] : 0.f;   // rows behind the end hold no sums
                    dD[i] = fmaf(dyp, x, dD[i]);
                    dbias[i] += odt[i];
                }
                constexpr int BCN = (BCW + 255) / 256;
                float bc[BCN];
#pragma unroll
                for (int j = 0; j < BCN; ++j) {
                    const float* p = lds + BC + j * 256 + threadIdx.x;
                    bc[j] = j * 256 + 255 < BCW || j * 256 + (int)threadIdx.x < BCW ? (p[0] + p[BCW]) + (p[2 * BCW] + p[3 * BCW]) : 0.f;
                }
                __syncthreads();
                // the next tile first: a wait for its rows behind these stores would be one for the stores, too
                if (tile > tiles.first) stage(TILE);
                store_row<VEC>((T*)q.dx + out, n, odx);
                store_row<VEC>((T*)q.ddt + out, n, odt);
                if (gated) store_row<VEC>((T*)q.dz + out, n, odz);
                out -= (int64_t)TILE * q.Dn;
#pragma unroll
                for (int j = 0; j < BCN; ++j) {
                    const int e = j * 256 + threadIdx.x;
                    if (e < rows * 2 * NP) bc_out[(int64_t)(e / (2 * NP)) * q.G * 2 * NP + e % (2 * NP)] = bc[j];
                }
                bc_out -= (int64_t)q.G * 2 * NP * TILE;
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
        for (int i = 0; i < VE; ++i) { at_row[DELTA + i * PITCH] = dD[i]; at_row[DY + i * PITCH] = dbias[i]; }
        __syncthreads();
        for (int i = threadIdx.x; i < w.nc; i += 256) {
            float u = 0.f, v = 0.f;
#pragma unroll
            for (int k = 0; k < TILE; ++k) { u += lds[DELTA + i * PITCH + k]; v += lds[DY + i * PITCH + k]; }
            q.part_d[slot * 2 * q.Dn + w.c0 + i] = u;
            q.part_d[slot * 2 * q.Dn + q.Dn + w.c0 + i] = v;
        }
    }
}

// The sums over workgroups: dB and dC over the channel tiles of a group, dA / dD / ddt_bias over slots and chunks.
struct ScanJoin {
    const float *part_bc, *part_a, *part_d;
    void *dB, *dC;
    float *dA, *dD, *dbias;
    const int32_t* off;
    int T, S, Dn, G, N, NP, tiles, parts, blocks_bc, blocks_a, zero_outside, vec;
};
// Sum of column `col` over `parts` rows `step` floats apart by the four quarters of the workgroup, 64 columns side by side;
// the first quarter gets it.
__device__ __forceinline__ float parts_sum(const float* p, int parts, int64_t step, bool inside, float (*red)[64]) {
    const int quarter = threadIdx.x >> 6;
    float s = 0.f;
    if (inside)
#pragma unroll 8
        for (int i = quarter; i < parts; i += 4) s += p[i * step];
    red[quarter][threadIdx.x & 63] = s;
    __syncthreads();
    return (red[0][threadIdx.x & 63] + red[1][threadIdx.x & 63]) + (red[2][threadIdx.x & 63] + red[3][threadIdx.x & 63]);
}
template <class T> __global__ __launch_bounds__(256) void scan_join_kernel(ScanJoin q) {
    __shared__ float red[4][64];
    int blk = blockIdx.x;
    if (blk < q.blocks_bc) {                            // four states of a row at a time
        const int64_t cols = (int64_t)q.T * q.G * 2 * q.NP;
        int begin = 0, end = q.T;                       // rows that a sequence holds
        if (q.off) {
            begin = min(max(q.off[0], 0), q.T);
            end = min(max(q.off[q.S], begin), q.T);
        }
        for (int64_t i = ((int64_t)blk * 256 + threadIdx.x) * 4; i < cols; i += (int64_t)q.blocks_bc * 1024) {
            const int at = (int)(i % (2 * q.NP)), isC = at >= q.NP, n = at - isC * q.NP;
            const int64_t rg = i / (2 * q.NP), row = rg / q.G;
            if (n >= q.N) continue;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row >= begin && row < end) {
#pragma unroll 8
                for (int p = 0; p < q.tiles; ++p) {
                    const float4 v = *(const float4*)(q.part_bc + (int64_t)p * cols + i);
                    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
                }
            } else if (!q.zero_outside) {
                continue;
            }
            const float o[4] = {s.x, s.y, s.z, s.w};
            store_some<4>((T*)(isC ? q.dC : q.dB) + rg * q.N + n, q.N - n, q.vec, o);
        }
        return;
    }
    blk -= q.blocks_bc;
    const int lane = threadIdx.x & 63;
    if (blk < q.blocks_a) {
        const int64_t i = (int64_t)blk * 64 + lane, all = (int64_t)q.Dn * q.N;
        const float s = parts_sum(q.part_a + i / q.N * q.NP + i % q.N, q.parts, (int64_t)q.Dn * q.NP, i < all, red);
        if (threadIdx.x < 64 && i < all) q.dA[i] = s;
        return;
    }
    blk -= q.blocks_a;
    const int i = blk * 64 + lane;                      // [2][D]: dD, then ddt_bias
    const float s = parts_sum(q.part_d + i, q.parts, 2 * (int64_t)q.Dn, i < 2 * q.Dn, red);
    float* out = i < q.Dn ? q.dD : q.dbias;
    if (threadIdx.x < 64 && i < 2 * q.Dn && out) out[i < q.Dn ? i : i - q.Dn] = s;
}

// One token for each of S sequences: bound by the states, read and written once.  P lanes a channel as above; a lane takes
// its channel in R sequences, whose states it has all in flight at once, and has them to itself, so `hT` may be `h0`.
template <class T, int P, int K, int R> __global__ __launch_bounds__(256) void scan_step_kernel(Scan q, int vec_state) {
    const int wide = (q.Dn * P + 255) / 256;           // workgroups side by side over the channels
    const int d = (blockIdx.x % wide * 256 + threadIdx.x) / P, n0 = threadIdx.x % P * K;
    const int s0 = blockIdx.x / wide * R;
    if (d >= q.Dn) return;                             // whole groups of P lanes
    const int g = d / (q.Dn / q.G);
    float h[R][K], A[K], x[R], v[R], z[R], b[R][K], c[R][K];
    const float bias = q.bias ? q.bias[d] : 0.f, skip = q.D ? q.D[d] : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int s = min(s0 + i, q.S - 1);
        if (vec_state) load_vec<K>(q.h0 + ((int64_t)s * q.Dn + d) * q.N + n0, h[i]);
        else load_state<K>(q.h0, s, q, d, n0, h[i]);
        x[i] = (float)((const T*)q.x)[s * q.ldx + d];
        v[i] = (float)((const T*)q.dt)[s * q.lddt + d] + bias;
        z[i] = q.z ? (float)((const T*)q.z)[s * q.ldz + d] : 0.f;
        load_some<K>((const T*)q.B + s * q.ldb + g * q.N + n0, q.N - n0, q.vec, b[i]);
        load_some<K>((const T*)q.C + s * q.ldc + g * q.N + n0, q.N - n0, q.vec, c[i]);
    }
    if (vec_state) load_vec<K>(q.A + (int64_t)d * q.N + n0, A);
    else load_state<K>(q.A, 0, q, d, n0, A);
    scale_rates<K>(A);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int s = s0 + i;
        if (s >= q.S) return;
        float delta = v[i], slope, y = 0.f;
        if (q.softplus) delta = softplus_slope(v[i], slope);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            h[i][k] = fmaf(__builtin_amdgcn_exp2f(delta * A[k]), h[i][k], delta * x[i] * b[i][k]);
            if (n0 + k < q.N) y = fmaf(h[i][k], c[i][k], y);
        }
        y = lanes_add<P>(y);
        if (vec_state) {
            // past the caches, which the states of a serving batch outgrow: 256 x 4096 in place 28.0 -> 26.5 us, 512 x 4096
            // 51.5 -> 48.4 (loads past them, too: 30.5 and 57.4, the next step finds less there)
            typename VecOf<float, K>::type v4;
#pragma unroll
            for (int k = 0; k < K; ++k) v4[k] = h[i][k];
            __builtin_nontemporal_store(v4, (typename VecOf<float, K>::type*)(q.hT + ((int64_t)s * q.Dn + d) * q.N + n0));
        } else save_state<K>(q.hT, s, q, d, n0, h[i]);
        if (n0 == 0) {
            y = fmaf(skip, x[i], y);
            if (q.z) y *= z[i] * sigmoidf(z[i]);
            ((T*)q.y)[s * q.ldy + d] = (T)y;
        }
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
    // Chunks: the two-pass form computes every exponential twice, so it is taken only where workgroups of whole sequences are
    // fewer than two for every CU (16 x 1024 x 2048, 16 states: 512 workgroups in one piece 174 us forward, 673 a training pass;
    // in two 202 and 747).  Then there are four for every CU at least, as near above a whole number of them as 5 % where twice
    // as many pieces reach that, and a piece has four tiles on average.  Prompt and training pass in us, * the rule's choice:
    //   12 x 1365 x 2048 (384 workgroups): one piece 230 and 878, two 230 and 823, three 229 and 838, four* 221 and 788, six 221 and 790
    //   8 x 2048 x 2048 (256): one 282 and 974, two 260 and 849, three 229 and 821, four* 222 and 789, six 219 and 780, eight 220 and 794
    //   4 x 4096 x 2048 (128): four 288 and 908, eight* 243 and 832, sixteen 232 and 821, thirty-two 239 and 865
    //   5 x 1024 x 1004, 64 states (315): one 159 and 631, three 136 and 518, four* 126 and 498, six 131 and 523, eight 126 and 511
    // The host knows the number of sequences and rows and not the lengths, so every sequence counts as one of the mean length: a
    // long one among many short ones is walked in too few pieces (8191 rows and 100 of 30, width 512: one piece 1094 and 3634,
    // sixteen 337 and 953); the option scan_chunks helps a caller who knows them.
    const int64_t whole = (int64_t)p.blocks * (S > 0 ? S : 1), tiles = (T + TILE - 1) / TILE;
    int64_t c = 1;
    if (whole < 512) {
        const int64_t least = (1024 + whole - 1) / whole;
        double best = 2.;
        for (int64_t i = least; i <= 2 * least && best > 1.05; ++i) {
            const double each = (double)(whole * i) / 256, idle = (double)((whole * i + 255) / 256) / each;
            if (idle < best) { best = idle; c = i; }
        }
    }
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
    const int bc = p.NP > 16 ? p.NP / 16 : 1;          // B and C are read NBC states at a time
    q.vec = a->N % bc == 0 && rows_vec(a->B, a->ldb, bc, a->dtype) && rows_vec(a->C, a->ldc, bc, a->dtype) &&
            a->D / a->G % p.VE == 0 && rows_vec(a->x, a->ldx, p.VE, a->dtype) && rows_vec(a->dt, a->lddt, p.VE, a->dtype) &&
            rows_vec(a->z, a->ldz, p.VE, a->dtype);
    return q;
}

template <class T, int P, int K, bool VEC> int fwd_run_as(hipStream_t s, const Scan& q, const Plan& p) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<T, P, K, VEC, true>), dim3(p.blocks, p.slots, p.chunks - 1), dim3(256), 0, s, q);
        PSVAE_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, P, K, VEC, false>), dim3(p.blocks, p.slots, p.chunks + q.zero_outside), dim3(256), 0, s, q);
    PSVAE_LAUNCH_CHECK();
    return 0;
}
template <class T, int P, int K, bool VEC> int bwd_run_as(hipStream_t s, const Scan& q, const Plan& p) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_bwd_kernel<T, P, K, VEC, true>), dim3(p.blocks, p.slots, p.chunks - 1), dim3(256), 0, s, q);
        PSVAE_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, P, K, VEC, false>), dim3(p.blocks, p.slots, p.chunks + q.zero_outside), dim3(256), 0, s, q);
    PSVAE_LAUNCH_CHECK();
    return 0;
}
template <class T, int P, int K> int fwd_run(hipStream_t s, const Scan& q, const Plan& p) {
    return q.vec ? fwd_run_as<T, P, K, true>(s, q, p) : fwd_run_as<T, P, K, false>(s, q, p);
}
template <class T, int P, int K> int bwd_run(hipStream_t s, const Scan& q, const Plan& p) {
    return q.vec ? bwd_run_as<T, P, K, true>(s, q, p) : bwd_run_as<T, P, K, false>(s, q, p);
}
template <class T, int P, int K> int step_run(hipStream_t s, const Scan& whole, const Plan& p) {
    Scan q = whole;
    const int vec = q.N == P * K && rows_vec(q.A, 0, K, PSVAE_F32) && rows_vec(q.h0, 0, K, PSVAE_F32) && rows_vec(q.hT, 0, K, PSVAE_F32);
    const int64_t wide = (q.Dn * P + 255) / 256, most = MOST_BLOCKS / wide;
    if (q.S > most) {                                   // more than one launch holds: the others in further ones
        q.S = (int)most;
        PSVAE_TRY((step_run<T, P, K>(s, q, p)));
        q.S = (int)(whole.S - most);
        const auto on = [&](const void* v, int64_t ld) -> const void* { return v ? (const T*)v + most * ld : nullptr; };
        q.x = on(q.x, q.ldx); q.dt = on(q.dt, q.lddt); q.z = on(q.z, q.ldz); q.B = on(q.B, q.ldb); q.C = on(q.C, q.ldc);
        q.y = (T*)q.y + most * q.ldy;
        q.h0 += most * q.Dn * q.N;
        q.hT += most * q.Dn * q.N;
        return step_run<T, P, K>(s, q, p);
    }
    // four sequences a lane where that leaves two workgroups for every CU
    if (wide * ((q.S + 3) / 4) >= 512)
        hipLaunchKernelGGL((scan_step_kernel<T, P, K, 4>), dim3((unsigned)(wide * ((q.S + 3) / 4))), dim3(256), 0, s, q, vec);
    else
        hipLaunchKernelGGL((scan_step_kernel<T, P, K, 1>), dim3((unsigned)(wide * q.S)), dim3(256), 0, s, q, vec);
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
    return (size_t)(T / HALF + S) * D * scan_plan(T, S, D, G, N).NP * sizeof(float);
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
    if (lddy < a->D) return PSVAE_E_SHAPE;
    const Plan p = scan_plan(a->T, a->S, a->D, a->G, a->N);
    Scan q = scan_args(a, p);
    const BwdScratch o = bwd_scratch(p, a->T, a->S, a->D, a->G);
    if (!aligned16(scratch) || (saved && !aligned16(saved))) return PSVAE_E_ALIGN;
    if (scratch_bytes < o.total * sizeof(float)) return PSVAE_E_WORKSPACE;
    float* base = (float*)scratch;
    q.dy = dy; q.lddy = lddy; q.dhT = dhT; q.kept = (float*)saved;
    q.dx = g->dx; q.ddt = g->ddt; q.dz = g->dz; q.dh0 = g->dh0;
    q.part_bc = base + o.bc; q.part_a = base + o.a; q.part_d = base + o.d;
    q.chunk_h = base + o.chunk;
    q.chunk_s = q.chunk_h + (size_t)(p.chunks - 1) * a->S * a->D * p.NP;
    q.vec = q.vec && rows_vec(dy, lddy, p.VE, a->dtype) && rows_vec(g->dx, a->D, p.VE, a->dtype) &&
            rows_vec(g->ddt, a->D, p.VE, a->dtype) && (!a->z || rows_vec(g->dz, a->D, p.VE, a->dtype));
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SCAN_BWD, (double)a->T * a->D * (a->z ? 7 : 5) * dtype_bytes(a->dtype));
    if (a->S > 0) {
        const int rc = PSVAE_SCAN_RUN(bwd_run, a->dtype, s, q, p);
        PSVAE_TRY(rc);
    }
    ScanJoin j{q.part_bc, q.part_a, q.part_d, g->dB, g->dC, g->dA, g->d_skip, g->d_dt_bias, a->seq_off,
               q.T, a->S, a->D, a->G, a->N, p.NP, p.tiles, a->S > 0 ? p.slots * p.chunks : 0, 0, 0, q.zero_outside, 0};
    const int64_t cols = (int64_t)a->T * a->G * 2 * p.NP;
    j.vec = a->N % 4 == 0 && rows_vec(g->dB, 0, 4, a->dtype) && rows_vec(g->dC, 0, 4, a->dtype);
    j.blocks_bc = (int)((cols + 1023) / 1024 < 8192 ? (cols + 1023) / 1024 : 8192);
    j.blocks_a = (int)(((int64_t)a->D * a->N + 63) / 64);
    PSVAE_BY_TYPE(a->dtype, T, {
        hipLaunchKernelGGL((scan_join_kernel<T>), dim3(j.blocks_bc + j.blocks_a + (2 * a->D + 63) / 64), dim3(256), 0, s, j);
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
    q.vec = a->N % p.K == 0 && rows_vec(a->B, a->ldb, p.K, a->dtype) && rows_vec(a->C, a->ldc, p.K, a->dtype);   // of B and C
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SCAN_FWD, (double)a->S * a->D * a->N * 8);
    return PSVAE_SCAN_RUN(step_run, a->dtype, s, q, p);
}
