// Attention with a window and sinks: the exponential kernel exp(scale q.k) summed over the last `window` positions and the
// first `sinks` positions, each row divided by its sum; and its gradients.
//
// The rows of the Hq / Hkv query heads that share one k/v head are one list of rows (row r = token r / G, head r % G), so
// a tile of keys is read once for all of them, and the gradients of a shared head are sums over one list.  A piece of rows sees two runs of
// keys, the sinks and the window; they are walked as one run of "slots" (slot u < s_hi: key u, then the window), so that a
// few sinks do not cost a tile of their own.
#include "f3m_tile.h"

#include "f3m_sequence.h"

namespace f3m {

struct AttnArgs {
    const char *q, *k, *v, *o, *dout;
    char *out, *dq, *dk, *dv;
    const float *lse_in;
    float *lse, *part, *delta;
    const int *q_lens, *kv_lens;
    long long qs[3], ks[3], vs[3], ds[3];   // strides in bytes: batch, token, head
    int B, Nq, Nk, Hq, Hkv, G, D;
    int window, sinks;                       // window: Nk or more sees everything
    float scale, scale2;                     // scale2 = scale * log2(e)
    int mtiles, splits, items;
    int ktiles, sink_tiles, sink_splits;
};

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;

// token and head of a packed row
struct Row { int i, g; };
__device__ __forceinline__ Row row_of(const AttnArgs &a, int r) { const int i = r / a.G; return Row{i, r - i * a.G}; }

// What a sequence and a piece of its rows see.
struct Seen {
    int q_len, kv_len, lo, s_hi, slots;      // slots = sinks + window of the piece; slot u >= s_hi is key u - s_hi + lo
    __device__ __forceinline__ int key(int u) const { return u < s_hi ? u : u - s_hi + lo; }
};
__device__ __forceinline__ int clamp_len(const int *lens, int b, int n) { return lens == nullptr ? n : min(max(lens[b], 0), n); }
__device__ __forceinline__ Seen seen_by(const AttnArgs &a, int b, int r0, int rows)
{
    Seen s;
    s.q_len = clamp_len(a.q_lens, b, a.Nq);
    s.kv_len = clamp_len(a.kv_lens, b, a.Nk);
    const int i0 = r0 / a.G, i1 = min(s.q_len - 1, (r0 + rows - 1) / a.G);
    const int p0 = s.kv_len - s.q_len + i0, p1 = s.kv_len - s.q_len + i1;
    s.lo = max(0, p0 - a.window + 1);
    const int hi = i1 < i0 ? 0 : max(0, p1 + 1);             // p1 < kv_len
    s.s_hi = min(min(a.sinks, s.lo), hi);
    s.slots = hi <= s.lo ? 0 : s.s_hi + hi - s.lo;
    return s;
}

// Loads four rows x 16 bytes of k or v for the transposing or row-major store: slots u0..u0+3 of the piece, zero behind
// the last slot and behind the head's columns.
__device__ __forceinline__ void load_slots(u32x4 *x, const char *base, long long stride, const Seen &s, int u0, int byte, int row_bytes)
{
#pragma unroll
    for (int n = 0; n < 4; n++) {
        const int u = u0 + n;
        x[n] = zero4();
        if (u < s.slots && byte < row_bytes) x[n] = *reinterpret_cast<const u32x4 *>(base + (long long)s.key(u) * stride + byte);
    }
}

// Forward.  One workgroup of four wavefronts: WM of them side by side along the rows (32 each), 4 / WM along the keys of a tile.  A wavefront
// forms S^T = K Q^T (rows: slots, columns: rows of q), so that a lane holds 16 slots of one row: maximum, sum and the factor of a new maximum stay in
// the lane (one exchange with the other half), and the exponentials are the operand of O^T += V^T P^T as they are.  V is transposed on its way into LDS.
// P is rounded to the type of v (bf16: 2^-9 of each weight, as much as the rounding of the output itself); its sum is taken before the rounding.
template <class T, int DP, int WM>
__global__ void __launch_bounds__(256, 2) attn_forward_kernel(AttnArgs a)
{
    constexpr int WK = 4 / WM, KW = WM == 4 ? 64 : 32, BK = KW * WK, BM = 32 * WM, CPR = DP / kPer16<T>;
    constexpr int KU = BK * kRowUnits<T, DP>, VU = DP * kLineUnits<T, BK>;
    constexpr int MERGE = WK > 1 ? (WK - 1) * WM * (DP / 32 * 16 + 2) * 64 / 4 : 0;      // units of 16 bytes
    __shared__ u32x4 lds[KU + VU > MERGE ? KU + VU : MERGE];
    u32x4 *kt = lds, *vt = lds + KU;
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;

    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    const int split = item % a.splits, mt = a.mtiles - 1 - (item / a.splits) % a.mtiles, bh = item / (a.splits * a.mtiles);
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int r0 = mt * BM, R = a.Nq * a.G;
    const Seen s = seen_by(a, b, r0, BM);
    const int tiles = (s.slots + BK - 1) / BK, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);

    // this lane's row
    const int r = r0 + 32 * wm + l;
    const Row row = row_of(a, min(r, R - 1));
    const bool live = r < R && row.i < s.q_len;
    const int p = s.kv_len - s.q_len + row.i;
    // its slots: [0, u_s) and [u_lo, u_hi)
    const int u_hi = live ? min(s.slots, max(0, p + 1 - s.lo + s.s_hi)) : 0;
    const int u_lo = max(0, p - a.window + 1 - s.lo) + s.s_hi;
    const int u_s = max(s.s_hi, min(a.sinks, s.kv_len) - s.lo + s.s_hi);
    // bounds over the wavefront's rows, from its first and last row (positions grow with the row)
    const int first_hi = wave_readlane(u_hi, 0), last_hi = wave_uniform(max(wave_readlane(u_hi, 31), first_hi));
    const int first_lo = wave_readlane(u_lo, 0), last_lo = wave_readlane(u_lo, 31);
    // a wavefront whose last rows are dead has first_hi > last: rows in between are found per lane
    const bool ragged = wave_ballot(!live) != 0ull;
    const int most_hi = ragged ? s.slots : last_hi;

    const char *qrow = a.q + (long long)b * a.qs[0] + (long long)row.i * a.qs[1] + (long long)(hk * a.G + row.g) * a.qs[2];
    typename T::Frag qf[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        qf[n] = zero_frag<T>();
        if (live && 16 * n + 8 * h < a.D) qf[n] = *reinterpret_cast<const typename T::Frag *>(qrow + (16 * n + 8 * h) * T::kBytes);
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) o[n] = zero_acc();
    float m = -INFINITY, sum = 0.f;                          // of this lane's half of the slots; m is the row's

    const char *kb = a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2], *vb = a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2];
    constexpr int UNITS = BK / 4 * CPR, PER = (UNITS + 255) / 256;
    u32x4 kx[PER][4], vx[PER][4];
    auto load = [&](int t) {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, g = unit / CPR, c = unit % CPR;
            if (unit >= UNITS) break;
            load_slots(kx[n], kb, a.ks[1], s, t * BK + 4 * g, 16 * c, a.D * T::kBytes);
            load_slots(vx[n], vb, a.vs[1], s, t * BK + 4 * g, 16 * c, a.D * T::kBytes);
        }
    };
    if (t0 < t1) load(t0);
    for (int t = t0; t < t1; t++) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, g = unit / CPR, c = unit % CPR;
            if (unit >= UNITS) break;
#pragma unroll
            for (int j = 0; j < 4; j++) Tile<T>::template put_row<DP>(kt, kx[n][j], 4 * g + j, c);
            Tile<T>::template put_transposed<BK>(vt, vx[n], g, c);
        }
        __syncthreads();
        if (t + 1 < t1) load(t + 1);
        const int base = wk * KW, u0 = t * BK + base;          // first slot of this wavefront in the tile
        if (u0 >= most_hi || (u0 + KW <= first_lo && u0 >= u_s)) continue;
        const bool masked = ragged || u0 + KW > first_hi || u0 < last_lo;
        f32x16 st[KW / 32];
#pragma unroll
        for (int x = 0; x < KW / 32; x++) {
            st[x] = zero_acc();
#pragma unroll
            for (int n = 0; n < DP / 16; n++)
                st[x] = mma<T>(Tile<T>::template row<DP>(kt, base + 32 * x + tile_row(l), 16 * n + 8 * h), qf[n], st[x]);
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KW / 32; x++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float z = st[x][e] * a.scale2;
                if (masked) {
                    const int u = u0 + 32 * x + 16 * (e / 8) + 8 * h + e % 8;
                    z = u < u_hi && (u >= u_lo || u < u_s) ? z : -INFINITY;
                }
                st[x][e] = z;
                top = fmaxf(top, z);
            }
        top = half_max(top);
        if (wave_ballot(top > m) != 0ull) {
            const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : fast_exp2(m - m2);
            sum *= f;
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[n][e] *= f;
            m = m2;
        }
        const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int x = 0; x < KW / 32; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) { w[e] = fast_exp2(st[x][8 * y + e] - m0); sum += w[e]; }
                const typename T::Frag pf = to_frag<T>(w);
#pragma unroll
                for (int n = 0; n < DP / 32; n++)
                    o[n] = mma<T>(Tile<T>::template line<BK>(vt, 32 * n + l, base + 32 * x + 16 * y + 8 * h), pf, o[n]);
            }
    }
    sum = half_sum(sum);

    if constexpr (WK > 1) {                                  // join the wavefronts that shared the rows
        float *mem = reinterpret_cast<float *>(lds);
        constexpr int REC = (DP / 32 * 16 + 2) * 64;
        __syncthreads();
        if (wk > 0) {
            float *mine = mem + ((wk - 1) * WM + wm) * REC;
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) mine[(n * 16 + e) * 64 + lane] = o[n][e];
            mine[(DP / 32 * 16) * 64 + lane] = m;
            mine[(DP / 32 * 16 + 1) * 64 + lane] = sum;
        }
        __syncthreads();
        if (wk > 0) return;
        for (int w = 1; w < WK; w++) {
            const float *his = mem + ((w - 1) * WM + wm) * REC;
            const float mh = his[(DP / 32 * 16) * 64 + lane], m2 = fmaxf(m, mh);
            const float f = m2 == -INFINITY ? 1.f : fast_exp2(m - m2), fh = m2 == -INFINITY ? 0.f : fast_exp2(mh - m2);
            sum = sum * f + his[(DP / 32 * 16 + 1) * 64 + lane] * fh;
            m = m2;
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[n][e] = o[n][e] * f + his[(n * 16 + e) * 64 + lane] * fh;
        }
    }
    if (r >= R) return;
    if (a.splits > 1) {                                      // a record of DP + 2 floats: sums, maximum, total
        float *rec = a.part + (((long long)bh * a.splits + split) * R + r) * (DP + 4);
        if (h == 0) { rec[DP] = m; rec[DP + 1] = sum; }
        if (sum > 0.f || sum != sum)
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int y = 0; y < 4; y++)
                    store4<Fp32>(rec, 32 * n + 8 * y + 4 * h, o[n][4 * y], o[n][4 * y + 1], o[n][4 * y + 2], o[n][4 * y + 3]);
        return;
    }
    const long long at = ((long long)b * a.Nq + row.i) * a.Hq + hk * a.G + row.g;
    if (a.lse != nullptr && h == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    char *orow = a.out + at * a.D * T::kBytes;
#pragma unroll
    for (int n = 0; n < DP / 32; n++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int d = 32 * n + 8 * y + 4 * h;
            if (d < a.D) store4<T>(orow, d, o[n][4 * y] * inv, o[n][4 * y + 1] * inv, o[n][4 * y + 2] * inv, o[n][4 * y + 3] * inv);
        }
}

// Joins the splits of a row: a wavefront per row, lanes along the head.
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_combine_kernel(AttnArgs a)
{
    const long long rows = (long long)a.Nq * a.G, all = rows * a.B * a.Hkv;
    const long long n = (long long)blockIdx.x * 4 + wave_uniform(threadIdx.x / 64);
    if (n >= all) return;
    const int lane = threadIdx.x % 64, bh = (int)(n / rows), r = (int)(n % rows), b = bh / a.Hkv, hk = bh % a.Hkv;
    const float *rec = a.part + ((long long)bh * a.splits * rows + r) * (DP + 4);
    const long long step = rows * (DP + 4);
    float m = -INFINITY;
    for (int x = 0; x < a.splits; x++) m = fmaxf(m, rec[x * step + DP]);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
    for (int x = 0; x < a.splits; x++) {
        const float part = rec[x * step + DP + 1];
        if (part == 0.f) continue;                           // nothing seen: the record holds no sums
        const float f = fast_exp2(rec[x * step + DP] - m);
        sum += part * f;
        if (2 * lane < DP) { o0 += rec[x * step + 2 * lane] * f; o1 += rec[x * step + 2 * lane + 1] * f; }
    }
    const Row row = row_of(a, r);
    const long long at = ((long long)b * a.Nq + row.i) * a.Hq + hk * a.G + row.g;
    if (a.lse != nullptr && lane == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (2 * lane >= a.D) return;
    if constexpr (T::kBytes == 2) reinterpret_cast<uint32_t *>(a.out)[at * (a.D / 2) + lane] = T::pack(o0 * inv, o1 * inv);
    else reinterpret_cast<u32x2 *>(a.out)[at * (a.D / 2) + lane] = u32x2{as_bits(o0 * inv), as_bits(o1 * inv)};
}

// Gradients.  delta_i = dout_i . out_i; 16 lanes per row.  lse in units of log 2, +inf where the row sees nothing (its weights are then 0).
template <class T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnArgs a)
{
    const long long all = (long long)a.B * a.Nq * a.Hq, n = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    const int x = threadIdx.x % 16;
    float sum = 0.f;
    if (n < all) {
        const int hq = (int)(n % a.Hq), i = (int)(n / a.Hq % a.Nq), b = (int)(n / a.Hq / a.Nq);
        if (i < clamp_len(a.q_lens, b, a.Nq))
            for (int e = 8 * x; e < a.D; e += 128) {
                float u[8], w[8];
                from_frag<T>(*reinterpret_cast<const typename T::Frag *>(a.o + (n * a.D + e) * T::kBytes), u);
                from_frag<T>(*reinterpret_cast<const typename T::Frag *>(a.dout + (long long)b * a.ds[0] + (long long)i * a.ds[1] +
                                                                         (long long)hq * a.ds[2] + e * T::kBytes), w);
#pragma unroll
                for (int j = 0; j < 8; j++) sum += u[j] * w[j];
            }
    }
    for (int y = 8; y >= 1; y >>= 1) sum += wave_shfl_xor_f(sum, y);
    if (n < all && x == 0) {
        a.delta[2 * n] = a.lse_in[n] == -INFINITY ? INFINITY : a.lse_in[n] * kLog2e;
        a.delta[2 * n + 1] = sum;
    }
}

// dq: the forward kernel's walk over the keys; dS^T = P^T (V dout^T - delta) is the operand of dq^T += K^T dS^T as it is.  k lies in LDS twice,
// row-major for S and transposed for dq.
template <class T, int DP>
__global__ void __launch_bounds__(256, 2) attn_dq_kernel(AttnArgs a)
{
    constexpr int BK = T::kBytes == 2 ? 64 : 32, BM = 128, CPR = DP / kPer16<T>;
    __shared__ u32x4 kt[BK * kRowUnits<T, DP>], vt[BK * kRowUnits<T, DP>], ktr[DP * kLineUnits<T, BK>];
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    const int mt = a.mtiles - 1 - item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hkv, hk = bh % a.Hkv;
    const int r0 = mt * BM, R = a.Nq * a.G;
    const Seen s = seen_by(a, b, r0, BM);
    const int tiles = (s.slots + BK - 1) / BK;

    const int r = r0 + 32 * wave + l;
    const Row row = row_of(a, min(r, R - 1));
    const bool live = r < R && row.i < s.q_len;
    const int p = s.kv_len - s.q_len + row.i;
    const int u_hi = live ? min(s.slots, max(0, p + 1 - s.lo + s.s_hi)) : 0;
    const int u_lo = max(0, p - a.window + 1 - s.lo) + s.s_hi;
    const int u_s = max(s.s_hi, min(a.sinks, s.kv_len) - s.lo + s.s_hi);
    const int first_hi = wave_readlane(u_hi, 0), last_hi = wave_uniform(max(wave_readlane(u_hi, 31), first_hi));
    const int first_lo = wave_readlane(u_lo, 0), last_lo = wave_readlane(u_lo, 31);
    const bool ragged = wave_ballot(!live) != 0ull;
    const int most_hi = ragged ? s.slots : last_hi;

    const int hq = hk * a.G + row.g;
    const char *qrow = a.q + (long long)b * a.qs[0] + (long long)row.i * a.qs[1] + (long long)hq * a.qs[2];
    const char *drow = a.dout + (long long)b * a.ds[0] + (long long)row.i * a.ds[1] + (long long)hq * a.ds[2];
    typename T::Frag qf[DP / 16], df[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        qf[n] = zero_frag<T>();
        df[n] = zero_frag<T>();
        if (live && 16 * n + 8 * h < a.D) {
            qf[n] = *reinterpret_cast<const typename T::Frag *>(qrow + (16 * n + 8 * h) * T::kBytes);
            df[n] = *reinterpret_cast<const typename T::Frag *>(drow + (16 * n + 8 * h) * T::kBytes);
        }
    }
    const long long at = ((long long)b * a.Nq + row.i) * a.Hq + hq;
    const float lse2 = live ? a.delta[2 * at] : INFINITY, delta = live ? a.delta[2 * at + 1] : 0.f;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) dq[n] = zero_acc();

    const char *kb = a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2], *vb = a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2];
    constexpr int UNITS = BK / 4 * CPR, PER = (UNITS + 255) / 256;
    u32x4 kx[PER][4], vx[PER][4];
    auto load = [&](int t) {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, g = unit / CPR, c = unit % CPR;
            if (unit >= UNITS) break;
            load_slots(kx[n], kb, a.ks[1], s, t * BK + 4 * g, 16 * c, a.D * T::kBytes);
            load_slots(vx[n], vb, a.vs[1], s, t * BK + 4 * g, 16 * c, a.D * T::kBytes);
        }
    };
    if (tiles > 0) load(0);
    for (int t = 0; t < tiles; t++) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, g = unit / CPR, c = unit % CPR;
            if (unit >= UNITS) break;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                Tile<T>::template put_row<DP>(kt, kx[n][j], 4 * g + j, c);
                Tile<T>::template put_row<DP>(vt, vx[n][j], 4 * g + j, c);
            }
            Tile<T>::template put_transposed<BK>(ktr, kx[n], g, c);
        }
        __syncthreads();
        if (t + 1 < tiles) load(t + 1);
#pragma unroll
        for (int x = 0; x < BK / 32; x++) {
            const int u0 = t * BK + 32 * x;
            if (u0 >= most_hi || (u0 + 32 <= first_lo && u0 >= u_s)) continue;
            const bool masked = ragged || u0 + 32 > first_hi || u0 < last_lo;
            f32x16 st = zero_acc(), dp = zero_acc();
#pragma unroll
            for (int n = 0; n < DP / 16; n++) {
                st = mma<T>(Tile<T>::template row<DP>(kt, 32 * x + tile_row(l), 16 * n + 8 * h), qf[n], st);
                dp = mma<T>(Tile<T>::template row<DP>(vt, 32 * x + tile_row(l), 16 * n + 8 * h), df[n], dp);
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float pr = fast_exp2(st[8 * y + e] * a.scale2 - lse2);
                    if (masked) {
                        const int u = u0 + 16 * y + 8 * h + e;
                        pr = u < u_hi && (u >= u_lo || u < u_s) ? pr : 0.f;
                    }
                    w[e] = pr * (dp[8 * y + e] - delta);
                }
                const typename T::Frag sf = to_frag<T>(w);
#pragma unroll
                for (int n = 0; n < DP / 32; n++)
                    dq[n] = mma<T>(Tile<T>::template line<BK>(ktr, 32 * n + l, 32 * x + 16 * y + 8 * h), sf, dq[n]);
            }
        }
    }
    if (r >= R) return;
    char *out = a.dq + at * a.D * T::kBytes;
#pragma unroll
    for (int n = 0; n < DP / 32; n++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int d = 32 * n + 8 * y + 4 * h;
            if (d < a.D)
                store4<T>(out, d, dq[n][4 * y] * a.scale, dq[n][4 * y + 1] * a.scale, dq[n][4 * y + 2] * a.scale, dq[n][4 * y + 3] * a.scale);
        }
}

// dk and dv: a workgroup holds 128 keys (32 per wavefront, the lanes' columns) and walks the rows that see them, in tiles of 32: S = Q K^T, dP = dout V^T,
// dv^T += dout^T P, dk^T += Q^T dS.  q and dout lie in LDS row-major and transposed.  A tile of keys that holds sinks is seen by all rows
// behind it, many times the rows of any other under a window: its rows are dealt to sink_splits workgroups, whose sums are joined by attn_join_kernel.
template <class T, int DP>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1) attn_dkv_kernel(AttnArgs a)
{
    constexpr int BR = 32, BN = 128, CPR = DP / kPer16<T>;
    __shared__ u32x4 qt[BR * kRowUnits<T, DP>], dt[BR * kRowUnits<T, DP>], qtr[DP * kLineUnits<T, BR>], dtr[DP * kLineUnits<T, BR>];
    __shared__ u32x4 stat4[BR / 2], pos4[BR / 4];             // per row: lse, delta; position (-1: no row)
    float *stat = reinterpret_cast<float *>(stat4);
    int *pos = reinterpret_cast<int *>(pos4);
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    // items of a head: the splits of its sink tiles, then its other tiles
    const int sink_items = a.sink_tiles * a.sink_splits, each = sink_items + a.ktiles - a.sink_tiles;
    const int bh = item / each, rest = item % each, b = bh / a.Hkv, hk = bh % a.Hkv;
    const bool split = rest < sink_items;
    const int ktile = split ? rest / a.sink_splits : rest - sink_items + a.sink_tiles, part = split ? rest % a.sink_splits : 0;
    const int q_len = clamp_len(a.q_lens, b, a.Nq), kv_len = clamp_len(a.kv_lens, b, a.Nk), off = kv_len - q_len;
    const int j0 = ktile * BN, key = j0 + 32 * wave + l;
    // rows that see some key of the tile: position j0 .. last
    const int last = min(kv_len - 1, j0 < a.sinks ? kv_len - 1 : (int)min((long long)kv_len - 1, (long long)j0 + BN - 1 + a.window - 1));
    const int ia = max(0, j0 - off), ib = j0 < kv_len ? min(q_len, last - off + 1) : 0;
    int ra = ia * a.G, rb = max(ra, ib * a.G);
    if (split) {
        const int tiles = (rb - ra + BR - 1) / BR, per = (tiles + a.sink_splits - 1) / a.sink_splits;
        const int from = min(rb, ra + part * per * BR);
        rb = min(rb, from + per * BR);
        ra = from;
    }
    const bool have = key < kv_len;
    const char *krow = a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2] + (long long)min(key, a.Nk - 1) * a.ks[1];
    const char *vrow = a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2] + (long long)min(key, a.Nk - 1) * a.vs[1];
    typename T::Frag kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        kf[n] = zero_frag<T>();
        vf[n] = zero_frag<T>();
        if (have && ra < rb && 16 * n + 8 * h < a.D) {
            kf[n] = *reinterpret_cast<const typename T::Frag *>(krow + (16 * n + 8 * h) * T::kBytes);
            vf[n] = *reinterpret_cast<const typename T::Frag *>(vrow + (16 * n + 8 * h) * T::kBytes);
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) { dk[n] = zero_acc(); dv[n] = zero_acc(); }

    // units of 4 rows x 16 bytes of q, then of dout
    constexpr int UNITS = BR / 4 * CPR, PER = (2 * UNITS + 255) / 256;
    u32x4 x[PER][4];
    float st_lse = 0.f, st_delta = 0.f;
    int st_pos = -1;
    const char *qb = a.q + (long long)b * a.qs[0] + (long long)(hk * a.G) * a.qs[2];
    const char *db = a.dout + (long long)b * a.ds[0] + (long long)(hk * a.G) * a.ds[2];
    auto load = [&](int rt) {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, which = unit / UNITS, g = unit % UNITS / CPR, c = unit % CPR;
            if (unit >= 2 * UNITS) break;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = rt + 4 * g + j;
                x[n][j] = zero4();
                if (r < rb && 16 * c < a.D * T::kBytes) {
                    const Row row = row_of(a, r);
                    const char *at = which == 0 ? qb + (long long)row.i * a.qs[1] + (long long)row.g * a.qs[2]
                                                : db + (long long)row.i * a.ds[1] + (long long)row.g * a.ds[2];
                    x[n][j] = *reinterpret_cast<const u32x4 *>(at + 16 * c);
                }
            }
        }
        if (tid < BR) {
            const int r = rt + tid;
            st_lse = INFINITY;
            st_delta = 0.f;
            st_pos = -1;
            if (r < rb) {
                const Row row = row_of(a, r);
                const long long at = ((long long)b * a.Nq + row.i) * a.Hq + hk * a.G + row.g;
                st_lse = a.delta[2 * at];
                st_delta = a.delta[2 * at + 1];
                st_pos = off + row.i;
            }
        }
    };
    const int jw = j0 + 32 * wave;                            // this wavefront's keys: jw .. jw + 31
    if (ra < rb) load(ra);
    for (int rt = ra; rt < rb; rt += BR) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int unit = tid + 256 * n, which = unit / UNITS, g = unit % UNITS / CPR, c = unit % CPR;
            if (unit >= 2 * UNITS) break;
#pragma unroll
            for (int j = 0; j < 4; j++) Tile<T>::template put_row<DP>(which == 0 ? qt : dt, x[n][j], 4 * g + j, c);
            Tile<T>::template put_transposed<BR>(which == 0 ? qtr : dtr, x[n], g, c);
        }
        if (tid < BR) { stat[tid] = st_lse; stat[BR + tid] = st_delta; pos[tid] = st_pos; }
        __syncthreads();
        if (rt + BR < rb) load(rt + BR);
        // positions of the tile's first and last row
        const int pa = off + rt / a.G, pb = off + (min(rb, rt + BR) - 1) / a.G;
        if (pb < jw || jw >= kv_len || (jw >= a.sinks && pa - (jw + 31) >= a.window)) continue;
        const bool masked = rt + BR > rb || jw + 31 > pa || (pb - jw >= a.window && jw + 31 >= a.sinks);
        f32x16 st = zero_acc(), dp = zero_acc();
#pragma unroll
        for (int n = 0; n < DP / 16; n++) {
            st = mma<T>(Tile<T>::template row<DP>(qt, tile_row(l), 16 * n + 8 * h), kf[n], st);
            dp = mma<T>(Tile<T>::template row<DP>(dt, tile_row(l), 16 * n + 8 * h), vf[n], dp);
        }
#pragma unroll
        for (int y = 0; y < 2; y++) {
            float lse[8], del[8], pw[8], sw[8];
            const int at = 16 * y + 8 * h;
            from_frag<Fp32>(Frag32{{stat4[at / 4], stat4[at / 4 + 1]}}, lse);
            from_frag<Fp32>(Frag32{{stat4[(BR + at) / 4], stat4[(BR + at) / 4 + 1]}}, del);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float pr = fast_exp2(st[8 * y + e] * a.scale2 - lse[e]);
                if (masked) {
                    const int p = pos[at + e];
                    pr = key <= p && (p - key < a.window || key < a.sinks) ? pr : 0.f;
                }
                pw[e] = pr;
                sw[e] = pr * (dp[8 * y + e] - del[e]);
            }
            const typename T::Frag pf = to_frag<T>(pw), sf = to_frag<T>(sw);
#pragma unroll
            for (int n = 0; n < DP / 32; n++) {
                dv[n] = mma<T>(Tile<T>::template line<BR>(dtr, 32 * n + l, at), pf, dv[n]);
                dk[n] = mma<T>(Tile<T>::template line<BR>(qtr, 32 * n + l, at), sf, dk[n]);
            }
        }
    }
    if (key >= a.Nk) return;
    if (split && a.sink_splits > 1) {
        // record of a key and split: dk, dv as fp32
        float *rec = a.part + ((((long long)bh * a.sink_splits + part) * a.sink_tiles * BN) + j0 + 32 * wave + l) * (2 * DP);
#pragma unroll
        for (int n = 0; n < DP / 32; n++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int d = 32 * n + 8 * y + 4 * h;
                store4<Fp32>(rec, d, dk[n][4 * y], dk[n][4 * y + 1], dk[n][4 * y + 2], dk[n][4 * y + 3]);
                store4<Fp32>(rec, DP + d, dv[n][4 * y], dv[n][4 * y + 1], dv[n][4 * y + 2], dv[n][4 * y + 3]);
            }
        return;
    }
    const long long at = (((long long)b * a.Nk + key) * a.Hkv + hk) * a.D * T::kBytes;
#pragma unroll
    for (int n = 0; n < DP / 32; n++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int d = 32 * n + 8 * y + 4 * h;
            if (d >= a.D) continue;
            store4<T>(a.dk + at, d, dk[n][4 * y] * a.scale, dk[n][4 * y + 1] * a.scale, dk[n][4 * y + 2] * a.scale, dk[n][4 * y + 3] * a.scale);
            store4<T>(a.dv + at, d, dv[n][4 * y], dv[n][4 * y + 1], dv[n][4 * y + 2], dv[n][4 * y + 3]);
        }
}

// Joins the splits of the sink tiles' keys, in order: a thread per four elements.
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a)
{
    const int keys = a.sink_tiles * 128;
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
    const int e = (int)(n % (2 * DP / 4)) * 4;
    const long long kk = n / (2 * DP / 4);
    if (kk >= (long long)a.B * a.Hkv * keys) return;
    const int key = (int)(kk % keys), bh = (int)(kk / keys), b = bh / a.Hkv, hk = bh % a.Hkv, d = e % DP;
    if (key >= a.Nk || d >= a.D) return;
    const float *rec = a.part + ((long long)bh * a.sink_splits * keys + key) * (2 * DP) + e;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < a.sink_splits; x++) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(rec + (long long)x * keys * (2 * DP));
        for (int j = 0; j < 4; j++) s[j] += as_float(w[j]);
    }
    const float f = e < DP ? a.scale : 1.f;
    store4<T>((e < DP ? a.dk : a.dv) + (((long long)b * a.Nk + key) * a.Hkv + hk) * a.D * T::kBytes, d, s[0] * f, s[1] * f, s[2] * f, s[3] * f);
}

// ---- host ------------------------------------------------------------------------------------------------
namespace {

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

AttnArgs attn_args(const f3m_attn_params *p)
{
    F3M_REQUIRE(p != nullptr, 8, "params is NULL");
    F3M_REQUIRE(p->dtype >= F3M_BF16 && p->dtype <= F3M_F32, 61, "dtype must be F3M_BF16, F3M_F16 or F3M_F32 (got %d)", p->dtype);
    F3M_REQUIRE(p->D >= 8 && p->D <= 128 && p->D % 8 == 0, 2, "head size must be a multiple of 8 up to 128 (got %d)", p->D);
    F3M_REQUIRE(p->Hq >= 1 && p->Hkv >= 1 && p->Hq % p->Hkv == 0, 3, "query heads (%d) must be a multiple of key heads (%d)", p->Hq, p->Hkv);
    F3M_REQUIRE(p->B >= 0 && p->Nq >= 0 && p->Nk >= 0, 3, "bad shape");
    F3M_REQUIRE(p->window >= 0 && p->sinks >= 0, 61, "window and sinks must not be negative");
    F3M_REQUIRE(std::isfinite(p->scale), 61, "scale must be finite");
    const long long G = p->Hq / p->Hkv, most = 1ll << 30;
    F3M_REQUIRE(p->B * p->Hq <= most && p->Nk <= most && p->Nq <= most && p->Nq * G <= most, 3, "more than 2^30 rows, keys or heads");
    AttnArgs a = {};
    const long long e = p->dtype == F3M_F32 ? 4 : 2;
    for (int i = 0; i < 3; i++) {
        a.qs[i] = p->q_stride[i] * e;
        a.ks[i] = p->k_stride[i] * e;
        a.vs[i] = p->v_stride[i] * e;
        a.ds[i] = p->dout_stride[i] * e;
    }
    a.B = (int)p->B; a.Nq = (int)p->Nq; a.Nk = (int)p->Nk; a.Hq = p->Hq; a.Hkv = p->Hkv; a.G = (int)G; a.D = p->D;
    a.window = p->window == 0 || p->window > p->Nk ? (int)std::max<int64_t>(1, p->Nk) : (int)p->window;
    a.sinks = (int)std::min(p->sinks, p->Nk);
    a.scale = p->scale;
    a.scale2 = p->scale * kLog2e;
    return a;
}

// Wavefronts side by side along the rows: a call with few rows per k/v head (single tokens) gives its wavefronts the keys to share instead.
int row_waves(const AttnArgs &a, int dtype)
{
    const long long R = (long long)a.Nq * a.G;
    return R <= 32 && dtype != F3M_F32 ? 1 : R <= 64 ? 2 : 4;
}

// Two workgroups fit a compute unit: 512 fill the card.  A call with fewer row tiles splits the keys, at least two tiles of keys to a split.
void forward_shape(AttnArgs &a, int dtype)
{
    const int wm = row_waves(a, dtype), bm = 32 * wm, bk = wm == 4 ? 64 : 32 * (4 / wm);
    const long long R = (long long)a.Nq * a.G, heads = (long long)a.B * a.Hkv;
    a.mtiles = (int)((R + bm - 1) / bm);
    const long long tokens = std::min<long long>(a.Nq, bm / a.G + 2), slots = std::min<long long>(a.Nk, (long long)a.window + tokens + a.sinks);
    const long long tiles = (slots + bk - 1) / bk, base = std::max<long long>(1, heads * a.mtiles);
    a.splits = (int)std::max<long long>(1, std::min<long long>({512 / base, tiles / 2, 64}));
    F3M_REQUIRE(heads * a.mtiles * a.splits <= (1ll << 30), 3, "too many rows for one call");
    a.items = (int)(heads * a.mtiles * a.splits);
}

// The rows that see a sink tile, in parts of about what an ordinary tile of keys is seen by.
void grad_shape(AttnArgs &a)
{
    a.ktiles = (a.Nk + 127) / 128;
    a.sink_tiles = std::min((a.sinks + 127) / 128, a.ktiles);
    a.sink_splits = 1;
    if (a.window < a.Nk) a.sink_splits = (int)std::max<long long>(1, std::min<long long>(64, a.Nk / ((long long)a.window + 128)));
    else a.sink_tiles = 0;                                   // every row sees all before it: sinks are like other keys
}

size_t attn_workspace(const f3m_attn_params *p, bool grad)
{
    AttnArgs a = attn_args(p);
    const size_t dp = padded(a.D);
    if (!grad) {
        forward_shape(a, p->dtype);
        return a.splits == 1 ? 0 : (size_t)a.B * a.Hkv * a.splits * a.Nq * a.G * (dp + 4) * 4;
    }
    grad_shape(a);
    const size_t delta = ((size_t)a.B * a.Nq * a.Hq * 8 + 255) & ~size_t(255);
    return delta + (a.sink_splits == 1 ? 0 : (size_t)a.B * a.Hkv * a.sink_splits * a.sink_tiles * 128 * 2 * dp * 4);
}

template <class T, int DP> void forward(const AttnArgs &a, hipStream_t s)
{
    const int wm = row_waves(a, T::kId);
    const unsigned grid = xcd_grid(a.items);
    if (wm == 4) F3M_LAUNCH((attn_forward_kernel<T, DP, 4>), grid, 256, 0, s, a);
    else if (wm == 2) F3M_LAUNCH((attn_forward_kernel<T, DP, 2>), grid, 256, 0, s, a);
    else if constexpr (T::kBytes == 2) F3M_LAUNCH((attn_forward_kernel<T, DP, 1>), grid, 256, 0, s, a);
    check_launch("attention");
    if (a.splits > 1) {
        F3M_LAUNCH((attn_combine_kernel<T, DP>), cdiv((long long)a.B * a.Hkv * a.Nq * a.G, 4), 256, 0, s, a);
        check_launch("attention's join");
    }
}

template <class T, int DP> void backward(AttnArgs a, hipStream_t s)
{
    const long long heads = (long long)a.B * a.Hkv;
    if (a.Nq > 0) {
        F3M_LAUNCH((attn_delta_kernel<T>), cdiv((long long)a.B * a.Nq * a.Hq, 16), 256, 0, s, a);
        check_launch("attention's row sums");
        a.mtiles = (int)(((long long)a.Nq * a.G + 127) / 128);
        a.items = (int)(heads * a.mtiles);
        F3M_LAUNCH((attn_dq_kernel<T, DP>), xcd_grid(a.items), 256, 0, s, a);
        check_launch("attention's dq");
    }
    if (a.Nk > 0) {
        const long long items = heads * (a.sink_tiles * a.sink_splits + a.ktiles - a.sink_tiles);
        F3M_REQUIRE(items <= (1ll << 30), 3, "too many keys for one call");
        a.items = (int)items;
        F3M_LAUNCH((attn_dkv_kernel<T, DP>), xcd_grid(a.items), 256, 0, s, a);
        check_launch("attention's dk, dv");
        if (a.sink_splits > 1 && a.sink_tiles > 0) {
            F3M_LAUNCH((attn_join_kernel<T, DP>), cdiv(heads * a.sink_tiles * 128 * (2 * DP / 4), 256), 256, 0, s, a);
            check_launch("attention's sinks");
        }
    }
}

template <typename F> void with_size(int D, F f)
{
    const int dp = padded(D);
    if (dp == 32) f(std::integral_constant<int, 32>{});
    else if (dp == 64) f(std::integral_constant<int, 64>{});
    else if (dp == 96) f(std::integral_constant<int, 96>{});
    else f(std::integral_constant<int, 128>{});
}

void check_qkv(const f3m_attn_params *p, const void *q, const void *k, const void *v)
{
    const int e = p->dtype == F3M_F32 ? 4 : 2;
    if (p->B > 0 && p->Nq > 0) check_16(q, "q");
    if (p->B > 0 && p->Nk > 0) { check_16(k, "k"); check_16(v, "v"); }
    check_strides(p->q_stride, e, "q");
    check_strides(p->k_stride, e, "k");
    check_strides(p->v_stride, e, "v");
}

}  // namespace
}  // namespace f3m

using namespace f3m;

extern "C" {

int f3m_window_attention_workspace(const f3m_attn_params *params, int grad, size_t *bytes)
{
    return guarded_async([&] {
        F3M_REQUIRE(bytes != nullptr, 8, "bytes is NULL");
        *bytes = attn_workspace(params, grad != 0);
    });
}

int f3m_window_attention(const f3m_attn_params *params, const void *q, const void *k, const void *v, const int32_t *q_lens,
                         const int32_t *kv_lens, void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    return guarded_async([&] {
        AttnArgs a = attn_args(params);
        check_qkv(params, q, k, v);
        if (a.B == 0 || a.Nq == 0) return;
        check_16(out, "out");
        forward_shape(a, params->dtype);
        const size_t need = attn_workspace(params, false);
        if (need > 0) check_16(workspace, "workspace");
        F3M_REQUIRE(workspace_bytes >= need, 62, "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
        a.q = (const char *)q; a.k = (const char *)k; a.v = (const char *)v; a.out = (char *)out; a.lse = lse;
        a.q_lens = q_lens; a.kv_lens = kv_lens; a.part = (float *)workspace;
        with_type(params->dtype, [&](auto t) {
            with_size(a.D, [&](auto d) { forward<decltype(t), decltype(d)::value>(a, (hipStream_t)stream); });
        });
    });
}

int f3m_window_attention_grad(const f3m_attn_params *params, const void *q, const void *k, const void *v, const void *out,
                              const float *lse, const void *dout, const int32_t *q_lens, const int32_t *kv_lens, void *dq,
                              void *dk, void *dv, void *workspace, size_t workspace_bytes, void *stream)
{
    return guarded_async([&] {
        AttnArgs a = attn_args(params);
        check_qkv(params, q, k, v);
        if (a.B == 0) return;
        check_strides(params->dout_stride, params->dtype == F3M_F32 ? 4 : 2, "dout");
        if (a.Nq > 0) {
            check_16(out, "out"); check_16(dout, "dout"); check_16(dq, "dq");
            F3M_REQUIRE(lse != nullptr, 8, "lse is NULL");
        }
        if (a.Nk > 0) { check_16(dk, "dk"); check_16(dv, "dv"); }
        grad_shape(a);
        const size_t need = attn_workspace(params, true);
        if (need > 0) check_16(workspace, "workspace");
        F3M_REQUIRE(workspace_bytes >= need, 62, "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
        a.q = (const char *)q; a.k = (const char *)k; a.v = (const char *)v; a.o = (const char *)out; a.dout = (const char *)dout;
        a.lse_in = lse; a.q_lens = q_lens; a.kv_lens = kv_lens; a.dq = (char *)dq; a.dk = (char *)dk; a.dv = (char *)dv;
        a.delta = (float *)workspace;
        a.part = (float *)((char *)workspace + (((size_t)a.B * a.Nq * a.Hq * 8 + 255) & ~size_t(255)));
        with_type(params->dtype, [&](auto t) {
            with_size(a.D, [&](auto d) { backward<decltype(t), decltype(d)::value>(a, (hipStream_t)stream); });
        });
    });
}

}  // extern "C"
