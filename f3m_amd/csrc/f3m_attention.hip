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
    float scale, scale2;                     // scale2 = |scale| log2(e), not 0; the sign, or a scale of 0, is taken over by q (k in attn_dkv_kernel)
    unsigned keep, sign;                     // a word of elements & keep ^ sign: 0 if scale is 0, of the other sign if it is negative
    int near_rows;                           // rows of k and v lie near enough for 32-bit offsets
    int near_q;                              // so do 32 packed rows of q and dout
    int mtiles, splits, items;
    int paired;                              // odd heads take their tiles in the other order
    int ktiles, sink_tiles, sink_splits, tile_splits;
};

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;

// token and head of a packed row
struct Row { int i, g; };
__device__ __forceinline__ Row row_of(const AttnArgs &a, int r) { const int i = r / a.G; return Row{i, r - i * a.G}; }

// The n-th pair of sequence and k/v head in the order of the items.  An XCD takes a run of n; where they divide evenly its run holds every eighth pair, so that
// the heads of a long sequence are not all on one XCD (512 rows each of 4 sequences of 2048 to 8192 keys, 16 heads on 4: 174 -> 141 us on one card; 135 to 157 on others).
__device__ __forceinline__ int head_at(const AttnArgs &a, int n)
{
    const int heads = a.B * a.Hkv, per = heads / 8;
    return heads % 8 == 0 ? n % per * 8 + n / per : n;
}

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

// Moves rows of k or v from memory to LDS by way of registers.  A tile's rows are taken in PER turns of 256 / CPR rows: thread t takes the
// 16-byte piece t % CPR of row t / CPR of each.  Slots behind the last one and columns behind the head's are zero.
template <class T, int DP, int BK> struct SlotLoader {
    static constexpr int CPR = kRowUnits<T, DP>, ROWS = 256 / CPR, PER = BK / ROWS;
    static_assert(256 % CPR == 0 && BK % ROWS == 0, "");
    u32x4 x[PER];
    int off;                                                 // of this thread's piece in a turn of neighbouring rows
    const char *base;
    long long stride;
    int row_bytes;
    __device__ __forceinline__ void init(const char *p, long long step, int bytes)
    {
        base = p; stride = step; row_bytes = bytes;
        const int c = threadIdx.x % CPR;
        off = 16 * c < bytes ? (int)(threadIdx.x / CPR * step) + 16 * c : kOutside;
    }
    __device__ __forceinline__ void load(const Seen &s, int u0, bool near_rows)
    {
        if (near_rows && u0 >= s.s_hi) {                     // neighbouring rows of the window
            const char *at = base + (long long)s.key(u0) * stride;
#pragma unroll
            for (int n = 0; n < PER; n++) {
                const int rows = s.slots - u0 - n * ROWS;
                x[n] = load16(buffer(at + (long long)n * ROWS * stride, rows > 0 ? (int)((min(ROWS, rows) - 1) * stride) + row_bytes : 0), off);
            }
        } else {
#pragma unroll
            for (int n = 0; n < PER; n++) {
                const int u = u0 + n * ROWS + threadIdx.x / CPR, c = threadIdx.x % CPR;
                x[n] = zero4();
                if (u < s.slots && 16 * c < row_bytes) x[n] = *reinterpret_cast<const u32x4 *>(base + (long long)s.key(u) * stride + 16 * c);
            }
        }
    }
    __device__ __forceinline__ void store(u32x4 *tile) const
    {
        // columns behind the padded head (DP = 96 in 128) are stored too: their units are never read
#pragma unroll
        for (int n = 0; n < PER; n++) Tile<T, DP>::put(tile, x[n], n * ROWS + threadIdx.x / CPR, threadIdx.x % CPR);
    }
};

template <class T> __device__ __forceinline__ typename T::Frag signed_frag(typename T::Frag x, const AttnArgs &a)
{
    if constexpr (T::kBytes == 2) return (x & a.keep) ^ a.sign;
    else return Frag32{{(x.v[0] & a.keep) ^ a.sign, (x.v[1] & a.keep) ^ a.sign}};
}

// The row of a lane and the slots it sees: [0, u_s) and [u_lo, u_hi); and bounds over the rows of its wavefront.
struct LaneRow {
    Row row;
    bool live;
    int u_hi, u_lo, u_s;
    bool ragged;                                             // some row of the wavefront does not exist
    int first_hi, most_hi, first_lo, last_lo;
    __device__ __forceinline__ LaneRow(const AttnArgs &a, const Seen &s, int r, int R)
    {
        row = row_of(a, min(r, R - 1));
        live = r < R && row.i < s.q_len;
        const int p = s.kv_len - s.q_len + row.i;
        u_hi = live ? min(s.slots, max(0, p + 1 - s.lo + s.s_hi)) : 0;
        u_lo = max(0, p - a.window + 1 - s.lo) + s.s_hi;
        u_s = max(s.s_hi, min(a.sinks, s.kv_len) - s.lo + s.s_hi);
        // positions grow with the row
        ragged = wave_ballot(!live) != 0ull;
        first_hi = wave_readlane(u_hi, 0);
        const int last_hi = wave_readlane(u_hi, 31);
        most_hi = ragged ? s.slots : last_hi;
        first_lo = wave_readlane(u_lo, 0);
        last_lo = wave_readlane(u_lo, 31);
    }
    __device__ __forceinline__ bool sees(int u) const { return u < u_hi && (u >= u_lo || u < u_s); }
    // no row / not every row sees all of the n slots from u0
    __device__ __forceinline__ bool none(int u0, int n) const { return u0 >= most_hi || (u0 + n <= first_lo && u0 >= u_s); }
    __device__ __forceinline__ bool some(int u0, int n) const { return ragged || u0 + n > first_hi || u0 < last_lo; }
};

template <class T> constexpr int kUnitW = T::kId == Fp16::kId ? 7 : 0;

// Forward.  One workgroup of four wavefronts: WM of them side by side along the rows (32 each), 4 / WM along the keys of a tile.  A wavefront
// forms S^T = K Q^T (rows: slots, columns: rows of q), so that a lane holds 16 slots of one row: maximum, sum and the factor of a new maximum stay in
// the lane (one exchange with the other half), and the exponentials are the operand of O^T += V^T P^T as they are.
// P is rounded to the type of v, once (by up to 2^-8 of each weight in bf16, 2^-11 in fp16, as the output itself is; in two parts it would cost a third product); its sum
// is taken before the rounding.
// The maximum that weights are taken against is raised only when a row's passes it by a factor of 2^8: weights stay below 2^8 (fp16 holds 2^16),
// and the factor on the sums (DP / 2 multiplications a lane) is rarely due.  fp16: all weights and sums are 2^7 times as large (kUnitW; they stay below 2^15), so that
// a weight counts from 2^-32 of a row's largest on, not from 2^-25: thousands of small ones beside one large one are then not lost.
// Measured: 8192 tokens, 32 heads of 128 on 8, window 1024: 173 us, 757 TFLOP/s; its products and LDS reads alone take 116 (a large library product: 1123
// TFLOP/s), the rest is exponentials, loads and stores that two wavefronts a SIMD (255 registers) do not hide.  One token for each of 32 caches, window 8192: 214 us,
// 5.0 TB/s, memory.
template <class T, int DP, int WM>
__global__ void __launch_bounds__(256, T::kBytes == 4 && DP > 64 ? 1 : 2) attn_forward_kernel(AttnArgs a)
{
    constexpr int WK = 4 / WM, KW = WM == 4 ? 64 : 32, BK = KW * WK, BM = 32 * WM;
    constexpr int TU = BK * kRowUnits<T, DP>, NBUF = 4 * TU * 16 <= 80 * 1024 ? 2 : 1;      // two buffers where two workgroups still fit
    constexpr int REC = (DP / 32 * 16 + 2) * 64, MERGE = WK > 1 ? (WK - 1) * WM * REC / 4 : 0;
    __shared__ u32x4 lds[2 * NBUF * TU > MERGE ? 2 * NBUF * TU : MERGE];
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;

    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    const int split = item % a.splits, nth = (item / a.splits) % a.mtiles, nh = item / (a.splits * a.mtiles), bh = head_at(a, nh);
    const int mt = a.paired && (nh & 1) ? nth : a.mtiles - 1 - nth;       // the last rows see the most keys
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int r0 = mt * BM, R = a.Nq * a.G;
    const Seen s = seen_by(a, b, r0, BM);
    const int tiles = (s.slots + BK - 1) / BK, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);

    const int row_at = Tile<T, DP>::row_lane(tile_row(l), h);
    const typename Tile<T, DP>::ColLane col_at = Tile<T, DP>::col_lane(l, h);
    const int r = r0 + 32 * wm + l;
    const LaneRow me(a, s, r, R);
    const char *qrow = a.q + (long long)b * a.qs[0] + (long long)me.row.i * a.qs[1] + (long long)(hk * a.G + me.row.g) * a.qs[2];
    typename T::Frag qf[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        qf[n] = zero_frag<T>();
        if (me.live && 16 * n + 8 * h < a.D) qf[n] = signed_frag<T>(*reinterpret_cast<const typename T::Frag *>(qrow + (16 * n + 8 * h) * T::kBytes), a);
    }
#pragma unroll
    for (int n = 0; n < DP / 16; n++) settle(qf[n]);
    f32x16 o[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) o[n] = zero_acc();
    float m = -INFINITY, sum = 0.f;                          // maximum (of the products, before scale2); sum of this lane's half of the slots

    SlotLoader<T, DP, BK> kx, vx;
    kx.init(a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2], a.ks[1], a.D * T::kBytes);
    vx.init(a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2], a.vs[1], a.D * T::kBytes);
    if (t0 < t1) {
        kx.load(s, t0 * BK, a.near_rows);
        vx.load(s, t0 * BK, a.near_rows);
        if constexpr (NBUF == 2) {
            kx.store(lds);
            vx.store(lds + TU);
            if (t0 + 1 < t1) { kx.load(s, (t0 + 1) * BK, a.near_rows); vx.load(s, (t0 + 1) * BK, a.near_rows); }
        }
    }
    for (int t = t0; t < t1; t++) {
        // two buffers: tile t lies in one; tile t + 1, in registers, goes to the other, that tile t - 1 was read from before the barrier
        u32x4 *kt = lds + (NBUF == 2 ? ((t - t0) & 1) * 2 * TU : 0), *vt = kt + TU;
        __syncthreads();
        if constexpr (NBUF == 2) {
            if (t + 1 < t1) {
                u32x4 *next = lds + ((t - t0 + 1) & 1) * 2 * TU;
                kx.store(next);
                vx.store(next + TU);
            }
            if (t + 2 < t1) { kx.load(s, (t + 2) * BK, a.near_rows); vx.load(s, (t + 2) * BK, a.near_rows); }
        } else {
            kx.store(kt);
            vx.store(vt);
            __syncthreads();
            if (t + 1 < t1) { kx.load(s, (t + 1) * BK, a.near_rows); vx.load(s, (t + 1) * BK, a.near_rows); }
        }
        const int base = wk * KW, u0 = t * BK + base;          // first slot of this wavefront in the tile
        if (me.none(u0, KW)) continue;
        f32x16 st[KW / 32];
#pragma unroll
        for (int x = 0; x < KW / 32; x++) {
            st[x] = zero_acc();
#pragma unroll
            for (int n = 0; n < DP / 16; n++)
                st[x] = mma<T>(Tile<T, DP>::row(kt, base + 32 * x, row_at, n), qf[n], st[x]);
        }
        if constexpr (T::kBytes == 2) read_ahead<DP / 16 * (KW / 32), 1, DP / 16>();
        if (me.some(u0, KW)) {
#pragma unroll
            for (int x = 0; x < KW / 32; x++)
#pragma unroll
                for (int e = 0; e < 16; e++) st[x][e] = me.sees(u0 + 32 * x + 16 * (e / 8) + 8 * h + e % 8) ? st[x][e] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KW / 32; x++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, st[x][e]);
        top = half_max(top);
        if (wave_ballot((top - m) * a.scale2 > 8.f) != 0ull) {
            const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : fast_exp2((m - m2) * a.scale2);
            sum *= f;
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[n][e] *= f;
            m = m2;
        }
        const float m0 = m == -INFINITY ? 0.f : kUnitW<T> - m * a.scale2;
#pragma unroll
        for (int x = 0; x < KW / 32; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) { w[e] = fast_exp2(fmaf(st[x][8 * y + e], a.scale2, m0)); sum += w[e]; }
                const typename T::Frag pf = to_frag<T>(w);
#pragma unroll
                for (int n = 0; n < DP / 32; n++)
                    o[n] = mma<T>(Tile<T, DP>::col(vt, base + 32 * x + 16 * y, col_at, n), pf, o[n]);
            }
        if constexpr (T::kBytes == 2) {                        // the fragments of the next 16 keys are read before the products of these
            F3M_NEXT_READS(DP / 16);
#pragma unroll
            for (int g = 0; g < KW / 16; g++) {
                if (g + 1 < KW / 16) F3M_NEXT_READS(DP / 16);
                F3M_NEXT_MMA(DP / 32);
            }
        }
    }
    sum = half_sum(sum);

    if constexpr (WK > 1) {                                  // join the wavefronts that shared the rows
        float *mem = reinterpret_cast<float *>(lds);
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
            const float f = m2 == -INFINITY ? 1.f : fast_exp2((m - m2) * a.scale2), fh = m2 == -INFINITY ? 0.f : fast_exp2((mh - m2) * a.scale2);
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
        if (sum != 0.f)
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int y = 0; y < 4; y++)
                    store4<Fp32>(rec, 32 * n + 8 * y + 4 * h, o[n][4 * y], o[n][4 * y + 1], o[n][4 * y + 2], o[n][4 * y + 3]);
        return;
    }
    const long long at = ((long long)b * a.Nq + me.row.i) * a.Hq + hk * a.G + me.row.g;
    if (a.lse != nullptr && h == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m * a.scale2 + log2f(sum * power_of_two(-kUnitW<T>))) * kLn2;
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
        const float f = fast_exp2((rec[x * step + DP] - m) * a.scale2);
        sum += part * f;
        if (2 * lane < DP) { o0 += rec[x * step + 2 * lane] * f; o1 += rec[x * step + 2 * lane + 1] * f; }
    }
    const Row row = row_of(a, r);
    const long long at = ((long long)b * a.Nq + row.i) * a.Hq + hk * a.G + row.g;
    if (a.lse != nullptr && lane == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m * a.scale2 + log2f(sum * power_of_two(-kUnitW<T>))) * kLn2;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (2 * lane >= a.D) return;
    if constexpr (T::kBytes == 2) reinterpret_cast<uint32_t *>(a.out)[at * (a.D / 2) + lane] = T::pack(o0 * inv, o1 * inv);
    else reinterpret_cast<u32x2 *>(a.out)[at * (a.D / 2) + lane] = u32x2{as_bits(o0 * inv), as_bits(o1 * inv)};
}

// lse, in units of log 2 and less kUnitP, then delta of the packed rows of one k/v head
__device__ __forceinline__ float *row_stats(const AttnArgs &a, int bh) { return a.delta + (long long)bh * 2 * a.Nq * a.G; }
// fp32 records of the sink tiles' parts, before those of the other tiles
__device__ __forceinline__ long long sink_records(const AttnArgs &a) { return a.sink_splits > 1 ? (long long)a.B * a.Hkv * a.sink_splits * a.sink_tiles * 128 : 0; }

// dS, the operand of dq and dk, as a sum of two parts: rounded once, its error and those of P and out in delta together made the gradients 1.6 times as far
// from 64 bits as a 32-bit computation rounded at its end; in two parts 1.2 times.
template <class T> constexpr int kSplitS = T::kBytes == 2 ? 2 : 1;

// fp16: P, the operand of dv, is packed with its 1 at 2^15: what is below 2^-39 of a row is lost, not what is below 2^-24 (a key that every row sees
// with less than that has an ordinary dv under a large dout).  attn_dq_kernel takes it off the stored lse; dv and dk, whose dS then carries it too, give it back at the end.
template <class T> constexpr int kUnitP = T::kId == Fp16::kId ? 15 : 0;

// fp16: dS is packed in units of a power of two, one for each column of the product (a row of q for dq, a key for dk), which is a lane's own, as
// dS = P (dP - delta) passes 65504 under a loss scale and falls below 2^-24 without one while the gradients are ordinary numbers.  As with a softmax's maximum the unit is set by the
// largest seen (to 2^13 .. 2^14) and lowered when one passes it by more than a factor of two, the sums with it.  After that the largest is 2^13 or more, and the second part
// holds what is above 2^-38 of it.  Costs a multiplication and a maximum for each dS: 2 x 4096 tokens, 16 heads of 128 on 4, window 1024, forward and gradients: 452 -> 491 us.
template <class T> struct UnitS {
    static constexpr bool kUsed = T::kId == Fp16::kId;
    int n = 113;                                             // dS is packed as dS 2^n; at first so that anything that counts lowers it
    // w: this lane's sixteen dS; sums: its accumulators
    template <int TILES> __device__ __forceinline__ void apply(f32x16 &w, f32x16 *sums)
    {
        if constexpr (kUsed) {
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(w[e]));
            top = half_max(top);
            const bool past = top > power_of_two(15 - n);
            if (wave_ballot(past) != 0ull) {
                const int to = past ? 13 - exponent_of(top) : n;
                const float f = power_of_two(to - n);
#pragma unroll
                for (int t = 0; t < TILES; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sums[t][e] *= f;
                n = to;
            }
            const float f = power_of_two(n);
#pragma unroll
            for (int e = 0; e < 16; e++) w[e] *= f;
        }
    }
    template <int TILES> __device__ __forceinline__ void undo(f32x16 *sums, int more = 0) const
    {
        if constexpr (kUsed) {
            const float f = power_of_two(-n - more);
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) sums[t][e] *= f;
        }
    }
};

// dq: the forward kernel's walk over the keys; dS^T = P^T (V dout^T - delta) is the operand of dq^T += K^T dS^T as it is.  delta_i = dout_i . out_i is
// formed here from the row of dout in registers and kept, with lse, for attn_dkv_kernel (as a kernel of its own it read dout once more: 15 of 450 us).  It is taken
// of the rounded out that the forward pass stored, in fp32: up to half a step of out's type of each of its terms, for no second pass over the keys.
// Measured: 2 x 4096 tokens, 16 heads of 128 on 4, window 1024: 150 us, 600 TFLOP/s without counting the second part of dS.
template <class T, int DP, int WM>
__global__ void __launch_bounds__(256, T::kBytes == 4 && DP > 64 ? 1 : 2) attn_dq_kernel(AttnArgs a)
{
    constexpr int WK = 4 / WM, KW = T::kBytes == 2 && WM == 4 ? 64 : 32, BK = KW * WK, BM = 32 * WM, TU = BK * kRowUnits<T, DP>;
    constexpr int REC = DP / 32 * 16 * 64;
    __shared__ u32x4 lds[4 * TU];                              // two buffers of k and v
    static_assert(WK == 1 || (WK - 1) * WM * REC / 4 <= 4 * TU, "the wavefronts' sums are joined there");
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5, wm = wave % WM, wk = wave / WM;
    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    const int nh = item / a.mtiles, bh = head_at(a, nh), b = bh / a.Hkv, hk = bh % a.Hkv;
    const int mt = a.paired && (nh & 1) ? item % a.mtiles : a.mtiles - 1 - item % a.mtiles;
    const int r0 = mt * BM, R = a.Nq * a.G;
    const Seen s = seen_by(a, b, r0, BM);
    const int tiles = (s.slots + BK - 1) / BK;

    const int row_at = Tile<T, DP>::row_lane(tile_row(l), h);
    const typename Tile<T, DP>::ColLane col_at = Tile<T, DP>::col_lane(l, h);
    const int r = r0 + 32 * wm + l;
    const LaneRow me(a, s, r, R);
    const int hq = hk * a.G + me.row.g;
    const char *qrow = a.q + (long long)b * a.qs[0] + (long long)me.row.i * a.qs[1] + (long long)hq * a.qs[2];
    const char *drow = a.dout + (long long)b * a.ds[0] + (long long)me.row.i * a.ds[1] + (long long)hq * a.ds[2];
    typename T::Frag qf[DP / 16], df[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        qf[n] = zero_frag<T>();
        df[n] = zero_frag<T>();
        if (me.live && 16 * n + 8 * h < a.D) {
            qf[n] = signed_frag<T>(*reinterpret_cast<const typename T::Frag *>(qrow + (16 * n + 8 * h) * T::kBytes), a);
            df[n] = *reinterpret_cast<const typename T::Frag *>(drow + (16 * n + 8 * h) * T::kBytes);
        }
    }
#pragma unroll
    for (int n = 0; n < DP / 16; n++) { settle(qf[n]); settle(df[n]); }
    const long long at_out = ((long long)b * a.Nq + me.row.i) * a.Hq + hq;
    float lse2 = INFINITY, delta = 0.f;                       // lse in units of log 2; +inf where the row sees nothing: its weights are then 0
    if (me.live) {
        const char *orow = a.o + at_out * a.D * T::kBytes;
#pragma unroll
        for (int n = 0; n < DP / 16; n++)
            if (16 * n + 8 * h < a.D) {
                float x[8], y[8];
                from_frag<T>(*reinterpret_cast<const typename T::Frag *>(orow + (16 * n + 8 * h) * T::kBytes), x);
                from_frag<T>(df[n], y);
#pragma unroll
                for (int e = 0; e < 8; e++) delta = fmaf(x[e], y[e], delta);
            }
        lse2 = a.lse_in[at_out] * kLog2e;
        if (lse2 == -INFINITY) lse2 = INFINITY;
    }
    delta = half_sum(delta);
    if (wk == 0 && h == 0 && r < R) {
        float *stats = row_stats(a, bh) + r;
        stats[0] = lse2 - kUnitP<T>;
        stats[(long long)R] = delta;
    }
    f32x16 dq[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) dq[n] = zero_acc();
    UnitS<T> unit;

    SlotLoader<T, DP, BK> kx, vx;
    kx.init(a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2], a.ks[1], a.D * T::kBytes);
    vx.init(a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2], a.vs[1], a.D * T::kBytes);
    if (tiles > 0) {
        kx.load(s, 0, a.near_rows);
        vx.load(s, 0, a.near_rows);
        kx.store(lds);
        vx.store(lds + TU);
        if (tiles > 1) { kx.load(s, BK, a.near_rows); vx.load(s, BK, a.near_rows); }
    }
    for (int t = 0; t < tiles; t++) {
        const u32x4 *kt = lds + (t & 1) * 2 * TU, *vt = kt + TU;
        __syncthreads();
        if (t + 1 < tiles) {
            u32x4 *next = lds + ((t + 1) & 1) * 2 * TU;
            kx.store(next);
            vx.store(next + TU);
        }
        if (t + 2 < tiles) { kx.load(s, (t + 2) * BK, a.near_rows); vx.load(s, (t + 2) * BK, a.near_rows); }
#pragma unroll
        for (int x = 0; x < KW / 32; x++) {
            const int at = wk * KW + 32 * x, u0 = t * BK + at;
            if (me.none(u0, 32)) continue;
            f32x16 st = zero_acc(), dp = zero_acc();
#pragma unroll
            for (int n = 0; n < DP / 16; n++) st = mma<T>(Tile<T, DP>::row(kt, at, row_at, n), qf[n], st);
#pragma unroll
            for (int n = 0; n < DP / 16; n++) dp = mma<T>(Tile<T, DP>::row(vt, at, row_at, n), df[n], dp);
            if constexpr (T::kBytes == 2) read_ahead<DP / 8, 1, DP / 32 + 1>();
#pragma unroll
            for (int e = 0; e < 16; e++) st[e] = fast_exp2(fmaf(st[e], a.scale2, -lse2));
            if (me.some(u0, 32)) {
#pragma unroll
                for (int e = 0; e < 16; e++) st[e] = me.sees(u0 + 16 * (e / 8) + 8 * h + e % 8) ? st[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) st[e] *= dp[e] - delta;
            unit.template apply<DP / 32>(st, dq);
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = st[8 * y + e];
                typename T::Frag sf[kSplitS<T>];
                split_frag<T, kSplitS<T>>(w, sf);
#pragma unroll
                for (int n = 0; n < DP / 32; n++) {
                    const typename T::Frag x = Tile<T, DP>::col(kt, at + 16 * y, col_at, n);
#pragma unroll
                    for (int p = 0; p < kSplitS<T>; p++) dq[n] = mma<T>(x, sf[p], dq[n]);
                }
            }
            if constexpr (T::kBytes == 2) {
                constexpr int N = DP / 16;
                F3M_NEXT_READS(4);
#pragma unroll
                for (int n = 0; n < N; n++) { F3M_NEXT_MMA(kSplitS<T>); if (n + 2 < N) F3M_NEXT_READS(2); }
            }
        }
    }
    unit.template undo<DP / 32>(dq);
    if constexpr (WK > 1) {                                  // add the sums of the wavefronts that shared the rows
        float *mem = reinterpret_cast<float *>(lds);
        __syncthreads();
        if (wk > 0) {
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) mem[((wk - 1) * WM + wm) * REC + (n * 16 + e) * 64 + lane] = dq[n][e];
        }
        __syncthreads();
        if (wk > 0) return;
        for (int w = 1; w < WK; w++)
#pragma unroll
            for (int n = 0; n < DP / 32; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) dq[n][e] += mem[((w - 1) * WM + wm) * REC + (n * 16 + e) * 64 + lane];
    }
    if (r >= R) return;
    char *out = a.dq + at_out * a.D * T::kBytes;
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
// dv^T += dout^T P, dk^T += Q^T dS.  k stays in registers, v in LDS: with both in registers only one wavefront fits a SIMD (2 x 4096 tokens, 16 heads of 128 on 4,
// window 1024: 604 us, now 240).  Two wavefronts a SIMD with all 256 registers wait half their time; P and dS are packed before the last products so that the
// next tile's rows can travel in their registers.  P is rounded once for dv, as in the forward pass, dS in two parts.  A tile of keys that holds sinks is seen by all rows behind it, many times the rows of any other under a window: its
// rows are dealt to sink_splits workgroups; calls with few keys deal the rows of every tile (tile_splits).  attn_join_kernel adds the parts in order.
template <class T, int DP>
__global__ void __launch_bounds__(256, T::kBytes == 2 ? (DP <= 64 ? 3 : 2) : 1) attn_dkv_kernel(AttnArgs a)
{
    constexpr int BR = 32, BN = 128, CPR = kRowUnits<T, DP>, TU = BR * CPR, VU = BN * CPR;
    __shared__ u32x4 lds[VU + 4 * TU];                        // v, two buffers of q and dout
    __shared__ u32x4 stat4[2][BR * 3 / 4];                 // per row: lse, -delta, position (-1: no row)
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int item = xcd_item(blockIdx.x, a.items);
    if (item >= a.items) return;
    // items of a head: the parts of its sink tiles, then those of its other tiles
    const int sink_items = a.sink_tiles * a.sink_splits, each = sink_items + (a.ktiles - a.sink_tiles) * a.tile_splits;
    const int nh = item / each, rest = item % each, bh = head_at(a, nh), b = bh / a.Hkv, hk = bh % a.Hkv;
    const bool sink = rest < sink_items;
    const int splits = sink ? a.sink_splits : a.tile_splits, nth = sink ? rest : rest - sink_items;
    const int part = nth % splits, at_tile = nth / splits + (sink ? 0 : a.sink_tiles);
    const int ktile = a.paired && (nh & 1) ? a.ktiles - 1 - at_tile : at_tile;       // paired: there are no sink tiles
    const int q_len = clamp_len(a.q_lens, b, a.Nq), kv_len = clamp_len(a.kv_lens, b, a.Nk), off = kv_len - q_len;
    const int j0 = ktile * BN, key = j0 + 32 * wave + tile_row(l);   // this order: v is read at the lane's address of q and dout
    // Rows that see some key of the tile: position j0 .. last.  0 <= ia <= ib <= q_len before the heads are counted, for tiles behind kv_len and before all windows
    // too: a row number beyond q_len, or before 0, times G may pass 32 bits and come back as a row.
    const int last = min(kv_len - 1, j0 < a.sinks ? kv_len - 1 : (int)min((long long)kv_len - 1, (long long)j0 + BN - 1 + a.window - 1));
    const int ia = j0 < kv_len ? max(0, j0 - off) : 0, ib = j0 < kv_len ? max(ia, min(q_len, last - off + 1)) : 0;
    int ra = ia * a.G, rb = ib * a.G;
    if (splits > 1) {
        const int tiles = (rb - ra + BR - 1) / BR, per = (tiles + splits - 1) / splits;
        ra = min(rb, ra + part * per * BR);
        rb = min(rb, ra + per * BR);
    }
    // keys before the first row's window are seen by no row and not read
    const int unseen = max(0, off - a.window + 1);
    const bool have = key < kv_len && ra < rb && (key >= unseen || key < a.sinks);
    const char *kb = a.k + (long long)b * a.ks[0] + (long long)hk * a.ks[2], *vb = a.v + (long long)b * a.vs[0] + (long long)hk * a.vs[2];
    typename T::Frag kf[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; n++) {
        kf[n] = zero_frag<T>();
        if (have && 16 * n + 8 * h < a.D)
            kf[n] = signed_frag<T>(*reinterpret_cast<const typename T::Frag *>(kb + (long long)key * a.ks[1] + (16 * n + 8 * h) * T::kBytes), a);
    }
    if (ra < rb)
        for (int unit = tid; unit < BN * CPR; unit += 256) {
            const int j = j0 + unit / CPR, c = unit % CPR;
            u32x4 x = zero4();
            if (j < kv_len && (j >= unseen || j < a.sinks) && 16 * c < a.D * T::kBytes) x = *reinterpret_cast<const u32x4 *>(vb + (long long)j * a.vs[1] + 16 * c);
            Tile<T, DP>::put(lds, x, unit / CPR, c);
        }
#pragma unroll
    for (int n = 0; n < DP / 16; n++) settle(kf[n]);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; n++) { dk[n] = zero_acc(); dv[n] = zero_acc(); }
    UnitS<T> unit;

    // a tile's rows in PER turns of ROWS rows: thread t takes the 16-byte piece t % CPR of row t / CPR of each
    constexpr int ROWS = 256 / CPR < BR ? 256 / CPR : BR, PER = BR / ROWS;
    const int turn = tid / CPR, piece = tid % CPR;
    const bool takes = turn < ROWS && 16 * piece < a.D * T::kBytes;
    struct Staged {                                           // a tile on its way
        u32x4 q[PER], d[PER];
        float st;                                             // threads 0 .. 31: lse of a row, 32 .. 63: -delta, 64 .. 95: position
    };
    const float *stats = row_stats(a, bh);
    const char *qb = a.q + (long long)b * a.qs[0] + (long long)(hk * a.G) * a.qs[2];
    const char *db = a.dout + (long long)b * a.ds[0] + (long long)(hk * a.G) * a.ds[2];
    const bool near_q = a.near_q && ROWS % a.G == 0;          // a turn starts with a token's first head: its offsets are the same in all
    const Row row0 = row_of(a, turn);
    const int qoff = (int)(row0.i * a.qs[1] + row0.g * a.qs[2]) + 16 * piece, doff = (int)(row0.i * a.ds[1] + row0.g * a.ds[2]) + 16 * piece;
    auto load = [&](Staged &x, int rt) {
        if (near_q) {
#pragma unroll
            for (int n = 0; n < PER; n++) {
                const long long i = (rt + n * ROWS) / a.G;
                const bool in = takes && rt + n * ROWS + turn < rb;
                x.q[n] = load16(buffer(qb + i * a.qs[1], kOutside - 16), in ? qoff : kOutside);
                x.d[n] = load16(buffer(db + i * a.ds[1], kOutside - 16), in ? doff : kOutside);
            }
        } else {
#pragma unroll
            for (int n = 0; n < PER; n++) {
                const int r = rt + n * ROWS + turn;
                x.q[n] = x.d[n] = zero4();
                if (takes && r < rb) {
                    const Row row = row_of(a, r);
                    x.q[n] = *reinterpret_cast<const u32x4 *>(qb + (long long)row.i * a.qs[1] + (long long)row.g * a.qs[2] + 16 * piece);
                    x.d[n] = *reinterpret_cast<const u32x4 *>(db + (long long)row.i * a.ds[1] + (long long)row.g * a.ds[2] + 16 * piece);
                }
            }
        }
        if (tid < 3 * BR) {
            const int r = rt + tid % BR;
            if (tid < BR) x.st = r < rb ? stats[r] : INFINITY;
            else if (tid < 2 * BR) x.st = r < rb ? -stats[(long long)a.Nq * a.G + r] : 0.f;
            else x.st = as_float((uint32_t)(r < rb ? off + row_of(a, r).i : -1));
        }
    };
    auto store = [&](const Staged &x, int buf) {
        u32x4 *qt = lds + VU + buf * 2 * TU, *dt = qt + TU;
#pragma unroll
        for (int n = 0; n < PER; n++)
            if (ROWS * CPR == 256 || turn < ROWS) {
                Tile<T, DP>::put(qt, x.q[n], n * ROWS + turn, piece);
                Tile<T, DP>::put(dt, x.d[n], n * ROWS + turn, piece);
            }
        if (tid < 3 * BR) reinterpret_cast<float *>(stat4[buf])[tid] = x.st;
    };
    const int jw = j0 + 32 * wave;                            // this wavefront's keys: jw .. jw + 31
    const int row_lane = Tile<T, DP>::row_lane(tile_row(l), h);
    const typename Tile<T, DP>::ColLane col_lane = Tile<T, DP>::col_lane(l, h);
    const int tiles = (rb - ra + BR - 1) / BR;
    if (tiles > 0) {
        Staged x;
        load(x, ra);
        store(x, 0);
    }
    for (int n = 0; n < tiles; n++) {
        Staged next;
        __syncthreads();
        const int rt = ra + n * BR, buf = n & 1;
        const u32x4 *qt = lds + VU + buf * 2 * TU, *dt = qt + TU, *stat = stat4[buf];
        // positions of the tile's first and last row
        const int pa = off + rt / a.G, pb = off + (min(rb, rt + BR) - 1) / a.G;
        const bool more = n + 1 < tiles, out = pb < jw || jw >= kv_len || (jw >= a.sinks && pa - (jw + 31) >= a.window);
        constexpr bool EARLY = DP <= 64;                       // room for the next tile beside everything else
        if (more && (EARLY || out)) load(next, rt + BR);
        if (!out) {
            const int row_at = in_loop(row_lane);
            const typename Tile<T, DP>::ColLane col_at{in_loop(col_lane.a), in_loop(col_lane.b)};
            f32x16 st = zero_acc();
#pragma unroll
            for (int n = 0; n < DP / 16; n++) st = mma<T>(Tile<T, DP>::row(qt, 0, row_at, n), kf[n], st);
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float lse[8];
                from_frag<Fp32>(Frag32{{stat[4 * y + 2 * h], stat[4 * y + 2 * h + 1]}}, lse);
#pragma unroll
                for (int e = 0; e < 8; e++) st[8 * y + e] = fast_exp2(fmaf(st[8 * y + e], a.scale2, -lse[e]));
            }
            if constexpr (T::kBytes == 2) read_ahead<DP / 16, 1, DP / 32, 4>();
            if (rt + BR > rb || jw + 31 > pa || (pb - jw >= a.window && jw + 31 >= a.sinks)) {
                const int *pos = reinterpret_cast<const int *>(stat) + 2 * BR + 8 * h;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int p = pos[16 * (e / 8) + e % 8];
                    st[e] = key <= p && (p - key < a.window || key < a.sinks) ? st[e] : 0.f;
                }
            }
            f32x16 dp;                                         // starts from -delta
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float del[8];
                from_frag<Fp32>(Frag32{{stat[BR / 4 + 4 * y + 2 * h], stat[BR / 4 + 4 * y + 2 * h + 1]}}, del);
#pragma unroll
                for (int e = 0; e < 8; e++) dp[8 * y + e] = del[e];
            }
#pragma unroll
            for (int n = 0; n < DP / 16; n++)
                dp = mma<T>(Tile<T, DP>::row(dt, 0, row_at, n), Tile<T, DP>::row(lds, 32 * wave, row_at, n), dp);
            typename T::Frag pf[2], sf[2][kSplitS<T>];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = st[8 * y + e];
                pf[y] = to_frag<T>(w);
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] *= dp[8 * y + e];
                if constexpr (!unit.kUsed) split_frag<T, kSplitS<T>>(w, sf[y]);
#pragma unroll
                for (int e = 0; e < 8; e++) st[8 * y + e] = w[e];
            }
            if constexpr (unit.kUsed) {
                unit.template apply<DP / 32>(st, dk);
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) w[e] = st[8 * y + e];
                    split_frag<T, kSplitS<T>>(w, sf[y]);
                }
            }
            // P and dS are packed here: their registers take the next tile while the last products run
#pragma unroll
            for (int y = 0; y < 2; y++) {
                settle(pf[y]);
#pragma unroll
                for (int p = 0; p < kSplitS<T>; p++) settle(sf[y][p]);
            }
            if (more && !EARLY) load(next, rt + BR);
#pragma unroll
            for (int y = 0; y < 2; y++) {
#pragma unroll
                for (int n = 0; n < DP / 32; n++) dv[n] = mma<T>(Tile<T, DP>::col(dt, 16 * y, col_at, n), pf[y], dv[n]);
#pragma unroll
                for (int n = 0; n < DP / 32; n++) {
                    const typename T::Frag x = Tile<T, DP>::col(qt, 16 * y, col_at, n);
#pragma unroll
                    for (int p = 0; p < kSplitS<T>; p++) dk[n] = mma<T>(x, sf[y][p], dk[n]);
                }
            }
            if constexpr (T::kBytes == 2) {                    // fragments DP / 32 products ahead
                F3M_NEXT_READS(DP / 16);
#pragma unroll
                for (int n = 0; n < DP / 32; n++) { F3M_NEXT_MMA(1); F3M_NEXT_READS(2); }
#pragma unroll
                for (int n = 0; n < DP / 32; n++) { F3M_NEXT_MMA(kSplitS<T>); F3M_NEXT_READS(2); }
#pragma unroll
                for (int n = 0; n < DP / 32; n++) { F3M_NEXT_MMA(1); F3M_NEXT_READS(2); }
                F3M_NEXT_MMA(DP / 32 * kSplitS<T>);
            }
        }
        if (more) store(next, buf ^ 1);
    }
    unit.template undo<DP / 32>(dk, kUnitP<T>);
    if constexpr (kUnitP<T> != 0) {
#pragma unroll
        for (int n = 0; n < DP / 32; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) dv[n][e] *= power_of_two(-kUnitP<T>);
    }
    if (key >= a.Nk) return;
    if (splits > 1) {                                         // record of a key and part: dk, dv as fp32
        const long long keys = sink ? a.sink_tiles * BN : (a.ktiles - a.sink_tiles) * BN;
        const long long first = sink ? 0 : sink_records(a);
        float *rec = a.part + (first + ((long long)bh * splits + part) * keys + (key - (sink ? 0 : a.sink_tiles * BN))) * (2 * DP);
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

// Joins the parts of the keys, in order: a thread per four elements.
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a)
{
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
    const int e = (int)(n % (2 * DP / 4)) * 4, d = e % DP;
    const long long kk = n / (2 * DP / 4);
    const int first = a.sink_tiles * 128, joined = (a.tile_splits > 1 ? a.ktiles : a.sink_tiles) * 128, key = (int)(kk % joined);
    if (kk / joined >= (long long)a.B * a.Hkv || key >= a.Nk || d >= a.D) return;
    const int bh = (int)(kk / joined), b = bh / a.Hkv, hk = bh % a.Hkv;
    const bool sink = key < first;
    const int splits = sink ? a.sink_splits : a.tile_splits, keys = sink ? first : a.ktiles * 128 - first;
    if (splits == 1) return;
    const float *rec = a.part + ((sink ? 0 : sink_records(a)) + (long long)bh * splits * keys + (sink ? key : key - first)) * (2 * DP) + e;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < splits; x++) {
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
    F3M_REQUIRE(p->B <= most && p->B * p->Hq <= most && p->Nk <= most && p->Nq <= most && p->Nq * G <= most, 3, "more than 2^30 rows, keys or heads");
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
    a.scale2 = p->scale == 0.f ? 1.f : std::fabs(p->scale) * kLog2e;          // -infinity times it has to stay -infinity
    F3M_REQUIRE(std::isfinite(a.scale2), 61, "scale %g is too large", p->scale);
    a.keep = p->scale == 0.f ? 0u : ~0u;
    a.sign = p->scale < 0.f ? (p->dtype == F3M_F32 ? 0x80000000u : 0x80008000u) : 0u;
    const long long row = p->D * e, most_step = 1 << 22;
    a.near_rows = a.ks[1] >= row && a.ks[1] <= most_step && a.vs[1] >= row && a.vs[1] <= most_step;
    auto near = [&](const long long *s) { return s[1] >= 0 && s[2] >= 0 && s[1] < (1 << 30) && s[2] < (1 << 30) && 32 / G * s[1] + G * s[2] + row < (1 << 30); };
    a.near_q = G <= 64 && near(a.qs) && near(a.ds);
    return a;
}

constexpr long long kMostItems = 1 << 23;                    // workgroups of 256 threads: a launch holds fewer than 2^32 threads

// Without a window the tiles' work differs from one to all of the keys.  Where all workgroups run at once the longest decides, and a
// compute unit that holds tiles of two heads is evened out by taking those of the second in the other order; with more
// workgroups the longest first is better (16 heads of 4096 tokens, 64 wide: forward and gradients 389 us in the same order, 313 in this).
int paired_order(const AttnArgs &a, long long items) { return a.window >= a.Nk && items <= 1024; }

// Wavefronts side by side along the rows: a call whose rows do not fill the card (512 workgroups) in pieces of 128, or of 64, gives its wavefronts
// the keys to share instead.
int row_waves(const AttnArgs &a)
{
    const long long R = (long long)a.Nq * a.G, heads = (long long)a.B * a.Hkv;
    return R > 64 && heads * ((R + 127) / 128) >= 256 ? 4 : R > 32 && heads * ((R + 63) / 64) >= 256 ? 2 : 1;
}

// A call whose rows do not fill the card either way splits the keys, at least two tiles of keys to a split.
void forward_shape(AttnArgs &a)
{
    const int wm = row_waves(a), bm = 32 * wm, bk = wm == 4 ? 64 : 32 * (4 / wm);
    const long long R = (long long)a.Nq * a.G, heads = (long long)a.B * a.Hkv;
    a.mtiles = (int)((R + bm - 1) / bm);
    const long long tokens = std::min<long long>(a.Nq, bm / a.G + 2), slots = std::min<long long>(a.Nk, (long long)a.window + tokens + a.sinks);
    const long long tiles = (slots + bk - 1) / bk, base = std::max<long long>(1, heads * a.mtiles);
    a.splits = (int)std::max<long long>(1, std::min<long long>({512 / base, tiles / 2, 64}));
    F3M_REQUIRE(heads * a.mtiles * a.splits <= kMostItems, 3, "too many rows for one call");
    a.items = (int)(heads * a.mtiles * a.splits);
    a.paired = paired_order(a, a.items);
}

// The rows of every tile of keys in parts where the tiles do not fill the card: with a window to 512 workgroups, what runs at once; without one, where the
// tiles' work differs from one to all rows, to three times as many, which evens it out.  (2 x 4096 tokens, 16 heads of 128 on 4, window 1024: dq,
// dk, dv and the forward pass 546 us with one part, 446 with two, 479 with three.  4096 tokens, 16 heads of 64, no window: 344, 321, 289, four 299.)
// A part is at least two tiles of rows; those of the sink tiles, which many more rows see, are as long as the others.
void grad_shape(AttnArgs &a)
{
    a.ktiles = (a.Nk + 127) / 128;
    a.sink_tiles = a.window < a.Nk ? std::min((a.sinks + 127) / 128, a.ktiles) : 0;     // without a window sinks are like other keys
    const long long heads = (long long)a.B * a.Hkv, items = std::max<long long>(1, heads * a.ktiles), want = a.window < a.Nk ? 512 : 1536;
    const long long rows = std::min<long long>(a.Nq, (long long)a.window + 128) * a.G, all = (long long)a.Nq * a.G;
    a.tile_splits = (int)std::max<long long>(1, std::min<long long>({(want + items / 2) / items, rows / 64, 64}));
    const long long part = std::max<long long>(1, (rows / 32 + a.tile_splits - 1) / a.tile_splits);
    a.sink_splits = (int)std::max<long long>(1, std::min<long long>(64, (all / 32 + part - 1) / part));
    F3M_REQUIRE(heads * ((long long)a.sink_tiles * a.sink_splits + (long long)(a.ktiles - a.sink_tiles) * a.tile_splits) <= kMostItems &&
                heads * ((all + 63) / 64) <= kMostItems && heads * a.sink_tiles * 128 <= (1 << 25), 3, "too many rows or keys for one call");
}
long long grad_records(const AttnArgs &a)
{
    const long long heads = (long long)a.B * a.Hkv;
    return heads * 128 * ((a.sink_splits > 1 ? a.sink_splits * a.sink_tiles : 0) + (a.tile_splits > 1 ? a.tile_splits * (a.ktiles - a.sink_tiles) : 0));
}

size_t attn_workspace(const f3m_attn_params *p, bool grad)
{
    AttnArgs a = attn_args(p);
    const size_t dp = padded(a.D);
    if (!grad) {
        forward_shape(a);
        return a.splits == 1 ? 0 : (size_t)a.B * a.Hkv * a.splits * a.Nq * a.G * (dp + 4) * 4;
    }
    grad_shape(a);
    const size_t delta = ((size_t)a.B * a.Nq * a.Hq * 8 + 255) & ~size_t(255);
    return delta + (size_t)grad_records(a) * 2 * dp * 4;
}

template <class T, int DP> void forward(const AttnArgs &a, hipStream_t s)
{
    const int wm = row_waves(a);
    const unsigned grid = xcd_grid(a.items);
    if (wm == 4) F3M_LAUNCH((attn_forward_kernel<T, DP, 4>), grid, 256, 0, s, a);
    else if (wm == 2) F3M_LAUNCH((attn_forward_kernel<T, DP, 2>), grid, 256, 0, s, a);
    else F3M_LAUNCH((attn_forward_kernel<T, DP, 1>), grid, 256, 0, s, a);
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
        const int wm = row_waves(a) == 4 ? 4 : 2;
        a.mtiles = (int)(((long long)a.Nq * a.G + 32 * wm - 1) / (32 * wm));
        a.items = (int)(heads * a.mtiles);
        a.paired = paired_order(a, a.items);
        if (wm == 4) F3M_LAUNCH((attn_dq_kernel<T, DP, 4>), xcd_grid(a.items), 256, 0, s, a);
        else F3M_LAUNCH((attn_dq_kernel<T, DP, 2>), xcd_grid(a.items), 256, 0, s, a);
        check_launch("attention's dq");
    }
    if (a.Nk > 0) {
        const int others = a.ktiles - a.sink_tiles;
        const long long items = heads * ((long long)a.sink_tiles * a.sink_splits + (long long)others * a.tile_splits);
        a.items = (int)items;
        a.paired = paired_order(a, items);
        F3M_LAUNCH((attn_dkv_kernel<T, DP>), xcd_grid(a.items), 256, 0, s, a);
        check_launch("attention's dk, dv");
        if (a.tile_splits > 1 || (a.sink_splits > 1 && a.sink_tiles > 0)) {
            const long long joined = (a.tile_splits > 1 ? a.ktiles : a.sink_tiles) * 128ll;
            F3M_LAUNCH((attn_join_kernel<T, DP>), cdiv(heads * joined * (2 * DP / 4), 256), 256, 0, s, a);
            check_launch("attention's join of gradients");
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
        forward_shape(a);
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
