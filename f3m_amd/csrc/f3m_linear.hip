// Linear attention with a decay for each head: out_t = scale sum_{s<=t} e^{g(t-s)} (q_t.k_s) v_s, a separable kernel whose
// sources are carried as moments S_t = e^g S_{t-1} + k_t v_t^T, and its gradients.
//
// A sequence is cut into chunks of C tokens.  With Z the moments of everything before a chunk, already shifted to its first token,
//     out_i  = scale (e^{g i} q_i Z + sum_{j<=i} e^{g(i-j)} (q_i.k_j) v_j)            (moments evaluated + exact sum inside the chunk)
//     Z_next = e^{g C} Z + sum_j e^{g(C-j)} k_j v_j^T                                   (moments shifted + the chunk's own)
// One workgroup walks the chunks of one head with Z in registers, a wavefront to 32 columns of v.  Sequences that are too few to
// fill the card are cut into segments that run at the same time: a first pass forms each segment's own moments, a
// scan shifts and adds them, and the walk starts from them.
//
// The gradients are the same sum: dq = product of (dout, v, k) with the moments transposed; dk and dv = products of (v, dout, q) and
// (k, q, dout) with time reversed.  Z starts from e^g S_0 forwards and from dS_T backwards, which is what makes both the same; backwards it is the gradient of the
// state, which holds scale: k_j v_j^T are then weighted with it, and q_i Z is not multiplied by it.
//
// Precision.  Z is fp32.  For the products it is split into two 16-bit parts (bf16: 2^-16 is lost).  The other operands that the inputs do not hold are rounded once where
// they reach out alone: the weights inside a chunk, and e^{g(C-j)} v_j, so that every pair of tokens meets one such rounding, an error like that of the output's own.  Final
// moments are fp32 outputs: the pass that forms them splits e^{g(C-j)} v_j into three parts (bf16) or two (fp16) and keeps fp32 accuracy (where that pass is the walk itself, with
// many heads, out gains by it a little).  fp16: each of these operands is in units of a power of two, as the results are ordinary numbers where they pass 65504 or fall below
// 2^-14: Z of a wavefront, a row of a tile of weights, a column of weighted v (with many heads of 1024 tokens, 64 wide: 80 -> 91 us; a prompt 134 -> 139).
#include "f3m_tile.h"

#include "f3m_sequence.h"

namespace f3m {

// One product: out = q (sums of k v^T).  Up to three (the gradients) run in the same launches.
struct LinearJob {
    const char *q, *k, *v;
    char *out;
    const float *init;                        // (B, H, Dk, Dv) of the product or, if transposed, (B, H, Dv, Dk); may be null
    float *fin;                               // final moments, stored as init is; may be null
    long long qs[3], ks[3], vs[3];            // strides in bytes: batch, token, head
    int reverse, transposed;                  // time reversed; init and fin are stored transposed
};
struct LinearArgs {
    LinearJob job[3];
    const float *log_decay;
    float *seg;                               // a segment's own moments, then those at the start of the next, for each product
    const int *lens;
    int jobs, B, N, H, Dk, Dv;                // Dk, Dv: of the products
    int segments, seglen, heads;              // heads = B * H
    float scale;
};
// What a workgroup works on: items run over heads, then products, then segments, so that those that read the same tokens are near each other.
struct LinearItem {
    int bh, b, head, job, sg, len, from, to;
    __device__ __forceinline__ LinearItem(const LinearArgs &a, int item, int segments)
    {
        sg = item % segments;
        job = item / segments % a.jobs;
        // an XCD takes a run of items: where they divide evenly it holds every eighth head, so that a long sequence's are spread
        const int n = item / (segments * a.jobs), per = a.heads / 8;
        bh = a.heads % 8 == 0 ? n % per * 8 + n / per : n;
        b = bh / a.H;
        head = bh % a.H;
        len = a.lens == nullptr ? a.N : min(max(a.lens[b], 0), a.N);
        from = sg * a.seglen;
        to = min(len, from + a.seglen);
    }
};
__device__ __forceinline__ float *segment_moments(const LinearArgs &a, int bh, int job, int sg, int moments)
{
    return a.seg + (((long long)bh * a.jobs + job) * a.segments + sg) * moments;
}

template <class T> constexpr int kChunk = T::kBytes == 2 ? 64 : 32;
template <class T> constexpr int kSplitZ = T::kBytes == 2 ? 2 : 1;
template <class T> constexpr int kSplitV = T::kId == 0 ? 3 : T::kId == 1 ? 2 : 1;

// e^{g n} and e^{g n} - 1; n = 0 also where g is -inf
__device__ __forceinline__ float power(float g, int n) { return n == 0 ? 1.f : expf(g * (float)n); }
__device__ __forceinline__ float power_m1(float g, int n) { return n == 0 ? 0.f : expm1f(g * (float)n); }
// z -> e^{g n} z.  Near 1 the factor's distance from 1 is what a long product of such factors lives on, and z + (e^{g n} - 1) z keeps it; far below 1 that
// difference would leave nothing of the factor's own digits (e^{-13} to 1 %).
struct Shift {
    float add, by;                            // z + add z, then times by: both in z's own registers (a branch, or z by + z add, and the walk spills)
    // e^{g n} - 1 and e^{g n}
    __device__ __forceinline__ Shift(float less1, float whole) : add(less1 > -0.5f ? less1 : 0.f), by(less1 > -0.5f ? 1.f : whole) {}
    __device__ __forceinline__ float operator()(float z) const { return fmaf(z, add, z) * by; }
};

// A sequence in walking order: token t of it is row t, or row len - 1 - t where time is reversed.
struct Walk {
    const char *base;
    long long step;
    __device__ __forceinline__ Walk(const char *p, const long long *s, int b, int h, int len, int reverse)
        : base(p + (long long)b * s[0] + (long long)h * s[2] + (reverse ? (long long)(len - 1) * s[1] : 0)), step(reverse ? -s[1] : s[1]) {}
    __device__ __forceinline__ const char *row(int t) const { return base + (long long)t * step; }
};

// Shared memory of one chunk.
template <class T, int DK, int DV, bool MAIN> struct ChunkLds {
    static constexpr int C = kChunk<T>;
    u32x4 k[C * kRowUnits<T, DK>], v[C * kRowUnits<T, DV>], q[MAIN ? C * kRowUnits<T, DK> : 1];
    u32x4 a[MAIN ? C * kRowUnits<T, C> : 1];                                     // weights inside the chunk, [q token][k token]
    float pw[C + 2];                                                             // scale e^{g n}; 0 for what is not seen
    float pz[C];                                                                 // the same for Z
    float whole;                                                                 // shift of Z over the chunk
    float unit[MAIN && T::kId == Fp16::kId ? 3 * 32 : 1];                        // fp16: of each row of each 32 x 32 tile of a
    u32x4 wt4[C / 4];                                                            // fp32: weight of token j in Z_next
    // the largest of the first n tokens: the last one's, or with a decay above 0 the first one's
    __device__ __forceinline__ float largest_weight(int n) const
    {
        const float *w = reinterpret_cast<const float *>(wt4);
        return fmaxf(fabsf(w[0]), fabsf(w[n - 1]));
    }
    __device__ __forceinline__ void set_weights(int tid, int threads, float g, int end, float by)
    {
        for (int j = tid; j < C; j += threads) {
            const float f = power(g, max(0, end - j));
            reinterpret_cast<float *>(wt4)[j] = f * by;
            if (j == 0) whole = f;
        }
    }
};

// Moves a chunk from memory to LDS by way of registers, in PER turns of ROWS tokens: thread t takes the 16-byte piece t % CPR of token t / CPR of
// each.  Tokens behind the last one and columns behind the head's are zero.
template <class T, int W, int NT> struct TokenLoader {
    static constexpr int C = kChunk<T>, CPR = kRowUnits<T, W>, ROWS = NT / CPR, PER = (C + ROWS - 1) / ROWS;
    static_assert(NT % CPR == 0, "");
    u32x4 x[PER];
    int off;                                                  // of this thread's piece in a turn
    bool near;                                                // a turn's offsets fit 32 bits
    __device__ __forceinline__ void init(const Walk &w, int row_bytes)
    {
        const int r = threadIdx.x / CPR, c = threadIdx.x % CPR;
        const long long s = w.step < 0 ? -w.step : w.step;
        near = s < (1 << 24);
        off = 16 * c >= row_bytes ? kOutside : (int)((w.step < 0 ? ROWS - 1 - r : r) * s) + 16 * c;
    }
    __device__ __forceinline__ void load(const Walk &w, int t0, int end, int row_bytes)
    {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int r = n * ROWS + threadIdx.x / CPR, c = threadIdx.x % CPR;
            const bool in = t0 + r < end && (C % ROWS == 0 || r < C);
            if (near) {                                       // from the turn's lowest address on
                const Buffer b = buffer(w.row(t0 + n * ROWS + (w.step < 0 ? ROWS - 1 : 0)), kOutside - 16);
                x[n] = load16(b, in ? off : kOutside);
            } else {
                x[n] = zero4();
                if (in && 16 * c < row_bytes) x[n] = *reinterpret_cast<const u32x4 *>(w.row(t0 + r) + 16 * c);
            }
        }
    }
    __device__ __forceinline__ void store(u32x4 *tile) const
    {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int r = n * ROWS + threadIdx.x / CPR;
            if (C % ROWS == 0 || r < C) Tile<T, W>::put(tile, x[n], r, threadIdx.x % CPR);
        }
    }
};

// fp16: a lane's column of Z is held as Z 2^n, so that the weighted v, which are rounded to fp16, have their largest at 2^8 to 2^15 in every chunk: as they stand, small
// values, and all of them under a strong decay, have few bits left or none, and Z, whose final form is an fp32 output, no more than they.  n goes up to 40 and keeps Z 2^n below 2^101.
template <class T> struct UnitZ {
    static constexpr bool kUsed = T::kId == Fp16::kId;
    int n = 0;
    // vf: N fragments of v; weight: the largest of a token; most: the largest n
    template <int TILES, int N> __device__ __forceinline__ void follow(f32x16 *z, const typename T::Frag *vf, float weight, int most)
    {
        if constexpr (kUsed) {
            const float top = half_max(largest(vf, N)) * weight;
            const bool move = n > most || top > power_of_two(15 - n) || (n < most && top > 0.f && top < power_of_two(8 - n));
            if (wave_ballot(move) != 0ull) {
                const int to = move ? min(13 - exponent_of(top), most) : n;
                const float f = power_of_two(to - n);
#pragma unroll
                for (int t = 0; t < TILES; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) z[t][e] *= f;
                n = to;
            }
        }
    }
    __device__ __forceinline__ float in() const { return kUsed ? power_of_two(n) : 1.f; }
    __device__ __forceinline__ float out() const { return kUsed ? power_of_two(-n) : 1.f; }
};
constexpr int kMostUnit = 40;

// Z += K^T (weights . V) for this wavefront's columns, the weighted v as a sum of NS parts; vf: its fragments of v, one per 16 tokens.  k's fragments
// are read AHEAD products before their use.
template <class T, int DK, int DV, int NS, class L>
__device__ __forceinline__ void add_moments(f32x16 *z, const UnitZ<T> &unit, const L &m, const typename T::Frag *vf, int l, int h)
{
    constexpr int C = kChunk<T>, TILES = DK / 32, N = C / 16 * TILES, AHEAD = T::kBytes == 4 ? 0 : N < 3 ? N : 3;
    const typename Tile<T, DK>::ColLane k_at = Tile<T, DK>::col_lane(l, h, true);
    typename T::Frag kf[N];
#pragma unroll
    for (int n = 0; n < AHEAD; n++) kf[n] = Tile<T, DK>::col(m.k, 16 * (n / TILES), k_at, n % TILES);
#pragma unroll
    for (int s = 0; s < C / 16; s++) {
        float f[8];
        from_frag<T>(vf[s], f);
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] *= as_float(m.wt4[4 * s + 2 * h + e / 4][e % 4]) * unit.in();
        typename T::Frag part[NS];
        split_frag<T, NS>(f, part);
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            const int at = s * TILES + t;
            if (at + AHEAD < N) kf[at + AHEAD] = Tile<T, DK>::col(m.k, 16 * ((at + AHEAD) / TILES), k_at, (at + AHEAD) % TILES);
            if constexpr (AHEAD > 0) F3M_FENCE();
#pragma unroll
            for (int n = 0; n < NS; n++) z[t] = mma<T>(kf[at], part[n], z[t]);
        }
    }
}

// The moments of one segment alone (from zero), shifted to the token behind it -- those of a sequence's last segment to where the final moments stand: the
// last token forwards, past it backwards -- in the wavefronts' own order: a register of all lanes at a time.
// Measured: 32 heads of 8192 tokens, 128 wide, 16 segments: 46 us, 3.6 TB/s; 38 without the products, which are not wholly hidden (three parts of v).
template <class T, int DK, int DV, bool FINAL>
__global__ void __launch_bounds__(DV * 2, DV >= 96 ? 2 : 1) linear_moments_kernel(LinearArgs a)
{
    constexpr int C = kChunk<T>, NT = DV * 2;
    __shared__ ChunkLds<T, DK, DV, false> m;
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int items = a.heads * a.jobs * a.segments, item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const LinearItem it(a, item, a.segments);
    const LinearJob &job = a.job[it.job];
    const int from = it.from, to = it.to;
    const bool last = it.len <= from + a.seglen;
    if (from >= it.len || (last && job.fin == nullptr)) return;
    const float g = a.log_decay[it.head];
    const Walk kw(job.k, job.ks, it.b, it.head, it.len, job.reverse), vw(job.v, job.vs, it.b, it.head, it.len, job.reverse);
    const typename Tile<T, DV>::ColLane v_at = Tile<T, DV>::col_lane(l, h);
    f32x16 z[DK / 32];
#pragma unroll
    for (int t = 0; t < DK / 32; t++) z[t] = zero_acc();
    UnitZ<T> unit;
    TokenLoader<T, DK, NT> kx;
    TokenLoader<T, DV, NT> vx;
    kx.init(kw, a.Dk * T::kBytes);
    vx.init(vw, a.Dv * T::kBytes);
    auto load = [&](int c0) { kx.load(kw, c0, to, a.Dk * T::kBytes); vx.load(vw, c0, to, a.Dv * T::kBytes); };
    load(from);
    int shifted = -1;
    float fm1 = 0.f;
    for (int c0 = from; c0 < to; c0 += C) {
        const int end = c0 + C < to || !last ? C : to - c0 - (job.reverse ? 0 : 1);
        __syncthreads();
        kx.store(m.k);
        vx.store(m.v);
        if (end != shifted) {
            shifted = end;
            fm1 = power_m1(g, end);
            m.set_weights(tid, NT, g, end, job.reverse ? a.scale : 1.f);
        }
        __syncthreads();
        if (c0 + C < to) load(c0 + C);
        typename T::Frag vf[C / 16];
#pragma unroll
        for (int s = 0; s < C / 16; s++) vf[s] = Tile<T, DV>::col(m.v, 16 * s, v_at, wave);
        const Shift shift(fm1, m.whole);
#pragma unroll
        for (int t = 0; t < DK / 32; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) z[t][e] = shift(z[t][e]);
        unit.template follow<DK / 32, C / 16>(z, vf, m.largest_weight(min(C, to - c0)), kMostUnit);
        add_moments<T, DK, DV, FINAL ? kSplitV<T> : 1>(z, unit, m, vf, in_loop(l), h);
    }
    float *out = segment_moments(a, it.bh, it.job, it.sg, DK * DV) + wave * DK * 32 + lane;
#pragma unroll
    for (int t = 0; t < DK / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) out[(t * 16 + e) * 64] = z[t][e] * unit.out();
}

// Where a moment in the wavefronts' order stands in init and fin; -1 if it is padding.
template <int DK, int DV> __device__ __forceinline__ int moment_index(const LinearArgs &a, const LinearJob &job, int t, int e, int wave, int lane)
{
    const int dk = 32 * t + 16 * (e / 8) + 8 * (lane / 32) + e % 8, dv = 32 * wave + lane % 32;
    return dk >= a.Dk || dv >= a.Dv ? -1 : job.transposed ? dv * a.Dk + dk : dk * a.Dv + dv;
}
// Z at the start of a sequence: e^g S_0 forwards, dS_T backwards.
__device__ __forceinline__ float first_moment(const LinearArgs &a, const LinearJob &job, int bh, float g, int at)
{
    if (job.init == nullptr || at < 0) return 0.f;
    const float s = job.init[(long long)bh * a.Dk * a.Dv + at];
    return job.reverse ? s : s * power(g, 1);
}

// From the segments' own moments to those at the start of the following segment, and the final ones; a thread per moment.  Bound by memory (32 heads,
// 16 segments of 128 x 128: 14 us for 67 MB).
template <int DK, int DV>
__global__ void __launch_bounds__(256) linear_scan_kernel(LinearArgs a)
{
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
    if (n >= (long long)a.heads * a.jobs * DK * DV) return;
    const int i = (int)(n % (DK * DV)), bj = (int)(n / (DK * DV)), bh = bj / a.jobs, nth = bj % a.jobs;
    const LinearJob &job = a.job[nth];
    const int len = a.lens == nullptr ? a.N : min(max(a.lens[bh / a.H], 0), a.N);
    const int index = moment_index<DK, DV>(a, job, i / 1024 % (DK / 32), i / 64 % 16, i / (DK * 32), i % 64);
    const float g = a.log_decay[bh % a.H];
    const Shift shift(power_m1(g, a.seglen), power(g, a.seglen));
    float z = first_moment(a, job, bh, g, index);
    float *seg = segment_moments(a, bh, nth, 0, DK * DV) + i;
    const int last = len == 0 ? 0 : (len - 1) / a.seglen;      // the segment that ends the sequence
    for (int s = 0; s < last; s += 4) {                        // four loads in flight
        float own[4];
#pragma unroll
        for (int x = 0; x < 4; x++) own[x] = s + x < last ? seg[(long long)(s + x) * (DK * DV)] : 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++)
            if (s + x < last) {
                z = own[x] + shift(z);
                seg[(long long)(s + x) * (DK * DV)] = z;
            }
    }
    if (job.fin == nullptr || index < 0) return;
    float *out = job.fin + (long long)bh * a.Dk * a.Dv + index;
    if (len == 0) *out = job.init == nullptr ? 0.f : job.init[(long long)bh * a.Dk * a.Dv + index];
    else {
        const float own = seg[(long long)last * (DK * DV)];
        const int rest = len - last * a.seglen - (job.reverse ? 0 : 1);
        *out = own + Shift(power_m1(g, rest), power(g, rest))(z);
    }
}

// The walk over the chunks of one segment: 48 of its 62 matrix instructions a chunk evaluate and carry the moments, and its vector instructions split them.
// Measured: 32 heads of 8192 tokens, 128 wide: 69 us, 63 without its loads: bound by the dependent steps of a chunk (three barriers) at two workgroups a compute unit.
// FINAL: it is the only one of a sequence and forms the final moments too.
template <class T, int DK, int DV, bool FINAL>
__global__ void __launch_bounds__(DV * 2, T::kBytes == 2 && DV >= 96 ? 2 : 1) linear_walk_kernel(LinearArgs a)
{
    constexpr int C = kChunk<T>, NT = DV * 2, NW = DV / 32, Q = C / 32;
    __shared__ ChunkLds<T, DK, DV, true> m;
    const int tid = threadIdx.x, wave = wave_uniform(tid / 64), lane = tid % 64, l = lane & 31, h = lane >> 5;
    const int items = a.heads * a.jobs * a.segments, item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const LinearItem it(a, item, a.segments);
    const LinearJob &job = a.job[it.job];
    const int bh = it.bh, sg = it.sg, len = it.len, from = it.from, to = it.to, all = min(a.N, from + a.seglen);
    const float g = a.log_decay[it.head];
    const Walk qw(job.q, job.qs, it.b, it.head, len, job.reverse), kw(job.k, job.ks, it.b, it.head, len, job.reverse), vw(job.v, job.vs, it.b, it.head, len, job.reverse);
    char *const orow = job.out + ((long long)it.b * a.N * a.H + it.head) * a.Dv * T::kBytes;
    const long long ostep = (long long)a.H * a.Dv * T::kBytes;

    // rows behind the last token
    const int line = a.Dv * T::kBytes / 16;
    for (int n = tid; n < max(0, all - max(from, to)) * line; n += NT)
        *reinterpret_cast<u32x4 *>(orow + (long long)(max(from, to) + n / line) * ostep + 16 * (n % line)) = zero4();

    f32x16 z[DK / 32];
    if (sg > 0) {
        const float *in = segment_moments(a, bh, it.job, sg - 1, DK * DV) + wave * DK * 32 + lane;
#pragma unroll
        for (int t = 0; t < DK / 32; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) z[t][e] = in[(t * 16 + e) * 64];
    } else {
#pragma unroll
        for (int t = 0; t < DK / 32; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) z[t][e] = first_moment(a, job, bh, g, moment_index<DK, DV>(a, job, t, e, wave, lane));
    }
    UnitZ<T> unit;
    for (int n = tid; n <= C + 1; n += NT) {
        const float f = n <= C ? power(g, n) : 0.f;
        m.pw[n] = f * a.scale;
        if (n < C) m.pz[n] = job.reverse ? f : f * a.scale;
    }
    TokenLoader<T, DK, NT> qx, kx;
    TokenLoader<T, DV, NT> vx;
    qx.init(qw, a.Dk * T::kBytes);
    kx.init(kw, a.Dk * T::kBytes);
    vx.init(vw, a.Dv * T::kBytes);
    int shifted = -1;
    float fm1 = 0.f;
    auto load = [&](int c0) { qx.load(qw, c0, to, a.Dk * T::kBytes); kx.load(kw, c0, to, a.Dk * T::kBytes); vx.load(vw, c0, to, a.Dv * T::kBytes); };
    if (from < to) load(from);
    const int q_lane = Tile<T, DK>::row_lane(l, h), k_lane = Tile<T, DK>::row_lane(tile_row(l), h);
    for (int c0 = from; c0 < to; c0 += C) {
        const int n = min(C, to - c0), q_at = in_loop(q_lane), k_at = in_loop(k_lane), l_in = in_loop(l);
        // forwards the final moments are those at the last token, not shifted past it
        const int end = c0 + C < to ? C : FINAL && job.fin != nullptr && !job.reverse ? n - 1 : n;
        __syncthreads();
        qx.store(m.q); kx.store(m.k); vx.store(m.v);
        if (end != shifted) {
            shifted = end;
            fm1 = power_m1(g, end);
            m.set_weights(tid, NT, g, end, job.reverse ? a.scale : 1.f);
        }
        __syncthreads();
        if (c0 + C < to) load(c0 + C);
        // weights inside the chunk: tiles of 32 k tokens x 32 q tokens on and above the diagonal, dealt to the wavefronts
#pragma unroll
        for (int pair = 0; pair < Q * (Q + 1) / 2; pair++) {
            if (pair % NW != wave) continue;
            const int kq = pair == 2 ? 1 : 0, qq = pair == 0 ? 0 : 1;
            f32x16 w = zero_acc();
#pragma unroll
            for (int s = 0; s < DK / 16; s++)
                w = mma<T>(Tile<T, DK>::row(m.k, 32 * kq, k_at, s), Tile<T, DK>::row(m.q, 32 * qq, q_at, s), w);
            if constexpr (T::kBytes == 2) read_ahead<DK / 16, 2, 2>();
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int d = 32 * (qq - kq) + l_in - (16 * (e / 8) + 8 * h + e % 8);
                w[e] *= m.pw[d < 0 ? C + 1 : d];
            }
            if constexpr (T::kId == Fp16::kId) {              // the row's largest to 2^13 .. 2^14
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(w[e]));
                const int n = exponent_of(half_max(top));
                const float f = power_of_two(13 - n);
#pragma unroll
                for (int e = 0; e < 16; e++) w[e] *= f;
                if (h == 0) m.unit[32 * pair + l] = power_of_two(n - 13);
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = w[8 * y + e];
                const typename T::Frag out = to_frag<T>(f);
                const int c = (32 * kq + 16 * y + 8 * h) / kPer16<T>;
                if constexpr (T::kBytes == 2) Tile<T, C>::put(m.a, out, 32 * qq + l, c);
                else { Tile<T, C>::put(m.a, out.v[0], 32 * qq + l, c); Tile<T, C>::put(m.a, out.v[1], 32 * qq + l, c + 1); }
            }
        }
        // moments evaluated at the chunk's tokens: out^T (rows: columns of v) = Z^T Q^T
        f32x16 o[Q];
#pragma unroll
        for (int y = 0; y < Q; y++) o[y] = zero_acc();
        float down = 1.f, up = 1.f;
        int most = kMostUnit;
        if constexpr (T::kId == Fp16::kId) {
            float top = 0.f;
#pragma unroll
            for (int t = 0; t < DK / 32; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(z[t][e]));
            top *= unit.out();
            for (int y = 32; y >= 1; y >>= 1) top = fmaxf(top, wave_shfl_xor_f(top, y));
            // one power of two for all of the wavefront's moments, which brings the largest to 2^13 .. 2^14
            const int ex = exponent_of(top);
            down = power_of_two(13 - ex - unit.n);
            up = power_of_two(ex - 13);
            most = min(most, 100 - ex);
        }
        {
            constexpr int N = Q * (DK / 16), AHEAD = T::kBytes == 4 ? 0 : N < 3 ? N : 3;
            typename T::Frag qf[N];
#pragma unroll
            for (int x = 0; x < AHEAD; x++) qf[x] = Tile<T, DK>::row(m.q, 32 * (x % Q), q_at, x / Q);
#pragma unroll
            for (int s = 0; s < DK / 16; s++) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = z[s / 2][8 * (s % 2) + e] * (unit.kUsed ? down : 1.f);
                typename T::Frag part[kSplitZ<T>];
                split_frag<T, kSplitZ<T>>(f, part);
#pragma unroll
                for (int y = 0; y < Q; y++) {
                    const int at = s * Q + y;
                    if (at + AHEAD < N) qf[at + AHEAD] = Tile<T, DK>::row(m.q, 32 * ((at + AHEAD) % Q), q_at, (at + AHEAD) / Q);
                    if constexpr (AHEAD > 0) F3M_FENCE();
#pragma unroll
                    for (int p = 0; p < kSplitZ<T>; p++) o[y] = mma<T>(part[p], qf[at], o[y]);
                }
            }
        }
#pragma unroll
        for (int y = 0; y < Q; y++) {
            const float f = m.pz[32 * y + l] * (unit.kUsed ? up : 1.f);
#pragma unroll
            for (int e = 0; e < 16; e++) o[y][e] *= f;
        }
        typename T::Frag vf[C / 16];
        const typename Tile<T, DV>::ColLane v_at = Tile<T, DV>::col_lane(l_in, h);
        const int a_at = Tile<T, C>::row_lane(l_in, h);
#pragma unroll
        for (int s = 0; s < C / 16; s++) vf[s] = Tile<T, DV>::col(m.v, 16 * s, v_at, wave);
        // moments at the end of the chunk
        const Shift shift(fm1, m.whole);
#pragma unroll
        for (int t = 0; t < DK / 32; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) z[t][e] = shift(z[t][e]);
        unit.template follow<DK / 32, C / 16>(z, vf, m.largest_weight(n), most);
        add_moments<T, DK, DV, FINAL ? kSplitV<T> : 1>(z, unit, m, vf, l_in, h);
        __syncthreads();
        // out^T += V^T A^T
#pragma unroll
        for (int y = 0; y < Q; y++) {
#pragma unroll
            for (int x = 0; x < y + 1; x++) {
                f32x16 sum = T::kId == Fp16::kId ? zero_acc() : o[y];
#pragma unroll
                for (int s = 2 * x; s < 2 * (x + 1); s++)
                    sum = mma<T>(vf[s], Tile<T, C>::row(m.a, 32 * y, a_at, s), sum);
                if constexpr (T::kId == Fp16::kId) {
                    const float f = m.unit[32 * (x + y) + l];  // pair of the tile: 0; 1, 2
#pragma unroll
                    for (int e = 0; e < 16; e++) o[y][e] = fmaf(sum[e], f, o[y][e]);
                } else o[y] = sum;
            }
            const int t = c0 + 32 * y + l;
            if (t < to) {
                char *row = orow + (long long)(job.reverse ? len - 1 - t : t) * ostep;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int d = 32 * wave + 8 * e + 4 * h;
                    if (d < a.Dv) store4<T>(row, d, o[y][4 * e], o[y][4 * e + 1], o[y][4 * e + 2], o[y][4 * e + 3]);
                }
            }
        }
    }
    if (!FINAL || job.fin == nullptr) return;
    if (len == 0) {                                          // nothing moved: what was given comes back
        const long long moments = (long long)a.Dk * a.Dv;
        for (long long n = tid; n < moments; n += NT) job.fin[bh * moments + n] = job.init == nullptr ? 0.f : job.init[bh * moments + n];
        return;
    }
    const float f = unit.out();
#pragma unroll
    for (int t = 0; t < DK / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int at = moment_index<DK, DV>(a, job, t, e, wave, lane);
            if (at >= 0) job.fin[(long long)bh * a.Dk * a.Dv + at] = z[t][e] * f;
        }
}

// One token, bound by reading and writing the state once (4096 states of 128 x 128: 107 us, 5.06 TB/s; 4 states of 64 x 64: 4 us): a workgroup per head, a thread to four columns of v and every (threads / columns)-th row of the state.
template <class T>
__global__ void __launch_bounds__(256) linear_step_kernel(LinearArgs a, float *state)
{
    const LinearJob &job = a.job[0];
    __shared__ u32x4 part[256];
    const int bh = blockIdx.x, b = bh / a.H, head = bh % a.H, tid = threadIdx.x;
    const int cols = a.Dv / 4, rows = 256 / cols, c = tid % cols, r0 = tid / cols;
    const float f = power(a.log_decay[head], 1);
    const char *q = job.q + (long long)b * job.qs[0] + (long long)head * job.qs[2], *k = job.k + (long long)b * job.ks[0] + (long long)head * job.ks[2];
    const char *v = job.v + (long long)b * job.vs[0] + (long long)head * job.vs[2];
    auto at = [](const char *p, int i) {
        if constexpr (T::kBytes == 4) return reinterpret_cast<const float *>(p)[i];
        else return T::lo(reinterpret_cast<const uint16_t *>(p)[i]);
    };
    float o[4] = {0.f, 0.f, 0.f, 0.f}, x[4];
    if (r0 < rows) {
        for (int j = 0; j < 4; j++) x[j] = at(v, 4 * c + j);
        u32x4 *s = reinterpret_cast<u32x4 *>(state + (long long)bh * a.Dk * a.Dv) + c;
        for (int r = r0; r < a.Dk; r += rows) {
            const float kr = at(k, r), qr = at(q, r);
            u32x4 w = s[(long long)r * cols];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float n = fmaf(as_float(w[j]), f, kr * x[j]);
                w[j] = as_bits(n);
                o[j] = fmaf(qr, n, o[j]);
            }
            s[(long long)r * cols] = w;
        }
    }
    part[tid] = u32x4{as_bits(o[0]), as_bits(o[1]), as_bits(o[2]), as_bits(o[3])};
    __syncthreads();
    if (tid >= cols) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < rows; r++)
        for (int j = 0; j < 4; j++) sum[j] += as_float(part[r * cols + c][j]);
    store4<T>(job.out + (long long)bh * a.Dv * T::kBytes, 4 * c, sum[0] * a.scale, sum[1] * a.scale, sum[2] * a.scale, sum[3] * a.scale);
}

// ---- host ------------------------------------------------------------------------------------------------
namespace {

int padded(int D) { return (D + 31) / 32 * 32; }

LinearArgs linear_args(const f3m_linear_params *p)
{
    F3M_REQUIRE(p != nullptr, 8, "params is NULL");
    F3M_REQUIRE(p->dtype >= F3M_BF16 && p->dtype <= F3M_F32, 61, "dtype must be F3M_BF16, F3M_F16 or F3M_F32 (got %d)", p->dtype);
    F3M_REQUIRE(p->Dk >= 8 && p->Dk <= 128 && p->Dk % 8 == 0 && p->Dv >= 8 && p->Dv <= 128 && p->Dv % 8 == 0, 2,
                "head sizes must be multiples of 8 up to 128 (got %d and %d)", p->Dk, p->Dv);
    F3M_REQUIRE(p->B >= 0 && p->N >= 0 && p->H >= 1, 3, "bad shape");
    F3M_REQUIRE(p->N <= (1ll << 30) && p->B <= (1ll << 22) && p->B * p->H <= (1ll << 22), 3, "more than 2^30 tokens or 2^22 sequences x heads");
    F3M_REQUIRE(std::isfinite(p->scale) && p->scale != 0.f, 61, "scale must be finite and not 0");
    LinearArgs a = {};
    a.B = (int)p->B; a.N = (int)p->N; a.H = p->H; a.Dk = p->Dk; a.Dv = p->Dv; a.heads = a.B * a.H; a.scale = p->scale;
    return a;
}

LinearJob linear_job(int bytes, const void *q, const int64_t *qs, const void *k, const int64_t *ks, const void *v, const int64_t *vs, void *out,
                     const float *init, float *fin, bool reverse, bool transposed)
{
    LinearJob j = {(const char *)q, (const char *)k, (const char *)v, (char *)out, init, fin, {}, {}, {}, reverse, transposed};
    for (int i = 0; i < 3; i++) { j.qs[i] = qs[i] * bytes; j.ks[i] = ks[i] * bytes; j.vs[i] = vs[i] * bytes; }
    return j;
}

// Segments: two workgroups fit a compute unit, 512 fill the card (32 heads of 8192 tokens, 128 wide: 144 us at half as many, 125, 140 at 768).  A
// segment costs another reading of k and v, its moments (fp32) and two more launches, so that from some number of products on one is better.  That number was found on
// the gradients of 64 heads of 2048 tokens, 192 products, with the forward pass (one segment 212 us, two 229, four 216), and there alone: for forward passes of 176
// to 255 heads, and other lengths, it is not measured.
void linear_shape(LinearArgs &a, int dtype, int jobs)
{
    const int C = dtype == F3M_F32 ? 32 : 64;
    const long long chunks = (a.N + C - 1) / C;
    const long long products = std::max(1, a.heads * jobs);
    const long long want = products >= 176 ? 1 : std::max<long long>(1, std::min<long long>(512 / products, chunks));
    const long long per = std::max<long long>(1, (chunks + want - 1) / want);
    a.seglen = (int)per * C;
    a.segments = (int)std::max<long long>(1, (chunks + per - 1) / per);
}

// The gradients are two launches of products where Dk and Dv differ, one after the other in the same memory: three products bound both.
size_t linear_workspace(const f3m_linear_params *p, bool grad)
{
    LinearArgs a = linear_args(p);
    const int jobs = grad ? 3 : 1;
    linear_shape(a, p->dtype, jobs);
    return a.segments == 1 ? 0 : (size_t)a.heads * jobs * a.segments * padded(a.Dk) * padded(a.Dv) * 4;
}

template <class T, int DK, int DV> void walk_sized(const LinearArgs &a, hipStream_t s)
{
    const long long products = (long long)a.heads * a.jobs;
    bool fin = false;
    for (int j = 0; j < a.jobs; j++) fin = fin || a.job[j].fin != nullptr;
    if (a.segments > 1) {
        if (fin) F3M_LAUNCH((linear_moments_kernel<T, DK, DV, true>), xcd_grid(products * a.segments), DV * 2, 0, s, a);
        else F3M_LAUNCH((linear_moments_kernel<T, DK, DV, false>), xcd_grid(products * a.segments), DV * 2, 0, s, a);
        check_launch("linear attention's moments");
        F3M_LAUNCH((linear_scan_kernel<DK, DV>), cdiv(products * DK * DV, 256), 256, 0, s, a);
        check_launch("linear attention's scan");
    }
    if (fin && a.segments == 1) F3M_LAUNCH((linear_walk_kernel<T, DK, DV, true>), xcd_grid(products), DV * 2, 0, s, a);
    else F3M_LAUNCH((linear_walk_kernel<T, DK, DV, false>), xcd_grid(products * a.segments), DV * 2, 0, s, a);
    check_launch("linear attention");
}

template <typename F> void with_32(int D, F f)
{
    const int dp = padded(D);
    if (dp == 32) f(std::integral_constant<int, 32>{});
    else if (dp == 64) f(std::integral_constant<int, 64>{});
    else if (dp == 96) f(std::integral_constant<int, 96>{});
    else f(std::integral_constant<int, 128>{});
}

void walk(const LinearArgs &a, int dtype, hipStream_t s)
{
    if (a.heads == 0) return;
    with_type(dtype, [&](auto t) {
        with_32(a.Dk, [&](auto dk) {
            with_32(a.Dv, [&](auto dv) { walk_sized<decltype(t), decltype(dk)::value, decltype(dv)::value>(a, s); });
        });
    });
}

void check_linear(const f3m_linear_params *p, const void *q, const void *k, const void *v, const float *log_decay)
{
    const int e = p->dtype == F3M_F32 ? 4 : 2;
    if (p->B > 0 && p->N > 0) { check_16(q, "q"); check_16(k, "k"); check_16(v, "v"); }
    F3M_REQUIRE(log_decay != nullptr, 8, "log_decay is NULL");
    check_strides(p->q_stride, e, "q");
    check_strides(p->k_stride, e, "k");
    check_strides(p->v_stride, e, "v");
}

void check_workspace(const f3m_linear_params *p, bool grad, const void *workspace, size_t bytes)
{
    const size_t need = linear_workspace(p, grad);
    if (need > 0) check_16(workspace, "workspace");
    F3M_REQUIRE(bytes >= need, 62, "workspace of %zu bytes, %zu are needed", bytes, need);
}

}  // namespace
}  // namespace f3m

using namespace f3m;

extern "C" {

int f3m_linear_attention_workspace(const f3m_linear_params *params, int grad, size_t *bytes)
{
    return guarded_async([&] {
        F3M_REQUIRE(bytes != nullptr, 8, "bytes is NULL");
        *bytes = linear_workspace(params, grad != 0);
    });
}

int f3m_linear_attention(const f3m_linear_params *params, const void *q, const void *k, const void *v, const float *log_decay,
                         const float *initial_state, const int32_t *lens, void *out, float *final_state, void *workspace,
                         size_t workspace_bytes, void *stream)
{
    return guarded_async([&] {
        LinearArgs a = linear_args(params);
        check_linear(params, q, k, v, log_decay);
        if (a.heads == 0) return;
        if (a.N > 0) check_16(out, "out");
        linear_shape(a, params->dtype, 1);
        check_workspace(params, false, workspace, workspace_bytes);
        a.job[0] = linear_job(params->dtype == F3M_F32 ? 4 : 2, q, params->q_stride, k, params->k_stride, v, params->v_stride, out, initial_state,
                              final_state, false, false);
        a.jobs = 1; a.log_decay = log_decay; a.lens = lens; a.seg = (float *)workspace;
        walk(a, params->dtype, (hipStream_t)stream);
    });
}

int f3m_linear_attention_grad(const f3m_linear_params *params, const void *q, const void *k, const void *v,
                              const float *log_decay, const float *initial_state, const void *dout, const float *dfinal_state,
                              const int32_t *lens, void *dq, void *dk, void *dv, float *dinitial_state, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    return guarded_async([&] {
        LinearArgs a = linear_args(params);
        check_linear(params, q, k, v, log_decay);
        const int e = params->dtype == F3M_F32 ? 4 : 2;
        check_strides(params->dout_stride, e, "dout");
        if (a.heads == 0) return;
        if (a.N > 0) { check_16(dout, "dout"); check_16(dq, "dq"); check_16(dk, "dk"); check_16(dv, "dv"); }
        linear_shape(a, params->dtype, 3);
        check_workspace(params, true, workspace, workspace_bytes);
        const int64_t *qs = params->q_stride, *ks = params->k_stride, *vs = params->v_stride, *os = params->dout_stride;
        const LinearJob of_q = linear_job(e, dout, os, v, vs, k, ks, dq, initial_state, nullptr, false, true);
        const LinearJob of_k = linear_job(e, v, vs, dout, os, q, qs, dk, dfinal_state, nullptr, true, true);
        const LinearJob of_v = linear_job(e, k, ks, q, qs, dout, os, dv, dfinal_state, dinitial_state, true, false);
        a.log_decay = log_decay; a.lens = lens; a.seg = (float *)workspace;
        const int Dk = a.Dk, Dv = a.Dv;
        if (Dk == Dv) {
            a.jobs = 3; a.job[0] = of_q; a.job[1] = of_k; a.job[2] = of_v;
            walk(a, params->dtype, (hipStream_t)stream);
        } else {
            a.jobs = 2; a.job[0] = of_q; a.job[1] = of_k;
            a.Dk = Dv; a.Dv = Dk;
            walk(a, params->dtype, (hipStream_t)stream);
            a.jobs = 1; a.job[0] = of_v;
            a.Dk = Dk; a.Dv = Dv;
            walk(a, params->dtype, (hipStream_t)stream);
        }
    });
}

int f3m_linear_attention_step(const f3m_linear_params *params, const void *q, const void *k, const void *v,
                              const float *log_decay, float *state, void *out, void *stream)
{
    return guarded_async([&] {
        LinearArgs a = linear_args(params);
        F3M_REQUIRE(a.N == 1, 3, "a step takes one token (N = %d)", a.N);
        check_linear(params, q, k, v, log_decay);
        if (a.heads == 0) return;
        check_16(state, "state"); check_16(out, "out");
        a.job[0] = linear_job(params->dtype == F3M_F32 ? 4 : 2, q, params->q_stride, k, params->k_stride, v, params->v_stride, out, nullptr, nullptr, false, false);
        a.log_decay = log_decay;
        with_type(params->dtype, [&](auto t) {
            F3M_LAUNCH((linear_step_kernel<decltype(t)>), a.heads, 256, 0, (hipStream_t)stream, a, state);
        });
        check_launch("linear attention's step");
    });
}

}  // extern "C"
