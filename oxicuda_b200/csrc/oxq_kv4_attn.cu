// Attention of query tokens over the paged 4-bit cache (layout: oxq_kv4.cuh), for few query rows per kv head.
//
// The mathematics.  With k^ = c s + m per group, the score of a query row q (in units of log2) is
//     x = scale log2(e) * sum over groups ( s * (q . c)_group + m * (sum of q)_group ),
// so the product runs on the codes themselves and scale and offset are applied to its result in f32: the keys are never
// rounded.  Likewise o = sum p v^ = sum (p s) c + sum p m: the second product's left factor is w = p s, its right factor
// the codes; the offsets' sum is kept beside it in f32.  A code is used as the f16 number with those bits, the subnormal
// c * 2^-24 (16 c * 2^-24 for a nibble four bits up): one AND per two codes, exact, and the power of two is taken out again
// in f32.  The matrix instruction lines products up by the operands' exponent fields, where a subnormal has the least normal
// one, and cuts them 2^-25 below that: the higher a code lies in the mantissa, the more of the other factor's bits are kept.
// So the keys' codes lie two bits up, 4 c * 2^-24 and 64 c * 2^-24: one shift a word more (1.4% of the large calls), and the
// log-sum-exp is off by 2e-7 of itself in place of 1.3e-6 (f16 queries, 4 keys; an f32 product of unpacked keys: 1.3e-7).
// The values' lie so for f16 outputs only; bf16's own step hides what is cut.  q enters as f16 scaled per row by a power of two, so that the row's largest element lies in
// [2^11, 2^12): exact, but for elements below 2^-21 of the row's largest, which are off by at most 2^-32 of it.
// The running reference M of a row is the maximum over its keys of x + log2(largest s of the value rows of the key and of
// its three companions 8, 16 and 24 places apart, rounded down, at least -15); it moves only when a key exceeds it by 2^5, which
// one vote per 32 keys finds out.  p is taken 2^10 above it: w stays below 2^16 whatever the scales are (s ends 2^-11 short of
// the next power of two, so at 65504 at most), and a group or a key whose s is small beside the others' keeps bits of its w.
// w is off by 2^-25, 2^-35 of the largest, at worst, and as much again is cut from each product: a group 2^-19 of the other
// one is as good as if it stood alone (tested; in the root mean square, bf16 outputs).  l = sum p, the
// offsets' sum and all accumulators are f32.  bf16 outputs take w rounded once to f16 (2^-11, an eighth of their own step).
// f16 outputs are finer than one f16 rounding of w; for them w is split into two f16 terms (two products).
//
// The shape.  mma.sync m16n8k16 with the keys as the 16 rows and 8 query rows as the columns (a kv head's query heads, and
// the tokens of a run): S^T = K Q^T, then O^T = V^T P^T; P^T moves from accumulator to operand layout by movmatrix.
// Four warps of a CTA take 32 keys each of a tile of 128, the other four of the next tile; bulk copies bring the tiles into a
// ring in shared memory, LEAD of them ahead, issued by the warps in turn (a warp for nothing else would cost the others a
// quarter of their registers).  All tiles of all (sequence, kv head, block of query rows) items lie on one line, which the
// CTAs cut into equal parts (lengths are known on the device only).  An item that lies inside one part is finished there; of a
// cut one every CTA leaves o, M and l in the workspace and a second kernel joins them, in the order of the keys, so
// results do not depend on timing.
//
// What bounds it: about 300 instructions per 16 keys at 16 warps on an SM, half of them on the logic pipe, which issues at
// half rate (32 sequences of 50 to 16000 keys, 8 kv heads of 128: 77 us, the tiles alone stream in 56, their bytes need 47;
// 4 x 131072 keys: 111, 87, 80).  f16 queries, with two products for a weight: 88 and 127, at 128 registers and 4 bytes spilled
// for two groups.  A single short call is latency: 3.5 us to find the work, 2 to the first tiles, 4 for the join.
#include "oxq_kv4_attn.cuh"
#include "oxq_tc.cuh"

namespace oxq {
namespace kv4 {

constexpr int TILE = 128;               // keys per tile: 4 warps x 32
constexpr int MIN_TILES = 2;            // tiles a CTA takes at least: a join of many small parts costs more than it brings
constexpr float ABOVE = 10.0f, MOVES = 5.0f;    // log2: how far above the reference p is taken, and by how much the reference may be exceeded
constexpr int SETUP = 6;                // what an item costs besides its tiles, in tiles (six ragged batches at 3, 4, 5, 6, 8: 79.1, 76.4, 76.9, 75.9, 77.2 us for the first)

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lo_f32(uint32_t v) { return __low2float(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float hi_f32(uint32_t v) { return __high2float(*reinterpret_cast<const __half2*>(&v)); }
// floor(log2(s)) of the largest of the words' low halves, non-negative f16 numbers; -15 for those below 2^-14
template <int NG> __device__ __forceinline__ float log2_floor(const uint32_t (&v)[4][NG]) {
    __half2 m = *reinterpret_cast<const __half2*>(&v[0][0]);
#pragma unroll
    for (int i = 1; i < 4 * NG; i++) m = __hmax2(m, *reinterpret_cast<const __half2*>(&v[i / NG][i % NG]));
    return (float)((int)((*reinterpret_cast<const uint32_t*>(&m) >> 10) & 31u) - 15);
}
template <int N> __device__ __forceinline__ void lds_words(uint32_t (&r)[N], const unsigned char* p) {
    if constexpr (N == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); r[0] = v.x; r[1] = v.y; }
    else r[0] = *reinterpret_cast<const uint32_t*>(p);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The tiles of one item (row block rt), and the steps of all items of a kv head: an item is p.setup steps and one for each tile.
struct Span { int first, tiles; int lo, hi; };          // first tile, how many (at least one), visible positions [lo, hi)
__device__ __forceinline__ Span item_span(const AttnParams& p, const SeqInfo& q, int rt, int nr) {
    Span s;
    const int j0 = p.by_per.div(rt * nr), j1 = p.by_per.div(min((rt + 1) * nr, q.n * p.per) - 1);
    s.hi = p.causal ? min(q.len, q.before + j1 + 1) : q.len;
    s.lo = max(0, window_start(p, q.before + j0));
    s.hi = max(s.hi, 0);
    s.first = min(s.lo, s.hi) / TILE;
    s.tiles = max(1, (s.hi + TILE - 1) / TILE - s.first);
    return s;
}
__device__ __forceinline__ int row_blocks(const AttnParams& p, const SeqInfo& q, int nr) { return (q.n * p.per + nr - 1) / nr; }
__device__ __forceinline__ int head_steps(const AttnParams& p, const SeqInfo& q, int nr) {
    int t = 0;
    for (int rt = 0, e = row_blocks(p, q, nr); rt < e; rt++) t += p.setup + item_span(p, q, rt, nr).tiles;
    return t;
}
// Rows of this kernel: those of sequences with at most row_limit of them (0: all); the other kernel takes the rest.
__device__ __forceinline__ SeqInfo small_seq(const AttnParams& p, int b) {
    SeqInfo q = seq_info(p, b);
    if (p.row_limit > 0 && (int64_t)q.n * p.per > p.row_limit) q.n = 0;
    return q;
}

// The line of steps, cut into `parts` parts that differ by one step at most.
struct Line {
    int total, parts, each, more;
    __device__ __forceinline__ int bound(int k) const { return each * k + min(k, more); }
    __device__ __forceinline__ int part_of(int step) const {
        const int wide = more * (each + 1);
        return step < wide ? step / (each + 1) : more + (step - wide) / each;
    }
};
struct Where { int b, at; };            // sequence, and the line's position of its first step

// The line, and the sequence that holds step bound(k), if k < parts.  Whole CTA of 256 threads: a scan over 256 sequences at a
// time, once for the total and, where there are more of them, once again for the place.
__device__ __forceinline__ Line find_part(const AttnParams& p, int nr, int ctas, int k, int* red, Where* found) {
    Line line;
    int want = -1;
    if (threadIdx.x == 0) *found = Where{0, 0};
    for (int pass = 0; pass < 2; pass++) {
        int base = 0, mine = 0, start = 0;
        for (int b0 = 0; b0 < p.s.seqs; b0 += 256) {
            const int b = b0 + (int)threadIdx.x;
            mine = b < p.s.seqs ? head_steps(p, small_seq(p, b), nr) * p.c.heads : 0;
            int x = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if ((threadIdx.x & 31) >= o) x += y;
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 31) red[threadIdx.x >> 5] = x;
            __syncthreads();
            start = base + x - mine;
#pragma unroll
            for (int w = 0; w < 8; w++) {
                const int v = red[w];
                if (w < (int)(threadIdx.x >> 5)) start += v;
                base += v;
            }
            if (pass == 1 && mine > 0 && start <= want && want < start + mine) { found->b = b; found->at = start; }
        }
        if (pass == 1) break;
        line.total = base;
        line.parts = base ? min(ctas, max(1, base / (MIN_TILES + p.setup))) : 0;
        line.each = line.parts ? (int)((unsigned)base / (unsigned)line.parts) : 0;
        line.more = base - line.each * line.parts;
        if (k >= line.parts) return line;
        want = line.bound(k);
        if (p.s.seqs <= 256) {
            if (mine > 0 && start <= want && want < start + mine) { found->b = threadIdx.x; found->at = start; }
            break;
        }
    }
    __syncthreads();
    return line;
}

// An item of a sequence: which one holds step `in_seq` of the sequence's own line.
struct Item { int head, rt, start; Span span; };
__device__ __forceinline__ Item find_item(const AttnParams& p, const SeqInfo& q, int nr, int in_seq) {
    Item it;
    const int per_head = head_steps(p, q, nr);
    it.head = (int)((unsigned)in_seq / (unsigned)per_head);
    it.start = it.head * per_head;
    for (it.rt = 0;; it.rt++) {
        it.span = item_span(p, q, it.rt, nr);
        if (in_seq < it.start + p.setup + it.span.tiles) return it;
        it.start += p.setup + it.span.tiles;
    }
}

template <int NT> struct Slot {         // what a cut item's CTA leaves: o [rows][D], then M, l
    static constexpr int ROWS = NT * 8;
    __host__ __device__ static constexpr int floats(int d) { return ROWS * (d + 2); }
};
// Each CTA's note for the join: the item that begins in its part and goes on in the next ones; last < 0: there is none.
struct alignas(16) Cut { int start, n, block, last; };     // the sequence's first row and how many, head * row blocks + row block

// Part of the tiles of one item that a CTA works on.
struct Work {
    Where w; SeqInfo seq; int seq_steps, at, end;
    Item it; int ta, tb;
    __device__ __forceinline__ bool next(const AttnParams& p, int nr) {
        while (at < end) {
            while (at >= w.at + seq_steps) {                          // on to the next sequence that has any
                w.at += seq_steps;
                if (++w.b >= p.s.seqs) return false;                  // cannot happen: `end` is within the line
                seq = small_seq(p, w.b);
                seq_steps = head_steps(p, seq, nr) * p.c.heads;
            }
            it = find_item(p, seq, nr, at - w.at);
            const int pos = at - w.at - it.start, all = p.setup + it.span.tiles, upto = min(all, pos + (end - at));
            ta = max(0, pos - p.setup);
            tb = max(0, upto - p.setup);
            at += upto - pos;
            if (tb > ta) return true;                                 // else only steps of its setup are here, and its tiles in the next part
        }
        return false;
    }
};

// One stage of the ring: a tile's codes and params, key after key, and for each 16 keys whether they are there.
template <int D, int NG> struct Stage {
    static constexpr int KC = 0, VC = KC + TILE * (D / 2), KP = VC + TILE * (D / 2), VP = KP + TILE * NG * 4, BYTES = VP + TILE * NG * 4;
};
template <int D, int NG, int NT>
struct Smem {
    static constexpr int ROWS = NT * 8, QPAD = D + 8, STAGES = 5, LEAD = 3;
    unsigned char ring[STAGES][Stage<D, NG>::BYTES];
    __half q[ROWS * QPAD];              // per eight elements in the order 0 4 1 5 2 6 3 7, the odd ones / 16
    float slab[4][ROWS * (D + 8)];
    float a[ROWS], bsum[ROWS][NG];      // scale log2(e) 2^(22 + e - 11), scale log2(e) * sum of q
    float m[8][ROWS], l[8][ROWS];
    uint64_t bars[2 * STAGES];
    unsigned char there[STAGES][8];
    int red[8];
    Where found;
    Work work[2];                       // this piece and the next: kept here, so that the main loop has the registers
};

template <typename T, int D, int NG, int NT>
__global__ void __launch_bounds__(256, NT == 1 ? 2 : 1) kv4_attn_rows_kernel(AttnParams p) {
    using Sm = Smem<D, NG, NT>;
    using St = Stage<D, NG>;
    constexpr bool SPLIT = Elem<T>::kDtype == OXQ_F16;
    constexpr int ROWS = NT * 8, NB = D / 32, NS = D / 64, QPAD = D + 8, OPAD = D + 8, STAGES = Sm::STAGES, LEAD = Sm::LEAD;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    const uint32_t bars = tc::smem_u32(sm.bars);
    const auto full = [&](int s) { return bars + 8 * s; };
    const auto empty = [&](int s) { return bars + 8 * (STAGES + s); };
    if (tid == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; s++) { tc::mbar_init(full(s), 1); tc::mbar_init(empty(s), 4); }
        tc::fence_barrier_init();
    }
    pdl_trigger();
    pdl_wait();

    const Line line = find_part(p, ROWS, gridDim.x, blockIdx.x, sm.red, &sm.found);
    if (tid == 0) reinterpret_cast<Cut*>(p.ws)[blockIdx.x] = Cut{0, 0, 0, -1};
    if ((int)blockIdx.x >= line.parts) return;
    float* slots = p.ws + gridDim.x * (sizeof(Cut) / sizeof(float));
    Work wk;
    wk.at = line.bound(blockIdx.x);
    wk.end = line.bound(blockIdx.x + 1);
    wk.w = sm.found;
    wk.seq = small_seq(p, wk.w.b);
    wk.seq_steps = head_steps(p, wk.seq, ROWS) * p.c.heads;
    bool ok = true;

    // One tile of `wk` into the ring as the CTA's tile number `number`, by this warp: lane = 4 * chunk + array.  The warps
    // take turns; the table's entry for a warp's next turn is fetched a turn ahead.
    const int chunk = min(1 << p.c.page_shift, TILE), arr = lane & 3, off = (lane >> 2) * chunk;
    int page = 0;
    struct { const int32_t* table; int head, first, lo, hi, tb; } src;                // of the piece whose tiles are being brought
    const auto fetch_page = [&](int i) {
        const int key = (src.first + i) * TILE + off;
        if (i < src.tb && off < TILE && key < src.hi && key + chunk > src.lo) page = src.table[key >> p.c.page_shift];
    };
    const auto bring = [&](int i, uint32_t number) {
        const int key = (src.first + i) * TILE + off, slot = number % STAGES;
        const bool wanted = off < TILE && key < src.hi && key + chunk > src.lo;
        const bool good = wanted && page >= 0 && page < p.c.pages;
        if (wanted && !good && arr == 0) *p.status = OXQ_ERR_INVALID_ARGUMENT;
        if (ok && !tc::mbar_wait_warp(empty(slot), (number / STAGES & 1) ^ 1)) { ok = false; if (lane == 0) *p.status = OXQ_ERR_DEVICE_TIMEOUT; }
        if (!ok) return;
        if (arr == 0 && off < TILE)
            for (int k = 0; k < chunk; k += 16) sm.there[slot][(off + k) >> 4] = good && key + k < src.hi && key + k + 16 > src.lo ? 1 : 0;
        const int row_bytes = arr < 2 ? D / 2 : NG * 4;
        const uint32_t bytes = good ? chunk * row_bytes : 0;
        const uint32_t all = __reduce_add_sync(0xffffffffu, bytes);
        __syncwarp();                                                 // what the lanes wrote goes before lane 0's arrival
        if (lane == 0) tc::mbar_arrive_expect_tx(full(slot), all);
        __syncwarp();
        if (good) {
            const unsigned char* from = arr == 0 ? p.c.kc : arr == 1 ? p.c.vc : reinterpret_cast<const unsigned char*>(arr == 2 ? p.c.kp : p.c.vp);
            const uint32_t to = arr == 0 ? St::KC : arr == 1 ? St::VC : arr == 2 ? St::KP : St::VP;
            const int64_t row = (((int64_t)page * p.c.heads + src.head) << p.c.page_shift) + (key & ((1 << p.c.page_shift) - 1));
            tc::bulk_load(tc::smem_u32(&sm.ring[slot][to]) + off * row_bytes, from + row * row_bytes, bytes, full(slot));
        }
    };
    uint32_t count = 0;                                               // of the CTA's tiles: the next one to use
    // Tile number t is for the group t & 1 of four warps; it is brought by warp (t >> 1) & 3 of the other group, LEAD = 3 tiles
    // before, when that group has just left the slot.
    const int group = warp >> 2;
    const auto prime = [&](const Work& wk) {                          // the first tiles of a new piece of work
        src = {p.s.table + (int64_t)wk.w.b * p.s.width, wk.it.head, wk.it.span.first, wk.it.span.lo, wk.it.span.hi, wk.tb};
        const int i = wk.ta + (int)((2 * (warp & 3) + 1 - group - count) & 7);
        fetch_page(i);
        if (i < wk.tb && i < wk.ta + LEAD) {
            bring(i, count + i - wk.ta);
            fetch_page(i + 8);
        }
    };

    // The rows of a piece of work, requested a piece ahead: D / 8 threads a row, eight elements each.
    Vec16<T> query;
    const auto fetch_rows = [&](const Work& wk) {
        const int row = wk.it.rt * ROWS + tid / (D / 8);
        *reinterpret_cast<uint4*>(&query) = make_uint4(0, 0, 0, 0);
        if (tid < ROWS * (D / 8) && row < wk.seq.n * p.per) {
            const T* src = (const T*)p.q + (int64_t)(wk.seq.start + p.by_per.div(row)) * p.q_ts + (int64_t)(wk.it.head * p.per + p.by_per.mod(row)) * p.q_hs + tid % (D / 8) * 8;
            if (p.q_vec) query = ld16_written(src);
            else
#pragma unroll
                for (int e = 0; e < 8; e++) query.v[e] = src[e];
        }
    };

    bool more = wk.next(p, ROWS);
    if (more) fetch_rows(wk);
    __syncthreads();                                                  // the barriers are set up
    if (more) prime(wk);
    for (int turn = 0; more; turn ^= 1) {
        const int ta = wk.ta, tb = wk.tb, len = wk.seq.len, before = wk.seq.before, first = wk.it.span.first;
        const int row0 = wk.it.rt * ROWS;
        // keys that every row of the block sees need no mask
        const int pos0 = before + p.by_per.div(row0), pos1 = before + p.by_per.div(min(row0 + ROWS, wk.seq.n * p.per) - 1);
        const int all_hi = p.causal ? min(len, pos0 + 1) : len, all_lo = window_start(p, pos1);

        // ---- the query rows
        __syncthreads();
        if (tid < ROWS * (D / 8)) {
            const int row = tid / (D / 8), g = tid % (D / 8);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = Elem<T>::to_f32(query.v[e]);
            float top = 0.0f, sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) { top = fmaxf(top, fabsf(f[e])); sum += f[e]; }
#pragma unroll
            for (int o = 1; o < D / 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
            for (int o = 1; o < D / 8 / NG; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int ex = max((int)(__float_as_uint(top) >> 23) - 127, -116);                      // 2^(11 - ex) has to be a number
            const float up = pow2_of(max(11 - ex, -126));
            uint4 o;
            o.x = pack_f16(f[0] * up, f[4] * up); o.y = pack_f16(f[1] * up * 0.0625f, f[5] * up * 0.0625f);
            o.z = pack_f16(f[2] * up, f[6] * up); o.w = pack_f16(f[3] * up * 0.0625f, f[7] * up * 0.0625f);
            *reinterpret_cast<uint4*>(&sm.q[row * QPAD + g * 8]) = o;
            if (g == 0) sm.a[row] = p.scale_log2 * pow2_of(min(ex, 127)) * 0x1p11f;       // 2^(22 - 11 + ex) itself may be beyond f32
            if (g % (D / 8 / NG) == 0) sm.bsum[row][g / (D / 8 / NG)] = p.scale_log2 * sum;
        }
        if (tid == 0) sm.work[turn] = wk;
        __syncthreads();

        // ---- this warp's constants and accumulators; columns 2 c and 2 c + 1 of each block of eight rows are this lane's
        float2 qa[NT], qb[NT][NG], M[NT], l[NT], po[NT][NG];
        float acc[NS * 4][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            qa[nt] = make_float2(sm.a[nt * 8 + 2 * c], sm.a[nt * 8 + 2 * c + 1]);
            M[nt] = both(-1e30f); l[nt] = both(0.0f);
#pragma unroll
            for (int g = 0; g < NG; g++) { qb[nt][g] = make_float2(sm.bsum[nt * 8 + 2 * c][g], sm.bsum[nt * 8 + 2 * c + 1][g]); po[nt][g] = both(0.0f); }
        }
#pragma unroll
        for (int i = 0; i < NS * 4; i++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][nt][e] = 0.0f;

        for (int i = ta + (int)((group - count) & 1); i < tb; i += 2) {
            const uint32_t number = count + i - ta;
            const int stage = number % STAGES;
            if (ok && !tc::mbar_wait(full(stage), number / STAGES & 1)) { ok = false; *p.status = OXQ_ERR_DEVICE_TIMEOUT; }
            __syncwarp();
            if (i + LEAD < tb && (int)((number + LEAD) >> 1 & 3) == (warp & 3)) {
                bring(i + LEAD, number + LEAD);
                fetch_page(i + LEAD + 8);
            }
            const uint32_t there = *reinterpret_cast<const uint16_t*>(&sm.there[stage][2 * (warp & 3)]);
            if (__all_sync(0xffffffffu, ok) && there) {
                const int t0 = (first + i) * TILE + (warp & 3) * 32;
                const unsigned char* ring = sm.ring[stage] + (warp & 3) * (32 * (D / 2));
                const unsigned char* kc = ring + St::KC + r * (D / 2) + c * (D / 8);
                const unsigned char* vc = ring + St::VC + 2 * c * (D / 2) + r * (D / 16);
                const unsigned char* pp = sm.ring[stage] + St::KP + ((warp & 3) * 32 + r) * (NG * 4);
                // ---- x = scores of keys t0 + r + 8 h; sixteen keys are one matrix instruction's
                float2 x[NT][4];
                uint32_t vp[4][NG];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t k[2][NB], kp[2][NG];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        lds_words(k[h], kc + (16 * u + 8 * h) * (D / 2));
                        lds_words(kp[h], pp + (16 * u + 8 * h) * (NG * 4));
                        lds_words(vp[2 * u + h], pp + (St::VP - St::KP) + (16 * u + 8 * h) * (NG * 4));
                    }
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        float s4[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) s4[nt][e] = 0.0f;
#pragma unroll
                        for (int i2 = 0; i2 < NB / NG; i2++) {
                            const int blk = g * (NB / NG) + i2;
                            const uint32_t w0 = k[0][blk] << 2, w1 = k[1][blk] << 2, u0 = k[0][blk] >> 6, u1 = k[1][blk] >> 6;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint4 qf = *reinterpret_cast<const uint4*>(&sm.q[(nt * 8 + r) * QPAD + blk * 32 + c * 8]);
                                mma_16816(s4[nt], w0 & 0x003C003Cu, w1 & 0x003C003Cu, w0 & 0x03C003C0u, w1 & 0x03C003C0u, qf.x, qf.y);
                                mma_16816(s4[nt], u0 & 0x003C003Cu, u1 & 0x003C003Cu, u0 & 0x03C003C0u, u1 & 0x03C003C0u, qf.z, qf.w);
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float ks = lo_f32(kp[h][g]), km = hi_f32(kp[h][g]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                x[nt][2 * u + h] = make_float2(fmaf(s4[nt][2 * h] * ks, qa[nt].x, g == 0 ? km * qb[nt][0].x : fmaf(km, qb[nt][g].x, x[nt][2 * u + h].x)),
                                                               fmaf(s4[nt][2 * h + 1] * ks, qa[nt].y, g == 0 ? km * qb[nt][0].y : fmaf(km, qb[nt][g].y, x[nt][2 * u + h].y)));
                        }
                    }
                }
                if (t0 < all_lo || t0 + 32 > all_hi || there != 0x0101u) {
                    const int lo = *reinterpret_cast<volatile int*>(&sm.work[turn].it.span.lo);        // the first key that the block sees; kept out of registers
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const int t = t0 + r + 8 * h;
                        const bool have = t < len && t >= lo && (there >> (8 * (h >> 1)) & 1u);
                        if (!have)                                    // places behind the last key, in front of the first one seen, and absent ones, hold anything
#pragma unroll
                            for (int g = 0; g < NG; g++) vp[h][g] = 0;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int pos = before + p.by_per.div(row0 + nt * 8 + 2 * c + e);      // the row's own position
                                const int vhi = p.causal ? min(len, pos + 1) : len, vlo = window_start(p, pos);
                                if (t < vlo || t >= vhi || !have) (e ? x[nt][h].y : x[nt][h].x) = -INFINITY;
                            }
                    }
                }
                // ---- the rows' reference
                float large = log2_floor(vp);                         // of this lane's four keys
                const float most = ABOVE + MOVES - large;
                bool over = false;
                float2 y[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float top = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        y[nt][h] = make_float2(x[nt][h].x - M[nt].x, x[nt][h].y - M[nt].y);
                        top = fmaxf(top, fmaxf(y[nt][h].x, y[nt][h].y));
                    }
                    over |= top > most;
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float2 top = make_float2(-INFINITY, -INFINITY);
#pragma unroll
                        for (int h = 0; h < 4; h++) top = make_float2(fmaxf(top.x, x[nt][h].x + large), fmaxf(top.y, x[nt][h].y + large));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            top.x = fmaxf(top.x, __shfl_xor_sync(0xffffffffu, top.x, o));
                            top.y = fmaxf(top.y, __shfl_xor_sync(0xffffffffu, top.y, o));
                        }
                        top = make_float2(fmaxf(top.x - ABOVE, M[nt].x), fmaxf(top.y - ABOVE, M[nt].y));
                        const float2 f = make_float2(exp2_approx(M[nt].x - top.x), exp2_approx(M[nt].y - top.y));
                        M[nt] = top;
                        l[nt].x *= f.x; l[nt].y *= f.y;
#pragma unroll
                        for (int g = 0; g < NG; g++) { po[nt][g].x *= f.x; po[nt][g].y *= f.y; }
#pragma unroll
                        for (int q = 0; q < NS * 4; q++) { acc[q][nt][0] *= f.x; acc[q][nt][1] *= f.y; acc[q][nt][2] *= f.x; acc[q][nt][3] *= f.y; }
#pragma unroll
                        for (int h = 0; h < 4; h++) y[nt][h] = make_float2(x[nt][h].x - top.x, x[nt][h].y - top.y);
                    }
                }
                // ---- p, its sums, and w = p s as the second product's operand
                uint32_t wb[NT][NG][4], wc[NT][NG][4];
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    float2 e2[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        e2[nt] = make_float2(exp2_approx(y[nt][h].x), exp2_approx(y[nt][h].y));
                        l[nt].x += e2[nt].x; l[nt].y += e2[nt].y;
                    }
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        const float vs = lo_f32(vp[h][g]), vm = hi_f32(vp[h][g]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            po[nt][g] = make_float2(fmaf(e2[nt].x, vm, po[nt][g].x), fmaf(e2[nt].y, vm, po[nt][g].y));
                            const float2 w = make_float2(e2[nt].x * vs, e2[nt].y * vs);
                            const uint32_t hi = pack_f16(w.x, w.y);
                            wb[nt][g][h] = transpose_8x8(hi);
                            if constexpr (SPLIT) wc[nt][g][h] = transpose_8x8(pack_f16(w.x - lo_f32(hi), w.y - hi_f32(hi)));
                        }
                    }
                }
                // ---- O^T: rows r and r + 8 of block (s, j) are elements 64 s + 8 r + 2 j and + 1, the second one times 16 (or the first, where the values are two bits down)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t v[4][NS];
#pragma unroll
                    for (int h = 0; h < 4; h++) lds_words(v[h], vc + (16 * u + (h & 1) + (h >> 1) * 8) * (D / 2));
#pragma unroll
                    for (int s = 0; s < NS; s++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            constexpr uint32_t kSel[4] = {0x4400u, 0x5511u, 0x6622u, 0x7733u};
                            const int g = NG == 1 ? 0 : s;
                            // every byte is there twice in its half; two bits down, its low nibble lies at the top of the mantissa
                            constexpr uint32_t kLow = SPLIT ? 0x03C003C0u : 0x000F000Fu, kHigh = SPLIT ? 0x003C003Cu : 0x00F000F0u;
                            const uint32_t b0 = __byte_perm(v[0][s], v[1][s], kSel[j]) >> (SPLIT ? 2 : 0), b1 = __byte_perm(v[2][s], v[3][s], kSel[j]) >> (SPLIT ? 2 : 0);
                            const uint32_t a0 = b0 & kLow, a1 = b0 & kHigh, a2 = b1 & kLow, a3 = b1 & kHigh;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma_16816(acc[s * 4 + j][nt], a0, a1, a2, a3, wb[nt][g][2 * u], wb[nt][g][2 * u + 1]);
                                if constexpr (SPLIT) mma_16816(acc[s * 4 + j][nt], a0, a1, a2, a3, wc[nt][g][2 * u], wc[nt][g][2 * u + 1]);
                            }
                        }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(empty(stage));
        }
        count += tb - ta;
        const Work done = sm.work[turn];
        if (tid == 0 && done.ta == 0 && done.tb < done.it.span.tiles)  // an item that begins here and goes on: the CTA's last piece
            reinterpret_cast<Cut*>(p.ws)[blockIdx.x] = Cut{done.seq.start, done.seq.n, done.it.head * row_blocks(p, done.seq, ROWS) + done.it.rt,
                                                           line.part_of(done.w.at + done.it.start + p.setup + done.it.span.tiles - 1)};
        wk = done;
        more = wk.next(p, ROWS);
        if (more) fetch_rows(wk);

        // ---- join the warps: common reference (M was ABOVE below it), then four slabs, two warps each one after the other
        constexpr float kDown = 0x1p-10f, kLow = (SPLIT ? 0x1p18f : 0x1p24f) * kDown, kHigh = (SPLIT ? 0x1p22f : 0x1p20f) * kDown;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            M[nt].x += ABOVE; M[nt].y += ABOVE;
            l[nt].x *= kDown; l[nt].y *= kDown;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l[nt].x += __shfl_xor_sync(0xffffffffu, l[nt].x, o);
                l[nt].y += __shfl_xor_sync(0xffffffffu, l[nt].y, o);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    po[nt][g].x += __shfl_xor_sync(0xffffffffu, po[nt][g].x, o);
                    po[nt][g].y += __shfl_xor_sync(0xffffffffu, po[nt][g].y, o);
                }
            }
            if (r == 0) {
                *reinterpret_cast<float2*>(&sm.m[warp][nt * 8 + 2 * c]) = M[nt];
                *reinterpret_cast<float2*>(&sm.l[warp][nt * 8 + 2 * c]) = l[nt];
            }
        }
        __syncthreads();
        // Only now, when every warp has left the ring: a parity wait tells a phase from the one before it, not from the one two
        // before, and nothing else keeps a warp that is done from running that far ahead of a slow one of its own group.  In the
        // loop above the order does it: tile t + 3 is brought after t has been seen, into the place of t - 2 that the same warp
        // has seen before, so whoever has seen t + 3 may wait for t + 5 in the place of t.
        if (more) prime(wk);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            if ((warp >> 2) == half) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int row = nt * 8 + 2 * c + e;
                        float top = sm.m[0][row];
#pragma unroll
                        for (int q = 1; q < 8; q++) top = fmaxf(top, sm.m[q][row]);
                        const float f = exp2_approx((e ? M[nt].y : M[nt].x) - top);
#pragma unroll
                        for (int s = 0; s < NS; s++) {
                            const float2 pg = po[nt][NG == 1 ? 0 : s];
                            const float off = (e ? pg.y : pg.x) * (f * kDown);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                float2& at = *reinterpret_cast<float2*>(&sm.slab[warp & 3][row * OPAD + 64 * s + 8 * r + 2 * j]);
                                float2 o;
                                o.x = fmaf(acc[s * 4 + j][nt][e] * kLow, f, off);
                                o.y = fmaf(acc[s * 4 + j][nt][e + 2] * kHigh, f, off);
                                if (half) { o.x += at.x; o.y += at.y; }
                                at = o;
                            }
                        }
                    }
            }
            __syncthreads();
        }
        const bool whole = done.ta == 0 && done.tb == done.it.span.tiles;
        const int rows = min(ROWS, done.seq.n * p.per - done.it.rt * ROWS);
        float* slot = whole ? nullptr : slots + (int64_t)(blockIdx.x * 2 + (done.ta > 0 ? 0 : 1)) * Slot<NT>::floats(D);
        for (int i = tid; i < ROWS * (D / 4); i += 256) {
            const int row = i / (D / 4), d = (i % (D / 4)) * 4;
            float top = sm.m[0][row];
#pragma unroll
            for (int q = 1; q < 8; q++) top = fmaxf(top, sm.m[q][row]);
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; q++) sum = fmaf(sm.l[q][row], exp2_approx(sm.m[q][row] - top), sum);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float4 v = *reinterpret_cast<const float4*>(&sm.slab[q][row * OPAD + d]);
                o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
            }
            if (slot) {
                *reinterpret_cast<float4*>(slot + row * D + d) = o;
                if (d == 0) { slot[ROWS * D + row] = top; slot[ROWS * D + ROWS + row] = sum; }
            } else if (row < rows) {
                store_row<T>(p, done.seq, done.it.head, done.it.rt * ROWS + row, d, make_float2(o.x, o.y), top, sum);
                store_row<T>(p, done.seq, done.it.head, done.it.rt * ROWS + row, d + 2, make_float2(o.z, o.w), top, sum);
            }
        }
    }
    if (!ok) {                                                        // a wait ran out: what was asked for still has to land, with a limit
        const uint64_t t0 = tc::globaltimer_ns();
        while (tc::globaltimer_ns() - t0 < 1000000ull) { }
    }
}

// Joins the parts of the items that the CTAs' boundaries cut: block x takes the one that begins in CTA x.  512 threads: eight
// rows at a time, and GROUPS sets of threads that share their parts.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(512) kv4_attn_join_kernel(AttnParams p) {
    constexpr int ROWS = NT * 8, D4 = D / 4, GROUPS = 512 / (8 * D4);
    __shared__ float4 part_o[GROUPS][8][D4];
    __shared__ float2 part_ml[GROUPS][8];
    pdl_trigger();
    pdl_wait();
    const int4 note = *reinterpret_cast<const int4*>(reinterpret_cast<const Cut*>(p.ws) + blockIdx.x);
    const int first = blockIdx.x, last = min(note.w, (int)gridDim.x - 1);
    if (last < 0) return;
    const SeqInfo seq = {note.x, note.y, 0, 0};
    const int blocks = row_blocks(p, seq, ROWS), head = note.z / blocks, row0 = (note.z - head * blocks) * ROWS, rows = min(ROWS, seq.n * p.per - row0);
    const float* slots = p.ws + (gridDim.x) * (sizeof(Cut) / sizeof(float));
    const auto slot = [&](int k) { return slots + (int64_t)(k * 2 + (k == first ? 1 : 0)) * Slot<NT>::floats(D); };
    const int group = threadIdx.x / (8 * D4), rr = threadIdx.x / D4 % 8, d = threadIdx.x % D4 * 4;
    for (int r0 = 0; r0 < rows; r0 += 8) {
        const int row = r0 + rr;
        float top = -1e30f, sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const auto take = [&](float m, float l, const float4& v) {
            const float now = fmaxf(top, m), f = exp2_approx(top - now), g = exp2_approx(m - now);
            top = now;
            sum = fmaf(sum, f, l * g);
            o.x = fmaf(o.x, f, v.x * g); o.y = fmaf(o.y, f, v.y * g); o.z = fmaf(o.z, f, v.z * g); o.w = fmaf(o.w, f, v.w * g);
        };
        for (int k0 = first + group; k0 <= last; k0 += 4 * GROUPS) {  // four parts' loads at a time
            float m[4], l[4];
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float* s = slot(min(k0 + u * GROUPS, last));
                m[u] = s[ROWS * D + row]; l[u] = s[ROWS * D + ROWS + row]; v[u] = *reinterpret_cast<const float4*>(s + row * D + d);
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (k0 + u * GROUPS <= last) take(m[u], l[u], v[u]);
        }
        __syncthreads();
        part_o[group][rr][d / 4] = o;
        if (d == 0) part_ml[group][rr] = make_float2(top, sum);
        __syncthreads();
        if (group == 0 && row < rows) {
#pragma unroll
            for (int g = 1; g < GROUPS; g++) take(part_ml[g][rr].x, part_ml[g][rr].y, part_o[g][rr][d / 4]);
            store_row<T>(p, seq, head, row0 + row, d, make_float2(o.x, o.y), top, sum);
            store_row<T>(p, seq, head, row0 + row, d + 2, make_float2(o.z, o.w), top, sum);
        }
    }
}

}  // namespace kv4
}  // namespace oxq

using namespace oxq;
using namespace oxq::kv4;

static int attn_ctas(const oxq_handle* h, int nt) { return h->sm_count * (nt == 1 ? 2 : 1); }

template <typename T, int D, int NG, int NT>
static int32_t launch_rows(oxq_handle* h, const AttnParams& p, int64_t most_tiles, int64_t item_tiles) {
    const int ctas = (int)(most_tiles < attn_ctas(h, NT) ? most_tiles : attn_ctas(h, NT));
    auto kernel = kv4_attn_rows_kernel<T, D, NG, NT>;
    constexpr int bytes = (int)sizeof(Smem<D, NG, NT>);
    static OxqPerDevice ready;
    if (!ready.get(h->device)) {
        OXQ_CUDA(h, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        ready.set(h->device, 1);
    }
    OXQ_CUDA(h, oxq_launch(kernel, ctas, 256, bytes, h->stream, p));
    if (ctas > 1 && item_tiles > MIN_TILES + SETUP) OXQ_CUDA(h, oxq_launch(kv4_attn_join_kernel<T, D, NT>, ctas, 512, 0, h->stream, p));
    return OXQ_OK;
}

template <typename T, int NT>
static int32_t launch_dims(oxq_handle* h, const oxq_kv4_cache* cc, const AttnParams& p, int64_t most_tiles, int64_t item_tiles) {
    if (cc->dim == 64) return launch_rows<T, 64, 1, NT>(h, p, most_tiles, item_tiles);
    if (cc->group == 64) return launch_rows<T, 128, 2, NT>(h, p, most_tiles, item_tiles);
    return launch_rows<T, 128, 1, NT>(h, p, most_tiles, item_tiles);
}

// Which kernels a call needs.  Up to ROWS_MOST query rows per sequence and kv head go to the kernel above, more to the tiles of
// oxq_kv4_tiles.cu.  A batch may hold both kinds, and only the device knows its sequences, so with more than one both kernels
// are launched and each takes its own; a single sequence goes whole to the one that its bound asks for, and so does a batch
// whose sequences must all be as long as the longest, by the number of tokens (3 x 1000 tokens: 218 us with the second kernel, 211
// without).
constexpr int64_t ROWS_MOST = 64;
struct Plan {
    int nt;                             // blocks of 8 or 16 query rows: 16 where a sequence has more than 8, because the codes are unpacked once for all of them
    bool rows, tiles;
    int64_t items; int parts;           // tile kernel: most pairs of blocks; CTAs an item
    size_t rows_bytes, bytes;
};
static Plan make_plan(const oxq_handle* h, const oxq_kv4_cache* cc, const oxq_kv4_batch* s, int64_t per, int64_t max_tokens) {
    Plan f;
    const int64_t all_rows = s->tokens * per, max_rows = (max_tokens > 0 && max_tokens < s->tokens ? max_tokens : s->tokens) * per;
    f.nt = max_rows <= 8 ? 1 : 2;
    f.tiles = max_rows > ROWS_MOST;
    const bool alike = s->seqs == 1 || (max_tokens > 0 && s->tokens / max_tokens >= s->seqs);
    f.rows = !f.tiles || !alike;
    f.rows_bytes = f.rows ? (size_t)attn_ctas(h, f.nt) * 2 * (f.nt == 1 ? Slot<1>::floats(cc->dim) : Slot<2>::floats(cc->dim)) * sizeof(float) + attn_ctas(h, f.nt) * sizeof(Cut) : 0;
    f.items = 0; f.parts = 1;
    if (f.tiles) {
        const int64_t with = all_rows / (ROWS_MOST + 1) < s->seqs ? all_rows / (ROWS_MOST + 1) : s->seqs;
        f.items = s->seqs == 1 ? (all_rows + 255) / 256 : all_rows / 256 + (f.rows ? with : s->seqs);
        // too few CTAs for the machine: several share an item's keys (at least four tiles each of the longest the table allows)
        const int64_t ctas = f.items * cc->heads, most = s->table_width * cc->page_size / (4 * TILE);
        int64_t parts = ctas > 0 && ctas * 2 <= h->sm_count ? h->sm_count / ctas : 1;
        if (parts > most) parts = most;
        if (parts > 16) parts = 16;
        f.parts = parts < 1 ? 1 : (int)parts;
    }
    f.bytes = f.rows_bytes + (f.parts > 1 ? (size_t)f.items * cc->heads * f.parts * oxq_kv4_tiles_slot_bytes(cc->dim) : 0);
    return f;
}

extern "C" {

int32_t oxq_kv4_attention_workspace_bytes(oxq_handle* h, const oxq_kv4_cache* cache, const oxq_kv4_batch* batch, int64_t q_heads, int64_t max_tokens,
                                          size_t* bytes_out) {
    OXQ_CHECK_HANDLE(h);
    Pool c; Batch s;
    if (int32_t rc = oxq_kv4_check(h, cache, batch, &c, &s)) return rc;
    if (!bytes_out) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "null size");
    if (q_heads <= 0 || q_heads % c.heads != 0) OXQ_FAIL(h, OXQ_ERR_DIMENSION_MISMATCH, "kv4 attention: %lld query heads over %d kv heads", (long long)q_heads, c.heads);
    if (max_tokens < 0) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 attention: negative max_tokens");
    *bytes_out = s.tokens == 0 || s.seqs == 0 ? 0 : make_plan(h, cache, batch, q_heads / c.heads, max_tokens).bytes;       // such a call does nothing
    return OXQ_OK;
}

int32_t oxq_kv4_attention(oxq_handle* h, const oxq_kv4_cache* cache, const oxq_kv4_batch* batch, const oxq_kv4_attention_args* a, void* workspace,
                          size_t workspace_bytes) {
    OXQ_CHECK_HANDLE(h);
    AttnParams p;
    memset(&p, 0, sizeof(p));
    if (int32_t rc = oxq_kv4_check(h, cache, batch, &p.c, &p.s)) return rc;
    if (!a) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: null arguments");
    if (a->dtype != OXQ_BF16 && a->dtype != OXQ_F16) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: queries are bf16 or f16, got dtype %d", a->dtype);
    if (a->q_heads <= 0 || a->q_heads % p.c.heads != 0)
        OXQ_FAIL(h, OXQ_ERR_DIMENSION_MISMATCH, "kv4 attention: %lld query heads over %d kv heads", (long long)a->q_heads, p.c.heads);
    if (a->window < 0 || (a->window > 0 && !a->causal)) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: a window must be positive, and needs the causal mask");
    if (!(a->scale > -3.0e38f && a->scale < 3.0e38f)) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: the scale is not finite");
    if (a->max_tokens < 0) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 attention: negative max_tokens");
    if (p.s.tokens == 0 || p.s.seqs == 0) return OXQ_OK;
    if (!a->q || !a->out) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: null queries or output");
    if (a->q == a->out) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: the output lies over the queries, which other CTAs may still read");
    if (a->q_token_stride < 0 || a->q_head_stride < 0 || a->out_token_stride < 0 || a->out_head_stride < 0)
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: negative stride");
    // the strides of a single token or head are never used
    const int64_t q_ts = p.s.tokens > 1 ? a->q_token_stride : 0, q_hs = a->q_heads > 1 ? a->q_head_stride : 0;
    const int64_t o_ts = p.s.tokens > 1 ? a->out_token_stride : 0, o_hs = a->q_heads > 1 ? a->out_head_stride : 0;
    // output rows that lie over one another would be written by several CTAs at once: the far stride has to pass all near rows
    const bool heads_near = p.s.tokens == 1 || (a->q_heads > 1 && o_hs <= o_ts);
    const int64_t near_rows = heads_near ? a->q_heads : p.s.tokens, near_stride = heads_near ? o_hs : o_ts;
    const int64_t far_rows = heads_near ? p.s.tokens : a->q_heads, far_stride = heads_near ? o_ts : o_hs;
    if ((near_rows > 1 && near_stride < cache->dim) ||
        (far_rows > 1 && (far_stride < cache->dim || (near_rows > 1 && (far_stride - cache->dim) / (near_rows - 1) < near_stride))))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: output rows overlap");
    if (((uintptr_t)a->out | (uintptr_t)(o_ts * 2) | (uintptr_t)(o_hs * 2)) & 3u)
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 attention: output rows must be 4-byte aligned");
    const int64_t per = a->q_heads / p.c.heads;
    if (p.s.tokens * per > INT32_MAX / 2) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 attention: too many query rows");
    const Plan plan = make_plan(h, cache, batch, per, a->max_tokens);
    if (plan.items * p.c.heads * plan.parts > INT32_MAX) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 attention: more row blocks than one call counts");
    if ((plan.bytes && !workspace) || workspace_bytes < plan.bytes || ((uintptr_t)workspace & 15u))
        OXQ_FAIL(h, OXQ_ERR_BUFFER_TOO_SMALL, "kv4 attention: workspace of %zu bytes (16-byte aligned), got %zu", plan.bytes, workspace ? workspace_bytes : (size_t)0);
    if (int32_t rc = oxq_require_sm100(h)) return rc;
    OxqDeviceGuard guard(h->device);
    p.q = a->q; p.q_ts = q_ts; p.q_hs = q_hs;
    p.q_vec = (((uintptr_t)a->q | (uintptr_t)(q_ts * 2) | (uintptr_t)(q_hs * 2)) & 15u) == 0;
    p.out = a->out; p.o_ts = o_ts; p.o_hs = o_hs; p.lse = a->lse;
    p.by_per.set((int)per);
    p.per = (int)per; p.q_heads = (int)a->q_heads;
    p.scale_log2 = a->scale * 1.44269504088896340736f;
    p.causal = a->causal ? 1 : 0;
    p.window = a->window > INT32_MAX ? INT32_MAX : (int)a->window;
    p.out_vec = (((uintptr_t)a->out | (uintptr_t)(o_ts * 2) | (uintptr_t)(o_hs * 2)) & 15u) == 0;
    p.status = h->dev_status;
    // the most tiles that there can be for the row kernel: every row block of every sequence over a whole table row
    const int nt = plan.nt;
    const int64_t item_tiles = (p.s.width * cache->page_size + TILE - 1) / TILE + 1 + SETUP;
    const int64_t blocks = plan.tiles ? p.s.seqs * (ROWS_MOST / (nt * 8)) : (p.s.tokens * per + nt * 8 - 1) / (nt * 8) + p.s.seqs;
    const int64_t items = plan.rows ? blocks * p.c.heads : 0;
    if (items > INT32_MAX / item_tiles) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 attention: more work than one call counts (2^31 tiles of %d keys)", TILE);
    const int64_t most = items * item_tiles;
    if (plan.tiles) {
        p.row_min = plan.rows ? (int)ROWS_MOST : 0;
        p.parts = plan.parts;
        p.ws = (float*)((char*)workspace + plan.rows_bytes);
        if (int32_t rc = oxq_kv4_tiles_launch(h, cache, p, a->dtype, plan.items)) return rc;
        if (!plan.rows) return OXQ_OK;
        p.row_limit = (int)ROWS_MOST;
    }
    p.ws = (float*)workspace;
    p.setup = most >= 8ll * attn_ctas(h, nt) ? SETUP : 0;             // where a CTA has a few tiles only, all count
    if (a->dtype == OXQ_BF16)
        return nt == 1 ? launch_dims<__nv_bfloat16, 1>(h, cache, p, most, item_tiles) : launch_dims<__nv_bfloat16, 2>(h, cache, p, most, item_tiles);
    return nt == 1 ? launch_dims<__half, 1>(h, cache, p, most, item_tiles) : launch_dims<__half, 2>(h, cache, p, most, item_tiles);
}

}  // extern "C"
