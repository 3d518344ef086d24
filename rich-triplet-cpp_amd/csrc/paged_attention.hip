// paged_attention.hip -- attention of the new tokens of many requests over a
// KV cache in pages.
//
// Row i of request s (n rows, len keys) has position len - n + i and sees the
// keys (position - window, position]:
//   out = sum_j softmax_j(scale q . k_j) v_j,
// zeros where it sees none.  Key j of the request is row j % page of page
// table[s][j / page].
//
// Work.  The rows of one request that share a KV head, (token, head of the
// group) in that order, are taken in blocks; an item is (request, KV head,
// block) and its tiles are the spans of keys the block's rows can see.  The
// sequence of all tiles of all items is cut into equal ranges, one per
// workgroup: the lengths are read on the device, so nothing is known of them
// when the launch is made, and a batch of very unequal requests still ends
// everywhere at once.  A workgroup finds its range by summing the requests'
// tiles itself.  An item cut between workgroups leaves its states (o, m, l) in
// the workspace; the last to arrive joins them in order, so results do not
// depend on who that is.
//
// Arithmetic.  Products on the matrix cores, online softmax per row:
//  * S^T = K Q^T, so that a lane holds one row's scores against several keys:
//    the row's maximum and sum are the lane's own and its partners' in the
//    other halves (32x32) or quarters (16x16) of the wave.
//  * O^T += V^T P^T: the lane that has a row's weights supplies them as they
//    are, for the keys its registers hold; V's fragments are read from LDS
//    transposed (ds_read_b64_tr_b16) for the same keys.
//  * 16-bit rows of q: products of 16-bit values, weights rounded to the type.
//    f16 weights are kept times 2^6, so that a weight of 2^-20 of the largest
//    still has all its bits.
//  * f32 rows over a 16-bit cache: q and the weights as limbs of the cache's
//    type, two of f16 (22 bits; q's row times a power of two that puts its
//    largest value at 2^14) or three of bf16 (24 bits), each multiplied with
//    the exact values of the cache.
//  * an f32 cache: f32 matrix steps.
//
// Bounds and times: at each of the two kernels.
//
// Infinities and NaN in v.  Keys a row does not see get weight 0, but 0 times an
// infinity or a NaN of their v would reach the row: in tiles with such pairs
// those values of v are made 0 in LDS, and added at the end to the rows that see
// them.  In the other tiles every row sees every key, but a product with a
// weight that has vanished, or with a limb that is 0 or negative, would turn an
// infinity into a NaN: a workgroup whose o has come out as something not finite
// walks its tiles again and does the same in all of them.  So whatever the tile,
// the limbs and the weight, such a value reaches the rows that see it as it is.
// (To look costs 0.1 to 0.3 us an item; to clean every tile from the start would
// cost each of them the reads and compares of all its values.)
#include "paged_core.hpp"

namespace rt_hip {
namespace {

constexpr int narrow_ring(int hd) { return hd == 256 ? 32768 : 16384; }

// ---- few rows: the waves split the keys ------------------------------------------
// Single tokens and drafts, bound by the bytes of keys and values.  A wave
// streams tiles of its own through its own LDS ring, no barrier between them,
// and the four waves' states are joined at the item's end.
// 64 requests of 100 to 16000 keys, 8 KV heads of 128 in bf16: 151 us for 782 MB
// (5.2 TB/s; a plain read of as much reaches 5.9).  16 requests of 5 tokens, a
// window of 1024, head_dim 256: 23 us for 48 MB.  One token over 777 keys: 11.2
// us, a chain of latencies: lengths, pages, keys, the waves' states, the join of
// the workgroups'.
template <class Q, class T, int HD, int RBLK>
__global__ __launch_bounds__(256, HD < 256 ? 2 : 1) void k_paged_narrow(PagedAttn p, Launch la) {
    constexpr int NW = 4, DB = 16, BM = DB * RBLK, BK = KindOf<T>::f32 ? 16 : 32, BN = NW * BK;
    using C = Core<Q, T, HD, DB, RBLK, BK>;
    constexpr int kRing = narrow_ring(HD);  // bytes of a wave's ring
    constexpr int D = kRing / 2 / C::TB;    // tiles of K, and of V, in the ring
    constexpr int H = BK / C::RPI;      // copies of a tile of K, or of V
    constexpr int G = BK / 8, PER = 8 / C::RPI;
    constexpr int kPart = part_floats(BM, HD);
    static_assert(BM * HD * 4 <= kRing && D >= 1, "a tile and a wave's state fit its ring");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float sm[NW][BM], sl[NW][BM];
    __shared__ int flag;
    __shared__ int dirty;  // the last of this workgroup's items whose o came out as something not finite
    if (threadIdx.x == 0) dirty = -1;
    int item = 0;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t* const ring = lds + wave * kRing;
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    // Tiles that take as long as an item's start and end, 6 us.  (0: 47 us where 2
    // takes 36 for 128 requests of 50 to 2000 keys, 380 where it takes 331 for 200
    // of up to 4000 at head_dim 256, 12 where it takes 14 for 16 of up to 900.)
    constexpr int EXTRA = 2;
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<256>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const uint32_t ring_at = uniform(static_cast<int>(lds_address(ring)));
    const float c1 = p.scale * kLog2e;
    C core;
    core.setup();
    bool all = false;  // the item once more, every tile of it as an edge tile
    while ((left = uniform(left)) > 0) {
        walk.pin();
        const int from = uniform(static_cast<int>(skip));
        const int to = uniform(static_cast<int>(min(static_cast<int64_t>(walk.tiles + EXTRA), skip + left)));
        skip = 0;
        left -= to - from;
        const int a = max(from - EXTRA, 0), b = max(to - EXTRA, 0);  // tiles
        if (a >= b) break;  // (the range ends before the item's first tile)
        int lo, hi;
        walk.span(walk.blk, &lo, &hi);
        const int rows = min(BM, walk.rows() - walk.blk * BM), row_first = walk.blk * BM;
        const int pos0 = walk.len - walk.n;
        // position of the block's first row (below every key: all tiles are edge tiles)
        const int low_pos = all ? -1 : pos0 + walk.token(row_first);
        const Pages pages = pages_of<T>(p, walk.s, walk.kvh, hi - 1);
        const int key0 = (walk.tile0 + a) * BN + wave * BK;
        int nt = b - a;
        if (key0 + (nt - 1) * BN >= hi) --nt;  // (the last tile's keys may end before this wave's)
        auto copy_k = [&](int i, const Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < H; ++j)
                C::template copy_rows<false>(g[j / PER].k, g[j / PER].row_bytes, g[j / PER].most, j / PER,
                                             j % PER * C::RPI, ring_at + (i % D) * C::TB + j * 1024);
        };
        auto copy_v = [&](int i, const Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < H; ++j)
                C::template copy_rows<true>(g[j / PER].k + g[j / PER].v, g[j / PER].row_bytes, g[j / PER].most, j / PER,
                                            j % PER * C::RPI, ring_at + (D + i % D) * C::TB + j * 1024);
        };
        auto groups = [&](int i, Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < G; ++j) g[j] = group_of(pages, key0 + i * BN + 8 * j);
        };
        for (int i = 0; i < D; ++i)
            if (i < nt) {
                Group g[G];
                groups(i, g);
                copy_k(i, g);
                copy_v(i, g);
            }
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n, row = row_first + r;
            const bool real = r < rows;
            const int t = walk.token(row);
            core.load_q(i, real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride +
                                      (walk.kvh * walk.group + walk.head(row, t)) * HD
                                : nullptr, c1);
            core.last[i] = real ? pos0 + t : -1;
            core.first[i] = walk.first_seen(core.last[i]);
        }
        // q is here: from now on only copies are in flight.  (The builtin, which the
        // compiler understands: it would wait for q's loads in every tile otherwise,
        // and with them for the copies.)
        wait_vmcnt<0>();
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        bool special = false;
        for (int i = 0; i < nt; ++i) {
            const int key = key0 + i * BN;
            const bool more = i + D < nt;
            const bool edge = is_edge(key);
            Group g[G];
            if (more) groups(i + D, g);
            // (what is in flight behind this tile's K: its V, and the later tiles in the ring)
            if (nt - i >= D) wait_copies<(2 * D - 1) * H>();
            else wait_copies<0>();
            core.scores(ring_at + (i % D) * C::TB);
            wait_lds();
            if (more) copy_k(i + D, g);
            core.softmax(key, edge);
            if (more) wait_copies<(2 * D - 1) * H>();
            else wait_copies<0>();
            const uint32_t v = ring_at + (D + i % D) * C::TB;
            if (edge) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < C::TB / 1024; ++j) any |= C::clean_at(v + j * 1024 + anew((tid & 63) * 16));
                special |= __builtin_amdgcn_ballot_w64(any) != 0;
                wait_lds();
            }
            core.pv(v);
            wait_lds();
            if (more) copy_v(i + D, g);
        }
        if (special) {
            for (int i = 0; i < nt; ++i)
                if (const int key = key0 + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j)
                        core.add_special(key + j, value_of(pages, key + j));
        }
        // The waves' states, joined in order.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        float* const mine = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n;
            const float l = C::across_sum(core.l[i]);
            if (core.kg == 0) {
                sm[wave][r] = core.m[i] * core.c[i];
                sl[wave][r] = l;
            }
#pragma unroll
            for (int j = 0; j < C::NC; ++j)
                *reinterpret_cast<f32x4*>(mine + r * HD + ((j * DB + 4 * core.kg) ^ (4 * (core.n & 7)))) = core.o[i][j];
        }
        __syncthreads();
        const int first_wg = static_cast<int>(item_at / per), last_wg = static_cast<int>((item_at + walk.tiles - 1) / per);
        const bool cut = first_wg != last_wg;
        float* const part = la.part + (static_cast<int64_t>(w) * 2 + (w == first_wg)) * kPart;
        for (int i = tid; i < rows * (HD / 4); i += 256) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float M = -kInf, L = 0.0f;
#pragma unroll
            for (int x = 0; x < NW; ++x) M = fmaxf(M, sm[x][r]);
            f32x4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = M == -kInf ? 1.0f : state_weight(sm[x][r] - M);
                L += sl[x][r] * f;
                O += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * kRing) + r * HD + (d ^ (4 * (r & 7)))) * f;
            }
            if (const f32x4 z = O * 0.0f; (z[0] + z[1]) + (z[2] + z[3]) != 0.0f) dirty = item;
            if (!cut) {
                const int row = row_first + r, t = walk.token(row);
                store_out(static_cast<Q*>(p.out) + (walk.row0 + t) * p.out_stride +
                              (walk.kvh * walk.group + walk.head(row, t)) * HD + d, O, L);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) st_dev(part + r * HD + d + e, O[e]);
                if (d == 0) {
                    st_dev(part + BM * HD + r, M);
                    st_dev(part + BM * HD + BM + r, L);
                }
            }
        }
        if (!all) {
            lds_barrier();
            if (uniform(dirty) == item) {
                all = true;
                skip = from, left += to - from;
                continue;
            }
        }
        ++item;
        if (cut) {
            if (arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag))
                join_parts<Q, BM, HD, 256>(walk, first_wg, last_wg, rows, reinterpret_cast<State*>(lds));
        }
        __syncthreads();  // the rings are free again
        all = false;
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// ---- many rows: the waves split the rows -------------------------------------------
// Chunks of prompts, bound by the matrix cores: every wave has 32 rows of its
// own, and K and V tiles are read from memory once for all of them.  Four waves
// or eight: enough_rows.
// 4096 tokens over 8192 keys before them, 24 heads of 128 in bf16: 490 to 535 us,
// 960 to 1050 TFLOP/s, by the clock that the card's power limit leaves (a library
// product of 8192^3: 1212); the matrix cores are busy half of the time, the VALU
// the other half.  900-token chunks of head_dim 64: 88 us for 43 GFLOP, the VALU
// busy 40% of it, the matrix cores 20%.  517 tokens over 1100 keys in f32: 106
// us, 81 TFLOP/s, the matrix cores busy 54% of it.
template <class Q, class T, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void k_paged_wide(PagedAttn p, Launch la) {
    constexpr int DB = 32, BM = DB * NW, BK = wide_keys<Q, T>(HD), BN = BK, NT = NW * 64;
    using C = Core<Q, T, HD, DB, 1, BK>;
    constexpr int PER = 8 / C::RPI;               // copies of a group of 8 keys
    constexpr int COPIES = BK / C::RPI / NW;      // copies of a tile of K, or of V, by each wave
    constexpr int GROUPS = COPIES < PER ? 1 : COPIES / PER;  // groups they are of
    constexpr int SLOTS = wide_slots(C::TB), L = SLOTS - 2;  // tiles of K, and of V, in LDS; copies run L steps further ahead
    constexpr int kPart = wide_part_floats(BM, HD);
    static_assert(COPIES >= 1 && COPIES * NW * C::RPI == BK && (COPIES < PER ? PER % COPIES : COPIES % PER) == 0,
                  "every wave copies alike, whole groups or part of one");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // SLOTS tiles of K, SLOTS of V
    __shared__ int page_ring[NW][128];
    __shared__ int special;  // the last of this workgroup's items whose v held what was made 0
    __shared__ int dirty;    // the last whose o came out as something not finite
    __shared__ int flag;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    // Tiles that take as long as an item's start and end, 5 us.  (35 requests, three
    // of them chunks of 800 to 900, head_dim 64 in bf16: 157 us with 0, 118 with
    // 6, 126 with 12; in f32 over f16, eight waves, 182 with 1, 144 with 6; one
    // chunk of 517 in f32, four waves: 120 with 1, 129 with 12.)
    constexpr int EXTRA = KindOf<T>::f32 ? (NW == 8 ? 3 : 1) : (NW == 8 ? 6 : 3);
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<NT>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const uint32_t lds_at = uniform(static_cast<int>(lds_address(lds)));
    const float c1 = p.scale * kLog2e;
    if (tid == 0) special = dirty = -1;
    int item = 0;
    C core;
    core.setup();
    bool all = false;  // the item once more, every tile of it as an edge tile
    while ((left = uniform(left)) > 0) {
        walk.pin();
        const int from = uniform(static_cast<int>(skip));
        const int to = uniform(static_cast<int>(min(static_cast<int64_t>(walk.tiles + EXTRA), skip + left)));
        skip = 0;
        left -= to - from;
        const int a = max(from - EXTRA, 0), b = max(to - EXTRA, 0);  // tiles
        if (a >= b) break;  // (the range ends before the item's first tile)
        int lo, hi;
        walk.span(walk.blk, &lo, &hi);
        const int rows = min(BM, walk.rows() - walk.blk * BM), row_first = walk.blk * BM;
        const int pos0 = walk.len - walk.n;
        const int low_pos = all ? -1 : pos0 + walk.token(row_first);  // (as above)
        const int r = wave * DB + core.n, row = row_first + r;
        const bool real = r < rows;
        const int t = walk.token(row);
        const int64_t head = (walk.kvh * walk.group + walk.head(row, t)) * HD;
        // the wave's rows see keys from wave_lo to wave_hi
        const int wave_low = pos0 + walk.token(row_first + min(wave * DB, rows - 1));
        const int wave_hi = pos0 + walk.token(row_first + min(wave * DB + DB, rows) - 1);
        const Pages pages = pages_of<T>(p, walk.s, walk.kvh, hi - 1);
        const int key0 = (walk.tile0 + a) * BN;
        const int nt = hi > 0 ? b - a : 0;
        // This wave's groups of the tiles whose K and whose V are copied next.
        PageWindow window;
        window.ring = uniform(static_cast<int>(lds_address(page_ring[wave])));
        Group grp_k[GROUPS], grp_v[GROUPS];
        const int group0 = wave * COPIES / PER;  // (the wave's copies start in it, at part0)
        const int part0 = COPIES < PER ? wave * COPIES % PER : 0;
        auto find_groups = [&](int i) {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) {
                const int at = group_at(pages, static_cast<uint32_t>(key0) + i * BN + 8 * (group0 + x));
                grp_k[x] = group_on(pages, at, window.at(pages, at >> pages.shift));
            }
        };
        // Copy x of this wave's of a tile of K, or V, into a slot.
        auto copy_k = [&](int slot, int x) {
            const Group& g = grp_k[x / PER];
            C::template copy_rows<false>(g.k, g.row_bytes, g.most, group0 + x / PER, (part0 + x % PER) * C::RPI,
                                         lds_at + slot * C::TB + (wave * COPIES + x) * 1024);
        };
        auto copy_v = [&](int slot, int x) {
            const Group& g = grp_v[x / PER];
            C::template copy_rows<true>(g.k + g.v, g.row_bytes, g.most, group0 + x / PER, (part0 + x % PER) * C::RPI,
                                        lds_at + (SLOTS + slot) * C::TB + (wave * COPIES + x) * 1024);
        };
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        int ahead = 0;  // the tile grp_k is of
        auto advance = [&] {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) grp_v[x] = grp_k[x];
            find_groups(++ahead);
        };
        lds_barrier();  // (every wave is done with the item before)
        if (nt > 0) {
            window.start(pages, group_at(pages, key0 + 8 * group0) >> pages.shift);
            wait_copies<0>();
            find_groups(0);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) copy_k(0, x);
            advance();
            if constexpr (L == 1) {
#pragma unroll
                for (int x = 0; x < COPIES; ++x) copy_v(0, x);
#pragma unroll
                for (int x = 0; x < COPIES; ++x) copy_k(1, x);
                advance();
            }
        }
        core.load_q(0, real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride + head : nullptr, c1);
        core.last[0] = real ? pos0 + t : -1;
        core.first[0] = walk.first_seen(core.last[0]);
        wait_vmcnt<0>();  // (the builtin: so that the compiler, too, knows that q is there)
        lds_barrier();
        // Step i in two halves: the products, O += P V of tile i - 1 and the
        // scores of tile i, and the weighing of tile i.  With eight waves, w and
        // w + 4 share a SIMD: the second four run a half behind the first, so
        // that one wave of a SIMD has the matrix cores while the other has the
        // VALU, a barrier between the halves.
        // Among its products a wave sends the copies of V of tile i + L and K of
        // tile i + 1 + L, into the slots of V of tile i - 2 and K of tile i - 1,
        // which every wave has read by then; it waits for them in step i + L,
        // before the barrier that step i + L + 1 lies behind.  (Past the last
        // tile they bring its last keys again, for no one.)
        constexpr bool kTwo = NW == 8;
        static_assert(!kTwo || L == 1, "the second four send their copies a half late");
        const bool second = kTwo && wave >= 4;
        // This wave's copies of V of tile i are there; of an edge tile's, cleaned.
        auto settle = [&](int i, int slot) {
            wait_copies<2 * COPIES * L>();
            if (is_edge(key0 + i * BN)) {
                bool any = false;
#pragma unroll
                for (int x = 0; x < COPIES; ++x)
                    any |= C::clean_at(lds_at + (SLOTS + slot) * C::TB + (wave * COPIES + x) * 1024 + anew((tid & 63) * 16));
                if (__builtin_amdgcn_ballot_w64(any) != 0) special = item;
            }
        };
        if (nt > 0) {
            if (second) lds_barrier();
            int now = 0;  // slot of tile i
            for (int i = 0; i <= nt; ++i) {
                const int before = now == 0 ? SLOTS - 1 : now - 1, behind = now + 1 == SLOTS ? 0 : now + 1;
                // (no branch around the products of what is not there or not seen: the
                // weights of a tile that no row of the wave sees are 0 and its V is
                // clean, being an edge tile; in step 0 the accumulator is cleared
                // after; scores of no tile are not used)
                __builtin_amdgcn_s_setprio(1);
                core.template products<2 * COPIES>(lds_at + now * C::TB, lds_at + (SLOTS + before) * C::TB, [&](int x) {
                    if (x < COPIES) copy_v(L ? behind : now, x);
                    else copy_k(before, x - COPIES);
                });
                __builtin_amdgcn_s_setprio(0);
                if (i == 0) core.no_values();
                if (second && i < nt) settle(i, now);
                if (kTwo) lds_barrier();
                // (behind the last tile: from hi on, keys that no row sees, which change nothing)
                const int key = i < nt ? key0 + i * BN : hi;
                core.softmax(key, i == nt || key + BK - 1 > wave_low || (p.window && wave_hi - key >= p.window));
                advance();
                if (!second && i < nt) settle(i, now);
                lds_barrier();
                now = behind;
            }
            if (kTwo && !second) lds_barrier();
            wait_copies<0>();
        }
        if (uniform(special) == item) {
            for (int i = 0; i < nt; ++i)
                if (const int key = key0 + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j)
                        core.add_special(key + j, value_of(pages, key + j));
        }
        float l = C::across_sum(core.l[0]);
        const int first_wg = static_cast<int>(item_at / per), last_wg = static_cast<int>((item_at + walk.tiles - 1) / per);
        bool whole = first_wg == last_wg;
        auto part = [&](int wg) { return la.part + (static_cast<int64_t>(wg) * 2 + (wg == first_wg)) * kPart + tid; };
        if (!whole) {
            // States as the registers are, a lane's values NT apart.
            float* const mine = part(w);
#pragma unroll
            for (int i = 0; i < C::NC; ++i)
#pragma unroll
                for (int e = 0; e < C::ACC; ++e) st_dev(mine + (i * C::ACC + e) * NT, core.o[0][i][e]);
            st_dev(mine + BM * HD, core.m[0] * core.c[0]);
            st_dev(mine + BM * HD + NT, l);
        }
        if (!all) {
            if (core.not_finite()) dirty = item;
            lds_barrier();
            if (uniform(dirty) == item) {
                all = true;
                skip = from, left += to - from;
                continue;
            }
        }
        ++item;
        if (!whole) {
            whole = arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag);
            if (whole) {
                float M = -kInf;
                l = 0.0f;
                core.no_values();
                for (int x = first_wg; x <= last_wg; ++x) {
                    // (all loads before the first use: they are served one latency after
                    // the other otherwise)
                    const float* const src = part(x);
                    const float m = ld_dev(src + BM * HD), sum = ld_dev(src + BM * HD + NT);
                    float o[C::NC * C::ACC];
#pragma unroll
                    for (int i = 0; i < C::NC * C::ACC; ++i) o[i] = ld_dev(src + i * NT);
                    __builtin_amdgcn_sched_barrier(0);
                    const float top = fmaxf(M, m);
                    const float fa = top == -kInf ? 0.0f : state_weight(M - top), fb = top == -kInf ? 0.0f : state_weight(m - top);
                    l = l * fa + sum * fb;
#pragma unroll
                    for (int i = 0; i < C::NC; ++i)
#pragma unroll
                        for (int e = 0; e < C::ACC; ++e)
                            core.o[0][i][e] = core.o[0][i][e] * fa + o[i * C::ACC + e] * fb;
                    M = top;
                }
            }
        }
        if (whole && real) {
            Q* const dst = static_cast<Q*>(p.out) + (walk.row0 + t) * p.out_stride + head;
#pragma unroll
            for (int i = 0; i < C::NC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    store_out(dst + core.dim_of(i, 4 * e),
                              f32x4{core.o[0][i][4 * e], core.o[0][i][4 * e + 1], core.o[0][i][4 * e + 2], core.o[0][i][4 * e + 3]}, l);
        }
        all = false;
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// Rows (tokens x group) of a request up to which its keys are split over the
// waves.  24 requests of 1500 to 5000 keys at head_dim 128, bf16, few-row form
// against many-row form: 16 rows 64 us; 32 rows 75 and 100; 48 rows 114 and 97;
// 64 rows 118 and 99.  (At head_dim 64 the two meet at 64 rows, with f32 rows
// over a bf16 cache at 40.)
constexpr int kNarrowRows = 32;
// Whether eight waves of 32 rows, two to a SIMD, have registers enough.  (Three
// limbs of q at head_dim 128 have not: 2048 tokens over 4000 keys take 367 us with
// eight, 372 with four, 64 over 500 45 and 28.)
template <class Q, class T>
constexpr bool eight_fit(int hd) {
    return hd == 64 || (hd == 128 && !(sizeof(Q) == 4 && !KindOf<T>::f32 && !KindOf<T>::f16));
}

// Blocks of 16 rows that a wave of the few-row form takes together where there
// are more than one: two, but for f32 rows over bf16, whose three limbs of two
// blocks do not fit the registers (24 requests of 32 rows, head_dim 128: 116 us
// with two, 102 with one, keys and values read twice; 294 and 205 at 256).
template <class Q, class T>
constexpr int narrow_blocks(int hd) {
    return hd > 64 && sizeof(Q) == 4 && !KindOf<T>::f32 && !KindOf<T>::f16 ? 1 : 2;
}

// Workgroups of the narrow form: those the CUs hold at once.  (With one to a CU
// 64 decoding requests take 166 us instead of 157, a mixed step 127 instead of 118.)
int narrow_slots(int hd) { return slots() * (hd == 256 ? 1 : 2); }

// Whether the many-row form takes blocks of 256 rows, eight waves, or of 128,
// four: where a request's rows fill more than one of the smaller, and all rows
// together are 40 to a CU (80 with an f32 cache), so that keys are read fewer
// times and one wave of a SIMD can work while the other waits.  Four and eight
// waves, us, head_dim 128, 24 heads, 3 to a KV head:
//   tokens over keys      bf16        f32 over f16   f32
//   64 over 500           25    31    27    36       36    56
//   256 over 1000         27    37    32    42       63    72
//   512 over 9000        108    86   150   131      509   478
//   1024 over 3000        88    70   119   108      397   374
//   2048 over 4000       209   148   296   241     1080   999
// 40 requests, 32 heads, 4 to a KV head: of 30 tokens (120 rows) 47 and 53, of
// 100 (400 rows) 164 and 115.  (The rule does not know the keys, so that 512 over
// 9000 in f32, 48 rows to a CU, takes four waves and loses 6%; and it counts the
// rows there is room for.)
bool enough_rows(const PagedAttn& p, int64_t rows) {
    const int64_t each = p.kv.dtype == RT_HIP_F32 ? 80 : 40;
    return rows > 128 && static_cast<int64_t>(p.n_tokens) * p.n_q >= slots() * each;
}

template <class Q, class T, int HD>
hipError_t run(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    Launch la = launch_of(p, part, counters);
    const int64_t rows = most_rows(p);
    const bool wide = rows > kNarrowRows, narrow = !wide || p.n_seq > 1;
    // (one workgroup to a CU, LDS holds no more; ranges of a single tile are worth
    // it: with 8 at least, 64 tokens over 500 keys took 65 us in f32 instead of 37)
    const unsigned grid = static_cast<unsigned>(slots());
    if (wide) {
        constexpr int BK = wide_keys<Q, T>(HD), LDS = 2 * wide_slots(BK * HD * sizeof(T)) * BK * HD * sizeof(T);
        constexpr int MOST = eight_fit<Q, T>(HD) ? 8 : 4;
        la.min_rows = narrow ? kNarrowRows : 0;
        la.max_rows = 0x7fffffff;
        const bool eight = MOST == 8 && enough_rows(p, rows);
        hipLaunchKernelGGL((eight ? k_paged_wide<Q, T, HD, MOST> : k_paged_wide<Q, T, HD, 4>), dim3(grid),
                           dim3(eight ? 512 : 256), LDS, s, p, la);
    }
    if (narrow) {
        la.min_rows = 0;
        la.max_rows = wide ? kNarrowRows : 0x7fffffff;
        const unsigned many = static_cast<unsigned>(narrow_slots(HD));
        const auto kernel = rows <= 16 ? k_paged_narrow<Q, T, HD, 1> : k_paged_narrow<Q, T, HD, narrow_blocks<Q, T>(HD)>;
        hipLaunchKernelGGL(kernel, dim3(many), dim3(256), 4 * narrow_ring(HD), s, p, la);
    }
    return hipGetLastError();
}

template <class Q, class T>
hipError_t run_hd(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    switch (p.kv.head_dim) {
        case 64: return run<Q, T, 64>(p, part, counters, s);
        case 128: return run<Q, T, 128>(p, part, counters, s);
        default: return run<Q, T, 256>(p, part, counters, s);
    }
}

}  // namespace

size_t paged_attention_workspace(const PagedAttn& p) {
    const int64_t rows = most_rows(p);
    const int hd = p.kv.head_dim, waves = hd < 256 ? 8 : 4;
    const size_t narrow = static_cast<size_t>(narrow_slots(hd)) * 2 * part_floats(rows <= 16 ? 16 : 32, hd);
    const size_t wide = rows > kNarrowRows ? static_cast<size_t>(slots()) * 2 * wide_part_floats(waves * 32, hd) : 0;
    return (narrow > wide ? narrow : wide) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttn& p, void* part, uint32_t* counters, hipStream_t s) {
    if (static_cast<size_t>(narrow_slots(64)) > kArrivalCounters) return hipErrorInvalidValue;
    float* const f = static_cast<float*>(part);
    if (p.dtype == RT_HIP_BF16) return run_hd<__bf16, __bf16>(p, f, counters, s);
    if (p.dtype == RT_HIP_F16) return run_hd<_Float16, _Float16>(p, f, counters, s);
    switch (p.kv.dtype) {
        case RT_HIP_F32: return run_hd<float, float>(p, f, counters, s);
        case RT_HIP_F16: return run_hd<float, _Float16>(p, f, counters, s);
        default: return run_hd<float, __bf16>(p, f, counters, s);
    }
}

}  // namespace rt_hip
