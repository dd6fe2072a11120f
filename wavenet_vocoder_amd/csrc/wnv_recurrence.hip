// wnv_recurrence.hip -- the gated linear recurrence: a scan over (B, T, C), its backward pass, and one step with the state in place.
//
//   z = (f | v | o) along the channels,  u = 1 - sigmoid(f)
//   h_t = a_t h_{t-1} + u_t v_t,  a = sigmoid(f)          y_t = h_t sigmoid(o_t)   (no o: y = h)
//
// a and u are each held to their own precision.  A gate that forgets leaves a h of the state, and h + u (v - h) would leave 2^-24 of h; a gate
// that remembers long has a next to 1, where 32 bits leave it 6e-8 off, and a state that goes through 1 / u such steps is 6e-8 / u off.  So
// steps are a h + u v only within a stretch of 8 of them, and what a stretch keeps of the state is 1 - U, with U summed up from its u, where
// that is the more exact of the two.  (An infinite v or state is infinite or NaN for the rest of its utterance.)
// h_{t-1} reads as zero at a step that begins an utterance of a packed slot (seg_start[b][t] == t).  Behind lengths[b] the state is
// handed on, y and the gradients are zero, and z is not looked at.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "wnv_hostutil.h"
#include "wnv_num.h"

#pragma clang fp contract(off)          // what is fused is written as fmaf: one kernel's arithmetic is another's

namespace {

struct RecArgs {
    int B, C, T, tiles, chunks;     // tiles of the channels, chunks of the time
    int part_bits;                  // a part is 1 << part_bits blocks
    long long zb, zt;               // batch and time stride of z, in elements
    long long h0b;
    const void* z;
    const float* h0;
    const int *lengths, *seg_start;
    void* y;
    float* h_last;
    float* saved;                   // [row][chunk][part][tile width]: the state before the part's first step
    unsigned long long* slots;      // workspace: of each row of tiles a counter, then its maps
    const void* dy;
    long long dyb, dyt;
    const float* dh_last;
    void* dz;
    float* dh0;
};

// ---- maps of the state --------------------------------------------------------------------------------------------------------
// A stretch of steps maps the state before it to the state behind it: h -> p h + b, with p the product of its gates; u = 1 - p is carried
// next to it (sums of products of gates, nothing is taken from anything), and p is 1 - u where u <= 1/2.  p < 0 says that the state behind
// is b whatever stood before, which only happens where utterances begin (SEG).  A stretch without steps hands any h on as it is, an
// infinite one too.  The backward pass maps what flows back by the same form.
struct Map { float p, u, b; };
constexpr Map NOTHING{1.f, 0.f, 0.f};

template <bool SEG> __device__ __forceinline__ float apply(Map m, float h) {
    const float r = fmaf(m.p, h, m.b);
    return SEG && m.p < 0.f ? m.b : r;
}
template <bool SEG> __device__ __forceinline__ Map join(Map first, Map then) {
    Map r;
    r.p = first.p * then.p;
    r.u = fmaf(first.p, then.u, first.u);
    r.b = apply<SEG>(then, first.b);
    if (SEG && (then.p < 0.f || first.p < 0.f)) r.p = -1.f;
    return r;
}

// A map is handed to the other workgroups as one 8-byte store that carries its own "valid": b, and p where it is at most 1/2, else -u (2:
// an utterance begins).  The workspace is filled with ones, and no map has that pattern (a NaN is rewritten to the usual one).  No fence
// is needed: nothing else is read on the strength of it.
constexpr unsigned EMPTY = 0xffffffffu;
template <bool SEG> __device__ __forceinline__ void publish(unsigned long long* slot, Map m) {
    float k = m.u <= 0.5f ? -m.u : m.p;
    if (SEG && m.p < 0.f) k = 2.f;
    const unsigned w = k != k ? 0x7fc00000u : __float_as_uint(k);
    __hip_atomic_store(slot, ((unsigned long long)__float_as_uint(m.b) << 32) | w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* slot) {
    return __hip_atomic_load(slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A map as it comes out of a slot.
template <bool SEG> __device__ __forceinline__ Map handed_on(Map m) {
    if (m.u <= 0.5f) m.p = SEG && m.p < 0.f ? m.p : 1.f - m.u;
    else m.u = 1.f - m.p;
    return m;
}
template <bool SEG> __device__ __forceinline__ Map unpacked(unsigned long long v) {
    const float k = __uint_as_float((unsigned)v), rest = 1.f - fabsf(k), b = __uint_as_float((unsigned)(v >> 32));
    const bool u = (int)(unsigned)v < 0;            // the sign, of a zero too
    Map m{u ? rest : k, u ? -k : rest, b};
    if (SEG && k > 1.f) m.p = -1.f;
    return m;
}

// Waits until the first n (uniform, N at most) of the slots that lie W apart hold maps, and hands them to `take` in their order.
// The wait ends: a workgroup draws its chunk from a counter, so the chunks before that of one that runs have all been started, and
// the lowest of them waits for nobody.  Should a slot stay empty for some seconds all the same, its map is NaN: the launch ends, and
// says so in its results.
template <int N, bool SEG, typename F> __device__ __forceinline__ void take_maps(const unsigned long long* slots, int W, int n, F take) {
    unsigned long long v[N];
    for (int tries = 0;; ++tries) {
        bool holds = true;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) v[i] = peek(slots + (long long)i * W);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n && (unsigned)v[i] == EMPTY) holds = false;
        if (holds || tries > (1 << 22)) break;
        __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) take(unpacked<SEG>(v[i]));   // the empty pattern itself is a NaN
}

// How a chunk learns the state before it, without a chain through all chunks and in one order of arithmetic whatever the timing:
// 16 chunks are a group, 16 groups a section.  Every chunk hands out its map; the last one of a group joins the 16 and hands out the
// group's; the last one of a section hands out the state behind it.  A chunk takes the section's state, runs it through the maps
// of the groups before its own and of the chunks before it in its group: two waits behind its own loads for 256 chunks (32768 steps),
// and one more for each further section.
constexpr int GROUP = 16, COUNTER = 16;      // a row's counter has 128 bytes of its own
struct Slots {                      // of one row of tiles, one channel
    unsigned long long *chunk, *group, *section;
};
__host__ __device__ __forceinline__ long long slots_of_row(int chunks, int W) {
    return COUNTER + (long long)W * (chunks + chunks / GROUP + chunks / (GROUP * GROUP));
}
__device__ __forceinline__ Slots slots_at(unsigned long long* all, int row, int chunks, int W, int ch) {
    unsigned long long* p = all + row * slots_of_row(chunks, W) + COUNTER + ch;
    return {p, p + (long long)W * chunks, p + (long long)W * (chunks + chunks / GROUP)};
}

// Hands out what others wait for of chunk k (counted in the order in which the chunks are drawn), and returns the map of the chunks
// before it in its group.
template <int W, bool SEG> __device__ __forceinline__ Map map_in_group(const Slots& s, int k, int chunks, Map own) {
    const int at = k % GROUP;
    const bool more = k + 1 < chunks, last = at == GROUP - 1;
    if (more && !last) publish<SEG>(s.chunk + (long long)k * W, own);
    Map all = NOTHING;
    for (int i = 0; i < at; i += GROUP / 2)         // 8 at a time: 15 at once cost 14 registers more, and a wave per SIMD with them
        take_maps<GROUP / 2, SEG>(s.chunk + (long long)(k - at + i) * W, W, min(at - i, GROUP / 2), [&](Map m) { all = join<SEG>(all, m); });
    if (more && last && k / GROUP % GROUP != GROUP - 1) publish<SEG>(s.group + (long long)(k / GROUP) * W, join<SEG>(all, own));
    return all;
}
// The state before the group of chunk k as far as the first 8 groups of its section lead, `first` before chunk 0, and the map of
// the section's other groups before it.
template <int W, bool SEG> __device__ __forceinline__ float state_before_groups(const Slots& s, int k, float first) {
    const int section = k / (GROUP * GROUP), g0 = section * GROUP, n = min(k / GROUP - g0, GROUP / 2);
    float h = first;
    if (section) take_maps<1, SEG>(s.section + (long long)(section - 1) * W, W, 1, [&](Map m) { h = m.b; });
    take_maps<GROUP / 2, SEG>(s.group + (long long)g0 * W, W, n, [&](Map m) { h = apply<SEG>(m, h); });
    return h;
}
template <int W, bool SEG> __device__ __forceinline__ Map map_of_groups(const Slots& s, int k) {
    const int g0 = k / (GROUP * GROUP) * GROUP + GROUP / 2, n = k / GROUP - g0;
    Map all = NOTHING;
    take_maps<GROUP / 2 - 1, SEG>(s.group + (long long)g0 * W, W, n, [&](Map m) { all = join<SEG>(all, m); });
    return all;
}
__device__ __forceinline__ bool ends_section(int k, int chunks) { return (k + 1) % (GROUP * GROUP) == 0 && k + 1 < chunks; }

// ---- the shape of a workgroup -------------------------------------------------------------------------------------------------
// 4 (or 8) waves of 4 stretches of L steps; a stretch is 16 lanes, a row of the wave, along the channels.  A lane holds V = 4 channels, so
// that a tile is 64 channels wide: 128 bytes of a 16-bit type, 256 of float32 (8 channels a lane and 4 steps, for rows of 256 bytes
// of a 16-bit type too, took 213 us forward when this took 185, and 506 backward for 316, bf16 8 x 24064 x 512: more maps to join per step).
// Registers decide how many workgroups share a CU: 3 forward (4 of 16-bit types) and 2 backward, each with 32 steps x channels a thread;
// half the steps and 3 workgroups backward took 356 us when this took 316.  The last lane of a tile that ends in no multiple of V starts earlier and shares
// channels with its neighbour (both compute and write the same); V = 1 is for rows narrower than 4.  Narrow tiles take stretches of 4
// lanes, 16 to a wave.
//
// Which cut runs goes by the amount of data too, and does not show in the results: 4 stretches are a quad, 4 quads a block of 128 steps, 1 block
// or, of rows up to 32 channels, 4 are a part.  The four of a quad and of a block are joined two and two, blocks within their part and
// parts one after the other, whether a workgroup holds one part, and the parts are chunks that hand each other their maps, or all of them.
constexpr int L = 8, BLOCK = 16 * L;
template <int LANES, int WAVES> struct Shape {
    static constexpr int STEPS = WAVES * (64 / LANES) * L;
    static constexpr int QUADS = STEPS / (4 * L), BLOCKS = QUADS / 4;
};

// V elements as they stand in memory, packed in as few registers; addresses are a uniform base and 32 bits of a lane's own.
template <typename E, int V> struct Vec {
    static constexpr int N = (V * (int)sizeof(E) + 3) / 4;
    uint32_t w[N];
    __device__ __forceinline__ float get(int i) const {
        if (sizeof(E) == 4) return __uint_as_float(w[i]);
        if (__is_same(E, wnv_bf16)) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        return (float)__builtin_bit_cast(wnv_f16, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
    }
};
// STREAM: past the caches, for data that no cache holds until its next use anyway (8 x 24064 x 512, with and without: float32 forward 285 and
// 301 us, backward 496 and 523; bf16 169 and 181, 290 and 312).  Rows that are no multiple of 128 bytes are left to the caches: their
// neighbours share a line, which the cache puts together (16 x 24064 x 100 float32: forward 195 with and 168 without, backward 376 and
// 307), and what fits the last level may be there for its next user.
template <int BYTES> struct Raw { typedef uint32_t T __attribute__((ext_vector_type(BYTES / 4), aligned(1))); };
template <> struct Raw<2> { typedef uint16_t T __attribute__((aligned(1))); };
template <> struct Raw<4> { typedef uint32_t T __attribute__((aligned(1))); };
template <typename E, int V, bool STREAM> __device__ __forceinline__ Vec<E, V> load(const E* base, uint32_t bytes) {        // at any alignment
    typedef typename Raw<V * sizeof(E)>::T R;
    const R* p = (const R*)((const char*)base + bytes);
    const R r = STREAM ? __builtin_nontemporal_load(p) : *p;
    Vec<E, V> v{};
    __builtin_memcpy(v.w, &r, sizeof r);
    return v;
}
template <typename E, int V, bool STREAM> __device__ __forceinline__ void store(E* base, uint32_t bytes, const float (&x)[V]) {
    typedef typename Raw<V * sizeof(E)>::T R;
    E e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float f = x[i];
        // a float32 product is rounded before it becomes f16, in every kernel: the compiler makes one mixed instruction of the two in some
        if (__is_same(E, wnv_f16)) asm("" : "+v"(f));
        e[i] = wnv_down<E>(f);
    }
    R r;
    __builtin_memcpy(&r, e, sizeof r);
    R* p = (R*)((char*)base + bytes);
    if (STREAM) __builtin_nontemporal_store(r, p);
    else *p = r;
}

// The maps of a quad's four stretches joined in time (BACK: the last one first): of all of them, and of those before the own one.
template <int LANES> __device__ __forceinline__ void exchange(float x, int stride, float& low, float& high) {     // of two stretches that lie `stride` apart
    if constexpr (LANES == 16) {        // two exchanges of registers, no LDS
        const uint32_t w = __float_as_uint(x);
        const auto r = stride == 1 ? __builtin_amdgcn_permlane16_swap(w, w, false, false) : __builtin_amdgcn_permlane32_swap(w, w, false, false);
        low = __uint_as_float(r[0]);
        high = __uint_as_float(r[1]);
    } else {
        const float other = __shfl_xor(x, stride * LANES);
        const bool second = threadIdx.x / LANES & stride;
        low = second ? other : x;
        high = second ? x : other;
    }
}
template <int LANES> __device__ __forceinline__ void exchange(Map x, int stride, Map& low, Map& high) {
    exchange<LANES>(x.p, stride, low.p, high.p);
    exchange<LANES>(x.u, stride, low.u, high.u);
    exchange<LANES>(x.b, stride, low.b, high.b);
}
template <int LANES, bool BACK, bool SEG> __device__ __forceinline__ void join_quad(Map x, Map& all, Map& before) {
    Map even, odd, low, high;
    exchange<LANES>(x, 1, even, odd);
    exchange<LANES>(BACK ? join<SEG>(odd, even) : join<SEG>(even, odd), 2, low, high);
    const int row = threadIdx.x / LANES & 3;
    all = BACK ? join<SEG>(high, low) : join<SEG>(low, high);
    before = (row & 1) != BACK ? (BACK ? odd : even) : NOTHING;
    if ((row >> 1) != BACK) before = join<SEG>(BACK ? high : low, before);
}
// What a forward pass keeps of its stretch's steps for the second run over them.  float32: a and u v.  16-bit types: the smaller of a and u,
// negative where that is u, next to v as it came; 16 registers less, which are a fourth wave per SIMD (bf16 8 x 24064 x 512: 171 us, with
// a and u v in three waves 178), and the arithmetic of wnv_blend.
template <typename E, int V> struct Steps {
    float keep[L][V], put[L][V];
    __device__ __forceinline__ void hold(int l, int i, float a, float, float uv) { keep[l][i] = a; put[l][i] = uv; }
    __device__ __forceinline__ float run(int l, int i, float h, float) const { return fmaf(keep[l][i], h, put[l][i]); }
};
template <typename E, int V> struct PackedSteps {
    float less[L][V];
    __device__ __forceinline__ void hold(int l, int i, float a, float u, float) { less[l][i] = u < a ? -u : a; }
    __device__ __forceinline__ float run(int l, int i, float h, float v) const {
        const bool keeps = (int)__float_as_uint(less[l][i]) < 0;
        const float more = keeps ? h : v, rest = keeps ? v : h, w = fabsf(less[l][i]);
        return fmaf(w, rest, fmaf(-w, more, more));
    }
};
template <int V> struct Steps<wnv_bf16, V> : PackedSteps<wnv_bf16, V> {};
template <int V> struct Steps<wnv_f16, V> : PackedSteps<wnv_f16, V> {};

// A stretch's map step by step, and at its end.
template <bool SEG> __device__ __forceinline__ void step(Map& m, float keep, float u, float put, bool begins) {
    if (SEG && begins) m.b = 0.f;
    m.b = fmaf(keep, m.b, put);
    m.u = fmaf(u, m.p, m.u);
    m.p *= keep;
}
template <bool SEG> __device__ __forceinline__ void finish(Map& m, int begins) {
    if (m.u <= 0.5f) m.p = 1.f - m.u;
    if (SEG && begins) m.p = -1.f;
}

struct Place { int b, tile, chunk, row; };

// Each row's tile has a counter from which its chunks are drawn, the order that the waits rely on.  (One for all tiles of a batch row is
// drawn from by too many at once: forward of 1 x 24064 x 512 bf16 42 us for 31, 1 x 24064 x 128 float32 19.5 for 17.9.)
// Workgroup i runs on XCD i % 8.  Units of one chunk in all tiles are dealt to the XCDs, so that the tiles' shares of a line meet in one
// L2 (tiles dealt by themselves: 5 x 3001 x 201 float32 forward 20.1 us for 18, 3 x 16749 x 113 bf16 25 for 22.5); within an XCD the
// tiles take turns, or each would stay on the same CUs and memory channels (float32 8 x 24064 x 512 both passes: 772 us for 758).
// False for the workgroups that fill up the last units.
template <bool BACK> __device__ __forceinline__ bool draw_place(const RecArgs& a, int W, Place& p) {
    __shared__ int drawn;
    const int i = blockIdx.x / 8, round = i / a.tiles, unit = round * 8 + blockIdx.x % 8;
    if (unit >= a.B * a.chunks) return false;
    p.b = unit % a.B;
    p.tile = (i + round) % a.tiles;
    p.row = p.b * a.tiles + p.tile;
    p.chunk = 0;
    if (a.chunks > 1) {
        if (threadIdx.x == 0) drawn = atomicAdd((int*)(a.slots + p.row * slots_of_row(a.chunks, W)), 1) + 1;     // it starts at -1
        __syncthreads();
        p.chunk = __builtin_amdgcn_readfirstlane(drawn);
    }
    if (BACK) p.chunk = a.chunks - 1 - p.chunk;
    return true;
}

template <bool BACK, bool SEG, int QUADS, int W> __device__ __forceinline__ Map block_of(const Map (&quads)[QUADS][W], int k, int ch) {
    const Map a = quads[4 * k][ch], b = quads[4 * k + 1][ch], c = quads[4 * k + 2][ch], d = quads[4 * k + 3][ch];
    return BACK ? join<SEG>(join<SEG>(d, c), join<SEG>(b, a)) : join<SEG>(join<SEG>(a, b), join<SEG>(c, d));
}
// The maps of a workgroup's quads joined to its chunk's, which the others get, to its blocks' where it has several, and to `prev`: of the
// parts before each of its own; one channel.  Returns the chunk's.
template <int W, int QUADS, bool BACK, bool SEG>
__device__ __forceinline__ Map join_blocks(const RecArgs& a, const Slots& slots, int order, int ch, const Map (&quads)[QUADS][W], Map (&blocks)[QUADS / 4][W],
                                            Map (&prev)[QUADS / 4][W]) {
    constexpr int BLOCKS = QUADS / 4;
    const int last = (1 << a.part_bits) - 1, parts = BLOCKS >> a.part_bits;
    Map all = NOTHING, own = NOTHING;
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
        const int mine = BACK ? BLOCKS - 1 - k : k;
        const Map block = block_of<BACK, SEG>(quads, mine, ch);
        if (BLOCKS == 1) {
            own = block;
        } else {
            blocks[mine][ch] = block;
            own = k & last ? join<SEG>(own, block) : block;
            if (parts > 1) {            // the only chunk
                if ((k & last) == 0) prev[mine >> a.part_bits][ch] = all;
                if ((k & last) == last) all = join<SEG>(all, handed_on<SEG>(own));
            }
        }
    }
    if (BLOCKS == 1 || parts == 1) prev[0][ch] = map_in_group<W, SEG>(slots, order, a.chunks, own);
    return own;
}
// The last chunk of a section hands out the state behind it as soon as it knows the one before it; one channel.
template <int W, bool SEG>
__device__ __forceinline__ void hand_out_section(const RecArgs& a, int row, int order, int ch, Map chunk, Map prev, Map groups, float base) {
    const float behind = apply<SEG>(chunk, apply<SEG>(prev, apply<SEG>(groups, base)));
    publish<SEG>(slots_at(a.slots, row, a.chunks, W, ch).section + (long long)(order / (GROUP * GROUP)) * W, {0.f, 1.f, behind});
}
// The state before a quad from that before its part, a lane's channels from ch on.  The quads' maps are all asked for before the first is used
// (2 x 300 x 128 float32 forward 8.1 us; one after the other 8.7).
template <int W, int V, int QUADS, bool BACK, bool SEG>
__device__ __forceinline__ void state_before_quad(const RecArgs& a, const Map (&quads)[QUADS][W], const Map (&blocks)[QUADS / 4][W], int quad, int ch, float (&h)[V]) {
    const int q = BACK ? QUADS - 1 - quad : quad, block = q / 4, in = q % 4;
    if (QUADS > 4)
        for (int k = block >> a.part_bits << a.part_bits; k < block; ++k)
#pragma unroll
            for (int c = 0; c < V; ++c) h[c] = apply<SEG>(blocks[BACK ? QUADS / 4 - 1 - k : k][ch + c], h[c]);
    Map three[3][V];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int c = 0; c < V; ++c) three[i][c] = quads[BACK ? QUADS - 1 - 4 * block - i : 4 * block + i][ch + c];
    if (QUADS == 4) {                   // a quad is a wave: one branch for all of it
        if (in == 0) return;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            Map before = three[0][c];
            if (in > 1) before = join<SEG>(before, three[1][c]);
            if (in > 2) before = join<SEG>(before, three[2][c]);
            h[c] = apply<SEG>(before, h[c]);
        }
    } else {
#pragma unroll
        for (int c = 0; c < V; ++c) {
            Map before = NOTHING;
#pragma unroll
            for (int i = 0; i < 3; ++i) before = join<SEG>(before, in > i ? three[i][c] : NOTHING);
            h[c] = apply<SEG>(before, h[c]);
        }
    }
}

// The number of a row's live steps.
__device__ __forceinline__ int live_to(const RecArgs& a, int b) { return a.lengths ? max(0, min(a.lengths[b], a.T)) : a.T; }
// The wave's entries of the map in one or two loads (asked for ahead of the data), a lane each; a stretch takes its 8 bits of a ballot.
template <int LANES> struct Entries { int e[(64 / LANES * L + 63) / 64]; };
template <int LANES, bool SEG> __device__ __forceinline__ Entries<LANES> map_entries(const RecArgs& a, int b, int from) {
    constexpr int N = 64 / LANES * L;
    Entries<LANES> r{};
    if (SEG) {
#pragma unroll
        for (int i = 0; i < (N + 63) / 64; ++i) {
            const int at = 64 * i + threadIdx.x % 64, t = from + threadIdx.x / 64 * N + at;
            r.e[i] = at < N && t < a.T ? a.seg_start[(long long)b * a.T + t] - t : 1;
        }
    }
    return r;
}
template <int LANES, bool SEG> __device__ __forceinline__ int begins_in(const Entries<LANES>& entries, int live) {
    static_assert(L == 8, "a stretch is a byte of a ballot");
    if (!SEG) return 0;
    const int row = threadIdx.x % 64 / LANES;
    unsigned long long bits = __ballot(entries.e[0] == 0);
    if constexpr (64 / LANES * L > 64) {
        const unsigned long long more = __ballot(entries.e[1] == 0);
        if (row >= 8) bits = more;
    }
    return (int)(bits >> (row % 8 * L)) & ((1 << live) - 1);
}

// One chunk of one tile.  Each thread reduces its stretch to a map, the wave joins its rows', wave 0 the chunk's and its group's while
// waves 1 and 2 find the state before the group; then each thread knows the state before its stretch and runs over it again, out of
// its registers.  z is read once.  Chunks that are live to their end (FULL) run without a test at every step: the steps' exponentials
// and reciprocals then overlap (8 x 24064 x 512: bf16 forward 169 us, with the tests 187, backward 290 and 330; float32, which waits for
// memory, 285 and 282).  In a packed slot most waves hold no beginning, and run as in any other row.
//
// What bounds it at 8 x 24064 x 512: float32 memory, 270 us for 1.58 GB, with the vector units issuing 30% of the time.  bf16 the vector units,
// 73% of the time in packed slots -- four transcendentals an element, at a quarter of the rate --, 171 us for 0.79 GB.
template <typename E, int G, int V, int LANES, int WAVES, bool SEG, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES, WAVES > 4 ? 2 : sizeof(E) == 2 ? 4 : 3) wnv_recurrence_fwd(RecArgs a) {
    typedef Shape<LANES, WAVES> S;
    constexpr int W = LANES * V, STEPS = S::STEPS;
    __shared__ Map quads[S::QUADS][W], blocks[S::BLOCKS][W], prev[S::BLOCKS][W], chunk[W], groups[W];
    __shared__ float base[W];
    const int tid = threadIdx.x, lane = tid % LANES, wave = __builtin_amdgcn_readfirstlane(tid / 64), at = lane * V;
    const int quad = LANES == 16 ? __builtin_amdgcn_readfirstlane(tid / 64) : tid / (4 * LANES), part = quad / 4 >> a.part_bits, parts = S::BLOCKS >> a.part_bits;
    Place p;
    if (!draw_place<false>(a, W, p)) return;
    const int c = min(p.tile * W + at, a.C - V), n = live_to(a, p.b);
    const int t0 = p.chunk * STEPS + tid / LANES * L, live = max(0, min(L, n - t0));
    const bool whole = p.chunk * STEPS + STEPS <= n;
    const Entries<LANES> entries = map_entries<LANES, SEG>(a, p.b, p.chunk * STEPS);
    const E* z = (const E*)a.z + (long long)p.b * a.zb + (long long)p.chunk * STEPS * a.zt;
    const uint32_t from = (uint32_t)(tid / LANES * L * a.zt + c) * (uint32_t)sizeof(E);

    Vec<E, V> f[L], v[L], o[L];
    Steps<E, V> steps;
    Map m[V], before[V];
    int begins = 0;
    const auto reduce = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || l < live) {
                f[l] = load<E, V, STREAM>(z + l * a.zt, from);
                v[l] = load<E, V, STREAM>(z + l * a.zt + a.C, from);
                if (G == 3) o[l] = load<E, V, STREAM>(z + l * a.zt + 2 * a.C, from);
            }
        begins = begins_in<LANES, SEG>(entries, live);
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = NOTHING;
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || l < live) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float u;
                    const float keep = wnv_gates(f[l].get(i), u), put = u * v[l].get(i);
                    steps.hold(l, i, keep, u, put);
                    step<false>(m[i], keep, u, put, false);
                }
            }
    };
    if (whole) reduce(std::true_type{});
    else reduce(std::false_type{});
    const bool any = SEG && __any(begins);
    const auto rows = [&](auto seg) {
        constexpr bool AT = decltype(seg)::value;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (AT && begins) {          // the state of its last utterance, from nothing
#pragma unroll
                for (int l = 0; l < L; ++l)
                    if (l < live) m[i].b = steps.run(l, i, begins >> l & 1 ? 0.f : m[i].b, v[l].get(i));
            }
            finish<AT>(m[i], begins);
            Map all;
            join_quad<LANES, false, AT>(m[i], all, before[i]);
            if (tid % (4 * LANES) < LANES) quads[quad][at + i] = all;
        }
    };
    if (any) rows(std::integral_constant<bool, SEG>{});
    else rows(std::false_type{});
    __syncthreads();
    const int ch = tid % 64;
    if (wave < 3 && ch < W) {
        const Slots slots = slots_at(a.slots, p.row, a.chunks, W, ch);
        if (wave == 0) {
            chunk[ch] = join_blocks<W, S::QUADS, false, SEG>(a, slots, p.chunk, ch, quads, blocks, prev);
        } else if (wave == 1) {
            base[ch] = state_before_groups<W, SEG>(slots, p.chunk, a.h0 ? a.h0[p.b * a.h0b + min(p.tile * W + ch / V * V, a.C - V) + ch % V] : 0.f);
        } else {
            groups[ch] = map_of_groups<W, SEG>(slots, p.chunk);
        }
    }
    __syncthreads();

    if (ends_section(p.chunk, a.chunks) && tid < W) hand_out_section<W, SEG>(a, p.row, p.chunk, tid, chunk[tid], prev[0][tid], groups[tid], base[tid]);
    float h[V];
    const int last_quad = parts > 1 ? (((a.T - 1) / BLOCK >> a.part_bits) + 1 << a.part_bits) * 4 - 1 : S::QUADS - 1;      // of the last part that is there
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = apply<SEG>(prev[part][at + i], apply<SEG>(groups[at + i], base[at + i]));
        if (a.saved && quad == part << a.part_bits + 2 && tid % (4 * LANES) < LANES)
            a.saved[(((long long)p.row * a.chunks + p.chunk) * parts + part) * W + at + i] = h[i];
    }
    state_before_quad<W, V, S::QUADS, false, SEG>(a, quads, blocks, quad, at, h);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = apply<SEG>(before[i], h[i]);
    }
    E* y = (E*)a.y + ((long long)p.b * a.T + (long long)p.chunk * STEPS) * a.C;
    const uint32_t to = (uint32_t)(tid / LANES * L * a.C + c) * (uint32_t)sizeof(E);
    const auto run = [&](auto full, auto seg) {
        constexpr bool FULL = decltype(full)::value, AT = decltype(seg)::value;
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || t0 + l < a.T) {
                float out[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float q = 0.f;
                    if (FULL || l < live) {
                        if (AT && begins >> l & 1) h[i] = 0.f;
                        h[i] = steps.run(l, i, h[i], v[l].get(i));
                        q = h[i];
                        if (G == 3) q *= wnv_gate(o[l].get(i));
                    }
                    out[i] = q;
                }
                store<E, V, STREAM>(y + (long long)l * a.C, to, out);
            }
    };
    if (whole && !any) run(std::true_type{}, std::false_type{});
    else if (SEG && whole) run(std::true_type{}, std::integral_constant<bool, SEG>{});
    else run(std::false_type{}, std::integral_constant<bool, SEG>{});
    if (p.chunk + 1 == a.chunks && quad == last_quad && tid % (4 * LANES) >= 3 * LANES) {       // its last stretch: the state behind it
#pragma unroll
        for (int i = 0; i < V; ++i) a.h_last[(long long)p.b * a.C + c + i] = h[i];
    }
}

// g_t = dy_t sigmoid(o_t);  dh_t = g_t + (what step t+1 hands back);  hands back r = a_t dh_t, nothing over a beginning
// df = dh (h_{t-1} - v) a u;  dv = dh u;  do = dy h sigmoid(o) (1 - sigmoid(o))
// The chunks run from the last to the first, r is found the way the forward pass finds h; h itself starts from the state that the
// forward pass saved before each chunk and is run through again.
template <typename E, int G, int V, int LANES, int WAVES, bool SEG, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES, 2) wnv_recurrence_bwd(RecArgs a) {
    typedef Shape<LANES, WAVES> S;
    constexpr int W = LANES * V, STEPS = S::STEPS;
    __shared__ Map ahead[S::QUADS][W], back[S::QUADS][W], ahead_blocks[S::BLOCKS][W], back_blocks[S::BLOCKS][W], prev[S::BLOCKS][W], chunk[W], groups[W];    // of h and of r
    __shared__ float base[W];
    const int tid = threadIdx.x, lane = tid % LANES, wave = __builtin_amdgcn_readfirstlane(tid / 64), at = lane * V;
    const int quad = LANES == 16 ? __builtin_amdgcn_readfirstlane(tid / 64) : tid / (4 * LANES), part = quad / 4 >> a.part_bits, parts = S::BLOCKS >> a.part_bits;
    Place p;
    if (!draw_place<true>(a, W, p)) return;
    const int order = a.chunks - 1 - p.chunk, c = min(p.tile * W + at, a.C - V), n = live_to(a, p.b);
    const int t0 = p.chunk * STEPS + tid / LANES * L, live = max(0, min(L, n - t0));
    const bool whole = p.chunk * STEPS + STEPS <= n;
    const Entries<LANES> entries = map_entries<LANES, SEG>(a, p.b, p.chunk * STEPS);
    const E* z = (const E*)a.z + (long long)p.b * a.zb + (long long)p.chunk * STEPS * a.zt;
    const E* dy = (const E*)a.dy + (long long)p.b * a.dyb + (long long)p.chunk * STEPS * a.dyt;
    const uint32_t from = (uint32_t)(tid / LANES * L * a.zt + c) * (uint32_t)sizeof(E);
    const uint32_t dfrom = (uint32_t)(tid / LANES * L * a.dyt + c) * (uint32_t)sizeof(E);

    Vec<E, V> f[L], v[L], o[L], d[L];
    Vec<float, V> saved;
    float keep[L][V], u[L][V], g[L][V], q[L][V];        // a, u; dy sigmoid(o); dy sigmoid(o) (1 - sigmoid(o))
    Map m[V], r[V];
    int begins = 0;
    const auto reduce = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || l < live) {
                f[l] = load<E, V, STREAM>(z + l * a.zt, from);
                v[l] = load<E, V, STREAM>(z + l * a.zt + a.C, from);
                if (G == 3) o[l] = load<E, V, STREAM>(z + l * a.zt + 2 * a.C, from);
                if (a.dy) d[l] = load<E, V, STREAM>(dy + l * a.dyt, dfrom);
            }
        saved = load<float, V, false>(a.saved + ((long long)p.row * a.chunks + p.chunk) * parts * W, (part * W + at) * 4);
        begins = begins_in<LANES, SEG>(entries, live);
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = r[i] = NOTHING;
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || l < live) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    keep[l][i] = wnv_gates(f[l].get(i), u[l][i]);
                    step<SEG>(m[i], keep[l][i], u[l][i], u[l][i] * v[l].get(i), begins >> l & 1);
                    g[l][i] = a.dy ? d[l].get(i) : 0.f;
                    if (G == 3) {
                        const float so = wnv_gate(o[l].get(i), q[l][i]);
                        q[l][i] *= g[l][i];
                        g[l][i] *= so;
                    }
                }
            }
#pragma unroll
        for (int l = L - 1; l >= 0; --l)
            if (FULL || l < live) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float dh = g[l][i] + r[i].b;
                    r[i].b = SEG && begins >> l & 1 ? 0.f : keep[l][i] * dh;
                }
            }
    };
    if (whole) reduce(std::true_type{});
    else reduce(std::false_type{});
    Map h_before[V], r_before[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        finish<SEG>(m[i], begins);
        r[i].p = m[i].p;
        r[i].u = m[i].u;
        Map all, all_back;
        join_quad<LANES, false, SEG>(m[i], all, h_before[i]);
        join_quad<LANES, true, SEG>(r[i], all_back, r_before[i]);
        if (tid % (4 * LANES) < LANES) ahead[quad][at + i] = all, back[quad][at + i] = all_back;
    }
    __syncthreads();
    const int ch = tid % 64;
    if (wave < (S::BLOCKS > 1 ? 4 : 3) && ch < W) {
        const Slots slots = slots_at(a.slots, p.row, a.chunks, W, ch);
        if (wave == 0) {
            chunk[ch] = join_blocks<W, S::QUADS, true, SEG>(a, slots, order, ch, back, back_blocks, prev);
        } else if (wave == 1) {
            base[ch] = state_before_groups<W, SEG>(slots, order, a.dh_last ? a.dh_last[(long long)p.b * a.C + min(p.tile * W + ch / V * V, a.C - V) + ch % V] : 0.f);
        } else if (wave == 2) {
            groups[ch] = map_of_groups<W, SEG>(slots, order);
        } else {
#pragma unroll
            for (int k = 0; k < S::BLOCKS; ++k) ahead_blocks[k][ch] = block_of<false, SEG>(ahead, k, ch);
        }
    }
    __syncthreads();

    if (ends_section(order, a.chunks) && tid < W) hand_out_section<W, SEG>(a, p.row, order, tid, chunk[tid], prev[0][tid], groups[tid], base[tid]);
    float h[V], x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = saved.get(i);
        x[i] = apply<SEG>(prev[part][at + i], apply<SEG>(groups[at + i], base[at + i]));
    }
    state_before_quad<W, V, S::QUADS, false, SEG>(a, ahead, ahead_blocks, quad, at, h);
    state_before_quad<W, V, S::QUADS, true, SEG>(a, back, back_blocks, quad, at, x);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = apply<SEG>(h_before[i], h[i]);
        x[i] = apply<SEG>(r_before[i], x[i]);
    }
    E* dz = (E*)a.dz + ((long long)p.b * a.T + (long long)p.chunk * STEPS) * (G * (long long)a.C);
    const uint32_t to = (uint32_t)(tid / LANES * L * G * a.C + c) * (uint32_t)sizeof(E);
    const auto run = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        float behind[L][V];
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (FULL || l < live) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float before = SEG && begins >> l & 1 ? 0.f : l ? behind[l - 1][i] : h[i];
                    behind[l][i] = fmaf(keep[l][i], before, u[l][i] * v[l].get(i));
                }
            }
#pragma unroll
        for (int l = L - 1; l >= 0; --l)
            if (FULL || t0 + l < a.T) {
                float df[V], dv[V], dg[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float xf = 0.f, xv = 0.f, xo = 0.f;
                    if (FULL || l < live) {
                        const float before = SEG && begins >> l & 1 ? 0.f : l ? behind[l - 1][i] : h[i];
                        const float slope = keep[l][i] * u[l][i], dh = g[l][i] + x[i];
                        xf = dh * fmaf(slope, before, -(slope * v[l].get(i)));      // the difference itself may overflow
                        xv = dh * u[l][i];
                        if (G == 3) xo = q[l][i] * behind[l][i];
                        x[i] = SEG && begins >> l & 1 ? 0.f : keep[l][i] * dh;
                    }
                    df[i] = xf;
                    dv[i] = xv;
                    dg[i] = xo;
                }
                E* row = dz + (long long)l * G * a.C;
                store<E, V, STREAM>(row, to, df);
                store<E, V, STREAM>(row + a.C, to, dv);
                if (G == 3) store<E, V, STREAM>(row + 2 * (long long)a.C, to, dg);
            }
    };
    if (whole) run(std::true_type{});
    else run(std::false_type{});
    if (p.chunk == 0 && a.dh0 && tid < LANES) {         // the first stretch: what flows out of it
#pragma unroll
        for (int i = 0; i < V; ++i) a.dh0[(long long)p.b * a.C + c + i] = x[i];
    }
}

__global__ void __launch_bounds__(256) wnv_recurrence_fill(uint4* p, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = uint4{EMPTY, EMPTY, EMPTY, EMPTY};
}

constexpr int RT = 64;

template <typename E>
__global__ void __launch_bounds__(RT) wnv_recurrence_one(const E* z, long long zb, float* state, E* y, int C, int gates) {
    const int c = blockIdx.x * RT + threadIdx.x, b = blockIdx.y;
    if (c >= C) return;
    z += (long long)b * zb + c;
    float h = state[(long long)b * C + c];
    h = wnv_blend(wnv_up(z[0]), h, wnv_up(z[C]));
    state[(long long)b * C + c] = h;
    if (gates == 3) h *= wnv_gate(wnv_up(z[2 * C]));
    y[(long long)b * C + c] = wnv_down<E>(h);
}

#define WNV_BY_TYPE(dtype, ...)                                                       \
    switch (dtype) {                                                                  \
        case WNV_F32: { using E = float; __VA_ARGS__; break; }                        \
        case WNV_BF16: { using E = wnv_bf16; __VA_ARGS__; break; }                    \
        default: { using E = wnv_f16; __VA_ARGS__; break; }                           \
    }

wnv_status check_shape(const char* who, int device, int64_t B, int64_t T, int64_t C, int gates, int dtype) {
    if (device < 0) return fail(WNV_ERR_INVALID_ARG, "%s: device must be >= 0", who);
    if (B <= 0 || T <= 0 || C <= 0) return fail(WNV_ERR_INVALID_ARG, "%s: B, T and C must be positive", who);
    if (T > (1 << 30)) return fail(WNV_ERR_UNSUPPORTED, "%s: at most 2^30 steps", who);
    if (B > 65535 || C > (1 << 20)) return fail(WNV_ERR_UNSUPPORTED, "%s: at most 65535 rows and 2^20 channels", who);
    if (gates != 2 && gates != 3) return fail(WNV_ERR_INVALID_ARG, "%s: gates must be 2 (f, v) or 3 (f, v, o)", who);
    if (!wnv_dtype_size(dtype)) return fail(WNV_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    return WNV_OK;
}

wnv_status launched(const char* who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WNV_OK : fail(WNV_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

// How B x T x C is cut.  Tiles are 64 channels and chunks 128 steps, or narrow ones of 16 channels (4 with V = 1) and 512 steps:
//  * where rows are narrow, lanes along the channels are idle, and with them go a quarter of the chunks to wait for (forward and
//    backward of 16 x 24064, us, narrow tiles and wide ones: float32 C = 20 99 and 126, C = 40 191 and 172; bf16 C = 32 87 and 121,
//    C = 48 119 and 135);
//  * where there is little data and that makes one chunk of several, which needs neither a filled workspace nor a wait: the host's
//    time falls by a launch and an allocation (2 x 300 x 128 float32 forward 10.1 us a call and 14.2, 2 x 400 x 512 10.3 and 14.6).
// Of narrow tiles two chunks become one of 8 waves, for the same reason (2 x 700 x 128 float32 forward 10.2 us a call and 14.6).
// More data is the GPU's time, and is read faster in whole lines by more workgroups (64 x 700 x 128 float32 forward 31 us in narrow
// tiles of 8 waves and 27 in wide ones, backward 43 and 42; 64 x 512 x 512 backward 119 and 97).
constexpr int NARROW_CHANNELS = 32, LITTLE_CHANNELS = 256;
constexpr int64_t LITTLE = 2 << 20;
struct Cut { int V, lanes, waves, W, tiles, chunks, part_bits, parts; };
Cut cut_of(int64_t B, int64_t T, int C) {
    constexpr int WIDE = Shape<16, 4>::STEPS, NARROW = Shape<4, 4>::STEPS;
    Cut c;
    const bool little = B * T * C <= LITTLE;
    const bool narrow = C <= NARROW_CHANNELS || (little && T > WIDE && T <= (C <= LITTLE_CHANNELS ? 2 * NARROW : NARROW));
    const bool joined = narrow && little && T > NARROW && T <= 2 * NARROW;
    const int steps = joined ? 2 * NARROW : narrow ? NARROW : WIDE;
    c.V = C < 4 ? 1 : 4;
    c.lanes = narrow ? 4 : 16;
    c.waves = joined ? 8 : 4;
    c.W = c.lanes * c.V;
    c.tiles = (C + c.W - 1) / c.W;
    c.chunks = (int)((T + steps - 1) / steps);
    c.part_bits = C <= NARROW_CHANNELS ? 2 : 0;
    c.parts = steps / BLOCK >> c.part_bits;
    return c;
}

wnv_status check_strides(const char* who, const wnv_recurrence_args* a, const Cut& c) {
    if (a->z_batch_stride < 0 || a->z_time_stride < 0 || (a->h0 && a->h0_batch_stride < 0) ||
        (a->dy && (a->dy_batch_stride < 0 || a->dy_time_stride < 0)))
        return fail(WNV_ERR_INVALID_ARG, "%s: negative stride", who);
    // a lane's offset within a chunk is 32 bits: of 1016 steps at most in narrow tiles, 120 in others, of 4 bytes an element
    const int64_t most = c.lanes == 4 ? 1 << 20 : 1 << 22;
    if (a->T > 1 && (a->z_time_stride >= most || (a->dy && a->dy_time_stride >= most)))
        return fail(WNV_ERR_UNSUPPORTED, "%s: time strides of %lld elements and more", who, (long long)most);
    return WNV_OK;
}

int64_t slot_bytes(int64_t B, const Cut& c) { return c.chunks > 1 ? B * c.tiles * slots_of_row(c.chunks, c.W) * 8 : 0; }

// The kernel's arguments; the workspace is filled on the way.
wnv_status prepare(const char* who, const wnv_recurrence_args* a, const Cut& c, RecArgs& k) {
    k.B = a->B; k.C = a->C; k.T = (int)a->T;
    k.tiles = c.tiles; k.chunks = c.chunks; k.part_bits = c.part_bits;
    k.zb = a->z_batch_stride; k.zt = a->T > 1 ? a->z_time_stride : 0; k.h0b = a->h0_batch_stride;
    k.z = a->z; k.h0 = a->h0; k.lengths = a->lengths; k.seg_start = a->seg_start;
    k.y = a->y; k.h_last = a->h_last; k.saved = (float*)a->saved; k.slots = (unsigned long long*)a->workspace;
    k.dy = a->dy; k.dyb = a->dy_batch_stride; k.dyt = a->T > 1 ? a->dy_time_stride : 0;
    k.dh_last = a->dh_last; k.dz = a->dz; k.dh0 = a->dh0;
    const int64_t threads = ((int64_t)k.B * k.chunks + 7) * k.tiles * c.waves * 64, bytes = slot_bytes(a->B, c);
    if (threads > UINT32_MAX) return fail(WNV_ERR_UNSUPPORTED, "%s: B x T x C is too large", who);
    if (bytes) {
        if (!a->workspace) return fail(WNV_ERR_INVALID_ARG, "%s: workspace is NULL", who);
        hipLaunchKernelGGL(wnv_recurrence_fill, dim3((unsigned)((bytes / 16 + 255) / 256)), dim3(256), 0, (hipStream_t)a->stream,
                           (uint4*)a->workspace, (long long)(bytes / 16));
        return launched(who);       // the chunks draw from what it writes: nothing runs without it
    }
    return WNV_OK;
}

template <typename E, int G, int V, int LANES, int WAVES, bool STREAM> void launch(bool back, const wnv_recurrence_args* a, const RecArgs& k) {
    const dim3 grid((unsigned)(((int64_t)k.B * k.chunks + 7) / 8 * 8 * k.tiles)), block(64 * WAVES);
    hipStream_t s = (hipStream_t)a->stream;
    if (back) {
        if (a->seg_start) hipLaunchKernelGGL((wnv_recurrence_bwd<E, G, V, LANES, WAVES, true, STREAM>), grid, block, 0, s, k);
        else hipLaunchKernelGGL((wnv_recurrence_bwd<E, G, V, LANES, WAVES, false, STREAM>), grid, block, 0, s, k);
    } else {
        if (a->seg_start) hipLaunchKernelGGL((wnv_recurrence_fwd<E, G, V, LANES, WAVES, true, STREAM>), grid, block, 0, s, k);
        else hipLaunchKernelGGL((wnv_recurrence_fwd<E, G, V, LANES, WAVES, false, STREAM>), grid, block, 0, s, k);
    }
}
// Whether data goes past the caches: more than the 256 MB of the last level, in whole lines.
bool streams(bool back, const wnv_recurrence_args* a) {
    const int64_t e = wnv_dtype_size(a->dtype), bytes = a->B * a->T * a->C * e * (back ? 2 * a->gates + 1 : a->gates + 1);
    uint64_t odd = (uint64_t)a->z | (uint64_t)(a->C * e) | (uint64_t)(a->z_time_stride * e) | (uint64_t)(a->z_batch_stride * e);
    if (back) odd |= (uint64_t)a->dz | (uint64_t)a->dy | (uint64_t)(a->dy_time_stride * e) | (uint64_t)(a->dy_batch_stride * e);
    else odd |= (uint64_t)a->y;
    return bytes > (256 << 20) && odd % 128 == 0;
}
template <typename E, int G> void launch(bool back, const wnv_recurrence_args* a, const Cut& c, const RecArgs& k) {
    if (c.lanes == 16) {
        streams(back, a) ? launch<E, G, 4, 16, 4, true>(back, a, k) : launch<E, G, 4, 16, 4, false>(back, a, k);
    } else if (c.V == 4) {              // rows of less than a line
        c.waves == 8 ? launch<E, G, 4, 4, 8, false>(back, a, k) : launch<E, G, 4, 4, 4, false>(back, a, k);
    } else {
        c.waves == 8 ? launch<E, G, 1, 4, 8, false>(back, a, k) : launch<E, G, 1, 4, 4, false>(back, a, k);
    }
}
template <typename E> void launch(bool back, const wnv_recurrence_args* a, const Cut& c, const RecArgs& k) {
    if (a->gates == 3) launch<E, 3>(back, a, c, k);
    else launch<E, 2>(back, a, c, k);
}

}  // namespace

extern "C" int64_t wnv_recurrence_saved_bytes(int32_t B, int64_t T, int32_t C, int32_t gates, int32_t dtype) {
    if (check_shape("wnv_recurrence_saved_bytes", 0, B, T, C, gates, dtype) != WNV_OK) return -1;
    const Cut c = cut_of(B, T, C);
    return (int64_t)B * c.tiles * c.chunks * c.parts * c.W * 4;
}

extern "C" int64_t wnv_recurrence_workspace_bytes(int32_t B, int64_t T, int32_t C, int32_t gates, int32_t dtype) {
    if (check_shape("wnv_recurrence_workspace_bytes", 0, B, T, C, gates, dtype) != WNV_OK) return -1;
    return slot_bytes(B, cut_of(B, T, C));
}

extern "C" wnv_status wnv_recurrence_forward(int32_t device, const wnv_recurrence_args* a) {
    if (!a || !a->z || !a->y || !a->h_last) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_forward: NULL argument");
    if (wnv_status st = check_shape("wnv_recurrence_forward", device, a->B, a->T, a->C, a->gates, a->dtype)) return st;
    const Cut c = cut_of(a->B, a->T, a->C);
    if (wnv_status st = check_strides("wnv_recurrence_forward", a, c)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_forward: cannot select device %d", device);
    RecArgs k{};
    if (wnv_status st = prepare("wnv_recurrence_forward", a, c, k)) return st;
    WNV_BY_TYPE(a->dtype, launch<E>(false, a, c, k));
    return launched("wnv_recurrence_forward");
}

extern "C" wnv_status wnv_recurrence_backward(int32_t device, const wnv_recurrence_args* a) {
    if (!a || !a->z || !a->saved || !a->dz) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_backward: NULL argument");
    if (wnv_status st = check_shape("wnv_recurrence_backward", device, a->B, a->T, a->C, a->gates, a->dtype)) return st;
    const Cut c = cut_of(a->B, a->T, a->C);
    if (wnv_status st = check_strides("wnv_recurrence_backward", a, c)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_backward: cannot select device %d", device);
    RecArgs k{};
    if (wnv_status st = prepare("wnv_recurrence_backward", a, c, k)) return st;
    WNV_BY_TYPE(a->dtype, launch<E>(true, a, c, k));
    return launched("wnv_recurrence_backward");
}

extern "C" wnv_status wnv_recurrence_step(int32_t device, const void* z, int64_t z_batch_stride, float* state, void* y, int32_t B,
                                          int32_t C, int32_t gates, int32_t dtype, void* stream) {
    if (!z || !state || !y) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_step: NULL argument");
    if (z_batch_stride < 0) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_step: negative stride");
    if (wnv_status st = check_shape("wnv_recurrence_step", device, B, 1, C, gates, dtype)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_step: cannot select device %d", device);
    const dim3 grid((C + RT - 1) / RT, B);
    WNV_BY_TYPE(dtype, hipLaunchKernelGGL(wnv_recurrence_one<E>, grid, dim3(RT), 0, (hipStream_t)stream, (const E*)z,
                                          (long long)z_batch_stride, state, (E*)y, C, gates));
    return launched("wnv_recurrence_step");
}
