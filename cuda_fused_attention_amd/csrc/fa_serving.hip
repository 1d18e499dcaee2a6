// Attention for serving: new tokens over a paged K/V cache, and queries over an
// encoder's states of another length. One kernel computes both; they differ in
// where the rows of a sequence and its keys lie.
//
//   O[i] = sum_j P_ij V_j / sum_j P_ij,  P_ij = exp(q_i . k_j / sqrt(D) - m_i),
//
// over the keys j < limit(i). The running base m_i and sum stay in 32 bits; the
// weights are rounded to the element type for the second matrix product (half a
// step of 16 bits each, as in the fused self-attention), and their sum uses the
// rounded values.
//
// Work: the query heads that share a key head are packed beside each other, row
// r of a sequence is token r / group and head r % group of the key head, so K and
// V are read once for all of them. A workgroup owns 32 * kWaves rows of one key
// head (a wave owns 32) and walks 32-key tiles that its waves copy HBM -> LDS
// together; with one new token only one wave has rows, and the others only copy.
// Few rows over many keys leave the device idle, so the keys of a row block are
// split into chunks over workgroups; their partial results (O, base, sum in 32 bits)
// are joined by a second kernel (3.5-7 us of a call's time). Two wave groups of a
// workgroup can take half of its keys each and meet in LDS, which spares the join.
//
// Measured on one MI355X, back to back (a large copy runs at 4.9 TB/s here, a large
// bf16 matrix product at 1.16-1.21 PFLOP/s):
//   64 sequences decode over 512 to 8192 keys, 32 heads on 8, dim 128: 220-230 us for
//   1.14 GB, 5.0-5.2 TB/s: bound by reading K and V;
//   2048 new tokens over 30720 cached, 32 heads on 8, dim 128: 876 us, 1.22 PFLOP/s, and
//   (4,8,2048) queries on 8192 states, dim 128: 230-237 us, 1.16-1.19 PFLOP/s: bound by
//   the matrix cores and the LDS reads of their operands, as the fused forward is;
//   one sequence, 8 heads, 2049 keys, dim 64: 9.1 us, all latency: 5.7 in the attention
//   kernel (2.1 until the first tile has come, 0.58 a step), 3.8 in the join.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fa_paged.hpp"
#include "fa_serving_core.hpp"

namespace {

using namespace fa::serving;
using fa::f32x16;
using fa::f32x4;
using fa::i32x4;

constexpr int kMaxSplits = 256;
constexpr long long kMaxKeys = 1LL << 30;  // of one sequence
constexpr long long kMaxRows = 1LL << 30;  // of one sequence and key head

// One launch. Strides and offsets are in elements.
struct Args
{
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* o;
    float* part;         // [row][split][D] of the split launches
    float* base_sum;     // [row][split][2]
    const int* table;    // paged: block table
    const int* starts;   // paged: first token of each sequence
    const int* lens;     // keys of each sequence (may be null where not paged)
    long long q_seq, q_head, q_row;
    long long o_seq, o_head, o_row;
    long long k_seq, k_head, k_row;  // k_seq: from page to page, or from sequence to sequence
    long long v_seq, v_head, v_row;
    long long table_stride;
    int table_width, num_blocks, block_shift;
    int seqs, tokens, heads_kv, group, max_queries, max_keys;
    int slots;      // row blocks of a key head over all sequences
    int per_seq;    // row blocks per sequence; 0: found from `starts`
    int splits, chunk;
    int causal;
    float c_log2;   // log2(e) / sqrt(D)
};

// What a row block works on.
struct Block
{
    int seq, head;       // sequence, key head
    int row0, rows;      // first row within the sequence, rows of the sequence
    int first_token;     // paged: the sequence's first row of q
    int keys;            // keys in reach
    int shift;           // token i sees the keys below shift + i + 1 (causal)
    int end;             // keys that the block's last row sees
    int splits;          // chunks of those keys
};

__device__ __forceinline__ int limit_of(const Args& a, const Block& b, int token)
{
    return a.causal ? max(0, min(b.keys, b.shift + token + 1)) : b.keys;
}

typedef const __attribute__((address_space(4))) int ConstInt;  // read through the scalar cache

// The block of `slot` (of R rows). False: it holds no row.
template <int R, bool kPaged>
__device__ __forceinline__ bool find_block(const Args& a, int slot, int head, Block& b)
{
    int rb, tokens;
    b.head = head;
    if constexpr (kPaged)
    {
        auto clamped = [&](int start) { return max(0, min(start, a.tokens)); };
        int start, end, len;
        if (a.per_seq > 0)
        {
            b.seq = slot / a.per_seq;
            rb = slot % a.per_seq;
            const ConstInt* const starts = (const ConstInt*)(a.starts + b.seq);
            start = starts[0];
            end = starts[1];
            len = *(const ConstInt*)(a.lens + b.seq);
        }
        else
        {
            // Sequence s owns the slots from floor(first row / R) + s on, at least
            // as many as it has blocks. 64 sequences are compared at a time, each time
            // one 64th of those left; the last time the lanes hold their ends and
            // lengths too.
            const int lane = threadIdx.x & 63;
            int lo = 0, hi = a.seqs, first = 0;
            while (true)
            {
                const int step = (hi - lo + 63) / 64;
                const int s = min(lo + lane * step, hi - 1);
                start = a.starts[s];
                end = a.starts[s + 1];
                len = a.lens[s];
                first = static_cast<int>(static_cast<long long>(clamped(start)) * a.group / R) + s;
                const int below = __popcll(__ballot(lo + lane * step < hi && first <= slot));
                const int at = max(1, below) - 1;
                if (step == 1)
                {
                    b.seq = lo + at;
                    start = __builtin_amdgcn_readlane(start, at);
                    end = __builtin_amdgcn_readlane(end, at);
                    len = __builtin_amdgcn_readlane(len, at);
                    rb = slot - __builtin_amdgcn_readlane(first, at);
                    break;
                }
                lo += at * step;
                hi = min(hi, lo + step);
            }
        }
        b.first_token = uniform(clamped(start));
        tokens = max(0, uniform(clamped(end)) - b.first_token);
        len = max(0, uniform(len));
        b.keys = static_cast<int>(min(static_cast<long long>(len), static_cast<long long>(a.table_width) << a.block_shift));
        b.shift = len - tokens;
        b.rows = min(tokens, a.max_queries) * a.group;
    }
    else
    {
        b.seq = slot / a.per_seq;
        rb = slot % a.per_seq;
        b.first_token = 0;
        b.keys = a.lens ? max(0, min(*(const ConstInt*)(a.lens + b.seq), a.max_keys)) : a.max_keys;
        b.shift = 0;
        b.rows = a.max_queries * a.group;
    }
    if (rb < 0 || static_cast<long long>(rb) * R >= b.rows) return false;
    b.seq = uniform(b.seq);
    b.keys = uniform(b.keys);
    b.rows = uniform(b.rows);
    b.row0 = uniform(rb * R);
    b.end = uniform(limit_of(a, b, (min(b.row0 + R, b.rows) - 1) / a.group));
    b.splits = uniform(max(1, min(a.splits, (b.end + a.chunk - 1) / a.chunk)));
    return true;
}

// Row r's place among all rows of q (the partial results' rows).
template <bool kPaged>
__device__ __forceinline__ long long part_row(const Args& a, const Block& b, int token, int h)
{
    const long long t = kPaged ? static_cast<long long>(b.first_token) + token
                               : static_cast<long long>(b.seq) * a.max_queries + token;
    return t * (static_cast<long long>(a.heads_kv) * a.group) + b.head * a.group + h;
}

// Where a block's keys lie. Sixteen keys from a multiple of 16 on lie in one
// page, so a copy's descriptor is scalar: the page's number comes through the
// scalar cache (the table is constant during a launch), a step before it is used.
template <int D, bool kPaged>
struct Keys
{
    // Sixteen keys: byte addresses of the first, and the bytes from it on that hold
    // keys. What a copy asks for past those reads as zero: keys past the end, and a
    // page outside the cache.
    struct Half
    {
        uint64_t k, v;
        uint32_t k_bytes, v_bytes;
    };

    const Args& a;
    uint64_t k_base, v_base;
    uint64_t table;
    uint32_t k_row_bytes, v_row_bytes;
    int end;

    __device__ __forceinline__ Keys(const Args& args, const Block& b) : a(args), end(b.end)
    {
        k_base = reinterpret_cast<uint64_t>(a.k) + static_cast<uint64_t>(b.head * a.k_head * 2);
        v_base = reinterpret_cast<uint64_t>(a.v) + static_cast<uint64_t>(b.head * a.v_head * 2);
        if constexpr (!kPaged)
        {
            k_base += static_cast<uint64_t>(b.seq * a.k_seq * 2);
            v_base += static_cast<uint64_t>(b.seq * a.v_seq * 2);
        }
        k_base = uniform(k_base);
        v_base = uniform(v_base);
        table = uniform(reinterpret_cast<uint64_t>(a.table) + static_cast<uint64_t>(b.seq * a.table_stride * 4));
        k_row_bytes = uniform(static_cast<uint32_t>(a.k_row * 2));
        v_row_bytes = uniform(static_cast<uint32_t>(a.v_row * 2));
    }

    // The page that holds `key` (the last one of the row for a key past it).
    // Only where the block sees a key, so the row has an entry.
    __device__ __forceinline__ int page_of(int key) const
    {
        if constexpr (!kPaged) return 0;
        const unsigned entry = static_cast<unsigned>(min(key >> a.block_shift, a.table_width - 1));
        return *(const ConstInt*)(table + static_cast<uint64_t>(entry) * 4);
    }

    // Pages are at most 2^34 elements apart and a page's rows within 2^30, in steps
    // of 16 bytes (host-side checks): 32-bit products but for the page's.
    __device__ __forceinline__ Half half_at(int key, int page) const
    {
        Half r;
        const int left = end - key;
        auto bytes = [&](uint32_t row_bytes) {
            return left >= 16 ? 16 * row_bytes : static_cast<uint32_t>(max(left, 0)) * row_bytes;
        };
        if constexpr (kPaged)
        {
            const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_blocks);
            const uint32_t at = there ? static_cast<uint32_t>(page) : 0u;
            const uint32_t in_page = static_cast<uint32_t>(key) & ((1u << a.block_shift) - 1);
            const uint64_t off = ((static_cast<uint64_t>(at) * static_cast<uint32_t>(a.k_seq >> 3)) << 4) +
                                 in_page * k_row_bytes;
            r.k = k_base + off;
            r.v = v_base + off;
            r.k_bytes = r.v_bytes = there ? bytes(k_row_bytes) : 0u;
        }
        else
        {
            r.k = k_base + static_cast<uint64_t>(static_cast<uint32_t>(key)) * k_row_bytes;
            r.v = v_base + static_cast<uint64_t>(static_cast<uint32_t>(key)) * v_row_bytes;
            r.k_bytes = bytes(k_row_bytes);
            r.v_bytes = bytes(v_row_bytes);
        }
        return r;
    }

    // Buffer descriptor of `bytes` bytes from `base` on (48-bit addresses, stride 0).
    static __device__ __forceinline__ i32x4 descriptor(uint64_t base, uint32_t bytes)
    {
        i32x4 r;
        r[0] = uniform(static_cast<int>(static_cast<uint32_t>(base)));
        r[1] = uniform(static_cast<int>(static_cast<uint32_t>(base >> 32) & 0xffffu));
        r[2] = uniform(static_cast<int>(bytes));
        r[3] = static_cast<int>(fa::kRawBufferConfig);
        return r;
    }

    // Address of a lane's key, for the rare path that reads keys outside the
    // pipeline; false: it holds zeros.
    __device__ __forceinline__ bool lane_key(int key, uint64_t& k) const
    {
        bool there = key < end;
        int page = 0;
        if constexpr (kPaged)
        {
            if (there) page = *reinterpret_cast<const int*>(table + static_cast<uint64_t>(key >> a.block_shift) * 4);
            there = there && static_cast<unsigned>(page) < static_cast<unsigned>(a.num_blocks);
        }
        k = half_at(key, there ? page : 0).k;
        return there;
    }
};

// The rows of a wave and what its lanes see of the keys.
struct Rows
{
    int row;      // the lane's row (at or past Block::rows: none)
    int token, qh;
    int limit;    // keys the lane's row sees; lanes past the last row repeat it
    int t_begin, t_end;  // the workgroup's tiles (equal where nothing is seen)
    int t_last;   // the wave's tiles end here
    int t_mask;   // first tile that some lane does not see whole
    bool unseen;  // some lane does not see keys that the block reads
};

template <int R>
__device__ __forceinline__ Rows wave_rows(const Args& a, const Block& b, int split, int wave, int i)
{
    Rows r;
    r.row = b.row0 + 32 * wave + i;
    const int row_in = min(r.row, b.rows - 1);
    r.token = row_in / a.group;
    r.qh = row_in - r.token * a.group;
    r.limit = limit_of(a, b, r.token);
    const int k_begin = split * a.chunk;
    const int k_end = split == b.splits - 1 ? b.end : k_begin + a.chunk;
    r.t_begin = k_begin / kTileKeys;
    r.t_end = (k_end + kTileKeys - 1) / kTileKeys;
    const int first = b.row0 + 32 * wave;
    const int wave_end = first < b.rows ? limit_of(a, b, min(first + 31, b.rows - 1) / a.group) : 0;
    r.t_last = uniform(min(r.t_end, (wave_end + kTileKeys - 1) / kTileKeys));
    const int least = uniform(limit_of(a, b, min(first, b.rows - 1) / a.group));
    r.t_mask = least / kTileKeys;
    r.unseen = least < b.end;
    return r;
}

template <bool kPaged>
__device__ __forceinline__ long long q_offset(const Args& a, const Block& b, const Rows& r)
{
    return (kPaged ? (b.first_token + static_cast<long long>(r.token)) * a.q_row : b.seq * a.q_seq + r.token * a.q_row) +
           (b.head * a.group + r.qh) * a.q_head;
}

template <bool kPaged>
__device__ __forceinline__ long long o_offset(const Args& a, const Block& b, int token, int qh)
{
    return (kPaged ? (b.first_token + static_cast<long long>(token)) * a.o_row : b.seq * a.o_seq + token * a.o_row) +
           (b.head * a.group + qh) * a.o_head;
}

// Per-lane LDS element offsets of a tile's operand reads.
template <int D>
__device__ __forceinline__ int k_read_offset(int i, int h, int ks)
{
    return i * D + (((2 * ks + h) ^ swz_k<D>(i)) << 3);
}
template <int D>
__device__ __forceinline__ int v_read_offset(int lane, int db)
{
    const int g16 = lane >> 4, s16 = lane & 15;
    const int row = 4 * (g16 >> 1) + (s16 >> 2);
    const int col = 32 * db + 16 * (g16 & 1) + 4 * (s16 & 3);
    return row * D + (((col >> 3) ^ swz_v<D>(row)) << 3) + (col & 7);
}

// A V operand: keys 16*half .. of head dims 32*db .. (`base`: the stage plus the
// lane's offset for db, in elements).
template <typename T, int D>
__device__ __forceinline__ typename Elem<T>::x8 read_v(const uint16_t* base, int half)
{
    const uint16_t* at = base + half * 16 * D;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 8 * D));
    return __builtin_bit_cast(typename Elem<T>::x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A wave's rows of O: the partial result of one chunk in 32 bits, or normalised to
// the element type. A lane holds pieces of 4 dims of its row. In 32 bits they are
// stored as they are. The 8-byte pieces of the whole rows would touch 32 rows at a
// time (2.1-2.5 us at the end of every workgroup of many rows): 128 bytes of each row
// at a time go through `buf` (4 KiB of LDS of the wave's own, 16-byte pieces swizzled
// by row) and leave as whole lines.
template <typename T, int D, bool kPaged>
__device__ __forceinline__ void store_rows(const Args& a, const Block& b, const Rows& r, int split, int lane,
                                           const f32x16 (&o)[D / 32], float m, float l, uint4* buf)
{
    const int i = lane & 31, h = lane >> 5;
    float la, lb;
    row_halves(l, la, lb);
    l = la + lb;
    if (b.splits > 1)
    {
        if (r.row >= b.rows) return;
        const long long pr = part_row<kPaged>(a, b, r.token, r.qh) * a.splits + split;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(a.part + pr * D + 32 * db + 8 * g + 4 * h) =
                    f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
        if (h == 0) *reinterpret_cast<float2*>(a.base_sum + 2 * pr) = float2{m, l};
        return;
    }
    // A row that saw nothing has the sum 0 and gives 0; a NaN sum leaves O's NaN.
    const float inv = l > 0.0f ? __builtin_amdgcn_rcpf(l) : 0.0f;
    // As they leave, lane / 8 of every 8 rows and 16 bytes of its 128: the place of
    // that row comes from the lane that holds it (-1: no row).
    const long long mine = r.row < b.rows ? o_offset<kPaged>(a, b, r.token, r.qh) : -1;
    const int piece = lane & 7;
    long long at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = __shfl(mine, 8 * u + (lane >> 3), 64);
#pragma unroll
    for (int half = 0; half < D / 64; ++half)
    {
#pragma unroll
        for (int x = 0; x < 8; ++x)
        {
            const f32x16& ob = o[2 * half + x / 4];
            uint2 w;
            w.x = pack_pair<T>(ob[4 * (x % 4)] * inv, ob[4 * (x % 4) + 1] * inv);
            w.y = pack_pair<T>(ob[4 * (x % 4) + 2] * inv, ob[4 * (x % 4) + 3] * inv);
            reinterpret_cast<uint2*>(buf + i * 8 + (x ^ (i & 7)))[h] = w;
        }
        fa::wait_vm_lgkm0<63>();  // the wave's own writes; nobody else touches `buf`
#pragma unroll
        for (int u = 0; u < 4; ++u)
        {
            const int row = 8 * u + (lane >> 3);
            const uint4 x = buf[row * 8 + (piece ^ (row & 7))];
            if (at[u] >= 0) *reinterpret_cast<uint4*>(a.o + at[u] + 64 * half + 8 * piece) = x;
        }
        fa::wait_vm_lgkm0<63>();
    }
}

// The block and the chunk of this workgroup; false: nothing to do.
template <int R, bool kPaged>
__device__ __forceinline__ bool take_block(const Args& a, Block& b, int& split)
{
    const int head = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.heads_kv));
    const int rest = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.heads_kv));
    // The heads lie next to each other in the grid, so where 8 divides their number all
    // blocks of a head run on one XCD and share its L2. Late rows see the most keys:
    // they start first. First chunks, which every block has, come before second ones: a
    // head of four has two XCDs, over which the slots alternate (chunk by chunk, the
    // chunks did, and the first ones of short sequences met on one: 76 us against 54 for
    // four chunks beside 29 decoding sequences).
    split = rest / a.slots;
    return find_block<R, kPaged>(a, a.slots - 1 - rest % a.slots, head, b) && split < b.splits;
}

// Keeps a value's producing instructions inside the current block: the compiler
// cannot sink them past the next branch.
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void pin(int& x) { asm volatile("" : "+v"(x)); }
template <typename x8>
__device__ __forceinline__ void pin8(x8& x)
{
    i32x4 bits = __builtin_bit_cast(i32x4, x);
    asm volatile("" : "+v"(bits));
    x = __builtin_bit_cast(x8, bits);
}

// Weights of scores s[kFirst + e], e < 8, against base m into p[e]; their rounded
// values are added to `sum`. kRounded: the product is rounded before the base is
// subtracted, so the score that set the base weighs exactly 2^kBias whatever its
// size; else one fused multiply-add.
template <typename T, bool kRounded>
__device__ __forceinline__ void weigh(const f32x16& s, int first, typename Elem<T>::x8& p, float m, float c_log2, float& sum)
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        float x;
        if constexpr (kRounded)
        {
#pragma clang fp contract(off)
            x = s[first + e] * c_log2 - m;
        }
        else x = fmaf(s[first + e], c_log2, -m);
        p[e] = static_cast<T>(__builtin_amdgcn_exp2f(x));
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) sum = Elem<T>::add_pair(p[e], p[e + 1], sum);
}

// step(masked, P, jj) for jj = 0 .. count-1 with P = jj modulo 6, a multiple of the
// stages and of the two score buffers, as a compile-time constant. Whole rounds in
// which no step's next tile is masked (jj < plain) take steps without the mask: where
// it is a branch, the compiler keeps the masked scores apart and copies all 16 on the
// path that masks nothing (a 2048 x 32768 chunk: 999 -> 908 us together with scalar
// copy addresses). Written out step by step: a recursive template keeps more
// registers live.
template <class Step>
__device__ __forceinline__ void walk(int count, int plain, Step&& step)
{
    int jj = 0;
    for (const int whole = min(count, plain) / 6 * 6; jj < whole; jj += 6)
    {
        step(std::false_type{}, std::integral_constant<int, 0>{}, jj);
        step(std::false_type{}, std::integral_constant<int, 1>{}, jj + 1);
        step(std::false_type{}, std::integral_constant<int, 2>{}, jj + 2);
        step(std::false_type{}, std::integral_constant<int, 3>{}, jj + 3);
        step(std::false_type{}, std::integral_constant<int, 4>{}, jj + 4);
        step(std::false_type{}, std::integral_constant<int, 5>{}, jj + 5);
    }
    while (jj < count)
    {
        step(std::true_type{}, std::integral_constant<int, 0>{}, jj);
        if (++jj >= count) break;
        step(std::true_type{}, std::integral_constant<int, 1>{}, jj);
        if (++jj >= count) break;
        step(std::true_type{}, std::integral_constant<int, 2>{}, jj);
        if (++jj >= count) break;
        step(std::true_type{}, std::integral_constant<int, 3>{}, jj);
        if (++jj >= count) break;
        step(std::true_type{}, std::integral_constant<int, 4>{}, jj);
        if (++jj >= count) break;
        step(std::true_type{}, std::integral_constant<int, 5>{}, jj);
        ++jj;
    }
}

// The step is the fused self-attention kernel's: in block A the matrix cores compute
// tile j+1's scores while the vector unit ends tile j's exponentials; past the step's
// one barrier, in block B, they add tile j's P V while the vector unit starts tile
// j+1's. K is copied three tiles ahead, V two. A lone wave per SIMD takes 0.60 us a
// step at head_dim 128 and 0.45 at 64 (its instructions in order), two 0.86 and 0.55:
// hence 256 rows of 8 waves where there are as many (head_dim 128: the 2048 x 32768
// chunk 876 us, 128 rows 1005-1116), and more than one workgroup on a CU else. (One
// tile a step without this overlap took 1251 us for that chunk.)
// The base is not followed tile by tile: it is set by the first tile and moved only
// when a tile's row sum passes kSumLimit, which bounds every weight (2^48 in bf16;
// 2^15 in fp16, whose largest value is near 2^16). The move is rare; it recomputes
// the tile's scores from memory.
template <typename T>
constexpr float kSumLimit = 281474976710656.0f;  // 2^48
template <>
constexpr float kSumLimit<_Float16> = 32768.0f;
// From here on the fused product's rounding against the base is no longer small
// (fp32's spacing at 2^28 is 32): every tile takes the exact path.
constexpr float kCoarseBase = 268435456.0f;

// Waves of a SIMD that the stages leave room for; the registers are kept to as many.
// Left to itself the compiler took 177 (head_dim 64) and 265 (128) for 64 rows of
// contiguous keys, and four and two workgroups ran on a CU where six and three fit:
// 64 x 32 heads of 60 queries on 77 keys take 19.4 us against 21.2 at head_dim 64 and
// 34.5 against 36.4 at 128, 256 x 32 heads on 512 keys 229 against 238.
template <int D>
constexpr int kWavesPerSimd = D == 64 ? 3 : 2;

template <typename T, int D, int kWaves, int kGroups, bool kPaged>
__global__ __launch_bounds__(64 * kWaves * kGroups)
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<D>, 8))) void
serving_attention_kernel(const Args a)
{
    using E = Elem<T>;
    using x8 = typename E::x8;
    using C = TileCopy<D, kWaves>;
    constexpr int R = 32 * kWaves;
    // LDS stages: three per tensor (four measured no faster). Two groups at head_dim 128
    // keep two of K, so that two workgroups fit a CU: K is then copied in block B.
    constexpr int kKStages = D == 128 && kGroups == 2 ? 2 : 3;
    constexpr int kVStages = 3;
    static_assert(6 % kKStages == 0 && 6 % kVStages == 0, "the walk's rounds");
    constexpr int kTile = kTileKeys * D;  // elements
    constexpr int kI = C::kIssues;
    // A wave's copies of a tile lie in one half of it, or in both.
    constexpr int kHalves = kI > 1 ? 2 : 1;
    constexpr int kGroupElems = (kKStages + kVStages) * kTile;
    // At the end the stages' room holds the second group's results (two groups) and
    // 4 KiB a wave for the stores.
    constexpr int kOtFloats = (D / 32) * 16 * 64;  // one wave's O^T
    constexpr int kMergeElems = kGroups == 1 ? 0 : kWaves * (kOtFloats + 128) * 2;
    constexpr int kEndElems = kMergeElems + kWaves * 2048;
    constexpr int kLdsElems = kGroups * kGroupElems > kEndElems ? kGroups * kGroupElems : kEndElems;
    __shared__ __attribute__((aligned(16))) uint16_t lds[kLdsElems];

    const int lane = threadIdx.x & 63;
    const int wave_all = uniform(static_cast<int>(threadIdx.x >> 6));
    const int grp = kGroups == 1 ? 0 : wave_all / kWaves;
    const int wave = kGroups == 1 ? wave_all : wave_all % kWaves;
    const int i = lane & 31;
    const int h = lane >> 5;
    Block b;
    int split;
    if (!take_block<R, kPaged>(a, b, split)) return;
    Rows r = wave_rows<R>(a, b, split, wave, i);
    const bool any_tile = r.t_begin < r.t_end;
    // Two groups: each walks half of the tiles, with the same number of steps.
    const int steps = (r.t_end - r.t_begin + kGroups - 1) / kGroups;
    r.t_begin += grp * steps;
    r.t_end = min(r.t_end, r.t_begin + steps);
    r.t_last = min(r.t_last, r.t_end);

    f32x16 o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
    float m = kEmptyBase, l = 0.0f;
    if (any_tile)
    {
        const Keys<D, kPaged> keys(a, b);
        const float c_log2 = a.c_log2;
        uint32_t koff[kI], voff[kI];  // a copy's lanes: row and chunk from the half's first row
        {
            const int sub = lane / C::kChunks;
            const int pchunk = lane % C::kChunks;
#pragma unroll
            for (int u = 0; u < kI; ++u)
            {
                const int row = (u * kWaves + wave) * C::kRows + sub;
                koff[u] = static_cast<uint32_t>(row & 15) * keys.k_row_bytes + ((pchunk ^ swz_k<D>(row)) * 16);
                voff[u] = static_cast<uint32_t>(row & 15) * keys.v_row_bytes + ((pchunk ^ swz_v<D>(row)) * 16);
            }
        }
        const uint32_t lds_base = fa::lds_addr(lds) + grp * (kGroupElems * 2);
        const int half0 = kHalves == 1 ? (wave * C::kRows) & 16 : 0;  // first key of the wave's (first) half
        struct Place
        {
            typename Keys<D, kPaged>::Half half[kHalves];
        };
        int pages[kHalves];  // of the tile whose place is computed next
        auto fetch_pages = [&](int t) {
#pragma unroll
            for (int x = 0; x < kHalves; ++x) pages[x] = keys.page_of(t * kTileKeys + half0 + 16 * x);
        };
        auto place_of = [&](int t) {
            Place p;
#pragma unroll
            for (int x = 0; x < kHalves; ++x) p.half[x] = keys.half_at(t * kTileKeys + half0 + 16 * x, pages[x]);
            return p;
        };
        auto copy_k = [&](const Place& p, int stage, int u) {
            const auto& half = p.half[kHalves == 1 ? 0 : (u * kWaves * C::kRows) >> 4];
            fa::dma16(keys.descriptor(half.k, half.k_bytes), koff[u],
                      lds_base + stage * (kTile * 2) + (u * kWaves + wave) * C::kBytes);
        };
        auto copy_v = [&](const Place& p, int stage, int u) {
            const auto& half = p.half[kHalves == 1 ? 0 : (u * kWaves * C::kRows) >> 4];
            fa::dma16(keys.descriptor(half.v, half.v_bytes), voff[u],
                      lds_base + (kKStages + stage) * (kTile * 2) + (u * kWaves + wave) * C::kBytes);
        };
        static_assert(kHalves == 1 || 16 % (kWaves * C::kRows) == 0, "every wave's copy u lies in the same half");

        const int t0 = r.t_begin;
        const int cnt = steps;
        const int lw = r.t_last - t0 - 1;             // last step this wave computes
        const int j_mask = min(lw, r.t_mask - t0 - 1);  // first step whose next tile is masked

        // Prologue: K 0, then K 1, V 0, K 2, V 1 in the order of their use (two stages of
        // K: K 2 follows when K 0 has been read). `ahead` is the place of tile 3 (K next,
        // V a step later), `behind` that of tile 2 (V next).
        Place ahead, behind;
        fetch_pages(t0);
        behind = place_of(t0);
        fetch_pages(t0 + 1);
#pragma unroll
        for (int u = 0; u < kI; ++u) copy_k(behind, 0, u);
#pragma unroll
        for (int x = 1; x < 3; ++x)
        {
            ahead = place_of(t0 + x);
            fetch_pages(t0 + x + 1);
#pragma unroll
            for (int u = 0; u < kI; ++u)
                if (x < kKStages) copy_k(ahead, x, u);
#pragma unroll
            for (int u = 0; u < kI; ++u) copy_v(behind, x - 1, u);
            behind = ahead;
        }
        ahead = place_of(t0 + 3);
        fetch_pages(t0 + 4);

        x8 qr[D / 16];
        const uint16_t* qp = a.q + q_offset<kPaged>(a, b, r);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qr[ks] = *reinterpret_cast<const x8*>(qp + 16 * ks + 8 * h);

        int k_at[D / 16], v_at[D / 32];  // byte offsets, pinned at each use: the stage then folds into the read
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) k_at[ks] = 2 * (grp * kGroupElems + k_read_offset<D>(i, h, ks));
#pragma unroll
        for (int db = 0; db < D / 32; ++db) v_at[db] = 2 * (grp * kGroupElems + kKStages * kTile + v_read_offset<D>(lane, db));
        x8 ka[D / 16], va[D / 32][2];
        auto load_k = [&](int stage, int first, int count) {
#pragma unroll
            for (int ks = first; ks < first + count; ++ks)
            {
                pin(k_at[ks]);
                ka[ks] = *reinterpret_cast<const x8*>(reinterpret_cast<const char*>(lds + stage * kTile) + k_at[ks]);
            }
        };
        auto load_v = [&](int stage, int first, int count) {
#pragma unroll
            for (int db = first; db < first + count; ++db)
            {
                pin(v_at[db]);
                const uint16_t* base = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(lds + stage * kTile) + v_at[db]);
                va[db][0] = read_v<T, D>(base, 0);
                va[db][1] = read_v<T, D>(base, 1);
            }
        };

        f32x16 sbuf[2];
        x8 p_lo[2], p_hi;
        float tsum = 0.0f;
        int limit_bits = __builtin_bit_cast(int, kSumLimit<T>);
        auto note_base = [&](float base) {
            if (__any(base != kEmptyBase && __builtin_fabsf(base) >= kCoarseBase)) limit_bits = __builtin_bit_cast(int, -1.0f);
            limit_bits = uniform(limit_bits);
        };
        // K 0 has landed: the other tiles of K and of V may fly.
        fa::wait_vm_lgkm0<(kKStages + 1) * kI>();
        barrier();
        if (lw >= 0)
        {
            load_k(0, 0, D / 16);
            sbuf[0] = f32x16{};
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) sbuf[0] = E::mfma(ka[ks], qr[ks], sbuf[0]);
            if (t0 >= r.t_mask) mask_tile(sbuf[0], r.limit - t0 * kTileKeys - 4 * h);
            m = __builtin_elementwise_maximum(m, row_max_raw(sbuf[0]) * c_log2 - E::kBias);
            weigh<T, false>(sbuf[0], 0, p_lo[0], m, c_log2, tsum);
            note_base(m);
        }
        // K 1 and V 0 have landed, K 0's stage is free.
        fa::wait_vm_lgkm0<(kKStages - 1) * kI>();
        barrier();
        load_k(1, 0, D / 16);
        if constexpr (kKStages == 2)
#pragma unroll
            for (int u = 0; u < kI; ++u) copy_k(behind, 0, u);

        // A weight of 0 times an infinity or a NaN is NaN. A tile that some lane does not
        // see whole (at most two of a wave: its rows' limits lie within 32 keys) is left
        // out where V holds such values, and added key by key after the walk, to the
        // lanes that see the key.
        unsigned left_out = 0;  // bit x: tile t_mask + x
        auto leave_out = [&](int t) __attribute__((always_inline)) {
            uint32_t found = 0;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) found |= not_finite<T>(va[x % (D / 32)][x / (D / 32)]);
            if (!__any(found != 0)) return false;
            left_out |= 1u << (t - r.t_mask);
            return true;
        };

        // The base lags (see above): tile jj's P was zeroed; its scores again, the base
        // at the row maximum, O and l rescaled, its P V from V's stage (intact until the
        // next step's copies), and the first half of the next tile's exponentials again.
        auto rebase = [&](auto par_tag, int jj) __attribute__((always_inline)) {
            constexpr int P = decltype(par_tag)::value;
            constexpr int B = P & 1;
            const int t = t0 + jj;
            uint64_t kp;
            const bool there = keys.lane_key(t * kTileKeys + i, kp);
            f32x16 st = {};
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
            {
                const x8 kr = there ? *reinterpret_cast<const x8*>(kp + (16 * ks + 8 * h) * 2) : x8{};
                st = E::mfma(kr, qr[ks], st);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (t >= r.t_mask) mask_tile(st, r.limit - t * kTileKeys - 4 * h);
            const float m_new = __builtin_elementwise_maximum(m, row_max_raw(st) * c_log2 - E::kBias);
            const float alpha = __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            note_base(m_new);
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
            float sum = 0.0f;
            x8 pr[2];
            weigh<T, true>(st, 0, pr[0], m, c_log2, sum);
            weigh<T, true>(st, 8, pr[1], m, c_log2, sum);
            l = l * alpha + sum;
            load_v(P % kVStages, 0, D / 32);
#pragma unroll
            for (int x = 0; x < D / 16; ++x) o[x % (D / 32)] = E::mfma(va[x % (D / 32)][x / (D / 32)], pr[x / (D / 32)], o[x % (D / 32)]);
            tsum = 0.0f;
            weigh<T, false>(sbuf[B ^ 1], 0, p_lo[B ^ 1], m, c_log2, tsum);
        };

        constexpr int kChunk = kI;                  // chunks per block, one copy each
        constexpr int kMfmaPer = (D / 16) / kChunk;  // products per chunk
        constexpr int kVPer = (D / 32) / kChunk;
        constexpr int kKPer = (D / 16) / kChunk;
        static_assert(kMfmaPer * kChunk == D / 16 && kVPer * kChunk == D / 32 && 8 % kChunk == 0, "chunks");
        constexpr int kExpPer = 8 / kChunk;
        // kExpPer weights of a half tile of scores, as weigh.
        auto weigh_part = [&](const f32x16& s, int first, x8& p, int at) {
#pragma unroll
            for (int e = at; e < at + kExpPer; ++e)
                p[e] = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(s[first + e], c_log2, -m)));
#pragma unroll
            for (int e = at; e < at + kExpPer; e += 2) tsum = E::add_pair(p[e], p[e + 1], tsum);
        };
        auto pv_part = [&](const x8 (&p)[2], int first, int count) {
#pragma unroll
            for (int x = first; x < first + count; ++x)
                o[x % (D / 32)] = E::mfma(va[x % (D / 32)][x / (D / 32)], p[x / (D / 32)], o[x % (D / 32)]);
        };
        auto qk_part = [&](f32x16& s, int first, int count) {
#pragma unroll
            for (int ks = first; ks < first + count; ++ks) s = E::mfma(ka[ks], qr[ks], s);
        };
        auto step = [&](auto masked_tag, auto par_tag, int jj) __attribute__((always_inline)) {
            constexpr int P = decltype(par_tag)::value;
            constexpr int B = P & 1;
            // Block A
            sbuf[B ^ 1] = f32x16{};
#pragma unroll
            for (int c = 0; c < kChunk; ++c)
            {
                qk_part(sbuf[B ^ 1], c * kMfmaPer, 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (kKStages == 3) copy_k(ahead, P % 3, c);
                __builtin_amdgcn_sched_barrier(0);
                load_v(P % kVStages, c * kVPer, kVPer);
                qk_part(sbuf[B ^ 1], c * kMfmaPer + 1, kMfmaPer - 1);
                weigh_part(sbuf[B], 8, p_hi, c * kExpPer);
                __builtin_amdgcn_sched_barrier(0);
            }
            pin8(p_hi);
            pin(tsum);
            // K jj+2 and V jj+1 have landed (what was issued after them may fly), every
            // LDS read is done.
            fa::wait_vm_lgkm0<(kKStages - 2) * kI>();
            barrier();
            // Block B
            bool rare = __any(tsum > __builtin_bit_cast(float, limit_bits));
            bool out = false;
            if constexpr (kPaged && decltype(masked_tag)::value)  // an encoder's states are seen by all rows
                if (r.unseen && t0 + jj >= r.t_mask && leave_out(t0 + jj))
                {
                    out = true;
                    rare = false;
                }
            if (rare || out)
            {
                asm volatile("");  // a branch, not selects on the common path
                p_lo[B] = x8{};
                p_hi = x8{};
                tsum = 0.0f;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) va[x % (D / 32)][x / (D / 32)] = x8{};  // 0 times an infinity is NaN
            }
            l += tsum;
            // Past the wave's last tile the next scores are of a stage that nobody needs.
            if constexpr (decltype(masked_tag)::value) mask_tile(sbuf[B ^ 1], jj == lw ? -kTileKeys : r.limit - (t0 + jj + 1) * kTileKeys - 4 * h);
            __builtin_amdgcn_sched_barrier(0);
            const x8 p_cur[2] = {p_lo[B], p_hi};
            tsum = 0.0f;
#pragma unroll
            for (int c = 0; c < kChunk; ++c)
            {
                pv_part(p_cur, c * kMfmaPer, 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (kKStages == 2) copy_k(ahead, (P + 3) % 2, c);
                copy_v(behind, (P + 2) % kVStages, c);
                __builtin_amdgcn_sched_barrier(0);
                load_k((P + 2) % kKStages, c * kKPer, kKPer);
                pv_part(p_cur, c * kMfmaPer + 1, kMfmaPer - 1);
                weigh_part(sbuf[B ^ 1], 0, p_lo[B ^ 1], c * kExpPer);
                __builtin_amdgcn_sched_barrier(0);
            }
            behind = ahead;
            ahead = place_of(t0 + jj + 4);
            fetch_pages(t0 + jj + 5);
            pin8(p_lo[B ^ 1]);
            pin(tsum);
            if (rare) rebase(par_tag, jj);
            pin(l);
        };
        const int active = max(0, min(cnt, lw + 1));
        walk(active, max(0, j_mask), step);
        // The steps past this wave's last tile: its share of the copies and the barriers.
        for (int jj = active; jj < cnt; ++jj)
        {
#pragma unroll
            for (int u = 0; u < kI; ++u)
                if constexpr (kKStages == 3) copy_k(ahead, jj % 3, u);
            fa::wait_vm_lgkm0<(kKStages - 2) * kI>();
            barrier();
#pragma unroll
            for (int u = 0; u < kI; ++u)
                if constexpr (kKStages == 2) copy_k(ahead, (jj + 3) % 2, u);
#pragma unroll
            for (int u = 0; u < kI; ++u) copy_v(behind, (jj + 2) % kVStages, u);
            behind = ahead;
            ahead = place_of(t0 + jj + 4);
            fetch_pages(t0 + jj + 5);
        }
        // The tiles that were left out, a key at a time.
        for (int t = r.t_mask; kPaged && left_out != 0; ++t, left_out >>= 1)
        {
            if ((left_out & 1u) == 0) continue;
            const int last = min(t * kTileKeys + kTileKeys, b.end);
            for (int key = t * kTileKeys; key < last; ++key)
            {
                const auto at = keys.half_at(key, keys.page_of(key));
                const bool there = at.k_bytes != 0;  // else a page of zeros
                float s = 0.0f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                {
                    const x8 kx = there ? *reinterpret_cast<const x8*>(at.k + (16 * ks + 8 * h) * 2) : x8{};
#pragma unroll
                    for (int e = 0; e < 8; ++e) s = fmaf(static_cast<float>(kx[e]), static_cast<float>(qr[ks][e]), s);
                }
                float sa, sb;
                row_halves(s, sa, sb);
                s = sa + sb;
                const bool sees = key < r.limit;
                const float m_new = __builtin_elementwise_maximum(m, sees ? s * c_log2 - E::kBias : m);
                const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                float x;
                {
#pragma clang fp contract(off)
                    x = s * c_log2 - m;
                }
                const T w = static_cast<T>(sees ? __builtin_amdgcn_exp2f(x) : 0.0f);
                // Each half of the lanes adds half of a row's keys to its sum: this one,
                // which both know, is the lower half's.
                l = l * alpha + (h == 0 ? static_cast<float>(w) : 0.0f);
#pragma unroll
                for (int db = 0; db < D / 32; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                    {
                        typedef T t4 __attribute__((ext_vector_type(4)));
                        const t4 vx = there ? *reinterpret_cast<const t4*>(at.v + (32 * db + 8 * g + 4 * h) * 2) : t4{};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            const float grown = o[db][4 * g + e] * alpha;
                            o[db][4 * g + e] = sees ? fmaf(static_cast<float>(w), static_cast<float>(vx[e]), grown) : grown;
                        }
                    }
            }
        }
        // Every copy has landed and every wave has read its last tile: the stages are free.
        fa::wait_vm_lgkm0<0>();
        barrier();
    }
    if constexpr (kGroups == 2)
    {
        // The second group hands its O^T, base and sum to the first.
        float* const part = reinterpret_cast<float*>(lds) + wave * (kOtFloats + 128);
        if (grp == 1)
        {
#pragma unroll
            for (int x = 0; x < D / 8; ++x)
            {
                const f32x16& ob = o[x / 4];
                *reinterpret_cast<f32x4*>(part + (x * 64 + lane) * 4) =
                    f32x4{ob[4 * (x % 4)], ob[4 * (x % 4) + 1], ob[4 * (x % 4) + 2], ob[4 * (x % 4) + 3]};
            }
            part[kOtFloats + lane] = m;
            part[kOtFloats + 64 + lane] = l;
        }
        fa::wait_vm_lgkm0<63>();
        barrier();
        if (grp == 1) return;
        const float m1 = part[kOtFloats + lane], l1 = part[kOtFloats + 64 + lane];
        const float top = __builtin_elementwise_maximum(m, m1);
        const float w0 = __builtin_amdgcn_exp2f(m - top), w1 = __builtin_amdgcn_exp2f(m1 - top);
        l = l * w0 + l1 * w1;
        m = top;
#pragma unroll
        for (int x = 0; x < D / 8; ++x)
        {
            const f32x4 y = *reinterpret_cast<const f32x4*>(part + (x * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x / 4][4 * (x % 4) + e] = o[x / 4][4 * (x % 4) + e] * w0 + y[e] * w1;
        }
    }
    if (b.row0 + 32 * wave < b.rows)
        store_rows<T, D, kPaged>(a, b, r, split, lane, o, m, l, reinterpret_cast<uint4*>(lds + kMergeElems) + wave * 256);
}

// Joins the chunks of a row: O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c with
// M the largest base, kept running. D/4 lanes read a chunk's 4 D bytes, so 256
// threads make 1024/D groups. For many chunks they all work on one row, chunk by chunk
// in turn, and meet in LDS (kAlone); for few each takes rows of its own. A whole call,
// alone against not: 33 chunks of one row a head 9.0 us against 10.0, 65 chunks of 16
// rows 16.4 against 26.9, 17 of 36 rows 46.2 against 50.6; 9 of 4 rows (64 sequences)
// 228.7 against 224.6, 17 chunks of 96 rows the same.
constexpr int kAloneChunks = 13;  // from this many on
constexpr int kAloneRows = 64;    // and up to as many rows of a block
constexpr int kJoinRows = 32;     // rows of a workgroup that are not kAlone

template <typename T, int D, int R, bool kPaged, bool kAlone>
__global__ __launch_bounds__(256) void serving_join_kernel(const Args a, int block_parts)
{
    constexpr int kLanes = D / 4;
    constexpr int kGroups = 256 / kLanes;
    const int head = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.heads_kv));
    const int rest = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.heads_kv));
    Block b;
    if (!find_block<R, kPaged>(a, rest / block_parts, head, b) || b.splits == 1) return;
    const int tid = threadIdx.x;
    const int group = tid / kLanes;
    const int d4 = (tid % kLanes) * 4;

    struct Sum
    {
        float top = kEmptyBase, total = 0.0f;
        f32x4 o = {};
        __device__ __forceinline__ void add(float m, float l, f32x4 x)
        {
            const float t = __builtin_elementwise_maximum(top, m);
            const float w0 = __builtin_amdgcn_exp2f(top - t), w1 = __builtin_amdgcn_exp2f(m - t);
            total = total * w0 + l * w1;
            o = o * w0 + x * w1;
            top = t;
        }
    };
    // kBatch chunks' values are under way together.
    auto join = [&](long long pr, int first, int step) {
        constexpr int kBatch = 8;
        Sum s;
        for (int c0 = first; c0 < b.splits; c0 += kBatch * step)
        {
            float2 ml[kBatch];
            f32x4 x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
            {
                const int c = c0 + u * step;
                ml[u] = float2{kEmptyBase, 0.0f};
                x[u] = f32x4{};
                if (c < b.splits)
                {
                    ml[u] = *reinterpret_cast<const float2*>(a.base_sum + 2 * (pr + c));
                    x[u] = *reinterpret_cast<const f32x4*>(a.part + (pr + c) * D + d4);
                }
            }
            float top = s.top;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) top = __builtin_elementwise_maximum(top, ml[u].x);
            const float w = __builtin_amdgcn_exp2f(s.top - top);
            s.total *= w;
            s.o *= w;
            s.top = top;
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
            {
                const float wu = __builtin_amdgcn_exp2f(ml[u].x - top);
                s.total += ml[u].y * wu;
                s.o += x[u] * wu;
            }
        }
        return s;
    };
    auto store = [&](const Sum& s, int token, int qh) {
        const float inv = s.total > 0.0f ? __builtin_amdgcn_rcpf(s.total) : 0.0f;
        uint2 w;
        w.x = pack_pair<T>(s.o[0] * inv, s.o[1] * inv);
        w.y = pack_pair<T>(s.o[2] * inv, s.o[3] * inv);
        *reinterpret_cast<uint2*>(a.o + o_offset<kPaged>(a, b, token, qh) + d4) = w;
    };
    if constexpr (kAlone)
    {
        __shared__ f32x4 parts[256];
        __shared__ float2 bases[256];
        const int row = b.row0 + rest % block_parts;
        if (row >= b.rows) return;
        const int token = row / a.group, qh = row % a.group;
        Sum s = join(part_row<kPaged>(a, b, token, qh) * a.splits, group, kGroups);
        parts[tid] = s.o;
        bases[tid] = float2{s.top, s.total};
        __syncthreads();
        if (tid >= kLanes) return;
#pragma unroll
        for (int g = 1; g < kGroups; ++g) s.add(bases[g * kLanes + tid].x, bases[g * kLanes + tid].y, parts[g * kLanes + tid]);
        store(s, token, qh);
    }
    else
    {
        const int first = b.row0 + rest % block_parts * kJoinRows;
        const int last = min(min(first + kJoinRows, b.row0 + R), b.rows);
        for (int row = first + group; row < last; row += kGroups)
        {
            const int token = row / a.group, qh = row % a.group;
            store(join(part_row<kPaged>(a, b, token, qh) * a.splits, 0, 1), token, qh);
        }
    }
}

// ---------------------------------------------------------------- host side

// Rows of a workgroup, row blocks and key chunks of a launch.
struct Plan
{
    int waves, groups;
    int per_seq;
    long long slots;
    int splits, chunk;
    size_t workspace;
};

// Which rows and chunks: the time of a launch is estimated (us) from what a
// workgroup of 32 * waves rows costs, workgroup + step * tiles. The step is the
// larger of a lone workgroup's and its share of a CU's rate where k workgroups are on
// the CU (up to per_cu).
//   one length   the rounds in which the device runs the workgroups;
//   ragged       the larger of the longest workgroup and the average over the
//                device's places, plus a share of the smaller (what remains of one
//                when the other ends). Only the device knows the lengths: their mean
//                is taken as `filled` of the longest.
// Not below what reading the keys once takes, plus the join's time. The constants are
// fits to 1150 drawn shapes (1 to 192 sequences, 1 to 32768 keys, 1 to 64 heads, one
// new token to chunks of 4096), each at every rows and chunks of the lists below. The
// choice takes 1.027 (head_dim 64) and 1.044 (128) times the best one's time in the
// geometric mean, more than 1.2 times it at 37 of the 1150. Without the two groups it
// would be 1.038 and 1.064; two groups of 128 rows gain 0.4 % and are not built, and
// 256 rows are of no use at head_dim 64.
struct RowsCost
{
    int waves, groups, per_cu;
    float workgroup, step, shared;
};

struct Costs
{
    RowsCost rows[4];
    int count;
    float filled, share, join, join_mb, launch, bytes_per_us;  // join_mb: per 10^6 floats of partial results
};

constexpr Costs kCosts64 = {
    {{2, 1, 6, 2.857f, 0.454f, 0.131f}, {4, 1, 3, 2.849f, 0.365f, 0.151f}, {2, 2, 3, 3.68f, 0.384f, 0.205f}},
    3, 0.9f, 0.507f, 4.118f, 1.335f, 1.95f, 5.958e6f};
constexpr Costs kCosts128 = {{{2, 1, 3, 3.479f, 0.586f, 0.286f},
                              {4, 1, 2, 3.318f, 0.551f, 0.392f},
                              {8, 1, 1, 4.233f, 0.57f, 0.631f},
                              {2, 2, 2, 3.748f, 0.704f, 0.452f}},
                             4, 0.852f, 0.44f, 2.596f, 1.533f, 4.251f, 5.109e6f};
constexpr int kSplitChoices[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};
static_assert(kSplitChoices[15] == kMaxSplits, "the joins' limit");

bool joins_alone(int block_rows, int splits) { return splits >= kAloneChunks && block_rows <= kAloneRows; }

// Workgroups of the join per row block of `block_rows` rows.
int join_parts(int block_rows, int splits)
{
    return joins_alone(block_rows, splits) ? block_rows : (block_rows + kJoinRows - 1) / kJoinRows;
}

constexpr double kMaxThreads = 2147483647.0;  // of a launch

Plan make_plan(long long seqs, long long tokens, int heads, int heads_kv, int head_dim, int max_queries, int max_keys,
               bool paged)
{
    const Costs& costs = head_dim == 64 ? kCosts64 : kCosts128;
    const int group = heads / heads_kv;
    const long long rows = std::min<long long>(max_queries, tokens) * group;
    const int tiles = static_cast<int>((std::min<long long>(max_keys, kMaxKeys) + kTileKeys - 1) / kTileKeys);
    const double cus = fa::device_compute_units();
    const bool ragged = paged && seqs > 1;
    const double filled = ragged ? costs.filled : 1.0;
    const double read = static_cast<double>(seqs) * tiles * kTileKeys * heads_kv * head_dim * 4.0 * filled / costs.bytes_per_us;
    const double read4 = read * read * read * read;
    Plan best{};
    double best_time = 0.0;
    for (int x = 0; x < costs.count; ++x)
    {
        const RowsCost& c = costs.rows[x];
        Plan p{};
        p.waves = c.waves;
        p.groups = c.groups;
        const int R = 32 * c.waves;
        const long long per_seq = (rows + R - 1) / R;
        p.per_seq = static_cast<int>(std::min<long long>(per_seq, 1 << 30));
        p.slots = seqs * per_seq;
        // Ragged batches: at most one slot per full block of rows and one per sequence.
        const long long packed = tokens * group / R + seqs;
        if (paged && per_seq > 1 && packed < p.slots)
        {
            p.per_seq = 0;
            p.slots = packed;
        }
        const double blocks = static_cast<double>(p.slots) * heads_kv;
        int last_chunk = 0;
        for (const int choice : kSplitChoices)
        {
            const int chunk = (tiles + choice - 1) / choice;  // tiles
            if (choice > 1 && (chunk < 2 || chunk == last_chunk)) continue;
            last_chunk = chunk;
            const int splits = chunk > 0 ? (tiles + chunk - 1) / chunk : 1;
            // Both grids have to hold it; the first choice stands where none fits, and its
            // launch is refused.
            const bool fits = blocks * splits * 64 * c.waves * c.groups <= kMaxThreads &&
                              (splits == 1 ||
                               blocks * join_parts(static_cast<int>(std::min<long long>(rows, R)), splits) * 256 <= kMaxThreads);
            if (!fits && best.waves > 0) continue;
            auto step_at = [&](double k) {
                return std::max<double>(c.step, c.shared * std::min<double>(std::max(k, 1.0), c.per_cu));
            };
            const double active = blocks * (splits == 1 ? 1.0 : ragged ? splits * filled : splits);
            const int steps = (chunk + c.groups - 1) / c.groups;
            double busy;
            if (ragged)
            {
                const double k = std::min<double>(std::max(active / cus, 1.0), c.per_cu);
                const double longest = c.workgroup + step_at(k) * steps;
                const double average = (active * c.workgroup + blocks * tiles / c.groups * filled * step_at(k)) / (cus * k);
                busy = std::max(longest, average) + costs.share * std::min(longest, average);
            }
            else
            {
                const double rounds = std::floor(active / (cus * c.per_cu));
                const double rest = active - rounds * cus * c.per_cu;
                busy = rounds * (c.workgroup + step_at(c.per_cu) * steps) +
                       (rest > 0.0 ? c.workgroup + step_at(rest / cus) * steps : 0.0);
            }
            const double fixed =
                costs.launch + (splits > 1 ? costs.join + costs.join_mb * 1e-6 * static_cast<double>(tokens) * heads *
                                                              head_dim * splits
                                           : 0.0);
            if (best_time > 0.0 && busy + fixed >= best_time) continue;
            // A smooth maximum: one of the two hides little of the other where they are close.
            const double busy2 = busy * busy;
            const double time = std::sqrt(std::sqrt(busy2 * busy2 + read4)) + fixed;
            if (best_time == 0.0 || time < best_time)
            {
                best_time = fits ? time : 0.0;
                best = p;
                best.splits = splits;
                best.chunk = std::max(chunk, 1) * kTileKeys;
            }
        }
    }
    if (best.splits > 1) best.workspace = static_cast<size_t>(tokens) * heads * best.splits * (head_dim + 2) * sizeof(float);
    return best;
}

template <typename T, int D, int kWaves, int kGroups, bool kPaged>
int launch_typed(const Args& a, const Plan& p, int head_rows, hipStream_t stream)
{
    const long long blocks = p.slots * a.heads_kv * p.splits;
    if (blocks > 0x7fffffffLL / (64 * kWaves * kGroups)) return hipErrorInvalidValue;
    const int block_rows = std::min(32 * kWaves, head_rows);
    const bool alone = joins_alone(block_rows, p.splits);
    const int parts = join_parts(block_rows, p.splits);
    const long long join_blocks = p.slots * a.heads_kv * parts;
    if (p.splits > 1 && join_blocks > 0x7fffffffLL / 256) return hipErrorInvalidValue;
    const hipError_t e = fa::launch_kernel(serving_attention_kernel<T, D, kWaves, kGroups, kPaged>,
                                           dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves * kGroups), stream, a);
    if (e != hipSuccess || p.splits == 1) return e;
    return fa::launch_kernel(alone ? serving_join_kernel<T, D, 32 * kWaves, kPaged, true>
                                   : serving_join_kernel<T, D, 32 * kWaves, kPaged, false>,
                             dim3(static_cast<unsigned>(join_blocks)), dim3(256), stream, a, parts);
}

template <typename T, int D, bool kPaged>
int launch_waves(const Args& a, const Plan& p, int head_rows, hipStream_t stream)
{
    if (p.waves == 2 && p.groups == 1) return launch_typed<T, D, 2, 1, kPaged>(a, p, head_rows, stream);
    if (p.waves == 4 && p.groups == 1) return launch_typed<T, D, 4, 1, kPaged>(a, p, head_rows, stream);
    if (p.waves == 2 && p.groups == 2) return launch_typed<T, D, 2, 2, kPaged>(a, p, head_rows, stream);
    if constexpr (D == 128)
        if (p.waves == 8 && p.groups == 1) return launch_typed<T, D, 8, 1, kPaged>(a, p, head_rows, stream);
    return hipErrorInvalidValue;  // make_plan names no others
}

template <bool kPaged>
int launch_any(const Args& a, const Plan& p, int head_rows, int head_dim, int dtype, hipStream_t stream)
{
    if (dtype == FA_DTYPE_BF16)
        return head_dim == 64 ? launch_waves<__bf16, 64, kPaged>(a, p, head_rows, stream)
                              : launch_waves<__bf16, 128, kPaged>(a, p, head_rows, stream);
    return head_dim == 64 ? launch_waves<_Float16, 64, kPaged>(a, p, head_rows, stream)
                          : launch_waves<_Float16, 128, kPaged>(a, p, head_rows, stream);
}

// Rows are read and written in pieces of 16 bytes: every stride keeps them aligned.
bool bad_strides(const fa_strides& s, bool with_batch)
{
    return ((with_batch ? s.batch : 0) | s.head | s.row) & 7;
}

// K and V: rows of a copy lie within 32-bit offsets of its first one, in rising order.
bool bad_key_row(long long row, int head_dim) { return row < head_dim || row >= (1LL << 26); }

int launch_paged(const void* q, const fa_paged_cache* cache, void* o, void* workspace, size_t workspace_bytes,
                 const int* block_table, long long table_stride, int table_width, const int* query_starts,
                 const int* kv_lens, int num_seqs, int tokens, int heads, int max_query_len, int max_kv_len, int causal,
                 const fa_strides* q_strides, const fa_strides* o_strides, void* stream)
{
    if (!cache) return hipErrorInvalidValue;
    if (cache->head_dim != 64 && cache->head_dim != 128) return FA_ERROR_UNSUPPORTED;
    const int D = cache->head_dim, heads_kv = cache->heads_kv;
    if (num_seqs < 0 || tokens < 0 || heads < 0 || max_query_len < 0 || max_kv_len < 0) return hipErrorInvalidValue;
    if (num_seqs == 0 || tokens == 0 || heads == 0 || max_query_len == 0) return hipSuccess;
    const int status = fa::check_paged_cache(*cache);
    if (status != hipSuccess) return status;
    if (heads_kv == 0 || heads % heads_kv != 0 || heads > 65536) return hipErrorInvalidValue;
    if (!q || !o || !query_starts || !kv_lens) return hipErrorInvalidValue;
    if (static_cast<long long>(std::min(max_query_len, tokens)) * (heads / heads_kv) > kMaxRows ||
        static_cast<long long>(table_width) * cache->block_size > kMaxKeys)
        return hipErrorInvalidValue;
    if (table_width < 0 || (table_width > 0 && !block_table) || table_stride < 0) return hipErrorInvalidValue;
    const fa_strides qs = q_strides ? *q_strides : fa_strides{0, D, static_cast<long long>(heads) * D};
    const fa_strides os = o_strides ? *o_strides : fa_strides{0, D, static_cast<long long>(heads) * D};
    if (fa::misaligned16(q) || fa::misaligned16(o) || bad_strides(qs, false) || bad_strides(os, false)) return hipErrorInvalidValue;
    const Plan p = make_plan(num_seqs, tokens, heads, heads_kv, D, max_query_len, max_kv_len, true);
    if (p.workspace > 0 && (!workspace || workspace_bytes < p.workspace || fa::misaligned16(workspace)))
        return hipErrorInvalidValue;
    Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(cache->k);
    a.v = static_cast<const uint16_t*>(cache->v);
    a.o = static_cast<uint16_t*>(o);
    a.part = static_cast<float*>(workspace);
    a.base_sum = a.part + static_cast<size_t>(tokens) * heads * p.splits * D;
    a.table = block_table;
    a.starts = query_starts;
    a.lens = kv_lens;
    a.q_head = qs.head, a.q_row = qs.row;
    a.o_head = os.head, a.o_row = os.row;
    a.k_seq = a.v_seq = cache->block_stride;
    a.k_head = a.v_head = cache->head_stride;
    a.k_row = a.v_row = cache->token_stride;
    a.table_stride = table_stride;
    a.table_width = table_width;
    a.num_blocks = cache->num_blocks;
    a.block_shift = __builtin_ctz(cache->block_size);
    a.seqs = num_seqs;
    a.tokens = tokens;
    a.heads_kv = heads_kv;
    a.group = heads / heads_kv;
    a.max_queries = max_query_len;
    a.slots = static_cast<int>(p.slots);
    a.per_seq = p.per_seq;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.causal = causal != 0;
    a.c_log2 = fa_default_scale(D) * fa::kLog2e;
    const int head_rows = static_cast<int>(std::min<long long>(1 << 20, static_cast<long long>(std::min(max_query_len, tokens)) * a.group));
    return launch_any<true>(a, p, head_rows, D, cache->dtype, static_cast<hipStream_t>(stream));
}

int launch_cross(const void* q, const void* k, const void* v, void* o, void* workspace, size_t workspace_bytes,
                 const int* kv_lens, int batch, int heads, int heads_kv, int q_len, int kv_len, int head_dim, int dtype,
                 const fa_strides* q_strides, const fa_strides* k_strides, const fa_strides* v_strides,
                 const fa_strides* o_strides, void* stream)
{
    if (head_dim != 64 && head_dim != 128) return FA_ERROR_UNSUPPORTED;
    if (batch < 0 || heads < 0 || heads_kv < 0 || q_len < 0 || kv_len < 0) return hipErrorInvalidValue;
    if (dtype != FA_DTYPE_BF16 && dtype != FA_DTYPE_FP16) return hipErrorInvalidValue;
    if (batch == 0 || heads == 0 || q_len == 0) return hipSuccess;
    if (heads_kv == 0 || heads % heads_kv != 0 || heads > 65536) return hipErrorInvalidValue;
    if (!q || !o || (kv_len > 0 && (!k || !v))) return hipErrorInvalidValue;
    if (static_cast<long long>(q_len) * (heads / heads_kv) > kMaxRows || kv_len > kMaxKeys) return hipErrorInvalidValue;
    auto contiguous = [&](int h, int n) {
        return fa_strides{static_cast<long long>(h) * n * head_dim, static_cast<long long>(n) * head_dim, head_dim};
    };
    const fa_strides qs = q_strides ? *q_strides : contiguous(heads, q_len);
    const fa_strides ks = k_strides ? *k_strides : contiguous(heads_kv, kv_len);
    const fa_strides vs = v_strides ? *v_strides : contiguous(heads_kv, kv_len);
    const fa_strides os = o_strides ? *o_strides : contiguous(heads, q_len);
    if (fa::misaligned16(q) || fa::misaligned16(k) || fa::misaligned16(v) || fa::misaligned16(o)) return hipErrorInvalidValue;
    if (bad_strides(qs, true) || bad_strides(ks, true) || bad_strides(vs, true) || bad_strides(os, true))
        return hipErrorInvalidValue;
    if (bad_key_row(ks.row, head_dim) || bad_key_row(vs.row, head_dim)) return hipErrorInvalidValue;
    const long long tokens = static_cast<long long>(batch) * q_len;
    const Plan p = make_plan(batch, tokens, heads, heads_kv, head_dim, q_len, kv_len, false);
    if (p.slots > 0x7fffffffLL) return hipErrorInvalidValue;
    if (p.workspace > 0 && (!workspace || workspace_bytes < p.workspace || fa::misaligned16(workspace)))
        return hipErrorInvalidValue;
    Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.o = static_cast<uint16_t*>(o);
    a.part = static_cast<float*>(workspace);
    a.base_sum = a.part + static_cast<size_t>(tokens) * heads * p.splits * head_dim;
    a.lens = kv_lens;
    a.q_seq = qs.batch, a.q_head = qs.head, a.q_row = qs.row;
    a.o_seq = os.batch, a.o_head = os.head, a.o_row = os.row;
    a.k_seq = ks.batch, a.k_head = ks.head, a.k_row = ks.row;
    a.v_seq = vs.batch, a.v_head = vs.head, a.v_row = vs.row;
    a.seqs = batch;
    a.heads_kv = heads_kv;
    a.group = heads / heads_kv;
    a.max_queries = q_len;
    a.max_keys = kv_len;
    a.slots = static_cast<int>(p.slots);
    a.per_seq = p.per_seq;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.c_log2 = fa_default_scale(head_dim) * fa::kLog2e;
    const int head_rows = static_cast<int>(std::min<long long>(1 << 20, static_cast<long long>(q_len) * a.group));
    return launch_any<false>(a, p, head_rows, head_dim, dtype, static_cast<hipStream_t>(stream));
}

}  // namespace

extern "C" {

size_t fa_attention_paged_workspace_bytes(int tokens, int num_seqs, int heads, int heads_kv, int head_dim,
                                          int max_query_len, int max_kv_len)
{
    if (tokens <= 0 || num_seqs <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || head_dim <= 0 ||
        max_query_len <= 0 || max_kv_len < 0)
        return 0;
    return make_plan(num_seqs, tokens, heads, heads_kv, head_dim, max_query_len, max_kv_len, true).workspace;
}

int fa_attention_paged_config(int tokens, int num_seqs, int heads, int heads_kv, int head_dim, int max_query_len,
                              int max_kv_len, int* rows_per_block, int* kv_groups, int* splits)
{
    if (!rows_per_block || !kv_groups || !splits) return fa::record_status(hipErrorInvalidValue);
    *rows_per_block = *kv_groups = *splits = 0;
    if (head_dim != 64 && head_dim != 128) return FA_ERROR_UNSUPPORTED;
    if (tokens <= 0 || num_seqs <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || max_query_len <= 0 ||
        max_kv_len < 0)
        return fa::record_status(hipErrorInvalidValue);
    const Plan p = make_plan(num_seqs, tokens, heads, heads_kv, head_dim, max_query_len, max_kv_len, true);
    *rows_per_block = 32 * p.waves;
    *kv_groups = p.groups;
    *splits = p.splits;
    return hipSuccess;
}

int fa_launch_attention_paged(const void* q, const fa_paged_cache* cache, void* o, void* workspace,
                              size_t workspace_bytes, const int* block_table, const int* query_starts,
                              const int* kv_lens, int num_seqs, int tokens, int heads, int table_width,
                              long long table_stride, int max_query_len, int max_kv_len, int causal,
                              const fa_strides* q_strides, const fa_strides* o_strides, void* stream)
{
    return fa::record_status(launch_paged(q, cache, o, workspace, workspace_bytes, block_table, table_stride, table_width,
                                          query_starts, kv_lens, num_seqs, tokens, heads, max_query_len, max_kv_len, causal,
                                          q_strides, o_strides, stream));
}

size_t fa_attention_cross_workspace_bytes(int batch, int heads, int heads_kv, int q_len, int kv_len, int head_dim)
{
    if (batch <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || q_len <= 0 || kv_len < 0 || head_dim <= 0)
        return 0;
    return make_plan(batch, static_cast<long long>(batch) * q_len, heads, heads_kv, head_dim, q_len, kv_len, false).workspace;
}

int fa_attention_cross_config(int batch, int heads, int heads_kv, int q_len, int kv_len, int head_dim,
                              int* rows_per_block, int* kv_groups, int* splits)
{
    if (!rows_per_block || !kv_groups || !splits) return fa::record_status(hipErrorInvalidValue);
    *rows_per_block = *kv_groups = *splits = 0;
    if (head_dim != 64 && head_dim != 128) return FA_ERROR_UNSUPPORTED;
    if (batch <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || q_len <= 0 || kv_len < 0)
        return fa::record_status(hipErrorInvalidValue);
    const Plan p = make_plan(batch, static_cast<long long>(batch) * q_len, heads, heads_kv, head_dim, q_len, kv_len, false);
    *rows_per_block = 32 * p.waves;
    *kv_groups = p.groups;
    *splits = p.splits;
    return hipSuccess;
}

int fa_launch_attention_cross(const void* q, const void* k, const void* v, void* o, void* workspace,
                              size_t workspace_bytes, const int* kv_lens, int batch, int heads, int heads_kv, int q_len,
                              int kv_len, int head_dim, int dtype, const fa_strides* q_strides,
                              const fa_strides* k_strides, const fa_strides* v_strides, const fa_strides* o_strides,
                              void* stream)
{
    return fa::record_status(launch_cross(q, k, v, o, workspace, workspace_bytes, kv_lens, batch, heads, heads_kv, q_len,
                                          kv_len, head_dim, dtype, q_strides, k_strides, v_strides, o_strides, stream));
}

}  // extern "C"
