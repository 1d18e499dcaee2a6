// Bookkeeping of a paged K/V cache: block tables and slot maps from request
// lengths, and the write of new K and V rows into their slots.
#include <algorithm>
#include <cstdint>

#include "fa_common.hpp"
#include "fa_paged.hpp"

namespace {

// ------------------------------------------------------------ tables and slots
//
//   starts[s] = sum_{t<s} n_t        kv_lens[s] = c_s + n_s
//   have_s = ceil(c_s / B), need_s = ceil((c_s + n_s) / B), at most the table's width
//   first_s = sum_{t<s} (need_t - have_t)
//   table[s][have_s + j] = free[first_s + j]
//   slot of token i of s, at position p = c_s + i: table[s][p / B] * B + p % B
//
// One launch: every workgroup sums all lengths for itself (8 bytes a sequence,
// from the L2) and then writes its share of the slots and the table entries, for
// which a token looks up its sequence among the sums in LDS. A slot in a new block
// takes its number from the free list, not from the table, so no workgroup reads
// what another writes. Latency alone: 3.4 us for 8 sequences, 5.6 for 1000 with 32768
// new tokens (a launch that does nothing takes about 2).
struct SlotArgs
{
    const int* cached;
    const int* fresh;
    int* table;
    const int* free_blocks;
    int* starts;
    int* kv_lens;
    long long* slots;
    int* taken;
    long long table_stride;
    int seqs, width, num_free, shift, max_tokens;
};

template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_slots_kernel(const SlotArgs a)
{
    constexpr int kWaves = kThreads / 64;
    __shared__ int s_start[kThreads], s_first[kThreads], s_cached[kThreads], s_have[kThreads];
    __shared__ int w_tokens[kWaves], w_blocks[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int mine = blockIdx.x * kThreads + tid;
    const int stride = gridDim.x * kThreads;
    int tokens = 0, blocks = 0;  // before the strip

    // Largest x < count with sums[x] <= value (sums rise, sums[0] <= value).
    auto find = [&](const int* sums, int count, int value) {
        int lo = 0;
        for (int step = kThreads / 2; step > 0; step >>= 1)
            if (lo + step < count && sums[lo + step] <= value) lo += step;
        return lo;
    };
    // First of this thread's items at or past `from`.
    auto first_item = [&](int from) {
        return from <= mine ? static_cast<long long>(mine)
                            : mine + (static_cast<long long>(from) - mine + stride - 1) / stride * stride;
    };

    for (int base = 0; base < a.seqs; base += kThreads)
    {
        const int s = base + tid;
        const int count = min(kThreads, a.seqs - base);
        const bool in = tid < count;
        const int c = in ? max(0, a.cached[s]) : 0;
        const int n = in ? max(0, a.fresh[s]) : 0;
        const long long kv = static_cast<long long>(c) + n;
        const long long round = (1LL << a.shift) - 1;
        const int have = static_cast<int>(min((c + round) >> a.shift, static_cast<long long>(a.width)));
        const int need = static_cast<int>(min((kv + round) >> a.shift, static_cast<long long>(a.width)));
        int x = n, y = need - have;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1)
        {
            const int px = __shfl_up(x, off, 64), py = __shfl_up(y, off, 64);
            if (lane >= off) x += px, y += py;
        }
        if (lane == 63) w_tokens[wave] = x, w_blocks[wave] = y;
        __syncthreads();
        int before_t = tokens, before_b = blocks, strip_t = 0, strip_b = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
        {
            if (w < wave) before_t += w_tokens[w], before_b += w_blocks[w];
            strip_t += w_tokens[w], strip_b += w_blocks[w];
        }
        s_start[tid] = before_t + x - n;
        s_first[tid] = before_b + y - (need - have);
        s_cached[tid] = c;
        s_have[tid] = have;
        if (in && blockIdx.x == 0)
        {
            a.starts[s] = before_t + x - n;
            a.kv_lens[s] = static_cast<int>(min(kv, 0x7fffffffLL));
        }
        __syncthreads();

        const long long t_end = min(tokens + strip_t, a.max_tokens);
        for (long long t = first_item(tokens); t < t_end; t += stride)
        {
            const int q = find(s_start, count, static_cast<int>(t));
            const long long p = static_cast<long long>(s_cached[q]) + (t - s_start[q]);
            const long long block = p >> a.shift;
            int page = -1;
            if (block < s_have[q]) page = a.table[(base + q) * a.table_stride + block];
            else if (block < a.width)
            {
                const long long f = s_first[q] + (block - s_have[q]);
                if (f >= 0 && f < a.num_free) page = a.free_blocks[f];
            }
            a.slots[t] = page < 0 ? -1 : (static_cast<long long>(page) << a.shift) + (p & round);
        }
        const long long b_end = static_cast<long long>(blocks) + strip_b;
        for (long long e = first_item(blocks); e < b_end; e += stride)
        {
            const int q = find(s_first, count, static_cast<int>(e));
            const long long column = s_have[q] + (e - s_first[q]);
            if (column < a.width)
                a.table[(base + q) * a.table_stride + column] = e < a.num_free ? a.free_blocks[e] : -1;
        }
        tokens += strip_t;
        blocks += strip_b;
        __syncthreads();
    }
    for (long long t = first_item(tokens); t < a.max_tokens; t += stride) a.slots[t] = -1;
    if (mine == 0)
    {
        a.starts[a.seqs] = tokens;
        *a.taken = blocks;
    }
}

int launch_slots(const int* cached, const int* fresh, int num_seqs, int* table, long long table_stride, int table_width,
                 const int* free_blocks, int num_free, int block_size, int* starts, int* kv_lens, long long* slots,
                 int max_tokens, int* taken, void* stream)
{
    if (num_seqs < 0 || table_width < 0 || num_free < 0 || max_tokens < 0 || table_stride < 0) return hipErrorInvalidValue;
    if (fa::bad_block_size(block_size)) return hipErrorInvalidValue;
    if (!starts || !taken || (num_seqs > 0 && (!cached || !fresh || !kv_lens))) return hipErrorInvalidValue;
    if ((num_seqs > 0 && table_width > 0 && (!table || table_stride < table_width)) || (num_free > 0 && !free_blocks) ||
        (max_tokens > 0 && !slots))
        return hipErrorInvalidValue;
    SlotArgs a{cached, fresh, table, free_blocks, starts, kv_lens, slots, taken, table_stride, num_seqs, table_width, num_free,
               __builtin_ctz(block_size), max_tokens};
    const int threads = num_seqs <= 256 ? 256 : 1024;
    const int grid = std::max(1, std::min(256, static_cast<int>((static_cast<long long>(max_tokens) + threads - 1) / threads)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return threads == 256 ? fa::launch_kernel(paged_slots_kernel<256>, dim3(grid), dim3(256), s, a)
                          : fa::launch_kernel(paged_slots_kernel<1024>, dim3(grid), dim3(1024), s, a);
}

// ------------------------------------------------------------ cache writes
//
// One thread moves 16 bytes of a K row and the same 16 of its V row, so a wave has
// 2 KiB of reads in flight at once. Bound by memory: 16384 tokens of 8 heads of 128
// take 27.8 us, 4.83 TB/s (a large copy runs at 4.9); 64 tokens 2.3 us, a launch.
struct AppendArgs
{
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* k_cache;
    uint16_t* v_cache;
    const long long* slots;
    long long k_row, k_head, v_row, v_head;
    long long block_stride, head_stride, token_stride;
    long long num_slots;
    long long items;  // 16-byte pieces of K
    int per_token, per_head, shift;
};

__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a)
{
    const long long step = static_cast<long long>(gridDim.x) * 256;
    for (long long x = blockIdx.x * 256LL + threadIdx.x; x < a.items; x += step)
    {
        const long long token = x / a.per_token;
        const int in_token = static_cast<int>(x - token * a.per_token);
        const int head = in_token / a.per_head;
        const int piece = (in_token - head * a.per_head) * 8;
        const long long slot = a.slots[token];
        if (static_cast<unsigned long long>(slot) >= static_cast<unsigned long long>(a.num_slots)) continue;
        const long long to = (slot >> a.shift) * a.block_stride + head * a.head_stride +
                             (slot & ((1LL << a.shift) - 1)) * a.token_stride + piece;
        const uint4 kx = *reinterpret_cast<const uint4*>(a.k + token * a.k_row + head * a.k_head + piece);
        const uint4 vx = *reinterpret_cast<const uint4*>(a.v + token * a.v_row + head * a.v_head + piece);
        *reinterpret_cast<uint4*>(a.k_cache + to) = kx;
        *reinterpret_cast<uint4*>(a.v_cache + to) = vx;
    }
}

int launch_append(const void* k, const void* v, const long long* slots, int tokens, const fa_paged_cache* cache,
                  const fa_strides* k_strides, const fa_strides* v_strides, void* stream)
{
    if (!cache || tokens < 0) return hipErrorInvalidValue;
    const int status = fa::check_paged_cache(*cache);
    if (status != hipSuccess) return status;
    if (tokens == 0 || cache->heads_kv == 0) return hipSuccess;
    if (!k || !v || !slots || fa::misaligned16(k) || fa::misaligned16(v)) return hipErrorInvalidValue;
    const fa_strides packed{0, cache->head_dim, static_cast<long long>(cache->heads_kv) * cache->head_dim};
    const fa_strides ks = k_strides ? *k_strides : packed;
    const fa_strides vs = v_strides ? *v_strides : packed;
    if ((ks.head | ks.row | vs.head | vs.row) & 7) return hipErrorInvalidValue;
    const long long per_token = static_cast<long long>(cache->heads_kv) * (cache->head_dim / 8);
    if (per_token > 0x7fffffffLL) return hipErrorInvalidValue;
    AppendArgs a{};
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.k_cache = static_cast<uint16_t*>(cache->k);
    a.v_cache = static_cast<uint16_t*>(cache->v);
    a.slots = slots;
    a.k_row = ks.row, a.k_head = ks.head, a.v_row = vs.row, a.v_head = vs.head;
    a.block_stride = cache->block_stride;
    a.head_stride = cache->head_stride;
    a.token_stride = cache->token_stride;
    a.num_slots = static_cast<long long>(cache->num_blocks) * cache->block_size;
    a.items = tokens * per_token;
    a.per_token = static_cast<int>(per_token);
    a.per_head = cache->head_dim / 8;
    a.shift = __builtin_ctz(cache->block_size);
    const long long grid = std::min<long long>((a.items + 255) / 256, 1 << 20);
    return fa::launch_kernel(paged_append_kernel, dim3(static_cast<unsigned>(grid)), dim3(256),
                             static_cast<hipStream_t>(stream), a);
}

}  // namespace

extern "C" {

int fa_launch_paged_slots(const int* cached_lens, const int* new_lens, int* block_table, const int* free_blocks,
                          int* query_starts, int* kv_lens, long long* slot_map, int* blocks_taken, int num_seqs,
                          int table_width, long long table_stride, int num_free, int block_size, int max_tokens,
                          void* stream)
{
    return fa::record_status(launch_slots(cached_lens, new_lens, num_seqs, block_table, table_stride, table_width,
                                          free_blocks, num_free, block_size, query_starts, kv_lens, slot_map, max_tokens,
                                          blocks_taken, stream));
}

int fa_launch_paged_append(const void* k, const void* v, const long long* slot_map, const fa_paged_cache* cache,
                           int tokens, const fa_strides* k_strides, const fa_strides* v_strides, void* stream)
{
    return fa::record_status(launch_append(k, v, slot_map, tokens, cache, k_strides, v_strides, stream));
}

}  // extern "C"
