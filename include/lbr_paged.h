/*
 * lbr_paged.h — op codes of the paged key/value cache and of drafted tokens, which
 * liblbr_executor.so has beside the reference's (lbr_executor.h); they are OpNodes like
 * the others, taken by every entry point.
 *
 * A cache is bytes [pages][page_bytes].  A page holds for each K/V head in turn the K
 * rows [page_size][hdp], the V rows [page_size/8][hdp][8], and a float scale for each K
 * row and each V row (hdp: head_dim rounded up to 16, the rest zeros); a stored value stands
 * for itself times its row's scale.  extra[0..5] of the three cache ops: page_size (a power
 * of two, 16 .. 32768), K/V heads, head_dim (1 .. 256), element type (0 float32, 1 float16,
 * 2 int8, 3 e4m3), pages of the cache, pages of a page-table row.
 *
 * page_table [B][pages of a row], start [B] and count [B] are int32 on the device.  What they
 * hold is checked there: rows outside the table or on a page that the cache does not have are not
 * written, and read as NaN; counts are taken as 0 .. S.  The cache starts on a 16-byte boundary.
 *
 *   CACHE_WRITE      inputs cache, K, V [B][heads][S][head_dim], table, start, count;
 *                    output = inputs[0], shape [pages, page_bytes], elem_size 1;
 *                    extra[6] = S, extra[7] = B.  Row i < count[b] goes to position start[b] + i
 *   CACHE_READ       inputs cache, table, start, count; output float [2, B, heads, T, head_dim]:
 *                    K and V of positions start[b] + i, zeros for i >= count[b]
 *   PAGED_ATTENTION  inputs Q [B][H][S][head_dim], cache, table, start, count; output as Q;
 *                    extra[6] = bits of the score scale.  Row i < count[b] attends to positions
 *                    0 .. start[b] + i, head h to K/V head h / (H / heads); the others are zeros
 *   VERIFY_DRAFT     inputs target [B][D+1][V], draft [B][D][V], tokens (int64) [B][D],
 *                    uniforms [B][D+1], count [B]; output int64 [B, D+1]; extra[0] = V.  Token i <
 *                    count[b] stands while uniforms[i] * draft[i][token] < target[i][token]; behind the n
 *                    that stand, one drawn with uniforms[D] from max(target[n] - draft[n], 0) or, where
 *                    all stand or that is zero, from target[n]; then -1
 */
#ifndef LBR_PAGED_H
#define LBR_PAGED_H

enum LbrPagedOp {
    OP_CACHE_WRITE = 1100, OP_CACHE_READ = 1101, OP_PAGED_ATTENTION = 1102, OP_VERIFY_DRAFT = 1103
};

#endif /* LBR_PAGED_H */
