/*
 * What the attention launch planner chooses, without a GPU: links the kernels'
 * object and launches nothing.
 *   attention_plan tokens heads kv_heads dim count page_size table_stride type
 * (page_size 0: prompts; type 0 f32, 1 f16, 2 bf16) prints
 *   rows target alike slots lists images items tiles grid
 */
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "qmv_kernels.h"

int main(int argc, char **argv)
{
    if (argc != 9) return 2;
    int a[8];
    for (int i = 0; i < 8; ++i) a[i] = atoi(argv[1 + i]);
    qmv::AttnTokens t = {};
    t.tokens = a[0];
    t.heads = a[1];
    t.kv_heads = a[2];
    t.dim = a[3];
    t.count = a[4];
    t.page_size = a[5];
    t.table_stride = a[6];
    const qmv::AttnPlan p = qmv::plan_attention(t, a[7]);
    printf("%d %d %d %d %d %lld %d %d %lld\n", p.rows, p.target, p.alike, p.slots, p.lists != 0, (long long)p.images, p.items,
           p.tiles, (long long)p.grid);
    return 0;
}
