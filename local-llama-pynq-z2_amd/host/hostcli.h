/* Shared pieces of the C host programs qwen_hip and runq_hip: prompt-id parsing, the cache's type.
 * Decoding (argmax or the sampler) runs on the device inside the step graph. */
#pragma once
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int *parse_ids(const char *arg, int *n) { /* qwen.c:771-777 */
    int *ids = calloc(strlen(arg) / 2 + 2, sizeof(int));
    *n = 0;
    for (const char *c = arg; *c;) {
        char *end;
        long v = strtol(c, &end, 10);
        if (end == c || (*end && *end != ',') || v < 0) { fprintf(stderr, "bad --ids\n"); exit(EXIT_FAILURE); }
        ids[(*n)++] = (int)v;
        c = *end ? end + 1 : end;
    }
    return ids;
}

/* --kv: the type of the K/V cache (llm_set_kv) */
static int parse_kv(const char *arg) {
    static const char *names[] = {"fp32", "bf16", "int8", "e4m3"};
    for (int i = 0; i < 4; i++)
        if (!strcmp(arg, names[i])) return i;
    fprintf(stderr, "bad --kv %s (fp32, bf16, int8 or e4m3)\n", arg);
    exit(EXIT_FAILURE);
}
