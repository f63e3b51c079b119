"""Pools that each have a thread of their own: host bookkeeping alone, without a GPU.  A child process, so that a crash names its test."""
import os
import subprocess
import sys

import pytest

from nvllm_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <pthread.h>
#include <stdio.h>
#include <stdlib.h>
#include "nvllm.h"
#include "ops.h"

enum { BLOCKS = 8, ROUNDS = ROUNDS_ };
static void die(const char* what) { fprintf(stderr, "%s\n", what); exit(1); }
static void attach(KVCacheManager* m, size_t at) {
    if (nvllm_attach_kv_pool(m, 16, BLOCKS, 2, 2, 32, 4, (void*)at, (void*)(at + 0x800000))) die("attach");
}
/* a pool without forks: what is given back lies on the stack */
static void* plain(void* arg) {
    KVCacheManager* m = arg;
    for (int i = 0; i < ROUNDS; i++) {
        const int a = alloc_block(m), b = alloc_block(m);
        free_block(m, b);
        free_block(m, a);
        if (a != 0 || b != 1 || m->free_blocks_count != BLOCKS) die("a block of the pool without forks is gone");
    }
    return 0;
}
/* a pool whose blocks are shared and let go of, again and again */
static void* forks(void* arg) {
    KVCacheManager* m = arg;
    int at[2][BLOCKS];
    BlockTable t = {at[0], 0}, child = {at[1], 0}, *to[1] = {&child};
    for (int i = 0; i < ROUNDS; i++) {
        for (t.num_blocks = 0; t.num_blocks < 3; t.num_blocks++) at[0][t.num_blocks] = alloc_block(m);
        if (nvllm_fork_tables(m, &t, 48, to, 1)) die("fork");
        for (int b = 0; b < BLOCKS; b++)
            if (nvllm_block_users(m, b) != (b < 3 ? 2 : 0)) die("users of a shared block");
        if (nvllm_free_table(m, &t) || m->free_blocks_count != BLOCKS - 3) die("a shared block came back early");
        if (nvllm_free_table(m, &child) || m->free_blocks_count != BLOCKS) die("a shared block did not come back");
    }
    return 0;
}
/* pools that come and go */
static void* pools(void* arg) {
    for (int i = 0; i < ROUNDS / 8; i++) {
        KVCacheManager m = {0};
        attach(&m, (size_t)arg + (size_t)(i % 64) * 0x1000000);
        int at[2][1] = {{alloc_block(&m)}, {-1}};
        BlockTable t = {at[0], 1}, child = {at[1], 0}, *to[1] = {&child};
        if (nvllm_fork_tables(&m, &t, 16, to, 1) || nvllm_block_users(&m, 0) != 2) die("fork in a new pool");
        free_kv_cache_manager(&m);
    }
    return 0;
}
int main(void) {
    static KVCacheManager m[4];
    pthread_t t[6];
    for (int i = 0; i < 4; i++) attach(&m[i], 0x100000000 + (size_t)i * 0x1000000);
    for (int i = 0; i < 4; i++) pthread_create(&t[i], 0, i % 2 ? forks : plain, &m[i]);
    for (int i = 0; i < 2; i++) pthread_create(&t[4 + i], 0, pools, (void*)(0x200000000 + (size_t)i * 0x100000000));
    for (int i = 0; i < 6; i++) pthread_join(t[i], 0);
    return 0;
}
"""


@pytest.mark.skipif(sys.platform != "linux", reason="needs a C compiler and POSIX threads")
def test_pools_of_several_threads(tmp_path):
    src, exe = tmp_path / "threads.c", tmp_path / "threads"
    src.write_text(SOURCE.replace("ROUNDS_", "100000"))
    subprocess.check_call(["gcc", "-O2", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), capi.HIP_LIB, "-lpthread", "-Wl,-rpath," + os.path.dirname(capi.HIP_LIB)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
