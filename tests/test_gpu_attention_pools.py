"""Paged attention's tile kernel and the append on pools past 2^32 bytes and past
2^32 halves (the kernel of single tokens: test_gpu_attention.py)."""
import numpy as np
import pytest

from attention_cases import Batch, attend64, check_attend, f32_word, from_half, pack_k, pack_v, to_half

pytestmark = pytest.mark.gpu

PAGE, DIM, KV = 1024, 256, 8
HALVES = PAGE * DIM * KV  # of a page: 4 MiB
PAGES = 2 ** 32 // HALVES + 3
# Past 2^32 bytes, and past 2^32 halves: where an offset of 32 bits would be too.
FAR = [(PAGES // 2 + 2, [(PAGES // 2 + 2) * HALVES % 2 ** 31 // HALVES]),
       (PAGES - 1, [(PAGES - 1) * HALVES % 2 ** 31 // HALVES, (PAGES - 1) * HALVES % 2 ** 32 // HALVES])]


@pytest.fixture(scope="module")
def pools(gpu):
    pair = [gpu.alloc(2 * PAGES * HALVES) for _ in range(2)]
    yield pair
    for b in pair:
        b.release()


def one_page(new, length, at):
    batch = Batch([new], [length], PAGE, spare=0)
    batch.table[0, 0], batch.pages = at, PAGES
    return batch


@pytest.mark.parametrize("at", [at for at, _ in FAR])
@pytest.mark.parametrize("plan", [128001, 128003])
def test_tiles(gpu, pools, at, plan):
    rng = np.random.default_rng(9)
    k, v = (to_half(rng.standard_normal((1, KV, PAGE, DIM)), "f16") for _ in range(2))
    new, length = 40, 700
    q = rng.standard_normal((new, KV, DIM)).astype(np.float32)
    # A value that only the later rows see, and that they get from the pool again.
    v[0, 3, 680, 17] = to_half(np.float32([np.nan]), "f16")[0]
    pools[0].write(pack_k(k), offset=2 * at * HALVES)
    pools[1].write(pack_v(v), offset=2 * at * HALVES)
    y = gpu.alloc_f32(new * KV * DIM)
    gpu.set_gemv_plan(-7, plan)
    gpu.dispatch("attn_paged_f16", [gpu.upload_f32(q), *one_page(new, length, at).upload(gpu), *pools, y],
                 [1, new, KV, KV, DIM, KV * DIM, KV * DIM, PAGE, PAGES, 1, PAGE, 1, 0, f32_word(0.0625)], group_size=64)
    assert gpu.last_hip_kernel() == "attn_tile_kernel"
    near = Batch([new], [length], PAGE, spare=0)
    want, bound = attend64(q, from_half(k, "f16"), from_half(v, "f16"), near, 0.0625)
    check_attend(gpu.read_f32(y, new * KV * DIM).reshape(new, KV, DIM), want, bound, f"page {at}")


@pytest.mark.parametrize("at,wrapped", FAR)
@pytest.mark.parametrize("new", [1, 21])
def test_append(gpu, pools, at, wrapped, new):
    # The same bytes as in the pool's eighth page, and nothing where an address of
    # 32 bits would be.
    rng = np.random.default_rng(new)
    rows = rng.standard_normal((new, 3 * KV * DIM)).astype(np.float32)
    blank = np.full(HALVES, 0x1234, np.uint16)
    width = 3 * KV * DIM
    kept = []
    for page in (7, at):
        for pool in pools:
            for p in (page, *wrapped):
                pool.write(blank, offset=2 * p * HALVES)
        batch = one_page(new, 700, page)
        qkv = gpu.upload_f32(rows.ravel())
        gpu.dispatch("kv_append_rope_f16",
                     [qkv, qkv, qkv, qkv, qkv, gpu.upload_bytes(np.arange(new, dtype=np.int32)),
                      gpu.upload_f32(np.ones(DIM // 2, np.float32)), *batch.upload(gpu), *pools,
                      gpu.alloc_f32(new * KV * DIM)],
                     [1, new, KV, KV, DIM, DIM, width, width, width, KV * DIM, 0, 0, 1, DIM // 2, 0, 0, 0, 0, PAGE,
                      PAGES, 1],
                     offsets=[0, 4 * KV * DIM, 8 * KV * DIM] + [0] * 10, group_size=64)
        kept.append([pool.read(np.uint16, HALVES, offset=2 * page * HALVES) for pool in pools])
        for pool in pools:
            for p in wrapped:
                assert (pool.read(np.uint16, HALVES, offset=2 * p * HALVES) == 0x1234).all(), (page, p)
    for near, far in zip(*kept):
        assert (near != 0x1234).sum() >= new * KV * DIM - new and np.array_equal(near, far)
