"""sharedkv_cache_append: queries that stay in place unturned, and rows that have no place."""

import pytest
import torch

from dsv4_planb_b200.cache import rope_table
from tests.test_gpu_cache import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_queries_without_rotation(cuda_device, interleaved, pool):
    """Without angles queries are copied, or stay where they are."""
    m = make([3, 40], [70, 200], pool=pool, heads=18, seed=61)
    for place in (False, True):
        q = m["q"].cuda()
        cache, scale, out = run(m, None, q=q, q_out=q if place else None, rope_interleaved=interleaved, check_status=True)
        check(m, cache, scale, None)
        assert torch.equal(out.cpu(), m["q"]) and (out is q) == place


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens", [([5], [3]), ([1, 2, 1], [4, 0, 9]), ([300], [40])])
def test_rows_before_the_start_are_reported(cuda_device, q_lens, kv_lens, pool):
    """Lengths that do not count the new rows in: rows before position 0 are skipped, and reported."""
    m = make(q_lens, [max(a, b) for a, b in zip(q_lens, kv_lens)], pool=pool, seed=60)
    m["seq"] = torch.tensor(kv_lens, dtype=torch.int32)
    m["where"] = [(b, kv_lens[b] - n + s) for b, n in enumerate(q_lens) for s in range(n)]
    rope = rope_table(400, 64)
    check(m, *run(m, rope)[:2], rope)
    with pytest.raises(RuntimeError, match="bad_position"):
        run(m, rope, check_status=True)


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_what_is_reported(cuda_device, pool):
    """Padding is not reported; an unmapped block and the end of the block table are."""
    m = make([3, 0, 66], [70, 0, 140], pool=pool, seed=62)
    rope = rope_table(200, 64)
    kv = torch.cat([m["kv"], m["kv"][:9]]).cuda()
    check(m, *run(m, rope, kv=kv, check_status=True)[:2], rope)
    for change in (lambda t: t[2].fill_(-1), lambda t: t.resize_(3, 1)):
        m = make([3, 0, 66], [70, 0, 140], pool=pool, seed=62)
        change(m["table"])
        check(m, *run(m, rope)[:2], rope)
        with pytest.raises(RuntimeError, match="bad_block"):
            run(m, rope, check_status=True)


def test_queries_beside_rows_in_one_buffer(cuda_device):
    """Queries turn in place in a buffer that holds kv too; a buffer whose heads are kv rows is refused."""
    rope = rope_table(300, 64)
    m = make([1], [77], heads=4, seed=63)
    want = run(m, rope, q=m["q"].cuda())
    buf = torch.cat([m["q"].reshape(1, -1), m["kv"]], dim=1).cuda()  # [1, (4 + 1) * 576]
    q = buf[:, :4 * 576].reshape(1, 4, 576)
    got = run(m, rope, kv=buf[:, 4 * 576:], q=q, q_out=q)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(q, want[2])
    m = make([3, 2], [77, 9], heads=4, seed=64)
    rows = torch.cat([m["q"].reshape(-1, 576), m["kv"]]).cuda()  # queries, then rows
    q = rows[:20].view(5, 4, 576)
    check(m, *run(m, rope, kv=rows[20:], q=q, q_out=q)[:2], rope)
    buf = torch.zeros((5, 4, 576), dtype=torch.bfloat16, device="cuda")
    for kv in (buf[:, 3], buf[:, 0], buf.view(20, 576)[-5:]):
        with pytest.raises(ValueError, match="nothing with kv"):
            run(m, rope, kv=kv, q=buf, q_out=buf)
        with pytest.raises(ValueError, match="nothing with kv"):
            run(m, rope, kv=kv, q=m["q"].cuda(), q_out=buf)
    one = make([1], [9], heads=4, seed=65)
    buf = torch.zeros((1, 4, 576), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="nothing with kv"):
        run(one, rope, kv=buf[0, 2].expand(1, 576), q=buf, q_out=buf)
    row = one["kv"][0].cuda().expand(1, 576)
    check(one, *run(one, rope, kv=row, q=buf, q_out=buf, check_status=True)[:2], rope)
    gaps = torch.zeros((5, 40 * 576), dtype=torch.bfloat16, device="cuda")  # q_out between two rows
    gaps[:, :576] = m["kv"].cuda()
    out = gaps[1, 576:21 * 576].view(5, 4, 576)
    got = run(m, rope, kv=gaps[:, :576], q=m["q"].cuda(), q_out=out, check_status=True)
    check(m, *got[:2], rope)
