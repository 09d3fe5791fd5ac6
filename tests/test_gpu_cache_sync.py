"""What a cache costs the runtime's other calls, and that its errors are found
all the same."""
import time

import numpy as np
import pytest

from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def test_synchronizing_calls_wait_once():
    """Two idle runtimes in turn, one of them with a cache: its synchronize
    needs no second trip to the device (20 us where a call takes 1)."""
    print("sync", flush=True)
    with rocm.Runtime(0) as a, rocm.Runtime(0) as b:
        c = b.cache(4, 1, 64, 2, 2)
        seen = ([], [])
        for _ in range(300):
            for i, r in enumerate((a, b)):
                t = time.perf_counter()
                r.synchronize()
                seen[i].append(time.perf_counter() - t)
        without, with_cache = (float(np.median(x)) for x in seen)
        assert with_cache <= 3 * without + 3e-6, (without, with_cache)
        c.close()


@pytest.mark.parametrize("how", ["synchronize", "download"])
def test_errors_are_reported_again_and_again(how):
    """Each report clears the flag and the word; a closed cache's error is
    still reported; two caches report into one runtime."""
    print("reports", how, flush=True)
    with rocm.Runtime(0) as rt:
        c, d = rt.cache(4, 1, 64, 2, 2), rt.cache(4, 1, 64, 2, 2)
        x = rt.to_device(np.zeros(4, np.int32))
        meet = rt.synchronize if how == "synchronize" else x.download
        for i in range(20):
            cache = (c, d)[i % 2]
            cache.release(rt.to_device(np.array([5 + i], np.int32)))
            with pytest.raises(_lib.MantaRocmError, match="cache sequence %d out of range" % (5 + i)):
                meet()
            meet()
        c.release(rt.to_device(np.array([7], np.int32)))
        c.close()
        with pytest.raises(_lib.MantaRocmError, match="cache sequence 7 out of range"):
            meet()
        meet()
        d.close()
        meet()
