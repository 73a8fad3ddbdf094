import fcntl
import multiprocessing.process
import os
import sys
import tempfile
import time

import pytest

# The GPU boxes of this pool show 256 logical CPUs but run under a cgroup quota of 16 cores (`/sys/fs/cgroup/cpu.max` = 1600000 100000).  torch's default of 128
# intra-op threads PER PROCESS -- the pytest process, every xdist worker, every spawned rank of the multi-process tests, each with its OpenMP workers
# spinning between parallel regions -- gets the whole job throttled: measured on twelve multi-rank tests, 202 s with the defaults against 32 s with four
# threads per process (`profiles/r04_gpu_suite_timing.md`).  Set before torch is imported anywhere, inherited by every child process.
for _k, _v in (("OMP_NUM_THREADS", "4"), ("MKL_NUM_THREADS", "4"), ("OMP_WAIT_POLICY", "PASSIVE")):
    os.environ.setdefault(_k, _v)
# Four xdist workers (and their spawned ranks) share ONE device: the engine's two memory-dependent switches (batched weight gradients, the kept SwiGLU product:
# engine.py `_mem_budget`) must not depend on what the neighbouring tests hold at that moment.  Under test they are decided from the device's total memory
# minus what THIS process holds; a test that then does not fit fails loudly (out of memory) instead of silently running another mode.
os.environ.setdefault("IE_MEM_BUDGET", "own")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def xport(port):
    """A rendezvous port private to this pytest-xdist worker (spawned ranks inherit PYTEST_XDIST_WORKER): tests that run at the same time are on
    different workers, so their process groups never meet on a port."""
    w = os.environ.get("PYTEST_XDIST_WORKER", "gw0")
    # (below the kernel's ephemeral range, 32768-60999: with `port + 1000 w` the fourth worker's ports sat inside it and a rendezvous once found its port taken by
    # a gloo pair connection -- EADDRINUSE in the round-6 suite; the tests' base ports lie in [29500, 30000))
    return 20000 + (int(port) - 29500) % 1000 + 1000 * (int(w[2:] or 0) % 12)


@pytest.hookimpl(tryfirst=True)
def pytest_cmdline_main(config):
    """Run the suite on four pytest-xdist workers by default (with the thread cap above: the whole GPU suite in ~100 s on one MI355X box, 860 s in round 3;
    the measurements behind it: profiles/r04_gpu_suite_timing.md).  `-n N` on the command line wins; IE_TEST_SERIAL=1 or a missing xdist plugin runs serially."""
    if (config.pluginmanager.hasplugin("xdist") and getattr(config.option, "numprocesses", None) is None and not os.environ.get("PYTEST_XDIST_WORKER")
            and os.environ.get("IE_TEST_SERIAL") != "1" and not getattr(config.option, "collectonly", False)):
        config.option.numprocesses = 4
        config.option.dist = "load"


# The longest tests first (eight ranks at 32 768 tokens / 7B width, the 8- and 4-rank layouts, the 7B-width engine runs), so that the short ones fill in
# around them instead of one of them forming the tail of the run.
_LONGEST_FIRST = ("test_isp_config3_layout_seq32768_sp8_at_7b_width", "test_sequence_parallel_sp4_sp8_equals_single_rank_step",
                  "test_llama2_tensor_parallel_2_with_hybrid_zero_on_8_ranks", "test_config3_shape_tensor2_weight4_on_internlm1_blocks_equals_one_rank",
                  "test_engine_7b_width_merged_benchmark_step_matches_oracle", "test_first_steps_of_the_benchmark_recipe_retrace_the_oracle_at_7b_width",
                  "test_engine_7b_shaped_layer_full_size_matches_oracle", "test_flash_attention_benchmark_regime_matches_oracle",
                  "test_weight_parallel_step_equals_resident_step", "test_moe_engine_expert_parallel_on_two_ranks_matches_the_reference_rules")


# ... and these LAST, when the other workers are running out of work: four staged ranks on one device (each imports torch and builds an engine) beside three
# busy workers hung once until its queue timeout (round 5); at the end of the run it has the box almost to itself.
_LAST = ("test_moe_engine_tensor_parallel_2_x_expert_parallel_2_on_four_ranks",)


def pytest_collection_modifyitems(config, items):
    rank = {n: i for i, n in enumerate(_LONGEST_FIRST)}
    rank.update({n: len(_LONGEST_FIRST) + 1 + i for i, n in enumerate(_LAST)})
    if os.environ.get("IE_TEST_FULL") != "1":   # parametrisations whose layout another test of the default run covers (each names it): IE_TEST_FULL=1 runs them too
        for it in items:
            if it.get_closest_marker("extended") is not None:
                it.add_marker(pytest.mark.skip(reason="extended parametrisation (its layout is covered by another test of the default run); IE_TEST_FULL=1 runs it"))
    items.sort(key=lambda it: rank.get(getattr(it, "originalname", None) or it.name, len(rank)))   # (stable: everything else keeps its file order)


def pytest_configure(config):
    if "torch" in sys.modules:   # (imported before this file by a plugin: the environment above came too late for this process)
        import torch

        torch.set_num_threads(int(os.environ["OMP_NUM_THREADS"]))
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    config.addinivalue_line("markers", "ranks(n): GPUs a multi-rank test needs for its RCCL (nccl backend) variant")
    config.addinivalue_line("markers", "extended: a parametrisation whose layout another default test covers; run with IE_TEST_FULL=1")


# A device takes few processes at once (16 where this suite was measured), and which tests of several ranks meet on the four workers changes with the number of
# tests.  So the ranks of all workers together draw from one pool of _SLOTS places: 4 workers + 10 ranks, whatever the order.  A test says how many it
# needs by the processes that it has made when it starts the first of them, and gives them back at its end; a place is a locked file, so that a dead worker's are free.
_SLOTS = 10
_SUBPROCESS_RANKS = 3   # a test that starts the benchmark program: two ranks and their parent
_made, _held = [], []
_process_init, _process_start = multiprocessing.process.BaseProcess.__init__, multiprocessing.process.BaseProcess.start


def _take_slots(n):
    folder = os.path.join(tempfile.gettempdir(), "ie_ranks_%s_%d" % (os.environ.get("PYTEST_XDIST_TESTRUNUID", "serial%d" % os.getpid()), os.getuid()))
    os.makedirs(folder, exist_ok=True)
    with open(os.path.join(folder, "turn"), "w") as turn:
        fcntl.flock(turn, fcntl.LOCK_EX)   # (one worker waits for places at a time: two that hold a part each cannot wait for each other)
        free = list(range(_SLOTS))
        while len(_held) < min(n, _SLOTS):
            for i in list(free):
                if len(_held) == min(n, _SLOTS):
                    break
                f = open(os.path.join(folder, str(i)), "w")
                try:
                    fcntl.flock(f, fcntl.LOCK_EX | fcntl.LOCK_NB)
                except OSError:
                    f.close()
                    continue
                _held.append(f)
                free.remove(i)
            if len(_held) < min(n, _SLOTS):
                time.sleep(0.05)


@pytest.hookimpl(hookwrapper=True)
def pytest_runtest_call(item):
    if item.get_closest_marker("gpu") is None:
        yield
        return

    def init(self, *args, **kw):
        _process_init(self, *args, **kw)
        _made.append(self)

    def start(self):
        if not _held:
            _take_slots(len(_made))
        _process_start(self)

    multiprocessing.process.BaseProcess.__init__, multiprocessing.process.BaseProcess.start = init, start
    try:
        if "subprocess" in getattr(getattr(item.obj, "__code__", None), "co_names", ()) + getattr(getattr(item.obj, "__code__", None), "co_varnames", ()):
            _take_slots(_SUBPROCESS_RANKS)
        yield
    finally:
        multiprocessing.process.BaseProcess.__init__, multiprocessing.process.BaseProcess.start = _process_init, _process_start
        for f in _held:
            f.close()
        _held.clear()
        _made.clear()


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")
