"""Records the token mixers' calls into HIP graphs through torch and replays them, with eager work between: every replay must
give the bits of the eager run, and new operand values in the same buffers must be picked up.  Run by
tests/test_gpu_mixers.py in a process of its own; exit code 77 = torch has no GPU."""
import os
import sys

try:
    import torch                      # before the library: the process keeps the first HIP runtime loaded
except ImportError:
    print("torch is not importable")
    sys.exit(77)
if not torch.cuda.is_available():
    print("torch sees no GPU")
    sys.exit(77)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "dragon-alpha-v1.2_amd"))
import dragon_hip as dh               # noqa: E402

A, L = dh.Cuda_attention, dh.Cuda_linear_attention


class Window:
    def __init__(self, N, H, G, QL, VL, d, window, sinks, train):
        self.sizes, self.tail = (N, H, G, QL, VL, d, d), (1, d ** -0.5, window, sinks)
        self.ins = [torch.empty(s, device="cuda") for s in ((N, QL, H, d), (N, VL, G, d), (N, VL, G, d), (N, QL, H, d))]
        self.lens = [torch.zeros(N, dtype=torch.int32, device="cuda") for _ in range(2)]
        need = A.window_bufsize(*self.sizes, window, sinks)
        if train:
            need = max(need, A.window_backward_bufsize(*self.sizes, window, sinks))
        self.need, self.buf, self.train = need, torch.empty(max(need // 4, 4), device="cuda"), train
        self.outs = [torch.empty_like(self.ins[0]), torch.empty(N, H, QL, device="cuda")] + \
            [torch.empty_like(x) for x in self.ins[:3] if train]

    def fill(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for x in self.ins:
            x.normal_(generator=g)
        N, QL, VL = self.sizes[0], self.sizes[3], self.sizes[4]
        self.lens[1].copy_(torch.tensor([max(0, VL - 17 * seed * i) for i in range(N)], dtype=torch.int32))
        self.lens[0].copy_(torch.clamp(self.lens[1], max=QL) if QL > 1 else torch.ones(N, dtype=torch.int32))

    def run(self):
        s = [torch.cuda.current_stream().cuda_stream]
        p = [x.data_ptr() for x in self.ins]
        o = [x.data_ptr() for x in self.outs]
        lens = [x.data_ptr() for x in self.lens]
        A.window_forward(s, 1, *p[:3], *o[:2], *lens, self.buf.data_ptr(), self.need, *self.sizes, *self.tail)
        if self.train:
            A.window_backward(s, 1, *p[:3], *o[:2], p[3], *o[2:], *lens, self.buf.data_ptr(), self.need, *self.sizes, *self.tail)


class Decay:
    def __init__(self, N, H, T, d, train):
        self.sizes, self.tail = (N, H, T, d, d), (1, d ** -0.5)
        self.ins = [torch.empty(N, T, H, d, device="cuda") for _ in range(4)] + [torch.empty(N, H, d, d, device="cuda") for _ in range(2)]
        self.g = -torch.linspace(0.01, 1.0, H, device="cuda")
        self.lens = torch.zeros(N, dtype=torch.int32, device="cuda")
        need = max(L.bufsize(*self.sizes), L.backward_bufsize(*self.sizes) if train else 0)
        self.need, self.buf, self.train = need, torch.empty(max(need // 4, 4), device="cuda"), train
        self.outs = [torch.empty_like(self.ins[0]), torch.empty_like(self.ins[4])]
        if train:
            self.outs += [torch.empty_like(x) for x in self.ins[:3]] + [torch.empty_like(self.ins[4])]

    def fill(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for x in self.ins:
            x.normal_(generator=g)
        N, T = self.sizes[0], self.sizes[2]
        self.lens.copy_(torch.tensor([max(0, T - 5 * seed * i) for i in range(N)], dtype=torch.int32))

    def run(self):
        s = [torch.cuda.current_stream().cuda_stream]
        q, k, v, dy, s0, ds1 = (x.data_ptr() for x in self.ins)
        o = [x.data_ptr() for x in self.outs]
        L.forward(s, 1, q, k, v, self.g.data_ptr(), s0, o[0], o[1], self.lens.data_ptr(), self.buf.data_ptr(), self.need, *self.sizes,
                  *self.tail)
        if self.train:
            L.backward(s, 1, q, k, v, self.g.data_ptr(), s0, dy, ds1, *o[2:6], self.lens.data_ptr(), self.buf.data_ptr(), self.need,
                       *self.sizes, *self.tail)


def main():
    ops = [Window(3, 8, 2, 1, 900, 64, 100, 4, False), Window(2, 4, 2, 300, 300, 64, 50, 3, True), Window(1, 2, 1, 260, 2600, 128, 0, 0, False),
           Decay(3, 4, 1, 64, False), Decay(2, 3, 400, 64, True)]
    graphs = []
    for op in ops:
        op.fill(1)
        op.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op.run()
        graphs.append(g)
    for seed in (1, 2, 3, 4):
        want = []
        for op in ops:
            op.fill(seed)
            op.run()
            want.append([x.clone() for x in op.outs])
        torch.cuda.synchronize()
        for _ in range(2):
            for op in ops:
                for x in op.outs:
                    x.fill_(7.0)
                op.buf.fill_(float("nan"))
            torch.cuda.synchronize()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for n, (op, w) in enumerate(zip(ops, want)):
                for i, (x, y) in enumerate(zip(op.outs, w)):
                    if not torch.equal(x, y):
                        print("call %d, output %d: a replay differs from the eager run (seed %d)" % (n, i, seed))
                        return 1
    print("ok")
    return 0


if __name__ == "__main__":
    sys.exit(main())
