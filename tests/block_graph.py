"""A small graph of pre-normalised gated blocks, for the tests."""
import numpy as np


class Block:
    def __init__(self, batch=21, width=24, hidden=20, inputs=13, classes=7, dropout=0.25, activations=("silu", "gelu"), seed=0):
        from tinyflow_b200 import autodiff as ad
        rng = np.random.RandomState(seed)
        self.X, self.y_ = ad.Placeholder("X"), ad.Placeholder("y_")
        self.values, self.residuals = {}, []

        def variable(name, *shape, around=0.0):
            node = ad.Variable(name)
            self.values[node] = (around + rng.randn(*shape) * (0.1 if len(shape) == 1 else shape[0] ** -0.5)).astype(np.float32)
            return node

        h = ad.matmul_op(self.X, variable("Win", inputs, width))
        branch = ad.matmul_op(self.X, variable("Wside", inputs, width))
        for i, activation in enumerate(activations):
            total, y = ad.dropout_add_layer_norm_op(branch, h, variable("g%d" % i, width, around=1.0), variable("b%d" % i, width), dropout)
            self.residuals.append(total)
            branch = ad.matmul_op(ad.gated_linear_op(y, variable("W%d" % i, width, 2 * hidden), activation), variable("V%d" % i, hidden, width))
            h = total
        y = ad.layer_norm_op(h + branch, variable("g", width, around=1.0), variable("b", width))
        self.y = ad.matmul_op(y, variable("Wout", width, classes))
        self.loss = ad.softmaxcrossentropy_op(self.y, self.y_)
        labels = np.zeros((batch, classes), np.float32)
        labels[np.arange(batch), rng.randint(0, classes, batch)] = 1
        self.values[self.X], self.values[self.y_] = rng.randn(batch, inputs).astype(np.float32), labels
        self.parameters = [n for n in self.values if n.isw == 1]
