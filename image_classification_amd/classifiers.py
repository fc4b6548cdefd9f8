"""`KNNScikit` with the reference's interface, brute-force search on the device, and
`SoftmaxClassifier`, a linear classifier trained on the device.

Mirrors model/classifiers.py:165-197: `KNNScikit(neighbors, metric, weights, **kw)`,
`train(features, labels)` fits once (later calls are ignored, the `_is_trained` guard at :175),
`get_neighbors(features, neighbors, dist=True)` returns what
`KNeighborsClassifier.kneighbors(features, n_neighbors, return_distance)` returns: distances
float64 [M, k] ascending and indices int64 [M, k], or the indices alone.  `test` and
`test_probability` (:180-193) vote over the neighbour lists as scikit-learn does.

Two searches sit behind it:
  * Euclidean, width <= 128, at most two neighbours (the descriptor matching of
    model/robust_matching.py:73-80): the matrix-core distance / top-2 kernel;
  * everything else (bag-of-words histograms of any width, 'manhattan' as configured in
    vision/logo_recognition/training.py:41, the `intersection` / `chisqr` functions of
    model/clustering.py passed as `metric`, more neighbours): distance matrix + row top-k.
Metrics without a device kernel raise NotImplementedError rather than running on the CPU.

The reference trains its discriminative classifiers over histograms with libsvm
(model/classifiers.py:218, vision/spatial_scene/spatial_scene_classifier.py:100-118);
`SoftmaxClassifier` takes that place here with the methods of the classes above it.
"""
import numpy as np
import torch

from . import clustering as _clustering
from .backend import default_backend
from .ops import MAX_TOP

__all__ = ["KNNScikit", "SoftmaxClassifier"]

_STRING_METRICS = {"euclidean": "euclidean", "l2": "euclidean", "manhattan": "manhattan",
                   "cityblock": "manhattan", "l1": "manhattan", "sqeuclidean": "sqeuclidean"}


def _device_metric(metric, kwargs):
    if callable(metric):
        if metric is _clustering.intersection:
            return "intersection"
        if metric is _clustering.chisqr:
            return "chisqr"
        raise NotImplementedError("only the `intersection` and `chisqr` functions of this package "
                                  "are supported as callable metrics")
    if metric == "minkowski":
        p = kwargs.get("p", 2)
        if p == 2:
            return "euclidean"
        if p == 1:
            return "manhattan"
        raise NotImplementedError("minkowski is supported for p = 1 and p = 2 only")
    if metric in _STRING_METRICS:
        return _STRING_METRICS[metric]
    raise NotImplementedError("KNNScikit on the device supports euclidean, manhattan, sqeuclidean, "
                              "intersection and chisqr (got %r)" % (metric,))


class KNNScikit(object):

    def __init__(self, neighbors=3, metric="euclidean", weights="distance", backend=None,
                 **distance_kwargs):
        self._is_trained = False
        self.n_neighbors = neighbors
        self.metric = metric
        self.weights = weights
        self.distance_kwargs = distance_kwargs
        self._backend = backend
        self._fit_X = None
        self._cb = None
        self._metric = _device_metric(metric, distance_kwargs)
        if weights not in ("distance", "uniform"):
            raise NotImplementedError("weights must be 'distance' or 'uniform'")

    def _b(self):
        return self._backend or default_backend()

    def train(self, features, labels):
        if not self._is_trained:
            features = np.asarray(features)
            if features.ndim != 2:
                raise ValueError("Expected 2D array, got %dD array instead" % features.ndim)
            labels = list(labels)
            if len(labels) != features.shape[0]:
                raise ValueError("Found input variables with inconsistent numbers of samples: "
                                 "[%d, %d]" % (features.shape[0], len(labels)))
            self.labels_map = sorted(list(set(labels)))
            self._labels = np.asarray(labels)
            self.classes_ = np.asarray(self.labels_map)
            self._fit_X = features
            self._cb = self._b().codebook(features)
            self._is_trained = True

    # Evaluation helpers of the reference (model/classifiers.py:199-215) over `DataBag`-like
    # objects with `.feats` and `.labs`; accuracy is the fraction of equal labels, as
    # sklearn.metrics.accuracy_score and KNeighborsClassifier.score compute it.
    @classmethod
    def score_proba(cls, train_bag, test_bag, neg_bag, min_prob_diff=0.4, **kwargs):
        knn = cls(**kwargs)
        knn.train(train_bag.feats, train_bag.labs)
        y_test_pred = knn.test_probability(test_bag.feats, min_prob_diff)
        test_score = float(np.mean(np.asarray(test_bag.labs) == np.asarray(y_test_pred)))
        y_neg_pred = knn.test_probability(neg_bag.feats, min_prob_diff)
        neg_score = 1 - float(np.mean(np.asarray(neg_bag.labs) == np.asarray(y_neg_pred)))
        return test_score, neg_score

    @classmethod
    def score(cls, train_bag, test_bag, **kwargs):
        knn = cls(**kwargs)
        knn.train(train_bag.feats, train_bag.labs)
        return float(np.mean(knn.test(test_bag.feats) == np.asarray(test_bag.labs)))

    def train_and_test(self, features, labels):
        """model/classifiers.py:49-51"""
        self.train(features, labels)
        return self.test(features)

    # The reference keeps a fitted index as a pickle of the object (model/classifiers.py:53-63;
    # vision/logo_recognition/model.py:23 loads the model directory's `knn` file with it).  Same
    # method names here, but the file is a numpy archive of the fitted rows, the labels and the
    # constructor arguments -- written under exactly the name given -- and nothing is unpickled.
    def save_to_file(self, file_name):
        if not self._is_trained:
            raise RuntimeError("This KNNScikit instance is not fitted yet.")
        import json
        metric = self.metric.__name__ if callable(self.metric) else str(self.metric)
        kwargs = {k: v for k, v in self.distance_kwargs.items()
                  if isinstance(v, (int, float, str, bool)) or v is None}
        with open(file_name, "wb") as f:
            np.savez(f, fit_x=np.asarray(self._fit_X), labels=np.asarray(self._labels),
                     neighbors=np.int64(self.n_neighbors), metric=np.str_(metric),
                     weights=np.str_(self.weights), kwargs=np.str_(json.dumps(kwargs)))

    @classmethod
    def load_from_file(cls, file_name, backend=None):
        import json
        with open(file_name, "rb") as f:
            data = np.load(f, allow_pickle=False)
            metric = str(data["metric"])
            if metric in ("intersection", "chisqr"):
                metric = getattr(_clustering, metric)
            kwargs = json.loads(str(data["kwargs"])) if "kwargs" in data.files else {}
            index = cls(neighbors=int(data["neighbors"]), metric=metric,
                        weights=str(data["weights"]), backend=backend, **kwargs)
            index.train(data["fit_x"], list(data["labels"]))
        return index

    def get_neighbors(self, features, neighbors, dist=True):
        if not self._is_trained:
            raise RuntimeError("This KNNScikit instance is not fitted yet.")
        neighbors = int(neighbors)
        n_fit = self._fit_X.shape[0]
        if neighbors < 1:
            raise ValueError("Expected n_neighbors > 0. Got %d" % neighbors)
        if neighbors > n_fit:
            raise ValueError("Expected n_neighbors <= n_samples_fit, but n_neighbors = %d, "
                             "n_samples_fit = %d, n_samples = %d"
                             % (neighbors, n_fit, np.asarray(features).shape[0]))
        features = np.asarray(features)
        if features.ndim == 1 and features.shape[0] == self._fit_X.shape[1]:
            # one sample given as a vector: the logo flow hands the histogram of its one image to
            # this step that way (vision/logo_recognition/matching_flow.py:37-38, then
            # `x[0].tolist()` on the result), which the scikit-learn of the reference's time took
            # as a single row; later versions refuse it
            features = features[None, :]
        if features.ndim != 2 or features.shape[1] != self._fit_X.shape[1]:
            raise ValueError("X has %s features, but KNNScikit is expecting %d features as input."
                             % (features.shape[1:] or "?", self._fit_X.shape[1]))
        b = self._b()
        if features.shape[0] == 0:
            ind = np.empty((0, neighbors), dtype=np.int64)
            return (np.empty((0, neighbors), dtype=np.float64), ind) if dist else ind
        if self._metric == "euclidean" and neighbors <= 2 and features.shape[1] <= 128:
            i1, d1, i2, d2, _ = b.assign_top2_np(features, self._cb)
            if neighbors == 1:
                ind = i1.cpu().numpy().astype(np.int64)[:, None]
                dd = d1.cpu().numpy().astype(np.float64)[:, None]
            else:
                ind = np.stack([i1.cpu().numpy(), i2.cpu().numpy()], axis=1).astype(np.int64)
                dd = np.stack([d1.cpu().numpy(), d2.cpu().numpy()], axis=1).astype(np.float64)
        else:
            dd, ind = b.knn_rows(b.f32(features), self._cb.c, neighbors, self._metric)
            dd = dd.cpu().numpy()
            ind = ind.cpu().numpy().astype(np.int64)
        return (dd, ind) if dist else ind

    # -- label votes over the neighbour lists (host side: [M, k] arrays) ---------------------------
    def _votes(self, features):
        dd, ind = self.get_neighbors(features, self.n_neighbors, dist=True)
        w = np.ones_like(dd)
        if self.weights == "distance":
            with np.errstate(divide="ignore"):
                w = 1.0 / dd
            zero = np.isinf(w)
            rows = zero.any(axis=1)
            w[rows] = zero[rows].astype(np.float64)
        col = np.searchsorted(self.classes_, self._labels[ind])
        votes = np.zeros((dd.shape[0], len(self.classes_)), dtype=np.float64)
        rows = np.arange(dd.shape[0])
        for j in range(ind.shape[1]):
            np.add.at(votes, (rows, col[:, j]), w[:, j])
        return votes

    def predict_proba(self, features):
        votes = self._votes(features)
        s = votes.sum(axis=1, keepdims=True)
        s[s == 0] = 1.0
        return votes / s

    def test(self, features):
        """Predicted label per row: the class with the largest vote, lowest class on ties."""
        return self.classes_[np.argmax(self._votes(features), axis=1)]

    def test_probability(self, features, min_prob_diff):
        """Best label when its probability leads the runner-up by `min_prob_diff`, else -1
        (model/classifiers.py:183-193)."""
        y_pred = []
        for row in self.predict_proba(features):
            idx = row.argsort()
            if row[idx[-1]] - row[idx[-2]] >= min_prob_diff:
                y_pred.append(self.labels_map[idx[-1]])
            else:
                y_pred.append(-1)
        return y_pred


class SoftmaxClassifier(object):
    """Linear softmax classifier over histograms or descriptors, with routed experts.

    logits = W_g [x, 1] for the nearest of `experts` centroids g (k-means over the training rows;
    one expert: an ordinary linear classifier; several: rows of at most 2048 columns), W_g classes x
    columns.  `rank`: W_g is a product B_g A_g through that many columns, for wide histograms with many
    classes.  Training minimises
    the mean negative log probability of the labels minus `entropy_weight` times the mean entropy,
    with AdamW steps over `epochs` passes in batches of `batch_size`; `state_bits=8` keeps the
    optimizer states in 8 bits.  Everything between the upload of the rows and the download of the
    answers runs on the device: the search routes, the grouped products, the log probabilities with
    their gradient and the step are one call each.

    Same methods as KNNScikit: `train` fits once (later calls are ignored), `test`,
    `predict_proba`, `test_probability`, `save_to_file` / `load_from_file`.  Equal seeds give equal
    weights.
    """

    def __init__(self, experts=1, rank=None, epochs=20, batch_size=4096, lr=0.05, weight_decay=1e-4,
                 entropy_weight=0.0, state_bits=32, seed=0, backend=None):
        if int(experts) < 1:
            raise ValueError("experts must be at least 1, got %r" % (experts,))
        if rank is not None and int(rank) < 1:
            raise ValueError("rank must be at least 1, got %r" % (rank,))
        if int(epochs) < 0 or int(batch_size) < 1:
            raise ValueError("epochs must not be negative and batch_size must be at least 1")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32, got %r" % (state_bits,))
        self.experts, self.rank = int(experts), None if rank is None else int(rank)
        self.epochs, self.batch_size = int(epochs), int(batch_size)
        self.lr, self.weight_decay = float(lr), float(weight_decay)
        self.entropy_weight = float(entropy_weight)
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._backend = backend
        self._is_trained = False
        self._weights = None           # [W] or [A, B], device
        self._centroids = None         # numpy [experts, columns], or None
        self._cb = None
        self.loss_ = []                # mean loss of every epoch

    def _b(self):
        return self._backend or default_backend()

    # The columns of a row on the device: the features, a one, zeros up to a multiple of four (whole
    # 16-byte pieces of float32 rows).
    @staticmethod
    def _padded(d):
        return (d + 1 + 3) // 4 * 4

    def _rows(self, features, columns):
        features = np.asarray(features)
        if features.ndim == 1 and columns is not None and features.shape[0] == columns:
            features = features[None, :]
        if features.ndim != 2:
            raise ValueError("Expected 2D array, got %dD array instead" % features.ndim)
        if columns is not None and features.shape[1] != columns:
            raise ValueError("X has %d features, but SoftmaxClassifier is expecting %d features as "
                             "input." % (features.shape[1], columns))
        if features.shape[1] < 1:
            raise ValueError("rows have no columns")
        x = self._b().f32(features)
        if not bool(torch.isfinite(x).all()):
            raise ValueError("Input X contains NaN or infinity.")
        rows = torch.zeros((x.shape[0], self._padded(x.shape[1])), dtype=torch.float32,
                           device=x.device)
        rows[:, :x.shape[1]] = x
        rows[:, x.shape[1]] = 1.0
        return x, rows

    def _route(self, x):
        if self._cb is None or x.shape[0] == 0:
            return torch.zeros(x.shape[0], dtype=torch.int32, device=x.device)
        return self._b().assign_top1(x.contiguous(), self._cb, False)[0]

    def _forward(self, rows, order, offsets):
        """(hidden rows or None, logits with padded columns)."""
        b = self._b()
        if self.rank is None:
            return None, b.grouped_matmul(rows, self._weights[0], offsets, order)
        h = b.grouped_matmul(rows, self._weights[0], offsets, order)
        return h, b.grouped_matmul(h, self._weights[1], offsets, order)

    def train(self, features, labels):
        if self._is_trained:
            return
        labels = list(labels)
        if len(labels) != np.asarray(features).shape[0]:
            raise ValueError("Found input variables with inconsistent numbers of samples: [%d, %d]"
                             % (np.asarray(features).shape[0], len(labels)))
        if not labels:
            raise ValueError("no rows to train on")
        b = self._b()
        x, rows = self._rows(features, None)
        n, d = x.shape
        if self.experts > n:
            raise ValueError("%d experts for %d rows" % (self.experts, n))
        self.labels_map = sorted(list(set(labels)))
        self.classes_ = np.asarray(self.labels_map)
        self._columns = int(d)
        classes = len(self.labels_map)
        target = b.i32(np.searchsorted(self.classes_, np.asarray(labels)).astype(np.int32))
        if self.experts > 1:
            self._centroids, _ = _clustering.kmeans_fit(
                np.asarray(features, dtype=np.float32), self.experts, iters=10, rng=self.seed,
                backend=b)
            self._cb = b.codebook(self._centroids)
        codes = self._route(x)
        gen = torch.Generator().manual_seed(self.seed)
        k, c = rows.shape[1], (classes + 3) // 4 * 4

        def zeros(*shape):
            return torch.zeros(shape, dtype=torch.float32, device=rows.device)

        if self.rank is None:
            self._weights = [zeros(self.experts, c, k)]
        else:
            # A is random and B zero: the first gradient reaches B alone, the next ones both
            r = (self.rank + 3) // 4 * 4
            a = zeros(self.experts, r, k)
            a[:, :self.rank, :d + 1] = (torch.randn(self.experts, self.rank, d + 1, generator=gen)
                                        * (d + 1) ** -0.5).to(rows.device)
            self._weights = [a, zeros(self.experts, c, r)]
        exp_avg, exp_avg_sq, scales = b.adamw_states(self._weights, self.state_bits)
        step = 0
        for _ in range(self.epochs):
            total = torch.zeros((), dtype=torch.float32, device=rows.device)
            pick = torch.randperm(n, generator=gen).to(rows.device)
            for lo in range(0, n, self.batch_size):
                at = pick[lo:lo + self.batch_size]
                xb, yb = rows[at], target[at]
                order, offsets = b.group_rows(codes[at], self.experts)
                h, z = self._forward(xb, order, offsets)
                logits = z[:, :classes]
                logp, entropy, lse, _, _ = b.label_logprobs(logits, yb)
                total += -logp.sum() - self.entropy_weight * entropy.sum()
                m = at.shape[0]
                d_logp = torch.full_like(logp, -1.0 / m)
                d_entropy = None if self.entropy_weight == 0.0 \
                    else torch.full_like(logp, -self.entropy_weight / m)
                # the gradient takes the logits' place; the padded columns stay zero
                b.label_logprobs_grad(logits, yb, lse, entropy, d_logp, d_entropy, out=logits)
                if self.rank is None:
                    grads = [b.grouped_matmul_dw(z, xb, offsets, order)]
                else:
                    dh = b.grouped_matmul_dx(z, self._weights[1], offsets, order)
                    grads = [b.grouped_matmul_dw(dh, xb, offsets, order),
                             b.grouped_matmul_dw(z, h, offsets, order)]
                step += 1
                b.adamw_step(self._weights, grads, exp_avg, exp_avg_sq, lr=self.lr, step=step,
                             weight_decay=self.weight_decay, scales=scales)
            self.loss_.append(float(total) / n)
        self._is_trained = True

    def train_and_test(self, features, labels):
        self.train(features, labels)
        return self.test(features)

    def _check_trained(self):
        if not self._is_trained:
            raise RuntimeError("This SoftmaxClassifier instance is not fitted yet.")

    def _logits(self, features):
        self._check_trained()
        x, rows = self._rows(features, self._columns)
        order, offsets = self._b().group_rows(self._route(x), self.experts)
        _, z = self._forward(rows, order, offsets)
        return z[:, :len(self.labels_map)]

    def alternatives(self, features, k=5):
        """(labels [n, k], log probabilities float64 [n, k]): the k (at most 32) likeliest classes of
        every row, likeliest first, equal ones in label order."""
        k = int(k)
        self._check_trained()
        most = min(len(self.labels_map), MAX_TOP)
        if not 1 <= k <= most:
            raise ValueError("k must be in [1, %d], got %d" % (most, k))
        z = self._logits(features)
        if z.shape[0] == 0:
            return self.classes_[np.empty((0, k), dtype=np.int64)], np.empty((0, k))
        _, _, _, logp, idx = self._b().label_logprobs(z, None, top=k)
        return self.classes_[idx.cpu().numpy()], logp.cpu().numpy().astype(np.float64)

    def log_probabilities(self, features, labels):
        """(log probability of each row's label, entropy of each row), float64 [n].  A label the
        classifier was not trained on has log probability 0."""
        z = self._logits(features)
        known = {c: i for i, c in enumerate(self.labels_map)}
        at = np.array([known.get(q, -1) for q in labels], dtype=np.int32)
        if at.shape[0] != z.shape[0]:
            raise ValueError("Found input variables with inconsistent numbers of samples: [%d, %d]"
                             % (z.shape[0], at.shape[0]))
        logp, entropy, _, _, _ = self._b().label_logprobs(z, self._b().i32(at))
        return logp.cpu().numpy().astype(np.float64), entropy.cpu().numpy().astype(np.float64)

    def predict_proba(self, features):
        z = self._logits(features)
        _, _, lse, _, _ = self._b().label_logprobs(z, None)
        p = np.exp(z.cpu().numpy().astype(np.float64) - lse.cpu().numpy().astype(np.float64)[:, None])
        return p / p.sum(axis=1, keepdims=True)

    def test(self, features):
        """Likeliest label per row, lowest class on ties."""
        return self.alternatives(features, 1)[0][:, 0]

    def test_probability(self, features, min_prob_diff):
        """Best label when its probability leads the runner-up by `min_prob_diff`, else -1
        (model/classifiers.py:183-193)."""
        self._check_trained()
        k = min(2, len(self.labels_map))
        best, logp = self.alternatives(features, k)
        p = np.exp(logp)
        lead = p[:, 0] - (p[:, 1] if k == 2 else 0.0)
        return [b if gap >= min_prob_diff else -1 for b, gap in zip(best[:, 0].tolist(), lead)]

    def save_to_file(self, file_name):
        """A numpy archive under exactly this name; nothing is pickled, so labels have to be numbers,
        strings or bytes."""
        self._check_trained()
        if self.classes_.dtype.hasobject:
            raise ValueError("labels of type %s cannot be saved without pickling them"
                             % type(self.labels_map[0]).__name__)
        arrays = {"weights_%d" % i: w.cpu().numpy() for i, w in enumerate(self._weights)}
        if self._centroids is not None:
            arrays["centroids"] = self._centroids
        with open(file_name, "wb") as f:
            np.savez(f, classes=self.classes_, columns=np.int64(self._columns),
                     experts=np.int64(self.experts), rank=np.int64(self.rank or 0), **arrays)

    @classmethod
    def load_from_file(cls, file_name, backend=None):
        with open(file_name, "rb") as f:
            data = np.load(f, allow_pickle=False)
            rank = int(data["rank"])
            c = cls(experts=int(data["experts"]), rank=rank or None, backend=backend)
            c.classes_ = data["classes"]
            c.labels_map = c.classes_.tolist()
            c._columns = int(data["columns"])
            b = c._b()
            c._weights = [b.f32(data["weights_%d" % i]) for i in range(2 if rank else 1)]
            if "centroids" in data.files:
                c._centroids = data["centroids"]
                c._cb = b.codebook(c._centroids)
        c._is_trained = True
        return c
